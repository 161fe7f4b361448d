// Column sums of every group's rows (the gradient of a grouped layer's bias), for kernels of their own and as a share of another launch.
#pragma once
#include "rp_grouped.h"

namespace rp {

struct GroupedSums {
    void* out;                     // [weights, cols] dense
    const void* x;
    RowGroups gr;
    int cols, accumulate;
    long long x_rs;
};
static inline long long sum_blocks(const GroupedSums& s) { return (long long)s.gr.weights * ((s.cols + 63) / 64); }

// Block `id`: 64 columns of one group, a vector of V of them a lane and so V rows a wave at a time.  Rows are dealt to 16 sums, whatever the number of waves, each in V parts that
// are added first; then the 16 in order.  Few groups are short of workgroups and bound by how long a load takes to come, so that 16 of them a wave are on their
// way at a time (bf16, 14949 rows of 3 groups, 427 columns, in the launch of all gradients, a column a lane and a vector: 163 us and 77).  A vector that straddles the end of its row is loaded
// early, where it ends with the row, and shifted into place.  parts: room for 16 x 64 sums.
template <typename T, int WAVES>
__device__ __forceinline__ void grouped_sums_block(const GroupedSums& s, long long id, typename traits<T>::acc* parts) {
    using A = typename traits<T>::acc;
    typedef unsigned int vector_t __attribute__((ext_vector_type(4), aligned(2)));        // (at any element)
    constexpr int PER = 16 / WAVES, V = 16 / (int)sizeof(T), LANES = 64 / V;
    const int strips = (s.cols + 63) / 64, w = (int)(id / strips), c0 = (int)(id % strips) * 64, lane = threadIdx.x & 63, q = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = c0 + lane % LANES * V, left = s.cols - c, by = left > 0 && left < V && s.cols >= V ? V - left : 0;
    const bool cut = c0 + 64 > s.cols && s.cols % V;
    A sum[PER][V] = {};
    const int e = s.gr.end(w);
    int i = s.gr.begin(w) + q * PER * V + lane / LANES;
    auto add = [&](A (&to)[V], const T* row) {
        T x[V];
        vector_t v = *(const vector_t*)(row + c - by);
        if (cut) v = __builtin_bit_cast(vector_t, __builtin_bit_cast(unsigned __int128, v) >> (8 * (int)sizeof(T) * by));
        __builtin_memcpy(x, &v, 16);
#pragma unroll
        for (int k = 0; k < V; k++) to[k] += widen(x[k]);
    };
    const T* x = (const T*)s.x;
    if (left > 0 && s.cols >= V) {
#pragma unroll WAVES
        for (; i + (PER - 1) * V < e; i += 16 * V)
#pragma unroll
            for (int j = 0; j < PER; j++) add(sum[j], x + (long long)(i + j * V) * s.x_rs);
#pragma unroll
        for (int j = 0; j < PER; j++)
            if (i + j * V < e) add(sum[j], x + (long long)(i + j * V) * s.x_rs);
    } else if (left > 0) {                                     // rows narrower than a vector
        for (; i < e; i += 16 * V)
            for (int j = 0; j < PER && i + j * V < e; j++)
                for (int k = 0; k < V; k++) sum[j][k] += k < left ? (A)widen(x[(long long)(i + j * V) * s.x_rs + c + k]) : (A)0;
    }
#pragma unroll
    for (int j = 0; j < PER; j++)
#pragma unroll
        for (int k = 0; k < V; k++) {
            A v = sum[j][k];
#pragma unroll
            for (int d = LANES; d < 64; d *= 2) v += __shfl_xor(v, d);
            if (lane < LANES) parts[(q * PER + j) * 64 + lane * V + k] = v;
        }
    __syncthreads();
    if (q || c0 + lane >= s.cols) return;
    A v = parts[lane];
#pragma unroll
    for (int r = 1; r < 16; r++) v += parts[r * 64 + lane];
    T* p = (T*)s.out + (long long)w * s.cols + c0 + lane;
    T y = round_to<T>(v);
    if (s.accumulate) y = round_to<T>(widen(*p) + widen(y));
    *p = y;
}

}  // namespace rp
