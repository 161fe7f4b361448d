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

// Block `id`: 64 columns of one group, a column a lane, the rows dealt to 16 sums that are added in order, whatever the number of waves.  Few groups are short of
// workgroups and bound by how long a load takes to come: 16 rows a wave are on their way at a time.  parts: room for 16 x 64 sums.
template <typename T, int WAVES>
__device__ __forceinline__ void grouped_sums_block(const GroupedSums& s, int id, typename traits<T>::acc* parts) {
    using A = typename traits<T>::acc;
    constexpr int PER = 16 / WAVES;
    const int strips = (s.cols + 63) / 64, w = id / strips, lane = threadIdx.x & 63, c = (id - w * strips) * 64 + lane, q = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    A sum[PER] = {};
    if (c < s.cols) {
        const int e = s.gr.end(w);
        const T* x = (const T*)s.x + c;
        int i = s.gr.begin(w) + q * PER;
#pragma unroll WAVES
        for (; i + PER <= e; i += 16)
#pragma unroll
            for (int j = 0; j < PER; j++) sum[j] += widen(x[(i + j) * s.x_rs]);
#pragma unroll
        for (int j = 0; j < PER; j++)
            if (i + j < e) sum[j] += widen(x[(i + j) * s.x_rs]);
    }
#pragma unroll
    for (int j = 0; j < PER; j++) parts[(q * PER + j) * 64 + lane] = sum[j];
    __syncthreads();
    if (q || c >= s.cols) return;
    A v = parts[lane];
#pragma unroll
    for (int i = 1; i < 16; i++) v += parts[i * 64 + lane];
    T* p = (T*)s.out + (long long)w * s.cols + c;
    T y = round_to<T>(v);
    if (s.accumulate) y = round_to<T>(widen(*p) + widen(y));
    *p = y;
}

}  // namespace rp
