// An adapter's narrow products and the gradients of its factors for fp32, fp64 and operands of any strides, on scalar multiply-adds in the accumulate type.
//
// h[i] = scale x[i] . A_a has rank outputs a row and k products each: 64 x 64 tiles of it would leave most CUs without one and each with a long chain.
// Here a workgroup owns eight rows and sixteen of the rank, and its 64 (float64: 32) groups of sixteen lanes share k: the chain of loads is what bounds it
// (fp32, 2 rows of 2293 and rank 64 14 us; 240 of 3672 and rank 16 in 44 segments 21).
// dB_a = sum of h[i]^T dy[i] (and dA_a^T = sum of u[i]^T x[i]): a workgroup owns 64 columns and sixteen of the rank, a column a lane, and its sixteen waves share the
// rows; the row's sixteen low values are uniform, one scalar load.
#include "rp_grouped.h"

#include <type_traits>

namespace rp {

constexpr int NR_ROWS = 8, NR_COLS = 16;                         // rows and columns of a workgroup
template <typename A> constexpr int nr_lanes() { return sizeof(A) == 8 ? 32 : 64; }         // lanes that share k
constexpr int NW_WAVES = 16;                                     // waves that share the rows

template <typename T>
__global__ void __launch_bounds__(NR_COLS * nr_lanes<typename traits<T>::acc>()) narrow_rows_kernel(GroupedArgs g, int col_blocks, long long first) {
    using A = typename traits<T>::acc;
    constexpr int NR_LANES = nr_lanes<A>();
    __shared__ A sums[NR_LANES][NR_ROWS][NR_COLS + 1];
    const long long id = first + blockIdx.x;
    const RowTile rt = find_row_tile_number(g.gr, NR_ROWS, (int)(id / col_blocks));
    if (rt.group < 0) return;
    const int c = threadIdx.x % NR_COLS, p = threadIdx.x / NR_COLS, col = (int)(id % col_blocks) * NR_COLS + c, last = rt.end - rt.begin - 1;
    const T* x = (const T*)g.A + rt.begin * g.a_rs;
    const T* f = (const T*)g.B + rt.weight * g.b_ws + (col < g.n ? col : g.n - 1) * g.b_cs;
    A acc[NR_ROWS];
#pragma unroll
    for (int r = 0; r < NR_ROWS; r++) acc[r] = 0;
#pragma unroll 4
    for (int k = p; k < g.k; k += NR_LANES) {
        const A fv = widen(f[k * g.b_rs]);
#pragma unroll
        for (int r = 0; r < NR_ROWS; r++) acc[r] += widen(x[(r < last ? r : last) * g.a_rs + k * g.a_cs]) * fv;       // (rows past the segment repeat its last and are not stored)
    }
#pragma unroll
    for (int r = 0; r < NR_ROWS; r++) sums[p][r][c] = acc[r];
    __syncthreads();
    const int r = threadIdx.x / NR_COLS;
    if (r >= NR_ROWS || r > last || col >= g.n) return;
    A s = sums[0][r][c];
#pragma unroll
    for (int q = 1; q < NR_LANES; q++) s += sums[q][r][c];
    ((A*)g.C)[(rt.begin + r) * g.c_rs + col] = g.scales ? (A)g.scales[rt.weight] * s : s;
}

// TRANSPOSED: dA; else dB
template <typename T, bool TRANSPOSED>
__global__ void __launch_bounds__(NW_WAVES * 64) narrow_weights_kernel(GroupedArgs g, int strips, int rank_blocks, long long first) {
    using A = typename traits<T>::acc;
    extern __shared__ __attribute__((aligned(16))) unsigned char nw_lds[];
    A (*sums)[NR_COLS][65] = (A (*)[NR_COLS][65])nw_lds;         // [NW_WAVES]
    const long long block = first + blockIdx.x;
    const int strip = (int)(block % strips), rb = (int)(block / strips % rank_blocks), w = (int)(block / strips / rank_blocks);
    const int width = TRANSPOSED ? g.k : g.n, rank = TRANSPOSED ? g.n : g.k;
    const T* s = (const T*)(TRANSPOSED ? g.A : g.B);
    const A* low = (const A*)(TRANSPOSED ? g.B : g.A);
    const long long s_rs = TRANSPOSED ? g.a_rs : g.b_rs, s_cs = TRANSPOSED ? g.a_cs : g.b_cs, l_rs = TRANSPOSED ? g.b_rs : g.a_rs;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = strip * 64 + lane, r0 = rb * NR_COLS;
    A acc[NR_COLS];
#pragma unroll
    for (int r = 0; r < NR_COLS; r++) acc[r] = 0;
    bool any = false;
    for_groups_of(g.gr, w, [&](int begin, int end) {
        any = true;
#pragma unroll 4
        for (int i = begin + wave; i < end; i += NW_WAVES) {
            const A v = col < width ? (A)widen(s[i * s_rs + col * s_cs]) : (A)0;
            const A* l = low + i * l_rs;
#pragma unroll
            for (int r = 0; r < NR_COLS; r++) acc[r] += v * l[r0 + r < rank ? r0 + r : rank - 1];
        }
    });
    if (!any) {                                                  // an adapter without rows: zeros, or what is there
        const int r = TRANSPOSED ? threadIdx.x % NR_COLS : threadIdx.x / 64, c = TRANSPOSED ? threadIdx.x / NR_COLS : threadIdx.x % 64;
        if (!g.accumulate && r0 + r < rank && strip * 64 + c < width) ((T*)g.C)[w * g.c_ws + (TRANSPOSED ? (strip * 64 + c) * g.c_rs + r0 + r : (r0 + r) * g.c_rs + strip * 64 + c)] = round_to<T>((A)0);
        return;
    }
#pragma unroll
    for (int r = 0; r < NR_COLS; r++) sums[wave][r][lane] = acc[r];
    __syncthreads();
    {
        const int id = threadIdx.x, r = TRANSPOSED ? id % NR_COLS : id / 64, c = TRANSPOSED ? id / NR_COLS : id % 64;       // a value a thread
        static_assert(NR_COLS == NW_WAVES, "as many values as threads");
        if (r0 + r >= rank || strip * 64 + c >= width) return;
        A t = sums[0][r][c];
#pragma unroll
        for (int p = 1; p < NW_WAVES; p++) t += sums[p][r][c];
        T* at = (T*)g.C + w * g.c_ws + (TRANSPOSED ? (strip * 64 + c) * g.c_rs + r0 + r : (r0 + r) * g.c_rs + strip * 64 + c);
        T y = round_to<T>(t);
        if (g.accumulate) y = round_to<T>(widen(*at) + widen(y));
        *at = y;
    }
}

int launch_narrow_rows(const GroupedArgs& g, int dtype) {
    const int col_blocks = (g.n + NR_COLS - 1) / NR_COLS;
    const long long all = row_tile_numbers(g.gr.rows, g.gr.groups, NR_ROWS) * col_blocks;
    RP_DISPATCH_DTYPE(dtype, {
        constexpr int threads = NR_COLS * nr_lanes<typename traits<T>::acc>();
        return in_launches(all, threads, [&](unsigned blocks, long long first) -> int {
            hipLaunchKernelGGL(narrow_rows_kernel<T>, dim3(blocks), dim3(threads), 0, current_stream(), g, col_blocks, first);
            return check_launch("narrow_rows_kernel") ? 0 : -1;
        });
    });
    return 0;
}

int launch_narrow_weights(const GroupedArgs& g, GroupedLow low, int dtype) {
    const bool transposed = low == LOW_B;
    const int width = transposed ? g.k : g.n, rank = transposed ? g.n : g.k, strips = (width + 63) / 64, rank_blocks = (rank + NR_COLS - 1) / NR_COLS;
    RP_DISPATCH_DTYPE(dtype, {
        constexpr int lds = NW_WAVES * NR_COLS * 65 * (int)sizeof(typename traits<T>::acc);
        auto launch = [&](auto kern) {
            if (!check_hip(hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, lds), "hipFuncSetAttribute")) return -1;
            return in_launches((long long)strips * rank_blocks * g.gr.weights, NW_WAVES * 64, [&](unsigned blocks, long long first) -> int {
                hipLaunchKernelGGL(kern, dim3(blocks), dim3(NW_WAVES * 64), lds, current_stream(), g, strips, rank_blocks, first);
                return check_launch("narrow_weights_kernel") ? 0 : -1;
            });
        };
        return transposed ? launch(narrow_weights_kernel<T, true>) : launch(narrow_weights_kernel<T, false>);
    });
    return 0;
}

}  // namespace rp
