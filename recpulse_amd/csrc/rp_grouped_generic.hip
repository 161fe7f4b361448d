// Grouped products for any strides, sizes and types: 64 x 64 tiles, 16 of k at a time through LDS, scalar multiply-adds, 4 x 4 outputs a
// thread.  What no other kernel takes comes here: the narrowest widths, operands without a unit stride, and the adapters' term of
// float32 and float64, whose rank is a few steps of k.  Sums in the accumulate type, rounded at the end, and once more where they are added to what the
// output holds (as a product of its own would be).
#include "rp_grouped_sums.h"

#include <type_traits>

namespace rp {

constexpr int GG_T = 64, GG_K = 16;

// One 64 x 64 tile: acc += A[0 .. m, 0 .. k] . B[0 .. k, 0 .. n], both masked past their extents.  Pointers at the tile's origin.
template <typename TA, typename TB, typename A>
__device__ __forceinline__ void generic_tile(A acc[4][4], A (*as)[GG_T + 4], A (*bs)[GG_T + 4], const TA* a, const TB* b, int m, int n, int k,
                                             long long a_rs, long long a_cs, long long b_rs, long long b_cs) {
    const int t = threadIdx.x, tr = (t >> 4) * 4, tc = (t & 15) * 4;
    for (int k0 = 0; k0 < k; k0 += GG_K) {
        A av[4], bv[4];
        // neighbouring threads along the axis with the smaller stride
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int id = t + 256 * i;
            const int ar = a_cs <= a_rs ? id / GG_K : id % GG_T, ak = a_cs <= a_rs ? id % GG_K : id / GG_T;
            const int bc = b_cs <= b_rs ? id % GG_T : id / GG_K, bk = b_cs <= b_rs ? id / GG_T : id % GG_K;
            av[i] = ar < m && k0 + ak < k ? (A)widen(a[ar * a_rs + (k0 + ak) * a_cs]) : (A)0;
            bv[i] = bc < n && k0 + bk < k ? (A)widen(b[(k0 + bk) * b_rs + bc * b_cs]) : (A)0;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int id = t + 256 * i;
            const int ar = a_cs <= a_rs ? id / GG_K : id % GG_T, ak = a_cs <= a_rs ? id % GG_K : id / GG_T;
            const int bc = b_cs <= b_rs ? id % GG_T : id / GG_K, bk = b_cs <= b_rs ? id / GG_T : id % GG_K;
            as[ak][ar] = av[i];
            bs[bk][bc] = bv[i];
        }
        __syncthreads();
#pragma unroll
        for (int kk = 0; kk < GG_K; kk++)
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) acc[i][j] += as[kk][tr + i] * bs[kk][tc + j];
    }
}

template <typename TA, typename T>
__global__ void __launch_bounds__(256) grouped_rows_generic_kernel(GroupedArgs g, int tiles_n, long long first) {
    using A = typename traits<T>::acc;
    __shared__ A as[GG_K][GG_T + 4], bs[GG_K][GG_T + 4];
    const long long id = first + blockIdx.x;
    const RowTile rt = find_row_tile_number(g.gr, GG_T, (int)(id / tiles_n));
    if (rt.group < 0) return;
    const int n0 = (int)(id % tiles_n) * GG_T, m = rt.end - rt.begin, n = g.n - n0 < GG_T ? g.n - n0 : GG_T;
    const int tr = (threadIdx.x >> 4) * 4, tc = (threadIdx.x & 15) * 4;
    A acc[4][4] = {};
    generic_tile<TA, T, A>(acc, as, bs, (const TA*)g.A + rt.begin * g.a_rs, (const T*)g.B + rt.weight * g.b_ws + n0 * g.b_cs, m, n, g.k, g.a_rs, g.a_cs, g.b_rs, g.b_cs);
    const T* bias = (const T*)g.bias;
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if (tr + i >= m || tc + j >= n) continue;
            T* p = (T*)g.C + (rt.begin + tr + i) * g.c_rs + n0 + tc + j;
            A v = acc[i][j];
            if (bias) v += widen(bias[(long long)rt.weight * g.n + n0 + tc + j]);
            if (g.accumulate == ACCUMULATE_JOINED) v += widen(*p);
            T y = round_to<T>(v);
            if (g.accumulate == ACCUMULATE) y = round_to<T>(widen(*p) + widen(y));
            *p = y;
        }
}

// A tile of C_w is a sum over the rows of group w
template <typename T>
__global__ void __launch_bounds__(256) grouped_weights_generic_kernel(GroupedArgs g, int tiles_k, int tiles_n, long long first) {
    using A = typename traits<T>::acc;
    __shared__ A as[GG_K][GG_T + 4], bs[GG_K][GG_T + 4];
    const long long id = first + blockIdx.x;
    const int tn = (int)(id % tiles_n), tk = (int)(id / tiles_n % tiles_k), w = (int)(id / tiles_n / tiles_k);
    const int m0 = tk * GG_T, n0 = tn * GG_T, m = g.k - m0 < GG_T ? g.k - m0 : GG_T, n = g.n - n0 < GG_T ? g.n - n0 : GG_T, b = g.gr.begin(w), e = g.gr.end(w);
    const int tr = (threadIdx.x >> 4) * 4, tc = (threadIdx.x & 15) * 4;
    A acc[4][4] = {};
    generic_tile<T, T, A>(acc, as, bs, (const T*)g.A + b * g.a_rs + m0 * g.a_cs, (const T*)g.B + b * g.b_rs + n0 * g.b_cs, m, n, e - b, g.a_cs, g.a_rs, g.b_rs, g.b_cs);
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if (tr + i >= m || tc + j >= n) continue;
            T* p = (T*)g.C + w * g.c_ws + (m0 + tr + i) * g.c_rs + n0 + tc + j;
            T y = round_to<T>(acc[i][j]);
            if (g.accumulate) y = round_to<T>(widen(*p) + widen(y));
            *p = y;
        }
}

template <typename T>
__global__ void __launch_bounds__(1024) grouped_sums_kernel(GroupedSums s, long long blocks) {
    __shared__ typename traits<T>::acc parts[16 * 64];
    for (long long id = blockIdx.x; id < blocks; id += gridDim.x) {
        grouped_sums_block<T, 16>(s, id, parts);
        __syncthreads();
    }
}

int launch_grouped_rows_generic(const GroupedArgs& g, bool low, int dtype) {
    const int tiles_n = (g.n + GG_T - 1) / GG_T;
    return in_launches(row_tile_numbers(g.gr.rows, g.gr.groups, GG_T) * tiles_n, 256, [&](unsigned blocks, long long first) -> int {
        RP_DISPATCH_DTYPE(dtype, {
            if (low) hipLaunchKernelGGL((grouped_rows_generic_kernel<typename traits<T>::acc, T>), dim3(blocks), dim3(256), 0, current_stream(), g, tiles_n, first);
            else hipLaunchKernelGGL((grouped_rows_generic_kernel<T, T>), dim3(blocks), dim3(256), 0, current_stream(), g, tiles_n, first);
        });
        return check_launch("grouped_rows_generic_kernel") ? 0 : -1;
    });
}

int launch_grouped_weights_generic(const GroupedArgs& g, int dtype) {
    const int tiles_k = (g.k + GG_T - 1) / GG_T, tiles_n = (g.n + GG_T - 1) / GG_T;
    return in_launches((long long)g.gr.weights * tiles_k * tiles_n, 256, [&](unsigned blocks, long long first) -> int {
        RP_DISPATCH_DTYPE(dtype, hipLaunchKernelGGL(grouped_weights_generic_kernel<T>, dim3(blocks), dim3(256), 0, current_stream(), g, tiles_k, tiles_n, first));
        return check_launch("grouped_weights_generic_kernel") ? 0 : -1;
    });
}

int launch_grouped_sums(const GroupedSums& s, int dtype) {
    const long long blocks = sum_blocks(s);
    RP_DISPATCH_DTYPE(dtype, hipLaunchKernelGGL(grouped_sums_kernel<T>, dim3((unsigned)(blocks < 1 << 20 ? blocks : 1 << 20)), dim3(1024), 0, current_stream(), s, blocks));
    return check_launch("grouped_sums_kernel") ? 0 : -1;
}

}  // namespace rp
