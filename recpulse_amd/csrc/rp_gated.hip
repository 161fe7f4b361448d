// Entry points of the gated linear layer, its kernels for any strides, sizes and types, and its backward pass.
//
//   z = x . W + b (columns [0, n): gate g, [n, 2 n): up u),  h = act(g) u
//   dz = [dh u act'(g) | dh act(g)],  dx = dz . W^T,  dW = x^T . dz,  db = sum of dz over the rows
//
// z is kept in the accumulate type (float32 for the 16-bit types), as the sums that they are: rounded to 16 bits, z's own error would reach dz beside dz's, and the gradients'
// error would be 1.3 times as large.  dz is rounded to the tensors' type, which is what the matrix cores multiply.
#include "rp_gated16.h"
#include "rp_grouped_sums.h"

namespace rp {

// Any strides and sizes: 64 rows x 32 columns of h a workgroup, 16 of k at a time through LDS, scalar multiply-adds
template <typename T, int GATE>
__global__ void __launch_bounds__(256) gated_any_kernel(GatedArgs g, int tiles_n, long long first) {
    using A = typename traits<T>::acc;
    constexpr int ROWS = 64, COLS = 32, K = 16;
    __shared__ A as[K][ROWS + 4], bs[K][2 * COLS + 4];
    const long long id = first + blockIdx.x;
    const int m0 = (int)(id / tiles_n) * ROWS, n0 = (int)(id % tiles_n) * COLS;
    const int t = threadIdx.x, tr = (t >> 4) * 4, tc = (t & 15) * 2;
    A acc[4][2][2] = {};
    for (int k0 = 0; k0 < g.k; k0 += K) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int e = t + 256 * i;
            const int ar = g.x_cs <= g.x_rs ? e / K : e % ROWS, ak = g.x_cs <= g.x_rs ? e % K : e / ROWS;
            const int bc = g.w_cs <= g.w_rs ? e % (2 * COLS) : e / K, bk = g.w_cs <= g.w_rs ? e / (2 * COLS) : e % K;
            const int col = n0 + bc % COLS;
            as[ak][ar] = m0 + ar < g.rows && k0 + ak < g.k ? (A)widen(((const T*)g.x)[(m0 + ar) * g.x_rs + (k0 + ak) * g.x_cs]) : (A)0;
            bs[bk][bc] = col < g.n && k0 + bk < g.k ? (A)widen(((const T*)g.w)[(k0 + bk) * g.w_rs + (col + (long long)(bc / COLS) * g.n) * g.w_cs]) : (A)0;
        }
        __syncthreads();
#pragma unroll
        for (int kk = 0; kk < K; kk++)
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    acc[i][j][0] += as[kk][tr + i] * bs[kk][tc + j];
                    acc[i][j][1] += as[kk][tr + i] * bs[kk][COLS + tc + j];
                }
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const int row = m0 + tr + i, col = n0 + tc + j;
            if (row >= g.rows || col >= g.n) continue;
            A gate = acc[i][j][0], up = acc[i][j][1];
            if (g.bias) {
                gate += widen(((const T*)g.bias)[col]);
                up += widen(((const T*)g.bias)[g.n + col]);
            }
            if (g.z) {
                ((A*)g.z)[(long long)row * 2 * g.n + col] = gate;
                ((A*)g.z)[(long long)row * 2 * g.n + g.n + col] = up;
            }
            ((T*)g.h)[row * g.h_rs + col] = round_to<T>(gate_value<GATE>(gate) * up);
        }
}

template <typename T>
static int launch_gated_any(const GatedArgs& g) {
    const int tiles_n = (g.n + 31) / 32;
    const long long blocks = (long long)((g.rows + 63) / 64) * tiles_n;
    return in_launches(blocks, 256, [&](unsigned count, long long first) {
        RP_DISPATCH_GATE(g.gate, hipLaunchKernelGGL((gated_any_kernel<T, GATE>), dim3(count), dim3(256), 0, current_stream(), g, tiles_n, first));
        return check_launch("gated_any_kernel") ? 0 : -1;
    });
}

// Element-wise passes: a workgroup takes 256 vectors of a row's columns at a time
constexpr int GATED_GRID = 1 << 20;

// h from z (float32 and float64, whose z comes from a product of its own)
template <typename T, int GATE>
__global__ void __launch_bounds__(256) gated_value_kernel(T* h, const typename traits<T>::acc* z, int rows, int n, long long h_rs, int across) {
    const long long total = (long long)rows * across;
    for (long long id = blockIdx.x; id < total; id += gridDim.x) {
        const int row = (int)(id / across), c = (int)(id % across) * 256 + threadIdx.x;
        if (c >= n) continue;
        const auto* zr = z + (long long)row * 2 * n;
        h[row * h_rs + c] = round_to<T>(gate_value<GATE>(zr[c]) * zr[n + c]);
    }
}

// dz from dh and z: N columns a thread where there are as many
template <typename T, int GATE>
__global__ void __launch_bounds__(256) gated_dz_kernel(T* dz, const T* dh, const typename traits<T>::acc* z, int rows, int n, long long dh_rs, int across) {
    using A = typename traits<T>::acc;
    constexpr int N = vec16<T>::N;
    const long long total = (long long)rows * across;
    for (long long id = blockIdx.x; id < total; id += gridDim.x) {
        const int row = (int)(id / across), c = ((int)(id % across) * 256 + (int)threadIdx.x) * N;
        const T* d = dh + row * dh_rs;
        const A* zr = z + (long long)row * 2 * n;
        T* out = dz + (long long)row * 2 * n;
        if (c >= n) continue;
        if (n >= N) {
            const RowVector<T> at(c, n);
            T dv[N], og[N], ou[N];
            A vg[N], vu[N];
            at.load(dv, d);
            A gate[N], up[N];
            __builtin_memcpy(gate, zr + at.at, sizeof(gate));
            __builtin_memcpy(up, zr + n + at.at, sizeof(up));
#pragma unroll
            for (int u = 0; u < N; u++) {
                const A v = widen(dv[u]);
                vg[u] = v * up[u] * gate_slope<GATE>(gate[u]);
                vu[u] = v * gate_value<GATE>(gate[u]);
            }
            round_vector<T>(og, vg);
            round_vector<T>(ou, vu);
            at.store(out, og);
            at.store(out + n, ou);
        } else {
            for (int u = 0; u < n; u++) {
                const A v = widen(d[u]), gate = zr[u], up = zr[n + u];
                out[u] = round_to<T>(v * up * gate_slope<GATE>(gate));
                out[n + u] = round_to<T>(v * gate_value<GATE>(gate));
            }
        }
    }
}

// dz and, in 16 bits, db from what has not been rounded yet (of the rounded dz, the error of sums of few rows was 1.5 times as large).  A workgroup makes 256 columns of each half of `per` rows and leaves
// their sums as a row of `parts` [chunks][2 n], which a second launch adds up in order: z and dh are read once.
template <typename T, int GATE>
__global__ void __launch_bounds__(256) gated_dz_sums_kernel(T* dz, float* parts, const T* dh, const float* z, int rows, int n, long long dh_rs, int strips, int per) {
    constexpr int N = vec16<T>::N, LANES = 32, WALK = 256 / LANES;
    __shared__ float room[WALK][LANES][2 * N + 1];
    const int strip = blockIdx.x % strips, chunk = blockIdx.x / strips, lane = threadIdx.x % LANES, slice = threadIdx.x / LANES, c = (strip * LANES + lane) * N;
    const RowVector<T> at(c < n ? c : n - N, n);
    float sums[2 * N] = {};
    const int end = rows - chunk * per < per ? rows : chunk * per + per;
    if (c < n)
#pragma unroll 2
        for (int row = chunk * per + slice; row < end; row += WALK) {
            const float* zr = z + (long long)row * 2 * n;
            T* out = dz + (long long)row * 2 * n;
            T dv[N], og[N], ou[N];
            float gate[N], up[N], vg[N], vu[N];
            at.load(dv, dh + row * dh_rs);
            __builtin_memcpy(gate, zr + at.at, sizeof(gate));
            __builtin_memcpy(up, zr + n + at.at, sizeof(up));
#pragma unroll
            for (int u = 0; u < N; u++) {
                const float v = widen(dv[u]);
                vg[u] = v * up[u] * gate_slope<GATE>(gate[u]);
                vu[u] = v * gate_value<GATE>(gate[u]);
                sums[u] += vg[u];
                sums[N + u] += vu[u];
            }
            round_vector<T>(og, vg);
            round_vector<T>(ou, vu);
            at.store(out, og);
            at.store(out + n, ou);
        }
#pragma unroll
    for (int u = 0; u < 2 * N; u++) room[slice][lane][u] = sums[u];
    __syncthreads();
    float* to = parts + (long long)chunk * 2 * n;
    for (int e = threadIdx.x; e < LANES * 2 * N; e += 256) {
        const int half = e / (LANES * N), l = e % (LANES * N) / N, u = e % N, col = (strip * LANES + l) * N;
        if (col >= n) continue;
        float sum = 0.f;
#pragma unroll
        for (int s = 0; s < WALK; s++) sum += room[s][l][half * N + u];
        to[half * n + RowVector<T>(col, n).at + u] = sum;      // (a last vector begins before its own columns and finds the same sums there)
    }
}
template <typename T> __device__ __forceinline__ void put_db(T* db, float sum, int accumulate) {
    const T y = round_to<T>(sum);
    *db = accumulate ? round_to<T>(widen(*db) + widen(y)) : y;
}
template <typename T>
__global__ void __launch_bounds__(1024) gated_db_kernel(T* db, const float* parts, int chunks, int width, int accumulate) {
    __shared__ float room[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x / 64, c = blockIdx.x * 64 + lane;
    float sum = 0.f;
    if (c < width)
#pragma unroll 8
        for (int i = wave; i < chunks; i += 16) sum += parts[(long long)i * width + c];
    room[wave][lane] = sum;
    __syncthreads();
    if (wave || c >= width) return;
#pragma unroll
    for (int w = 1; w < 16; w++) sum += room[w][lane];
    put_db(db + c, sum, accumulate);
}
// The same without memory for the parts, and for less than a vector of columns: z and dh are read again
template <typename T, int GATE>
__global__ void __launch_bounds__(1024) gated_db_any_kernel(T* db, const T* dh, const float* z, int rows, int n, long long dh_rs, int accumulate) {
    __shared__ float room[2][16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x / 64, c = blockIdx.x * 64 + lane;
    float sg = 0.f, su = 0.f;
    if (c < n)
        for (int row = wave; row < rows; row += 16) {
            const float v = widen(dh[row * dh_rs + c]), gate = z[(long long)row * 2 * n + c];
            sg += v * z[(long long)row * 2 * n + n + c] * gate_slope<GATE>(gate);
            su += v * gate_value<GATE>(gate);
        }
    room[0][wave][lane] = sg;
    room[1][wave][lane] = su;
    __syncthreads();
    if (wave || c >= n) return;
#pragma unroll
    for (int w = 1; w < 16; w++) { sg += room[0][w][lane]; su += room[1][w][lane]; }
    put_db(db + c, sg, accumulate);
    put_db(db + n + c, su, accumulate);
}

template <typename T>
static int launch_gated_dz(void* dz, const void* dh, const void* z, int rows, int n, int gate, long long dh_rs) {
    using A = typename traits<T>::acc;
    const int across = (n + 256 * vec16<T>::N - 1) / (256 * vec16<T>::N);
    const long long blocks = (long long)rows * across;
    RP_DISPATCH_GATE(gate, hipLaunchKernelGGL((gated_dz_kernel<T, GATE>), dim3((unsigned)(blocks < GATED_GRID ? blocks : GATED_GRID)), dim3(256), 0, current_stream(), (T*)dz, (const T*)dh, (const A*)z, rows, n, dh_rs, across));
    return check_launch("gated_dz_kernel") ? 0 : -1;
}
// dz and db in 16 bits
template <typename T>
static int launch_gated_dz_sums(void* dz, void* db, const void* dh, const void* z, int rows, int n, int gate, long long dh_rs, int accumulate) {
    // Two workgroups a CU, of at least eight rows, whose sums find room (fp16, us for both launches with 1, 2, 4 and 8 a CU, silu: 1999 x 1031 11.1 / 10.8 / 11.7 / 11.2, 8192 x 8192 165 / 165 / 176 / 176,
    // 8192 x 512 13.0 / 13.5 / 14.2 / 16.1; the exact gelu 16.7 / 14.5 / 16.0 / 14.9, 289 / 177 / 185 / 186, 21.4 / 17.4 / 16.4 / 19.5; dz alone, silu: 6.4, 163, 10.0)
    const int cus = device_cu_count() > 0 ? device_cu_count() : 256, strips = (n + 255) / 256;
    long long chunks = 2ll * cus / strips, room = (long long)(CallScratch::MOST / (8 * (size_t)n));
    if (chunks < 1) chunks = 1;
    if (chunks > (rows + 7) / 8) chunks = (rows + 7) / 8;
    if (chunks > room) chunks = room;
    if (n >= vec16<T>::N && chunks >= 1) {
        const int per = (int)((rows + chunks - 1) / chunks + 7) / 8 * 8;
        chunks = (rows + per - 1) / per;
        const CallScratch memory((size_t)chunks * 8 * n);
        if (memory.ptr) {
            RP_DISPATCH_GATE(gate, hipLaunchKernelGGL((gated_dz_sums_kernel<T, GATE>), dim3((unsigned)(strips * chunks)), dim3(256), 0, current_stream(), (T*)dz, (float*)memory.ptr, (const T*)dh, (const float*)z, rows, n, dh_rs, strips, per));
            if (!check_launch("gated_dz_sums_kernel")) return -1;
            hipLaunchKernelGGL((gated_db_kernel<T>), dim3((2 * n + 63) / 64), dim3(1024), 0, current_stream(), (T*)db, (const float*)memory.ptr, (int)chunks, 2 * n, accumulate);
            return check_launch("gated_db_kernel") ? 0 : -1;
        }
    }
    if (launch_gated_dz<T>(dz, dh, z, rows, n, gate, dh_rs) != 0) return -1;
    const int blocks = (n + 63) / 64;
    RP_DISPATCH_GATE(gate, hipLaunchKernelGGL((gated_db_any_kernel<T, GATE>), dim3(blocks), dim3(1024), 0, current_stream(), (T*)db, (const T*)dh, (const float*)z, rows, n, dh_rs, accumulate));
    return check_launch("gated_db_any_kernel") ? 0 : -1;
}

// C (+)= A . B by the kernels of the plain products, their partial sums in memory of this stream's own; where k would be split and there is no memory for that, as one group of all rows
static int product(void* C, const void* A, const void* B, const void* bias, int m, int k, int n, long long a_rs, long long a_cs, long long b_rs, long long b_cs, long long c_rs, int accumulate, int dtype) {
    int rc;
    bool refused;
    {
        const CallScratch memory(CallScratch::MOST);
        const GemmWorkspaceLoan loan(memory.ptr, CallScratch::MOST);
        rc = rp_hip_gemm_strided_batched(C, A, B, bias, 1, m, k, n, 0, a_rs, a_cs, 0, b_rs, b_cs, 0, c_rs, 1, accumulate, dtype);
        refused = loan.refused;
    }
    if (refused) rc = launch_grouped_rows(GroupedArgs{C, A, B, bias, nullptr, RowGroups{nullptr, nullptr, 1, m, 1}, k, n, a_rs, a_cs, 0, b_rs, b_cs, 0, c_rs, accumulate ? ACCUMULATE : 0}, dtype);
    return rc;
}

struct GatedGradients {
    void *dx, *dw, *db;
    long long dx_rs, dw_rs, dw_cs;
    int accumulate_dx, accumulate_dw, accumulate_db;
};
// dx = dz . W^T, dW = x^T . dz, db = sum of dz (asked for here by float32 and float64 layers).  16-bit layers of 512 rows and more as one group of a grouped layer, whose launches make the gradients side by side (fp16, us for all three as products of
// their own and so: 1999 x 519 x 2062 51.9 / 33.1, 4096 x 1031 x 4098 199 / 135, 1000 x 4096 x 1024 39.1 / 27.5, 8192 x 4096 x 16384 1795 / 1746; 300 x 200 x 2062 8.9 / 14.9, 1024 x 512 x 2048 14.4 / 16.8,
// 8192 x 256 x 512 50.7 / 56.7), the others as a linear layer's.
static int gated_gradients(const GatedGradients& o, const void* dz, const GatedArgs& g, int dtype) {
    const int n2 = 2 * g.n;
    if (!o.dx && !o.dw && !o.db) return 0;
    if (dtype_size(dtype) == 2 && g.rows >= 512 && g.k > 512 && (!o.dw || (o.dw_cs == 1 && o.dw_rs == n2))) {
        const RowGroups all{nullptr, nullptr, 1, g.rows, 1};
        const GroupedArgs x{o.dx, dz, g.w, nullptr, nullptr, all, n2, g.k, n2, 1, 0, g.w_cs, g.w_rs, 0, o.dx_rs, o.accumulate_dx ? ACCUMULATE : 0};
        const GroupedArgs w{o.dw, g.x, dz, nullptr, nullptr, all, g.k, n2, g.x_rs, g.x_cs, 0, n2, 1, 0, n2, o.accumulate_dw ? ACCUMULATE : 0};
        return launch_grouped_backward(x, w, GroupedSums{o.db, dz, all, n2, o.accumulate_db, n2}, dtype);
    }
    if (o.dw_cs == 1 && !o.accumulate_dx && !o.accumulate_dw && !o.accumulate_db) {      // (what it has made before it is refused memory is made again)
        const CallScratch memory(CallScratch::MOST);
        const GemmWorkspaceLoan loan(memory.ptr, CallScratch::MOST);
        const int rc = rp_hip_linear_backward(o.dx, o.dw, o.db, dz, g.x, g.w, g.rows, g.k, n2, g.x_rs, g.x_cs, g.w_rs, g.w_cs, o.dx_rs, 1, o.dw_rs, 1, 0, 0, 0, dtype);
        if (!loan.refused) return rc;
    }
    if (o.dx && product(o.dx, dz, g.w, nullptr, g.rows, n2, g.k, n2, 1, g.w_cs, g.w_rs, o.dx_rs, o.accumulate_dx, dtype) != 0) return -1;
    if (o.dw) {
        // (a transposed dW is the transposed product)
        const int rc = o.dw_cs == 1 ? product(o.dw, g.x, dz, nullptr, g.k, g.rows, n2, g.x_cs, g.x_rs, n2, 1, o.dw_rs, o.accumulate_dw, dtype)
                                    : product(o.dw, dz, g.x, nullptr, n2, g.rows, g.k, 1, n2, g.x_rs, g.x_cs, o.dw_cs, o.accumulate_dw, dtype);
        if (rc != 0) return -1;
    }
    return o.db ? rp_hip_reduce_rows(o.db, dz, g.rows, n2, o.accumulate_db, dtype) : 0;
}

// float32 and float64: z by a plain product, then h.  Without room for z, as many rows at a time as the stream's own memory holds.
template <typename T>
static int launch_gated_by_product(const GatedArgs& g, int dtype, bool* taken) {
    using A = typename traits<T>::acc;
    auto values = [&](void* h, const void* z, int rows) {
        const int across = (g.n + 255) / 256;
        const long long blocks = (long long)rows * across;
        RP_DISPATCH_GATE(g.gate, hipLaunchKernelGGL((gated_value_kernel<T, GATE>), dim3((unsigned)(blocks < GATED_GRID ? blocks : GATED_GRID)), dim3(256), 0, current_stream(), (T*)h, (const A*)z, rows, g.n, g.h_rs, across));
        return check_launch("gated_value_kernel") ? 0 : -1;
    };
    *taken = true;
    if (g.z) {
        if (product(g.z, g.x, g.w, g.bias, g.rows, g.k, 2 * g.n, g.x_rs, g.x_cs, g.w_rs, g.w_cs, 2ll * g.n, 0, dtype) != 0) return -1;
        return values(g.h, g.z, g.rows);
    }
    // (the memory's other half is for the product's own partial sums)
    constexpr size_t HALF = CallScratch::MOST / 2;
    const long long most = (long long)(HALF / (2 * (size_t)g.n * sizeof(A)));
    if (most < 1) { *taken = false; return 0; }
    const int chunk = most < g.rows ? (int)most : g.rows;
    const CallScratch memory(CallScratch::MOST);
    if (!memory.ptr) { *taken = false; return 0; }
    for (int row = 0; row < g.rows; row += chunk) {
        const int rows = g.rows - row < chunk ? g.rows - row : chunk;
        const T* x = (const T*)g.x + row * g.x_rs;
        bool refused;
        int rc;
        {
            const GemmWorkspaceLoan loan((char*)memory.ptr + HALF, HALF);
            rc = rp_hip_gemm_strided_batched(memory.ptr, x, g.w, g.bias, 1, rows, g.k, 2 * g.n, 0, g.x_rs, g.x_cs, 0, g.w_rs, g.w_cs, 0, 2ll * g.n, 1, 0, dtype);
            refused = loan.refused;
        }
        if (refused) rc = launch_grouped_rows(GroupedArgs{memory.ptr, x, g.w, g.bias, nullptr, RowGroups{nullptr, nullptr, 1, rows, 1}, g.k, 2 * g.n, g.x_rs, g.x_cs, 0, g.w_rs, g.w_cs, 0, 2ll * g.n, 0}, dtype);
        if (rc != 0 || values((T*)g.h + row * g.h_rs, memory.ptr, rows) != 0) return -1;
    }
    return 0;
}

// bf16 and fp16 on MFMA tiles: operands with a unit stride and rows of at least a 16-byte vector
static int gated16_forward(const GatedArgs& g, int dtype, bool* taken) {
    *taken = false;
    if (g.x_cs != 1 || (g.w_cs != 1 && g.w_rs != 1) || path_disabled("mfma")) return 0;
    const bool b_mc = g.w_cs == 1;
    const long long w_stride = b_mc ? g.w_rs : g.w_cs;
    // rows as long as they have to be, no further apart than the tiles' 32-bit offsets reach
    if (g.k < 8 || g.x_rs < g.k || g.x_rs >= (1 << 22) || w_stride >= (1 << 22)) return 0;
    if (b_mc ? g.n < 8 || w_stride < 2ll * g.n : w_stride < g.k || (2ll * g.n + 256) * w_stride * 2 > 0x7fffffffll) return 0;
    *taken = true;
    const bool ragged = ((uintptr_t)g.x & 15) || ((uintptr_t)g.w & 15) || g.x_rs % 8 || w_stride % 8 || g.k % 8 || (b_mc && g.n % 8);
    Plan p{FAM_MFMA16, 64, 64, false, b_mc, true, ""};
    p.ragged = ragged;
    choose_tile16(p, 1, g.rows, g.k, 2 * g.n);
    // (of four slabs the epilogue is most of the work, and tiles of 128 have two workgroups a CU for it: fp16, z kept, us on 256 and on 128: 256 -> 2048 of 1999 rows 36.9 / 18.9, of 4000 36.1 / 29.8,
    // of 8192 55.0 / 53.9; 256 -> 8192 of 4000 133 / 106, of 8192 221 / 231; 512 -> 4096 of 2500 44.4 / 46.7)
    if (p.bm == 256 && g.k <= 4 * M16_BK) p.bm = p.bn = 128;
    if (!ragged && p.bm == 256 && p.bn == 256) {
        const int edge = g.rows % 256 || g.n % 128 || g.k % M16_BK ? M16_EDGE : M16_WHOLE;
        return dtype == RP_DTYPE_BFLOAT16 ? launch_gated16_256_bf16(g, edge) : launch_gated16_256_f16(g, edge);
    }
    const int edge = ragged ? M16_RAGGED : M16_EDGE;
    if (g.rows > 64 && p.bm >= 128 && p.bn >= 128) return launch_gated16_128(g, edge, dtype);
    // Few tiles: k in shares of at least eight slabs, a workgroup a CU where that keeps seven eighths of them busy, else two (bf16, us with one, two and three a CU: 16 rows, 4096 -> 8192 32.4 / 32.1 / 36.7
    // (one share: 40), -> 5120 18.9 / 19.8 / 23.0, -> 6144 31.2 / 25.4 / 29.7, -> 10240 53.2 / 41.3 / 50.1; 64 rows, -> 8192 34.2 / 38.8 / 38.8, -> 6144 33.4 / 31.7 / 31.5)
    const long long tiles = (long long)((g.rows + 63) / 64) * ((g.n + 63) / 64), share_bytes = 8ll * g.rows * g.n;
    const int cus = device_cu_count() > 0 ? device_cu_count() : 256, slabs = (g.k + M16_BK - 1) / M16_BK;
    long long count = cus / tiles;
    if (8 * count * tiles < 7ll * cus) count = 2ll * cus / tiles;
    if (count > slabs / 8) count = slabs / 8;
    if (count > (long long)CallScratch::MOST / share_bytes) count = (long long)CallScratch::MOST / share_bytes;
    if (count >= 2 && !path_disabled("gated_shares")) {
        const int per = (int)((slabs + count - 1) / count), shares = (slabs + per - 1) / per;
        const CallScratch memory((size_t)(shares * share_bytes));
        if (memory.ptr) return launch_gated16_64x128(g, GatedShares{shares, per * M16_BK, (float*)memory.ptr}, edge, dtype);
    }
    return launch_gated16_64x128(g, GatedShares{1, 0, nullptr}, edge, dtype);
}

static bool gated_args_ok(const char* who, bool pointers, int rows, int k, int n, int gate, std::initializer_list<long long> strides, int dtype) {
    if (!pointers || rows <= 0 || k <= 0 || n <= 0 || rows > (1 << 29) || n > (1 << 26)) {
        set_error("%s: null operand, non-positive extent, more than 2^29 rows or 2^26 columns (rows=%d k=%d n=%d)", who, rows, k, n);
        return false;
    }
    if (!dtype_size(dtype)) { set_error("%s: unsupported dtype %d", who, dtype); return false; }
    if (gate < RP_GATE_SILU || gate > RP_GATE_SIGMOID) { set_error("%s: unknown gate %d", who, gate); return false; }
    for (long long s : strides)
        if (s < 0) { set_error("%s: negative stride", who); return false; }
    return true;
}
static bool gated_rows_apart(const char* who, const char* what, int rows, int width, long long rs) {
    if (rows == 1 || rs >= width) return true;
    set_error("%s: rows of %s are %lld elements apart and hold %d", who, what, rs, width);
    return false;
}

}  // namespace rp

using namespace rp;

extern "C" {

int rp_hip_gated_linear_forward(void* h, void* z, const void* x, const void* w, const void* bias, int rows, int k, int n, int gate,
                                long long x_rs, long long x_cs, long long w_rs, long long w_cs, long long h_rs, int dtype) {
    const char* who = "rp_hip_gated_linear_forward";
    if (!gated_args_ok(who, h && x && w, rows, k, n, gate, {x_rs, x_cs, w_rs, w_cs, h_rs}, dtype) || !gated_rows_apart(who, "h", rows, n, h_rs)) return -1;
    const GatedArgs g{h, z, x, w, bias, rows, k, n, gate, x_rs, x_cs, w_rs, w_cs, h_rs};
    if (dtype == RP_DTYPE_FLOAT32 || dtype == RP_DTYPE_FLOAT64) {
        bool taken;
        const int rc = dtype == RP_DTYPE_FLOAT32 ? launch_gated_by_product<float>(g, dtype, &taken) : launch_gated_by_product<double>(g, dtype, &taken);
        if (rc != 0 || taken) return rc;
    } else {
        bool taken;
        const int rc = gated16_forward(g, dtype, &taken);
        if (rc != 0 || taken) return rc;
    }
    RP_DISPATCH_DTYPE(dtype, return launch_gated_any<T>(g));
    return -1;
}

int rp_hip_gated_linear_backward(void* dx, void* dw, void* db, void* dz, const void* dh, const void* z, const void* x, const void* w, int rows, int k, int n, int gate,
                                 long long dh_rs, long long x_rs, long long x_cs, long long w_rs, long long w_cs, long long dx_rs, long long dw_rs, long long dw_cs,
                                 int accumulate_dx, int accumulate_dw, int accumulate_db, int dtype) {
    const char* who = "rp_hip_gated_linear_backward";
    if (!gated_args_ok(who, dz && dh && z && (!dx || w) && (!dw || x), rows, k, n, gate, {dh_rs, x_rs, x_cs, w_rs, w_cs, dx_rs, dw_rs, dw_cs}, dtype)) return -1;
    if (dx && !gated_rows_apart(who, "dx", rows, k, dx_rs)) return -1;
    if (dw && !(dw_cs == 1 && (k == 1 || dw_rs >= 2ll * n)) && !(dw_rs == 1 && dw_cs >= k)) { set_error("%s: dw has unit stride along one axis and rows that do not overlap along the other", who); return -1; }
    if (db && dtype_size(dtype) == 2) {
        const int rc = dtype == RP_DTYPE_BFLOAT16 ? launch_gated_dz_sums<bf16_t>(dz, db, dh, z, rows, n, gate, dh_rs, accumulate_db) : launch_gated_dz_sums<f16_t>(dz, db, dh, z, rows, n, gate, dh_rs, accumulate_db);
        if (rc != 0) return -1;
        db = nullptr;
    } else {
        RP_DISPATCH_DTYPE(dtype, if (launch_gated_dz<T>(dz, dh, z, rows, n, gate, dh_rs) != 0) return -1);
    }
    return gated_gradients(GatedGradients{dx, dw, db, dx_rs, dw_rs, dw_cs, accumulate_dx, accumulate_dw, accumulate_db}, dz, GatedArgs{nullptr, nullptr, x, w, nullptr, rows, k, n, gate, x_rs, x_cs, w_rs, w_cs, 0}, dtype);
}

}  // extern "C"
