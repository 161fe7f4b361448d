// Layer norm of rows and its gradients, all types.
//
//   mean = sum x / d,  r = 1 / sqrt(sum (x - mean)^2 / d + eps),  h = (x - mean) r,  y = h w + b
//   g = dy w,  dx = r (g - sum g / d - h sum(g h) / d),  dw = sum over the rows of dy h,  db = sum over the rows of dy
//
// What bounds it is memory: x and y once, dy, x and dx once.  A team of threads (a wave, or a workgroup) holds a row in registers, so that the second sum over a row (of the
// squares of x - mean: the difference of two large sums would lose the variance of rows far from zero) costs no second read.  Backward, a team walks rows with its columns' sums of dw and db in
// registers and leaves them as one row of partial sums, which a second launch adds up in order.  Sums and the values between are float32 (float64 for float64), each output is rounded once.
#include "rp_teams.h"

namespace rp {

constexpr int NORM_BLOCKS = 512;        // most workgroups of a backward launch, each of which leaves a row of partial sums
constexpr int NORM_GRID = 1 << 20;      // and of those for rows that are not held in registers, which walk on from there (a launch has fewer than 2^32 threads)
static int norm_grid(int blocks) { return blocks < NORM_GRID ? blocks : NORM_GRID; }

template <typename A> struct NormArgs {
    void *y, *dx, *dw, *db;
    const void *x, *w, *b, *dy;
    A *stats, *partials;
    int rows, d;
    long long y_rs, x_rs, dy_rs, dx_rs;
    A eps;
    int accumulate_dx, accumulate_dw, accumulate_db;
};

__device__ __forceinline__ float one_over_root(float v) { return 1.f / sqrtf(v); }
__device__ __forceinline__ double one_over_root(double v) { return 1.0 / sqrt(v); }

// Rows of up to four vectors a thread, two of 1024 threads: the next row's loads fly while a row is added up, and weight and bias are loaded once.  Up to a width of 8192 (16 bits) that fits the registers.
// Wider, the sums of dw and db beside it do not: 122 registers of a thread lie in scratch memory from 8193 on in bf16, 326 from 16385 and 846 from 32769 (8192 rows, us and TB/s backward with dw and db, and for
// dx alone: width 8192 117, 3.4 and 78, 5.2; 12288 779, 0.8 and 113, 5.4; 16384 816, 1.0 and 145, 5.6; float32, 4096 rows, 12288 309, 2.0 and 114, 5.3)
constexpr bool norm_ahead(int lanes, int steps, int elem) { return elem < 8 && steps * (lanes == 1024 ? 4 : 2) <= 8; }

template <typename T, int LANES, int STEPS>
__global__ void __launch_bounds__(LANES < 256 ? 256 : LANES) layer_norm_kernel(NormArgs<typename traits<T>::acc> g) {
    using A = typename traits<T>::acc;
    constexpr int TEAMS = LANES < 256 ? 256 / LANES : 1, N = vec16<T>::N;
    constexpr bool AHEAD = norm_ahead(LANES, STEPS, sizeof(T));
    __shared__ A room[2][LANES / 64];
    const int lane = threadIdx.x % LANES, stride = (int)gridDim.x * TEAMS;
    int row = (int)blockIdx.x * TEAMS + (TEAMS > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / LANES) : 0);
    RowVector<T> at[STEPS];
    T next[STEPS][N], w[STEPS][N], b[STEPS][N];
#pragma unroll
    for (int s = 0; s < STEPS; s++) at[s] = RowVector<T>((s * LANES + lane) * N, g.d);
    auto load_row = [&](int r) {
        const T* x = (const T*)g.x + (r < g.rows ? r : g.rows - 1) * g.x_rs;      // (a row again rather than none)
#pragma unroll
        for (int s = 0; s < STEPS; s++) at[s].load(next[s], x);
    };
    auto load_weights = [&]() {
#pragma unroll
        for (int s = 0; s < STEPS; s++) {
            if (g.w) at[s].load(w[s], (const T*)g.w);
            if (g.b) at[s].load(b[s], (const T*)g.b);
        }
    };
    if (AHEAD) load_row(row);
    if (AHEAD) load_weights();
    // (whole teams; a workgroup of several has no barriers)
    for (; row < g.rows; row += stride) {
        T raw[STEPS][N];
        if (!AHEAD) load_row(row);
        __builtin_memcpy(raw, next, sizeof(raw));
        if (AHEAD) load_row(row + stride);
        A sum[1] = {};
#pragma unroll
        for (int s = 0; s < STEPS; s++)
#pragma unroll
            for (int u = 0; u < N; u++) sum[0] += at[s].has(u) ? widen(raw[s][u]) : (A)0;
        team_sums_in_turn<LANES>(sum, room[0]);
        const A mean = sum[0] / (A)g.d;
        A squares[1] = {};
#pragma unroll
        for (int s = 0; s < STEPS; s++)
#pragma unroll
            for (int u = 0; u < N; u++) {
                const A c = at[s].has(u) ? widen(raw[s][u]) - mean : (A)0;
                squares[0] += c * c;
            }
        if (!AHEAD) load_weights();
        team_sums_in_turn<LANES>(squares, room[1]);
        const A r = one_over_root(squares[0] / (A)g.d + g.eps);
        if (g.stats && lane == 0) {
            g.stats[2 * (long long)row] = mean;
            g.stats[2 * (long long)row + 1] = r;
        }
        T* y = (T*)g.y + row * g.y_rs;
#pragma unroll
        for (int s = 0; s < STEPS; s++) {
            T out[N];
            A value[N];
#pragma unroll
            for (int u = 0; u < N; u++) {
                A h = (widen(raw[s][u]) - mean) * r;
                if (g.w) h *= widen(w[s][u]);
                if (g.b) h += widen(b[s][u]);
                value[u] = h;
            }
            round_vector<T>(out, value);
            at[s].store(y, out);
        }
    }
}

template <typename T, int LANES, int STEPS, bool WEIGHTS>
__global__ void __launch_bounds__(LANES < 256 ? 256 : LANES) layer_norm_backward_kernel(NormArgs<typename traits<T>::acc> g) {
    using A = typename traits<T>::acc;
    constexpr int TEAMS = LANES < 256 ? 256 / LANES : 1, N = vec16<T>::N;
    constexpr bool AHEAD = norm_ahead(LANES, STEPS, sizeof(T));
    extern __shared__ __attribute__((aligned(16))) char lds[];       // 4 LANES / 64 values; with WEIGHTS and several teams 2 d more
    A* room = (A*)lds;
    const int lane = threadIdx.x % LANES, team = TEAMS > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / LANES) : 0, stride = (int)gridDim.x * TEAMS;
    RowVector<T> at[STEPS];
    T w[STEPS][N], next_x[STEPS][N], next_dy[STEPS][N];
    A sw[STEPS][N], sb[STEPS][N], next_mean = 0, next_r = 0;
#pragma unroll
    for (int s = 0; s < STEPS; s++) {
        at[s] = RowVector<T>((s * LANES + lane) * N, g.d);
        if (g.w) at[s].load(w[s], (const T*)g.w);
#pragma unroll
        for (int u = 0; u < N; u++) {
            if (!g.w) w[s][u] = round_to<T>((A)1);
            sw[s][u] = sb[s][u] = (A)0;
        }
    }
    auto load_row = [&](int r) {
        r = r < g.rows ? r : g.rows - 1;             // (a row again rather than none)
        const T* x = (const T*)g.x + r * g.x_rs;
        const T* dy = (const T*)g.dy + r * g.dy_rs;
#pragma unroll
        for (int s = 0; s < STEPS; s++) {
            at[s].load(next_x[s], x);
            at[s].load(next_dy[s], dy);
        }
        next_mean = g.stats[2 * (long long)r];
        next_r = g.stats[2 * (long long)r + 1];
    };
    int row = (int)blockIdx.x * TEAMS + team;
    if (AHEAD) load_row(row);
    for (int turn = 0; row < g.rows; row += stride, turn ^= 1) {
        T rx[STEPS][N], rg[STEPS][N];
        if (!AHEAD) load_row(row);
        __builtin_memcpy(rx, next_x, sizeof(rx));
        __builtin_memcpy(rg, next_dy, sizeof(rg));
        const A mean = next_mean, r = next_r;
        if (AHEAD) load_row(row + stride);
        A sums[2] = {};
#pragma unroll
        for (int s = 0; s < STEPS; s++)
#pragma unroll
            for (int u = 0; u < N; u++) {
                const A h = at[s].has(u) ? (widen(rx[s][u]) - mean) * r : (A)0, d = at[s].has(u) ? widen(rg[s][u]) : (A)0, dw = d * widen(w[s][u]);
                sums[0] += dw;
                sums[1] += dw * h;
                if constexpr (WEIGHTS) {
                    sw[s][u] += d * h;
                    sb[s][u] += d;
                }
            }
        if (!g.dx) continue;
        team_sums_in_turn<LANES>(sums, room + turn * 2 * (LANES / 64));
        const A c0 = sums[0] / (A)g.d, c1 = sums[1] / (A)g.d;
        T* dx = (T*)g.dx + row * g.dx_rs;
#pragma unroll
        for (int s = 0; s < STEPS; s++) {
            T out[N], was[N];
            A value[N];
            if (g.accumulate_dx) at[s].load(was, dx);
#pragma unroll
            for (int u = 0; u < N; u++) {
                const A h = (widen(rx[s][u]) - mean) * r;
                A v = r * (widen(rg[s][u]) * widen(w[s][u]) - c0 - h * c1);
                if (g.accumulate_dx) v += widen(was[u]);
                value[u] = v;
            }
            round_vector<T>(out, value);
            at[s].store(dx, out);
        }
    }
    if constexpr (WEIGHTS) {
        A* part = g.partials + (long long)blockIdx.x * 2 * g.d;
        if constexpr (TEAMS > 1) {                 // the teams add to the workgroup's row one after the other
            A* sum = room + 4 * (LANES / 64);
            for (int i = 0; i < TEAMS; i++) {
                if (team == i)
#pragma unroll
                    for (int s = 0; s < STEPS; s++)
#pragma unroll
                        for (int u = 0; u < N; u++)
                            if (at[s].has(u)) {
                                const int c = at[s].at + u;
                                sum[c] = (i ? sum[c] : (A)0) + sw[s][u];
                                sum[g.d + c] = (i ? sum[g.d + c] : (A)0) + sb[s][u];
                            }
                __syncthreads();
            }
            for (int c = threadIdx.x; c < 2 * g.d; c += 256) part[c] = sum[c];
        } else {
#pragma unroll
            for (int s = 0; s < STEPS; s++)
#pragma unroll
                for (int u = 0; u < N; u++)
                    if (at[s].has(u)) {
                        part[at[s].at + u] = sw[s][u];
                        part[g.d + at[s].at + u] = sb[s][u];
                    }
        }
    }
}

// dw and db from the workgroups' rows of partial sums: 64 columns to a workgroup, sixteen waves that take every sixteenth row, added in wave order
template <typename T>
__global__ void __launch_bounds__(1024) norm_columns_kernel(NormArgs<typename traits<T>::acc> g, int parts) {
    using A = typename traits<T>::acc;
    __shared__ A room[16][64];
    const int wave = threadIdx.x / 64, c = (int)blockIdx.x * 64 + (int)(threadIdx.x & 63);
    A sum = 0;
    if (c < 2 * g.d) {
#pragma unroll 8
        for (int i = wave; i < parts; i += 16) sum += g.partials[(long long)i * 2 * g.d + c];
    }
    room[wave][threadIdx.x & 63] = sum;
    __syncthreads();
    if (wave || c >= 2 * g.d) return;
#pragma unroll
    for (int i = 1; i < 16; i++) sum += room[i][threadIdx.x];
    const bool is_b = c >= g.d;
    T* out = (T*)(is_b ? g.db : g.dw);
    if (!out) return;
    out += is_b ? c - g.d : c;
    *out = round_to<T>((is_b ? g.accumulate_db : g.accumulate_dw) ? widen(*out) + sum : sum);
}

// Rows shorter than a vector, or longer than a workgroup's registers: a workgroup walks its row once for each sum
template <typename T>
__global__ void __launch_bounds__(256) layer_norm_any_kernel(NormArgs<typename traits<T>::acc> g) {
    using A = typename traits<T>::acc;
    __shared__ A room[4];
    for (int row = blockIdx.x; row < g.rows; row += gridDim.x) {
    const T* x = (const T*)g.x + row * g.x_rs;
    A sum[1] = {}, squares[1] = {};
    for (int c = threadIdx.x; c < g.d; c += 256) sum[0] += widen(x[c]);
    team_sums<256>(sum, room);
    const A mean = sum[0] / (A)g.d;
    for (int c = threadIdx.x; c < g.d; c += 256) { const A v = widen(x[c]) - mean; squares[0] += v * v; }
    team_sums<256>(squares, room);
    const A r = one_over_root(squares[0] / (A)g.d + g.eps);
    if (g.stats && threadIdx.x == 0) { g.stats[2 * (long long)row] = mean; g.stats[2 * (long long)row + 1] = r; }
    T* y = (T*)g.y + row * g.y_rs;
    for (int c = threadIdx.x; c < g.d; c += 256) {
        A h = (widen(x[c]) - mean) * r;
        if (g.w) h *= widen(((const T*)g.w)[c]);
        if (g.b) h += widen(((const T*)g.b)[c]);
        y[c] = round_to<T>(h);
    }
    }
}

template <typename T>
__global__ void __launch_bounds__(256) layer_norm_any_dx_kernel(NormArgs<typename traits<T>::acc> g) {
    using A = typename traits<T>::acc;
    __shared__ A room[8];
    for (int row = blockIdx.x; row < g.rows; row += gridDim.x) {
    const T* x = (const T*)g.x + row * g.x_rs;
    const T* dy = (const T*)g.dy + row * g.dy_rs;
    const A mean = g.stats[2 * (long long)row], r = g.stats[2 * (long long)row + 1];
    A sums[2] = {};
    for (int c = threadIdx.x; c < g.d; c += 256) {
        const A v = widen(dy[c]) * (g.w ? widen(((const T*)g.w)[c]) : (A)1);
        sums[0] += v;
        sums[1] += v * ((widen(x[c]) - mean) * r);
    }
    team_sums<256>(sums, room);
    const A c0 = sums[0] / (A)g.d, c1 = sums[1] / (A)g.d;
    T* dx = (T*)g.dx + row * g.dx_rs;
    for (int c = threadIdx.x; c < g.d; c += 256) {
        A v = r * (widen(dy[c]) * (g.w ? widen(((const T*)g.w)[c]) : (A)1) - c0 - (widen(x[c]) - mean) * r * c1);
        if (g.accumulate_dx) v += widen(dx[c]);
        dx[c] = round_to<T>(v);
    }
    }
}

// A workgroup's partial sums of every column, its rows those of equal number modulo the workgroups; `across` threads to a row, a power of two
template <typename T>
__global__ void __launch_bounds__(256) layer_norm_any_columns_kernel(NormArgs<typename traits<T>::acc> g, int across) {
    using A = typename traits<T>::acc;
    __shared__ A room[2][256];
    const int lane = threadIdx.x % across, slice = threadIdx.x / across, slices = 256 / across;
    for (int c0 = 0; c0 < g.d; c0 += across) {
        const int c = c0 + lane;
        A sw = 0, sb = 0;
        if (c < g.d)
            for (int row = (int)blockIdx.x * slices + slice; row < g.rows; row += (int)gridDim.x * slices) {
                const A d = widen(((const T*)g.dy)[row * g.dy_rs + c]);
                sw += d * ((widen(((const T*)g.x)[row * g.x_rs + c]) - g.stats[2 * (long long)row]) * g.stats[2 * (long long)row + 1]);
                sb += d;
            }
        __syncthreads();
        room[0][threadIdx.x] = sw;
        room[1][threadIdx.x] = sb;
        __syncthreads();
        if (slice == 0 && c < g.d) {
            for (int i = 1; i < slices; i++) { sw += room[0][i * across + lane]; sb += room[1][i * across + lane]; }
            g.partials[(long long)blockIdx.x * 2 * g.d + c] = sw;
            g.partials[(long long)blockIdx.x * 2 * g.d + g.d + c] = sb;
        }
    }
}

// How a row of d elements is held: threads to a row and 16-byte vectors to a thread; steps 0: not in registers
struct NormPlan { int lanes, steps; };
static NormPlan norm_plan(int d, size_t elem) {
    const int n = (int)(16 / elem);
    if (d < n) return {256, 0};
    for (int lanes : {64, 256, 1024})
        for (int steps : {1, 2, 4}) {
            if (lanes == 256 && steps == 1) continue;      // (a wave holds those)
            if ((long long)lanes * steps * n >= d) return {lanes, steps};
        }
    return (long long)1024 * 8 * n >= d ? NormPlan{1024, 8} : NormPlan{256, 0};
}
static int norm_blocks(int rows, const NormPlan& p) {
    const int teams = p.lanes < 256 ? 256 / p.lanes : 1, most = (rows + teams - 1) / teams;
    return most < NORM_BLOCKS ? most : NORM_BLOCKS;
}

template <typename T, int LANES, int STEPS>
static int launch_norm_team(const NormArgs<typename traits<T>::acc>& g, bool backward) {
    using A = typename traits<T>::acc;
    constexpr int TEAMS = LANES < 256 ? 256 / LANES : 1, THREADS = LANES < 256 ? 256 : LANES;
    if (!backward) {
        const int cus = device_cu_count() > 0 ? device_cu_count() : 256, all = (g.rows + TEAMS - 1) / TEAMS, resident = cus * (2048 / THREADS);
        hipLaunchKernelGGL((layer_norm_kernel<T, LANES, STEPS>), dim3(all < resident ? all : resident), dim3(THREADS), 0, current_stream(), g);
        return check_launch("layer_norm_kernel") ? 0 : -1;
    }
    const bool weights = g.dw || g.db;
    const int blocks = norm_blocks(g.rows, NormPlan{LANES, STEPS});
    const size_t lds = sizeof(A) * (4 * (LANES / 64) + (weights && TEAMS > 1 ? 2 * (size_t)g.d : 0));
    if (weights) hipLaunchKernelGGL((layer_norm_backward_kernel<T, LANES, STEPS, true>), dim3(blocks), dim3(THREADS), lds, current_stream(), g);
    else hipLaunchKernelGGL((layer_norm_backward_kernel<T, LANES, STEPS, false>), dim3(blocks), dim3(THREADS), lds, current_stream(), g);
    if (!check_launch("layer_norm_backward_kernel")) return -1;
    if (!weights) return 0;
    hipLaunchKernelGGL((norm_columns_kernel<T>), dim3((2 * g.d + 63) / 64), dim3(1024), 0, current_stream(), g, blocks);
    return check_launch("norm_columns_kernel") ? 0 : -1;
}

template <typename T>
static int launch_norm(const NormArgs<typename traits<T>::acc>& g, bool backward) {
    const NormPlan p = norm_plan(g.d, sizeof(T));
    switch (p.lanes * 16 + p.steps) {
        case 64 * 16 + 1: return launch_norm_team<T, 64, 1>(g, backward);
        case 64 * 16 + 2: return launch_norm_team<T, 64, 2>(g, backward);
        case 64 * 16 + 4: return launch_norm_team<T, 64, 4>(g, backward);
        case 256 * 16 + 2: return launch_norm_team<T, 256, 2>(g, backward);
        case 256 * 16 + 4: return launch_norm_team<T, 256, 4>(g, backward);
        case 1024 * 16 + 2: return launch_norm_team<T, 1024, 2>(g, backward);
        case 1024 * 16 + 4: return launch_norm_team<T, 1024, 4>(g, backward);
        case 1024 * 16 + 8: return launch_norm_team<T, 1024, 8>(g, backward);
    }
    if (!backward) {
        hipLaunchKernelGGL((layer_norm_any_kernel<T>), dim3(norm_grid(g.rows)), dim3(256), 0, current_stream(), g);
        return check_launch("layer_norm_any_kernel") ? 0 : -1;
    }
    if (g.dx) {
        hipLaunchKernelGGL((layer_norm_any_dx_kernel<T>), dim3(norm_grid(g.rows)), dim3(256), 0, current_stream(), g);
        if (!check_launch("layer_norm_any_dx_kernel")) return -1;
    }
    if (!g.dw && !g.db) return 0;
    const int blocks = norm_blocks(g.rows, p);
    int across = 1;
    while (across < 256 && across < g.d) across *= 2;
    hipLaunchKernelGGL((layer_norm_any_columns_kernel<T>), dim3(blocks), dim3(256), 0, current_stream(), g, across);
    if (!check_launch("layer_norm_any_columns_kernel")) return -1;
    hipLaunchKernelGGL((norm_columns_kernel<T>), dim3((2 * g.d + 63) / 64), dim3(1024), 0, current_stream(), g, blocks);
    return check_launch("norm_columns_kernel") ? 0 : -1;
}

static bool norm_args_ok(const char* who, bool pointers, int rows, int d, std::initializer_list<long long> strides, int dtype) {
    if (!pointers || rows <= 0 || d <= 0 || rows > (1 << 30) || d > (1 << 26)) { set_error("%s: null operand, non-positive extent, more than 2^30 rows or a width above 2^26 (rows=%d d=%d)", who, rows, d); return false; }
    if (!dtype_size(dtype)) { set_error("%s: unsupported dtype %d", who, dtype); return false; }
    for (long long s : strides)
        if (s < 0) { set_error("%s: negative stride", who); return false; }
    return true;
}
static bool norm_rows_apart(const char* who, const char* what, int rows, int d, long long rs) {
    if (rows == 1 || rs >= d) return true;
    set_error("%s: rows of %s are %lld elements apart and hold %d", who, what, rs, d);
    return false;
}

}  // namespace rp

using namespace rp;

extern "C" {

int rp_hip_layer_norm_forward(void* y, void* stats, const void* x, const void* w, const void* b, int rows, int d, long long y_rs, long long x_rs, double eps, int dtype) {
    const char* who = "rp_hip_layer_norm_forward";
    if (!norm_args_ok(who, y && x, rows, d, {y_rs, x_rs}, dtype) || !norm_rows_apart(who, "y", rows, d, y_rs)) return -1;
    if (!(eps >= 0)) { set_error("%s: eps is not negative", who); return -1; }
    RP_DISPATCH_DTYPE(dtype, using A = typename traits<T>::acc; return launch_norm<T>(NormArgs<A>{y, nullptr, nullptr, nullptr, x, w, b, nullptr, (A*)stats, nullptr, rows, d, y_rs, x_rs, 0, 0, (A)eps, 0, 0, 0}, false));
    return -1;
}

long long rp_hip_layer_norm_workspace(int rows, int d, int dtype) {
    if (!norm_args_ok("rp_hip_layer_norm_workspace", true, rows, d, {}, dtype)) return -1;
    return (long long)norm_blocks(rows, norm_plan(d, dtype_size(dtype))) * 2 * d * (dtype == RP_DTYPE_FLOAT64 ? 8 : 4);
}

int rp_hip_layer_norm_backward(void* dx, void* dw, void* db, const void* dy, const void* x, const void* w, const void* stats, void* workspace, int rows, int d,
                               long long dy_rs, long long x_rs, long long dx_rs, int accumulate_dx, int accumulate_dw, int accumulate_db, int dtype) {
    const char* who = "rp_hip_layer_norm_backward";
    if (!norm_args_ok(who, dy && x && stats && (workspace || (!dw && !db)), rows, d, {dy_rs, x_rs, dx_rs}, dtype) || (dx && !norm_rows_apart(who, "dx", rows, d, dx_rs))) return -1;
    if (!dx && !dw && !db) return 0;
    RP_DISPATCH_DTYPE(dtype, using A = typename traits<T>::acc; return launch_norm<T>(NormArgs<A>{nullptr, dx, dw, db, x, w, nullptr, dy, (A*)const_cast<void*>(stats), (A*)workspace, rows, d, 0, x_rs, dy_rs, dx_rs, (A)0, accumulate_dx, accumulate_dw, accumulate_db}, true));
    return -1;
}

}  // extern "C"
