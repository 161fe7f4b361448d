// Distillation from a teacher's top logits, forward and backward, all types.
//
//   p = softmax(t / T) over the row's K entries of the teacher,  q = softmax(s / T) over all classes of the student
//   loss = T^2 sum over j of p_j (log p_j - log q[id_j]),   ds[v] = T f (q[v] - sum over id_j = v of p_j)
// with f the row's share of the result (1, or 1 / rows for the mean) times the upstream gradient.  A row without an entry is left out: its loss and gradient are zeros.
//
// What bounds it is memory: the student's logits once and, backward, their gradient once.  A workgroup holds a row in registers where it fits (131072 classes of 16 bits,
// 65536 of float32), so that the largest logit, the sum and the gradient cost one read together; longer rows are read once for each of the three.
// The K entries are handled beside: their classes' gradients are written a second time, after the row's, by the first entry of each class (a class may be named twice).
#include "rp_gemm.h"
#include "rp_teams.h"

namespace rp {

constexpr int DISTILL_MOST_K = 1024, DISTILL_GRID = 1 << 20;

template <typename A> struct DistillArgs {
    void* grad;
    const void *logits, *teacher, *upstream;
    const int* ids;
    A* stats;                                      // [rows] log sum exp(s / T), [rows] log sum exp(t / T), [rows] losses
    int rows, classes, k, reduction;
    long long logits_rs;
    A temperature;
};

// The K entries in LDS: classes (-1: none) and log p.  Returns whether there is an entry.
template <typename T, int THREADS, typename A>
__device__ __forceinline__ bool teacher_entries(const DistillArgs<A>& g, int row, int* ids, A* log_p, A* room, A scale, bool known, A& log_mass) {
    const int* id = g.ids + (long long)row * g.k;
    const T* t = (const T*)g.teacher + (long long)row * g.k;
    A top = -INFINITY;
    __syncthreads();                               // (the last row's entries are done with)
    for (int j = threadIdx.x; j < g.k; j += THREADS) {
        const int v = id[j];
        const bool in = v >= 0 && v < g.classes;
        const A u = in ? widen(t[j]) * scale : -(A)INFINITY;
        ids[j] = in && !(u == -(A)INFINITY) ? v : -1;
        log_p[j] = u;
        top = larger(top, u);
    }
    if (!known) {
        top = team_max<THREADS>(top, room);
        A mass[1] = {};
        for (int j = threadIdx.x; j < g.k; j += THREADS) mass[0] += ids[j] < 0 ? (A)0 : natural_exp(log_p[j] - top);
        team_sums<THREADS>(mass, room + THREADS / 64);
        log_mass = top == -(A)INFINITY ? -(A)INFINITY : top + natural_log(mass[0]);
    }
    __syncthreads();
    return !(log_mass == -(A)INFINITY);
}

// The gradients of the entries' classes, over what the row's own pass left there
template <typename T, int THREADS, typename A>
__device__ __forceinline__ void correct_entries(const DistillArgs<A>& g, const T* logits, T* grad, const int* ids, A* p, const ScaledExp<A>& q, A log_mass, A factor) {
    for (int j = threadIdx.x; j < g.k; j += THREADS) p[j] = ids[j] < 0 ? (A)0 : natural_exp(p[j] - log_mass);      // (log p until here)
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();                               // the row's stores are done: these come after
    for (int j = threadIdx.x; j < g.k; j += THREADS) {
        const int v = ids[j];
        if (v < 0) continue;
        A mass = 0;
        int before = 0;
#pragma unroll 8
        for (int i = 0; i < g.k; i++) {            // (in the order of the entries, whichever thread adds)
            const bool same = ids[i] == v;
            mass += same ? p[i] : (A)0;
            before += same && i < j;
        }
        if (!before) grad[v] = round_to<T>((q(widen(logits[v])) - mass) * factor);
    }
}

template <typename A> __device__ __forceinline__ A row_factor(const DistillArgs<A>& g, int row) {
    A f = g.upstream ? ((const A*)g.upstream)[g.reduction == 0 ? row : 0] : (A)1;
    if (g.reduction == 1) f /= (A)g.rows;
    return f * g.temperature;
}

// Vectors a thread holds up to which two workgroups of 1024 share a CU, 64 registers a thread: one's loads and stores fly while the other adds up
constexpr int DISTILL_SHARED_STEPS = 8;
constexpr int distill_waves(int threads, int steps, int elem) { return threads == 1024 ? (steps <= DISTILL_SHARED_STEPS && elem < 8 ? 8 : 4) : 1; }

// FORWARD: the row's sums and loss; with a gradient asked for, that too.  Otherwise the gradient from the sums that a forward call left.  STEPS 0: the row is read again for each.
template <typename T, int THREADS, int STEPS, bool FORWARD>
__global__ void __launch_bounds__(THREADS, distill_waves(THREADS, STEPS, sizeof(T))) distill_kernel(DistillArgs<typename traits<T>::acc> g) {
    using A = typename traits<T>::acc;
    constexpr int N = vec16<T>::N, HELD = STEPS ? STEPS : 1;
    __shared__ A room[2 * (THREADS / 64)];
    __shared__ A log_p[DISTILL_MOST_K];
    __shared__ int ids[DISTILL_MOST_K];
    const A scale = (A)1 / g.temperature;
    // Vector i of a thread begins at byte tid * 16 + i * THREADS * 16 of the row, which buffer descriptors end with its last whole 4 bytes: what lies behind reads as zeros and is not
    // written, and one offset does for all loads and stores.  step i is whole where every thread's vector lies in the row; an odd last element of 16 bits goes by itself.
    auto whole = [&](int i) { return (i + 1) * THREADS * N <= g.classes; };
    const int row_bytes = STEPS ? g.classes * (int)sizeof(T) / 4 * 4 : 0;
    const bool odd = STEPS && sizeof(T) == 2 && g.classes % 2;
    const int odd_tid = (g.classes - 1) / N % THREADS;
    for (int row = blockIdx.x; row < g.rows; row += gridDim.x) {
        const T* s = (const T*)g.logits + row * g.logits_rs;
        int tid = threadIdx.x;
        asm volatile("" : "+v"(tid));              // (the masks of a row's end are made again for each row: kept, they would take more registers than there are)
        u32x4_t raw[HELD];
        T last = round_to<T>((A)0);
        if constexpr (STEPS > 0) {
            const __amdgpu_buffer_rsrc_t from = buffer_rsrc(s, row_bytes);
#pragma unroll
            for (int i = 0; i < STEPS; i++) raw[i] = __builtin_amdgcn_raw_buffer_load_b128(from, tid * 16, i * THREADS * 16, 0);
            if (odd) last = s[g.classes - 1];
        }
        A lse, log_mass = FORWARD ? (A)0 : g.stats[g.rows + row];
        const bool some = teacher_entries<T, THREADS>(g, row, ids, log_p, room, scale, !FORWARD, log_mass);
        if constexpr (STEPS > 0) {
#pragma unroll
            for (int i = 0; i < STEPS; i++)
                if (!whole(i)) {
                    const int left = g.classes - (i * THREADS + tid) * N;
                    T x[N];
                    __builtin_memcpy(x, &raw[i], 16);
#pragma unroll
                    for (int u = 0; u < N; u++) {
                        if (odd && u + 1 == left) x[u] = last;
                        x[u] = u < left ? x[u] : round_to<T>(-(A)INFINITY);      // (no mask from here on: exp gives 0)
                    }
                    __builtin_memcpy(&raw[i], x, 16);
                }
        }
        auto each = [&](auto f) {
            if constexpr (STEPS > 0) {
#pragma unroll
                for (int i = 0; i < STEPS; i++) {
                    T x[N];
                    asm volatile("" : "+v"(raw[i]));      // (widened anew for each pass)
                    __builtin_memcpy(x, &raw[i], 16);
#pragma unroll
                    for (int u = 0; u < N; u++) f(widen(x[u]));
                }
            } else {
                for (int v = tid; v < g.classes; v += THREADS) f(widen(s[v]));
            }
        };
        if constexpr (FORWARD) {
            A top = -(A)INFINITY, sum[1] = {};
            each([&](A x) { top = plain_max(top, x); });      // (NaN shows in the sum)
            top = team_max<THREADS>(top, room);
            const A base = top == -(A)INFINITY ? (A)0 : top * scale;
            const ScaledExp<A> weight(scale, base);
            each([&](A x) { sum[0] += weight(x); });
            team_sums<THREADS>(sum, room + THREADS / 64);
            lse = base + natural_log(sum[0]);
            A loss[1] = {};
            if (some)
                for (int j = tid; j < g.k; j += THREADS) {
                    if (ids[j] < 0) continue;
                    const A lp = log_p[j] - log_mass, p = natural_exp(lp);
                    if (p != 0) loss[0] += p * (lp - scaled_less(widen(s[ids[j]]), scale, lse));
                }
            team_sums<THREADS>(loss, room);
            if (tid == 0) {
                g.stats[row] = lse;
                g.stats[g.rows + row] = log_mass;
                g.stats[2 * (long long)g.rows + row] = loss[0] * g.temperature * g.temperature;
            }
        } else {
            lse = g.stats[row];
        }
        if (!g.grad) continue;
        T* grad = (T*)g.grad + (long long)row * g.classes;
        const A factor = row_factor(g, row);
        const ScaledExp<A> q(scale, lse);
        auto share = [&](A x) { return round_to<T>(some ? q(x) * factor : (A)0); };
        if constexpr (STEPS > 0) {
            const __amdgpu_buffer_rsrc_t to = buffer_rsrc(grad, row_bytes);
#pragma unroll
            for (int i = 0; i < STEPS; i++) {
                T out[N];
                asm volatile("" : "+v"(raw[i]));
                __builtin_memcpy(out, &raw[i], 16);
#pragma unroll
                for (int u = 0; u < N; u++) out[u] = share(widen(out[u]));
                u32x4_t v;
                __builtin_memcpy(&v, out, 16);
                __builtin_amdgcn_raw_buffer_store_b128(v, to, tid * 16, i * THREADS * 16, 0);
                __builtin_amdgcn_sched_barrier(0);
            }
            if (odd && tid == odd_tid) grad[g.classes - 1] = share(widen(last));
        } else {
            for (int v = tid; v < g.classes; v += THREADS) grad[v] = share(widen(s[v]));
        }
        if (some) correct_entries<T, THREADS>(g, s, grad, ids, log_p, q, log_mass, factor);
    }
}

// The rows' losses as they are, or their sum or mean: one workgroup, in double, whose threads' sums are added in order
template <typename A>
__global__ void __launch_bounds__(1024) distill_loss_kernel(A* out, const A* losses, int rows, int reduction) {
    if (reduction == 0) {
        for (int i = (int)(blockIdx.x * 1024 + threadIdx.x); i < rows; i += (int)gridDim.x * 1024) out[i] = losses[i];
        return;
    }
    __shared__ double room[16];
    double sum[1] = {};
    for (int i = threadIdx.x; i < rows; i += 1024) sum[0] += (double)losses[i];
    team_sums<1024>(sum, room);
    if (threadIdx.x == 0) out[0] = (A)(reduction == 1 ? sum[0] / rows : sum[0]);
}

template <typename T, int THREADS, int STEPS>
static int launch_distill_row(const DistillArgs<typename traits<T>::acc>& g, bool forward) {
    const int blocks = g.rows < DISTILL_GRID ? g.rows : DISTILL_GRID;
    if (forward) hipLaunchKernelGGL((distill_kernel<T, THREADS, STEPS, true>), dim3(blocks), dim3(THREADS), 0, current_stream(), g);
    else hipLaunchKernelGGL((distill_kernel<T, THREADS, STEPS, false>), dim3(blocks), dim3(THREADS), 0, current_stream(), g);
    return check_launch("distill_kernel") ? 0 : -1;
}

template <typename T>
static int launch_distill(const DistillArgs<typename traits<T>::acc>& g, bool forward) {
    constexpr int N = vec16<T>::N;
    if (g.classes < N || (long long)g.classes > 1024ll * 16 * N) return launch_distill_row<T, 1024, 0>(g, forward);
    if (g.classes <= 256 * N) return launch_distill_row<T, 256, 1>(g, forward);
    if (g.classes <= 256 * 4 * N) return launch_distill_row<T, 256, 4>(g, forward);
    if (g.classes <= 1024 * 2 * N) return launch_distill_row<T, 1024, 2>(g, forward);
    if (g.classes <= 1024 * 4 * N) return launch_distill_row<T, 1024, 4>(g, forward);
    if (g.classes <= 1024 * 8 * N) return launch_distill_row<T, 1024, 8>(g, forward);
    return launch_distill_row<T, 1024, 16>(g, forward);
}

static bool distill_args_ok(const char* who, bool pointers, int rows, int classes, int k, long long logits_rs, double temperature, int reduction, int dtype) {
    if (!pointers || rows <= 0 || classes <= 0 || k <= 0 || rows > (1 << 30) || classes > (1 << 29)) {
        set_error("%s: null operand, non-positive extent, more than 2^30 rows or 2^29 classes (rows=%d classes=%d k=%d)", who, rows, classes, k);
        return false;
    }
    if (k > DISTILL_MOST_K) { set_error("%s: at most %d entries of the teacher (k=%d)", who, DISTILL_MOST_K, k); return false; }
    if (!dtype_size(dtype)) { set_error("%s: unsupported dtype %d", who, dtype); return false; }
    if (logits_rs < 0) { set_error("%s: negative stride", who); return false; }
    if (!(temperature > 0) || temperature > 1e30) { set_error("%s: the temperature is above 0 and finite", who); return false; }
    if (reduction < 0 || reduction > 2) { set_error("%s: reduction must be none (0), mean (1) or sum (2)", who); return false; }
    return true;
}

}  // namespace rp

using namespace rp;

extern "C" {

int rp_hip_distillation_forward(void* loss_out, void* grad_logits, void* stats, const void* logits, const int* ids, const void* teacher, const void* upstream_dev,
                                int rows, int classes, int k, long long logits_rs, double temperature, int reduction, int dtype) {
    if (!distill_args_ok("rp_hip_distillation_forward", loss_out && stats && logits && ids && teacher, rows, classes, k, logits_rs, temperature, reduction, dtype)) return -1;
    RP_DISPATCH_DTYPE(dtype, using A = typename traits<T>::acc;
        if (launch_distill<T>(DistillArgs<A>{grad_logits, logits, teacher, upstream_dev, ids, (A*)stats, rows, classes, k, reduction, logits_rs, (A)temperature}, true) != 0) return -1;
        const int blocks = reduction ? 1 : rows < (1 << 20) ? (rows + 1023) / 1024 : 1024;
        hipLaunchKernelGGL((distill_loss_kernel<A>), dim3(blocks), dim3(1024), 0, current_stream(), (A*)loss_out, (const A*)stats + 2 * (long long)rows, rows, reduction);
        return check_launch("distill_loss_kernel") ? 0 : -1);
    return -1;
}

int rp_hip_distillation_backward(void* grad_logits, const void* stats, const void* logits, const int* ids, const void* teacher, const void* upstream_dev,
                                 int rows, int classes, int k, long long logits_rs, double temperature, int reduction, int dtype) {
    if (!distill_args_ok("rp_hip_distillation_backward", grad_logits && stats && logits && ids && teacher, rows, classes, k, logits_rs, temperature, reduction, dtype)) return -1;
    RP_DISPATCH_DTYPE(dtype, using A = typename traits<T>::acc;
        return launch_distill<T>(DistillArgs<A>{grad_logits, logits, teacher, upstream_dev, ids, (A*)const_cast<void*>(stats), rows, classes, k, reduction, logits_rs, (A)temperature}, false));
    return -1;
}

}  // extern "C"
