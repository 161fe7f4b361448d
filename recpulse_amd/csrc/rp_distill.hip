// Distillation from a teacher's top logits, forward and backward, all types.
//
//   p = softmax(t / T) over the row's K entries of the teacher,  q = softmax(s / T) over all classes of the student
//   loss = T^2 sum over j of p_j (log p_j - log q[id_j]),   ds[v] = T f (q[v] - sum over id_j = v of p_j)
// with f the row's share of the result (1, or 1 / rows for the mean) times the upstream gradient.  A row without an entry is left out: its loss and gradient are zeros.
//
// What bounds it is memory: the student's logits once and, backward, their gradient once.  A workgroup holds a row in registers where it fits (131072 classes of 16 bits,
// 65536 of float32), so that the largest logit, the sum and the gradient cost one read together; longer rows are read once for the two sums and again for the gradient (from 2^27 classes on, whose byte offsets pass
// 32 bits, once for each of the three).
// The largest logit and the sum are kept apart, and every difference is one of two logits: a row far from zero would lose its digits to the rounding of a log sum (float32 around 4096: 1e-4 of every
// probability).  The K entries are handled beside, one a thread: their classes' gradients are written a second time, after the row's, by the first entry of each class (a class may be named twice).
#include "rp_gemm.h"
#include "rp_teams.h"

namespace rp {

constexpr int DISTILL_MOST_K = 1024;

template <typename A> struct DistillArgs {
    void* grad;
    const void *logits, *teacher, *upstream;
    const int* ids;
    A* stats;                                      // [rows] largest logit, [rows] sum of exp((s - that) / T) or, without entries, -1, [rows] losses
    int rows, classes, k, reduction;
    long long logits_rs;
    A temperature;
};

template <typename A> __device__ __forceinline__ A row_factor(const DistillArgs<A>& g, int row) {
    A f = g.upstream ? ((const A*)g.upstream)[g.reduction == 0 ? row : 0] : (A)1;
    if (g.reduction == 1) f /= (A)g.rows;
    return f * g.temperature;
}

// The gradients of the entries' classes, over what the row's own pass left there.  `v`, `value`: this thread's entry (-1: none) and its logit; `p`: exp((t - largest t) / T) of all entries
template <typename T, typename A>
__device__ __forceinline__ void correct_entries(int k, T* grad, const int* ids, const A* p, int v, A value, const ScaledExp<A>& weight, A share, A part, A factor) {
    if (v < 0) return;
    const int j = threadIdx.x;
    A mass = 0;
    int before = 0;
#pragma unroll 8
    for (int i = 0; i < k; i++) {                  // (in the order of the entries, whichever thread adds)
        const bool same = ids[i] == v;
        mass += same ? p[i] : (A)0;
        before += same && i < j;
    }
    if (!before) grad[v] = round_to<T>((weight(value) * share - mass * part) * factor);
}

// Vectors a thread holds up to which two workgroups of 1024 share a CU, 64 registers a thread: one's loads and stores fly while the other adds up
constexpr int DISTILL_SHARED_STEPS = 8;
constexpr int distill_waves(int threads, int steps, int elem) { return threads == 1024 ? (steps <= DISTILL_SHARED_STEPS && elem < 8 ? 8 : 4) : 1; }

// Whether a forward pass corrects a row's entries during the next row, whose loads it does not wait for then: not in the kernels whose row leaves no registers for it (bf16, us at once and later:
// 4096 x 32000 131 / 123, 2000 x 130000 286 / 271; 4096 x 65536 272 / 288)
constexpr bool distill_later(int threads, int steps, int elem) { return !(threads == 1024 && steps == DISTILL_SHARED_STEPS && elem < 8); }

// A value that all lanes have, in scalar registers
__device__ __forceinline__ float in_scalar(float v) { return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(v))); }
__device__ __forceinline__ double in_scalar(double v) { return __hiloint2double(__builtin_amdgcn_readfirstlane(__double2hiint(v)), __builtin_amdgcn_readfirstlane(__double2loint(v))); }
__device__ __forceinline__ float one_over(float v) { return __builtin_amdgcn_rcpf(v); }      // (off by one place)
__device__ __forceinline__ double one_over(double v) { return 1.0 / v; }
template <typename T> __device__ __forceinline__ void load_one(T& x, const __amdgpu_buffer_rsrc_t& from, int offset) {
    if constexpr (sizeof(T) == 2) { const uint16_t v = __builtin_amdgcn_raw_buffer_load_b16(from, offset, 0, 0); __builtin_memcpy(&x, &v, 2); }
    else if constexpr (sizeof(T) == 4) { const uint32_t v = __builtin_amdgcn_raw_buffer_load_b32(from, offset, 0, 0); __builtin_memcpy(&x, &v, 4); }
    else { const auto v = __builtin_amdgcn_raw_buffer_load_b64(from, offset, 0, 0); __builtin_memcpy(&x, &v, 8); }
}

// FORWARD: the row's sums and loss; with a gradient asked for, that too.  Otherwise the gradient from the largest logit and sum that a forward call left.  STEPS 0: the row is read again for each.
// A workgroup walks rows; the next row's loads are issued as soon as a row's registers are stored, and fly while its last steps wait for one another.  k <= THREADS: a thread has an entry or none.
template <typename T, int THREADS, int STEPS, bool FORWARD>
__global__ void __launch_bounds__(THREADS, distill_waves(THREADS, STEPS, sizeof(T))) distill_kernel(DistillArgs<typename traits<T>::acc> g) {
    using A = typename traits<T>::acc;
    constexpr int N = vec16<T>::N, HELD = STEPS ? STEPS : 1, WAVES = THREADS / 64;
    __shared__ A rooms[3][2][WAVES];
    __shared__ A entry_p[2][THREADS];              // (of this row and of the one before, which may still be read)
    __shared__ int entry_ids[2][THREADS];
    __shared__ A entry_value[2][THREADS];          // (the thread's own: registers are for the row.  With these and what all lanes share in scalar ones 4096 x 65536 bf16 288 us -> 272)
    const A scale = in_scalar((A)1 / g.temperature);
    // Vector i of a thread begins at byte tid * 16 + i * THREADS * 16 of the row, which buffer descriptors end with its last whole 4 bytes: what lies behind reads as zeros and is not
    // written, and one offset does for all loads.  Step i is whole where every thread's vector lies in the row; an odd last element of 16 bits goes by itself.
    auto whole = [&](int i) { return (i + 1) * THREADS * N <= g.classes; };
    const int row_bytes = STEPS ? g.classes * (int)sizeof(T) / 4 * 4 : 0;
    const bool odd = STEPS && sizeof(T) == 2 && g.classes % 2;
    u32x4_t raw[HELD];
    T last = round_to<T>((A)0), entry = round_to<T>((A)0);
    int id = -1;
    auto row_of = [&](int row) { return (const T*)g.logits + (row < g.rows ? row : g.rows - 1) * g.logits_rs; };      // (a row again rather than none)
    auto load_step = [&](const __amdgpu_buffer_rsrc_t& from, auto ic) {
        constexpr int i = decltype(ic)::value;
        raw[i] = __builtin_amdgcn_raw_buffer_load_b128(from, (int)threadIdx.x * 16, i * THREADS * 16, 0);
    };
    auto load_entry = [&](int row) {
        if (row >= g.rows) row = g.rows - 1;
        if (odd) last = row_of(row)[g.classes - 1];
        // (one offset a thread for either, no addresses)
        if ((int)threadIdx.x < g.k) {
            id = (int)__builtin_amdgcn_raw_buffer_load_b32(buffer_rsrc(g.ids + (long long)row * g.k, g.k * 4ll), (int)threadIdx.x * 4, 0, 0);
            load_one(entry, buffer_rsrc((const T*)g.teacher + (long long)row * g.k, g.k * (long long)sizeof(T)), (int)threadIdx.x * (int)sizeof(T));
        }
    };
    {
        const __amdgpu_buffer_rsrc_t from = buffer_rsrc(row_of(blockIdx.x), row_bytes);
        static_for<0, STEPS>([&](auto ic) { load_step(from, ic); });
        load_entry(blockIdx.x);
    }
    // The entries of the row before are corrected once this row's loads have been waited for, before which its stores were issued, and all threads have met
    A top_before = 0, share_before = 0, part_before = 0, factor_before = 0;
    bool some_before = false;
    auto correct_row = [&](T* grad, int turn, const ScaledExp<A>& weight, A share, A part, A factor) {
        const bool own = (int)threadIdx.x < g.k;
        correct_entries<T>(g.k, grad, entry_ids[turn], entry_p[turn], own ? entry_ids[turn][threadIdx.x] : -1, own ? entry_value[turn][threadIdx.x] : (A)0, weight, share, part, factor);
    };
    auto correct_before = [&](int row, int turn) {
        if (some_before) correct_row((T*)g.grad + (long long)row * g.classes, turn, ScaledExp<A>(scale, top_before), share_before, part_before, factor_before);
    };
    constexpr bool LATER = FORWARD && distill_later(THREADS, STEPS, sizeof(T));
    int row = blockIdx.x, turn = 0;
    for (; row < g.rows; row += gridDim.x, turn ^= 1) {
        const T* s = row_of(row);
        int tid = threadIdx.x;
        asm volatile("" : "+v"(tid));              // (the masks of a row's end are made again for each row: kept, they would take more registers than there are)
        // the entry: its class (-1: none), the teacher's logit and the student's
        A* p = entry_p[turn];
        int* ids = entry_ids[turn];
        A goal = id >= 0 && id < g.classes ? widen(entry) : -(A)INFINITY;
        int v = goal == -(A)INFINITY ? -1 : id;
        A value = v < 0 ? (A)0 : widen(s[v]);
        const T row_last = last;
        if (tid < g.k) {
            ids[tid] = v;
            p[tid] = goal;
            entry_value[turn][tid] = value;
        }
        if constexpr (STEPS > 0) {
#pragma unroll
            for (int i = 0; i < STEPS; i++)
                if (!whole(i)) {
                    const int left = g.classes - (i * THREADS + tid) * N;
                    T x[N];
                    __builtin_memcpy(x, &raw[i], 16);
#pragma unroll
                    for (int u = 0; u < N; u++) {
                        if (odd && u + 1 == left) x[u] = row_last;
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
                for (int c = tid; c < g.classes; c += THREADS) f(widen(s[c]));
            }
        };
        A top = -(A)INFINITY, sum, part = 0;       // part: 1 over the entries' sum
        bool some;                                 // an entry counts
        if constexpr (FORWARD) {
            bool again = false;
            if constexpr (STEPS > 0 && sizeof(T) == 2) {
                // Two values at a time as whole numbers: of those that are not negative the largest number is the largest value (and +NaN above all).  Rows without one are looked through again.
                typedef short __attribute__((ext_vector_type(2))) short2_t;
                u32x4_t most = raw[0];
#pragma unroll
                for (int i = 1; i < STEPS; i++)
#pragma unroll
                    for (int w = 0; w < 4; w++) most[w] = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(short2_t, (uint32_t)most[w]), __builtin_bit_cast(short2_t, (uint32_t)raw[i][w])));
                int first = -32768;
#pragma unroll
                for (int w = 0; w < 4; w++) {
                    const short2_t pair = __builtin_bit_cast(short2_t, (uint32_t)most[w]);
                    first = first > pair[0] ? first : pair[0];
                    first = first > pair[1] ? first : pair[1];
                }
                top = (A)first;
            } else {
                each([&](A x) { top = plain_max(top, x); });      // (NaN shows in the sum)
            }
            A tops[2] = {top, goal};
            if (LATER) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            team_tops_in_turn<THREADS>(tops, rooms[0][0]);
            if (LATER) correct_before(row - (int)gridDim.x, turn ^ 1);
            top = tops[0];
            if constexpr (STEPS > 0 && sizeof(T) == 2) {
                again = !(top >= (A)0);
                T x;
                x.bits = (uint16_t)(int)top;
                top = widen(x);
                if (again) {
                    top = -(A)INFINITY;
                    each([&](A x) { top = plain_max(top, x); });
                    __syncthreads();
                    A one[1] = {top};
                    team_tops_in_turn<THREADS>(one, rooms[0][0]);
                    top = one[0];
                }
            }
            top = in_scalar(top);
            const A goal_top = in_scalar(tops[1]);
            const ScaledExp<A> weight(scale, top);
            A sums[2] = {(A)0, v < 0 ? (A)0 : ScaledExp<A>(scale, goal_top)(goal)};
            each([&](A x) { sums[0] += weight(x); });
            team_sums_in_turn<THREADS>(sums, rooms[1][0]);
            sum = in_scalar(sums[0]);
            const A goal_sum = in_scalar(sums[1]);
            some = !(goal_top == -(A)INFINITY);
            // (from LDS again, two barriers later)
            v = tid < g.k ? ids[tid] : -1;
            goal = tid < g.k ? p[tid] : -(A)INFINITY;
            value = tid < g.k ? entry_value[turn][tid] : (A)0;
            const ScaledExp<A> goal_weight(scale, goal_top);
            part = in_scalar(one_over(goal_sum));
            const A own_weight = v < 0 ? (A)0 : goal_weight(goal), own_p = own_weight * part;
            if (tid < g.k) p[tid] = own_weight;
            A loss[1] = {own_p != 0 ? own_p * ((goal_weight.log(goal) - natural_log(goal_sum)) - (weight.log(value) - natural_log(sum))) : (A)0};
            if (g.k > 64) team_sums_in_turn<THREADS>(loss, rooms[2][0]);
            else loss[0] = wave_sum(loss[0]);          // (the first wave has all entries)
            if (tid == 0) {
                g.stats[row] = top;
                g.stats[g.rows + row] = some ? sum : (A)-1;
                g.stats[2 * (long long)g.rows + row] = some ? loss[0] * g.temperature * g.temperature : (A)0;
            }
        } else {
            top = g.stats[row];
            sum = g.stats[g.rows + row];
            some = !(sum < 0);
        }
        const __amdgpu_buffer_rsrc_t from = buffer_rsrc(row_of(row + gridDim.x), row_bytes);
        if (!g.grad) {
            static_for<0, STEPS>([&](auto ic) { load_step(from, ic); });
            load_entry(row + gridDim.x);
            continue;                              // (two barriers lie between a room's readers and its next writers)
        }
        T* grad = (T*)g.grad + (long long)row * g.classes;
        const ScaledExp<A> weight(scale, top);
        const A factor = in_scalar(row_factor(g, row)), share = in_scalar(one_over(sum)), scaled = in_scalar(share * factor);
        auto rest = [&](A x) { return some ? weight(x) * scaled : (A)0; };
        if constexpr (STEPS > 0) {
            const __amdgpu_buffer_rsrc_t to = buffer_rsrc(grad, row_bytes);
            static_for<0, STEPS>([&](auto ic) {
                constexpr int i = decltype(ic)::value;
                T out[N];
                A values[N];
                asm volatile("" : "+v"(raw[i]));
                __builtin_memcpy(out, &raw[i], 16);
#pragma unroll
                for (int u = 0; u < N; u++) values[u] = weight(widen(out[u])) * scaled;
                if (some) round_vector<T>(out, values);
                else __builtin_memset(out, 0, 16);           // (whatever the row's logits are)
                u32x4_t o;
                __builtin_memcpy(&o, out, 16);
                // (the whole offset in a vector register: behind a 16-byte store with part of it in a scalar one the compiler lets the next instruction write the data's registers, and zeros of such a
                // write have been stored here)
                __builtin_amdgcn_raw_buffer_store_b128(o, to, tid * 16 + i * THREADS * 16, 0, 2);      // (streaming: 4096 x 65536 bf16 297 us, 288 so)
                load_step(from, ic);
                __builtin_amdgcn_sched_barrier(0);
            });
            if (odd && tid == (g.classes - 1) / N % THREADS) grad[g.classes - 1] = round_to<T>(rest(widen(row_last)));
        } else if (g.classes >= N) {
            for (int c = tid * N; c < g.classes; c += THREADS * N) {
                const RowVector<T> at(c, g.classes);
                T x[N];
                A values[N];
                at.load(x, s);
#pragma unroll
                for (int u = 0; u < N; u++) values[u] = rest(widen(x[u]));
                round_vector<T>(x, values);
                at.store(grad, x);
            }
        } else {
            for (int c = tid; c < g.classes; c += THREADS) grad[c] = round_to<T>(rest(widen(s[c])));
        }
        load_entry(row + gridDim.x);
        if (LATER) {
            top_before = top;
            share_before = share;
            part_before = part;
            factor_before = factor;
            some_before = some;
            continue;
        }
        if (!FORWARD && some) {                    // the entries' weights, while the stores fly, added up in the order of a forward call
            goal = tid < g.k ? p[tid] : -(A)INFINITY;
            A most = wave_max(goal);
            if (g.k > 64) {
                if ((tid & 63) == 0) rooms[0][0][tid / 64] = most;
                __syncthreads();
                for (int w = 0; w < (g.k + 63) / 64; w++) most = larger(most, rooms[0][0][w]);
            }
            const A own_weight = goal == -(A)INFINITY ? (A)0 : ScaledExp<A>(scale, in_scalar(most))(goal), all = wave_sum(own_weight);
            if (tid < g.k) p[tid] = own_weight;
            if ((tid & 63) == 0) rooms[1][0][tid / 64] = all;
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();                           // the row's stores are done: the entries' classes come after
        if (!FORWARD && some) {
            A all = rooms[1][0][0];                // (of few entries the first wave, which has them all, is the only one that this is for)
            for (int w = 1; w < (g.k + 63) / 64; w++) all += rooms[1][0][w];
            part = one_over(all);
        }
        if (some) correct_row(grad, turn, weight, share, part, factor);
    }
    if (LATER && g.grad) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        correct_before(row - (int)gridDim.x, turn ^ 1);
    }
}

// The loss alone: nothing of a row is needed twice, so that a workgroup of 256 walks it with a running largest value and sum, and eight of them share a CU
template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS, sizeof(T) < 8 ? 8 : 4) distill_loss_rows_kernel(DistillArgs<typename traits<T>::acc> g) {
    using A = typename traits<T>::acc;
    constexpr int N = vec16<T>::N, U = 4, WAVES = THREADS / 64, PIECE = U * THREADS * N;
    __shared__ A rooms[3][2][WAVES];
    const A scale = in_scalar((A)1 / g.temperature);
    const int row_bytes = g.classes * (int)sizeof(T) / 4 * 4, tid = threadIdx.x;
    const bool odd = sizeof(T) == 2 && g.classes % 2;
    for (int row = blockIdx.x; row < g.rows; row += gridDim.x) {
        const T* s = (const T*)g.logits + row * g.logits_rs;
        const __amdgpu_buffer_rsrc_t from = buffer_rsrc(s, row_bytes);
        u32x4_t next[U];
        auto load = [&](int c0) {
#pragma unroll
            for (int i = 0; i < U; i++) next[i] = __builtin_amdgcn_raw_buffer_load_b128(from, (c0 + (i * THREADS + tid) * N) * (int)sizeof(T), 0, 0);
        };
        load(0);
        int v = -1;
        A goal = -(A)INFINITY, value = 0;
        if (tid < g.k) {
            const int id = g.ids[(long long)row * g.k + tid];
            if (id >= 0 && id < g.classes) goal = widen(((const T*)g.teacher)[(long long)row * g.k + tid]);
            if (!(goal == -(A)INFINITY)) { v = id; value = widen(s[id]); }
        }
        A top = -(A)INFINITY, sum = 0;
        if (odd && tid == 0) top = widen(s[g.classes - 1]);      // (an odd last element of 16 bits goes by itself)
        ScaledExp<A> weight(scale, top);
        if (odd && tid == 0) sum = weight(top);
        for (int c0 = 0; c0 < g.classes; c0 += PIECE) {
            T x[U][N];
            __builtin_memcpy(x, next, sizeof(x));
            if (c0 + PIECE < g.classes) load(c0 + PIECE);
            if (c0 + PIECE > g.classes) {
#pragma unroll
                for (int i = 0; i < U; i++)
#pragma unroll
                    for (int u = 0; u < N; u++) x[i][u] = c0 + (i * THREADS + tid) * N + u < g.classes - odd ? x[i][u] : round_to<T>(-(A)INFINITY);
            }
            A most = top;
#pragma unroll
            for (int i = 0; i < U; i++)
#pragma unroll
                for (int u = 0; u < N; u++) most = plain_max(most, widen(x[i][u]));
            const ScaledExp<A> next_weight(scale, most);
            sum *= top == -(A)INFINITY ? (A)0 : weight.as(next_weight);
            weight = next_weight;
#pragma unroll
            for (int i = 0; i < U; i++)
#pragma unroll
                for (int u = 0; u < N; u++) sum += weight(widen(x[i][u]));
            top = most;
        }
        A tops[2] = {top, goal};
        team_tops_in_turn<THREADS>(tops, rooms[0][0]);
        const ScaledExp<A> row_weight(scale, tops[0]), goal_weight(scale, tops[1]);
        A sums[2] = {top == -(A)INFINITY ? sum * 0 : sum * weight.as(row_weight), v < 0 ? (A)0 : goal_weight(goal)};
        team_sums_in_turn<THREADS>(sums, rooms[1][0]);
        const bool some = !(tops[1] == -(A)INFINITY);
        const A own_p = v < 0 ? (A)0 : goal_weight(goal) * one_over(sums[1]);
        A loss[1] = {own_p != 0 ? own_p * ((goal_weight.log(goal) - natural_log(sums[1])) - (row_weight.log(value) - natural_log(sums[0]))) : (A)0};
        if (g.k > 64) team_sums_in_turn<THREADS>(loss, rooms[2][0]);
        else loss[0] = wave_sum(loss[0]);
        if (tid == 0) {
            g.stats[row] = tops[0];
            g.stats[g.rows + row] = some ? sums[0] : (A)-1;
            g.stats[2 * (long long)g.rows + row] = some ? loss[0] * g.temperature * g.temperature : (A)0;
        }
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
    // as many workgroups as the CUs hold at a time, each of which walks rows
    const int cus = device_cu_count() > 0 ? device_cu_count() : 256, held = THREADS == 1024 ? distill_waves(THREADS, STEPS, sizeof(T)) / 4 : 8, blocks = g.rows < cus * held ? g.rows : cus * held;
    if (forward) hipLaunchKernelGGL((distill_kernel<T, THREADS, STEPS, true>), dim3(blocks), dim3(THREADS), 0, current_stream(), g);
    else hipLaunchKernelGGL((distill_kernel<T, THREADS, STEPS, false>), dim3(blocks), dim3(THREADS), 0, current_stream(), g);
    return check_launch("distill_kernel") ? 0 : -1;
}

template <typename T, int THREADS>
static int launch_distill_loss_rows(const DistillArgs<typename traits<T>::acc>& g) {
    const int cus = device_cu_count() > 0 ? device_cu_count() : 256, held = cus * (2048 / THREADS);
    hipLaunchKernelGGL((distill_loss_rows_kernel<T, THREADS>), dim3(g.rows < held ? g.rows : held), dim3(THREADS), 0, current_stream(), g);
    return check_launch("distill_loss_rows_kernel") ? 0 : -1;
}

template <typename T>
static int launch_distill(const DistillArgs<typename traits<T>::acc>& g, bool forward) {
    constexpr int N = vec16<T>::N;
    // (777 x 50021 fp16, the loss: rows held in registers 42 us, walked 25; byte offsets in 32 bits)
    if (forward && !g.grad && g.classes >= N && g.classes < (1 << 27)) return g.k <= 256 ? launch_distill_loss_rows<T, 256>(g) : launch_distill_loss_rows<T, 1024>(g);
    if (g.classes < N) return launch_distill_row<T, 1024, 0>(g, forward);
    if ((long long)g.classes > 1024ll * 16 * N) {
        // (rows longer than registers: walked once for the sums and once for the gradient)
        if (forward && g.classes < (1 << 27)) {
            DistillArgs<typename traits<T>::acc> loss = g;
            loss.grad = nullptr;
            if (launch_distill<T>(loss, true) != 0) return -1;
            forward = false;
        }
        return launch_distill_row<T, 1024, 0>(g, forward);
    }
    if (g.k > 256) {                               // (an entry a thread)
        if (g.classes <= 1024 * 2 * N) return launch_distill_row<T, 1024, 2>(g, forward);
    } else if (g.classes <= 256 * N) return launch_distill_row<T, 256, 1>(g, forward);
    if (g.k <= 256 && g.classes <= 256 * 4 * N) return launch_distill_row<T, 256, 4>(g, forward);
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
