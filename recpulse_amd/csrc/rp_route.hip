// Routing of tokens to experts, and the exchange of rows between tokens and their experts' groups.
//
// Routing.  Each token takes its k largest logits (equal ones in the order of their index, -inf never), and a weight for each:
//   w_j = exp(l_j - max) / sum,   the sum over the k taken ("normalize") or over all experts.
// A slot is (token, j), slot number token * k + j.  The slots are sorted by expert, in slot order within an expert:
//   offsets[e] .. offsets[e + 1]   the places of expert e's slots,   order[place] = slot,   position[slot] = place.
// The sort counts: it needs how many slots of each expert lie before a slot, no comparison.
//
// Exchange.  dispatch: out[position[t, j]] = x[t].  combine: y[t] = sum over j of w[t, j] z[position[t, j]].  Each is the other's
// gradient (with w = 1); the gradient of combine also has dw[t, j] = dy[t] . z[position[t, j]].
#include "rp_rows.h"

#include <type_traits>

namespace rp {

constexpr int ROUTE_MAX_K = 16, ROUTE_MAX_EXPERTS = 1024, ROUTE_MAX_SLOTS = 1 << 30;
constexpr int SORT_CHUNKS = 256;             // workgroups that a longer list is dealt to, at most

// ---- order-preserving integer keys: larger logit, larger key; equal logits (+0 and -0 too), equal keys ----
// 0 is "not there": an expert that is taken already, one past the last, or a logit of -inf.  NaN is above every number.
template <typename A> struct logit_key;
template <> struct logit_key<float> {
    using type = uint32_t;
    static __device__ __forceinline__ type of(float x) {
        if (x != x) return 0xFFFFFFFFu;
        const uint32_t b = __float_as_uint(x + 0.f);                       // (-0 + 0 = +0)
        return b == 0xFF800000u ? 0u : (b & 0x80000000u) ? ~b : b | 0x80000000u;
    }
    static __device__ __forceinline__ float value(type k) { return __uint_as_float((k & 0x80000000u) ? k & 0x7FFFFFFFu : ~k); }
};
template <> struct logit_key<double> {
    using type = uint64_t;
    static __device__ __forceinline__ type of(double x) {
        if (x != x) return ~0ull;
        const uint64_t b = __builtin_bit_cast(uint64_t, x + 0.0);
        return b == 0xFFF0000000000000ull ? 0ull : (b >> 63) ? ~b : b | (1ull << 63);
    }
    static __device__ __forceinline__ double value(type k) { return __builtin_bit_cast(double, (k >> 63) ? k & ~(1ull << 63) : ~k); }
};

// ---- reductions over the LANES (16 or 64) lanes of a token, the result in all of them ----
// Inside a row of 16 lanes by rotating it (DPP, no LDS); all lanes see the same tree, so sums are the same in every lane.
template <int ROT> __device__ __forceinline__ uint32_t row_rotate(uint32_t v) { return __builtin_amdgcn_update_dpp(v, v, 0x120 + ROT, 0xf, 0xf, false); }
template <int ROT, typename V> __device__ __forceinline__ V row_rotated(V v) {
    if constexpr (sizeof(V) == 4) return __builtin_bit_cast(V, row_rotate<ROT>(__builtin_bit_cast(uint32_t, v)));
    else {
        const uint64_t b = __builtin_bit_cast(uint64_t, v);
        return __builtin_bit_cast(V, (uint64_t)row_rotate<ROT>((uint32_t)b) | (uint64_t)row_rotate<ROT>((uint32_t)(b >> 32)) << 32);
    }
}
template <typename V> __device__ __forceinline__ V from_lane(V v, int lane) {
    if constexpr (sizeof(V) == 4) return __builtin_bit_cast(V, __builtin_amdgcn_readlane(__builtin_bit_cast(uint32_t, v), lane));
    else {
        const uint64_t b = __builtin_bit_cast(uint64_t, v);
        return __builtin_bit_cast(V, (uint64_t)(uint32_t)__builtin_amdgcn_readlane((uint32_t)b, lane) | (uint64_t)(uint32_t)__builtin_amdgcn_readlane((uint32_t)(b >> 32), lane) << 32);
    }
}
template <int LANES, typename V, typename F> __device__ __forceinline__ V reduce_lanes(V v, F f) {
    v = f(v, row_rotated<8>(v));
    v = f(v, row_rotated<4>(v));
    v = f(v, row_rotated<2>(v));
    v = f(v, row_rotated<1>(v));
    if constexpr (LANES == 64) v = f(f(from_lane(v, 0), from_lane(v, 16)), f(from_lane(v, 32), from_lane(v, 48)));
    return v;
}

// ---- a logit and its expert in one number: the largest is the largest logit's, the lowest index among equal ones ----
// Below 1: not there.  float32: key and 1023 - expert are the upper 32 and lower 10 bits of a whole number that float64 holds exactly, and a
// maximum is one instruction (the value is never NaN or negative; written as an instruction, the compiler would quiet both operands first).
// 16 bits: the same in a uint32.  float64 has no wider type: key and expert are found one after the other.
template <typename T> struct Candidate {
    using type = double;
    static __device__ __forceinline__ type of(float x, int e) {
        const uint32_t k = logit_key<float>::of(x);
        return k ? __builtin_fma((double)k, 1024.0, (double)(1023 - e)) : 0.0;
    }
    static __device__ __forceinline__ type largest(type a, type b) {
        double r;
        asm("v_max_f64 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
        return r;
    }
    static __device__ __forceinline__ bool there(type c) { return c >= 1.0; }
    static __device__ __forceinline__ type without(type c, type taken) {                   // (the upper word alone: what is left is below 1)
        const uint64_t b = __builtin_bit_cast(uint64_t, c);
        return __builtin_bit_cast(double, (uint64_t)(c == taken ? 0u : (uint32_t)(b >> 32)) << 32 | (uint32_t)b);
    }
    static __device__ __forceinline__ uint32_t key(type c) { return (uint32_t)(c * (1.0 / 1024.0)); }
    static __device__ __forceinline__ int expert(type c) { return 1023 - (int)(c - (double)key(c) * 1024.0); }
    static __device__ __forceinline__ float value(type c) { return logit_key<float>::value(key(c)); }
};
// DROP: bits of a 16-bit value's float32 key that say nothing (all zeros, of a negative value all ones)
template <int DROP> struct Candidate16 {
    using type = uint32_t;
    static __device__ __forceinline__ type of(float x, int e) {
        const uint32_t k = logit_key<float>::of(x) >> DROP;
        return k ? k << 10 | (uint32_t)(1023 - e) : 0u;
    }
    static __device__ __forceinline__ type largest(type a, type b) { return a > b ? a : b; }
    static __device__ __forceinline__ bool there(type c) { return c != 0; }
    static __device__ __forceinline__ type without(type c, type taken) { return c == taken ? 0u : c; }
    static __device__ __forceinline__ int expert(type c) { return 1023 - (int)(c & 1023u); }
    static __device__ __forceinline__ float value(type c) {
        const uint32_t k = c >> 10 << DROP;
        return logit_key<float>::value(k & 0x80000000u ? k : k | ((1u << DROP) - 1));
    }
};
template <> struct Candidate<bf16_t> : Candidate16<16> {};
template <> struct Candidate<f16_t> : Candidate16<13> {};

// The k largest of a token's logits by LANES lanes, V experts a lane (expert e sits in lane e % LANES).  Lane j < k returns slot j's
// expert (-1: none was left) and weight.
// What bounds it is the chain of k selections, each a maximum over the experts; rows of 16 lanes keep four tokens in a wave and every
// reduction inside a DPP row.  (With the largest key found first and then the lowest index that has it, 200000 tokens of 128 took 100 us, now 72.)
template <typename T, int LANES, int V>
__device__ __forceinline__ void route_token(const T* row, bool live, int experts, int k, bool normalize, int l, int& expert, typename traits<T>::acc& weight) {
    using A = typename traits<T>::acc;
    A x[V];
#pragma unroll
    for (int v = 0; v < V; v++) {
        const int e = v * LANES + l;
        x[v] = live && e < experts ? widen(row[e]) : (A)-INFINITY;
    }
    expert = -1;
    A value = 0, top = 0;
    if constexpr (sizeof(A) == 4) {
        using C = Candidate<T>;
        using P = typename C::type;
        P cand[V], mine = 0;
#pragma unroll
        for (int v = 0; v < V; v++) cand[v] = C::of(x[v], v * LANES + l);
        for (int j = 0; j < k; j++) {
            P best = cand[0];
#pragma unroll
            for (int v = 1; v < V; v++) best = C::largest(best, cand[v]);
            best = reduce_lanes<LANES>(best, [](P a, P b) { return C::largest(a, b); });
#pragma unroll
            for (int v = 0; v < V; v++) cand[v] = C::without(cand[v], best);
            if (j == 0) top = C::there(best) ? C::value(best) : (A)0;
            if (l == j) mine = best;
        }
        if (C::there(mine)) { expert = C::expert(mine); value = C::value(mine); }
    } else {
        using K = typename logit_key<A>::type;
        K key[V];
#pragma unroll
        for (int v = 0; v < V; v++) key[v] = logit_key<A>::of(x[v]);
        for (int j = 0; j < k; j++) {
            K best = key[0];
#pragma unroll
            for (int v = 1; v < V; v++) best = key[v] > best ? key[v] : best;
            best = reduce_lanes<LANES>(best, [](K a, K b) { return a > b ? a : b; });
            int at = 0x7fffffff;
#pragma unroll
            for (int v = V - 1; v >= 0; v--) at = key[v] == best ? v * LANES + l : at;
            at = reduce_lanes<LANES>(at, [](int a, int b) { return a < b ? a : b; });
            if (best == 0) continue;                          // (the same for all lanes of the token)
#pragma unroll
            for (int v = 0; v < V; v++) key[v] = at == v * LANES + l ? (K)0 : key[v];
            const A got = logit_key<A>::value(best);
            if (j == 0) top = got;
            if (l == j) { expert = at; value = got; }
        }
    }
    const A e = expert >= 0 ? exp(value - top) : (A)0;        // (an infinite or NaN top leaves NaN weights)
    A sum = 0;
    if (normalize) sum = e;
    else {
#pragma unroll
        for (int v = 0; v < V; v++) sum += x[v] == (A)-INFINITY ? (A)0 : exp(x[v] - top);
    }
    sum = reduce_lanes<LANES>(sum, [](A a, A b) { return a + b; });
    weight = expert >= 0 ? e / sum : (A)0;
}

// ---- the sort ----
// Slots [s0, s1) by a workgroup of WAVES waves, each a run of whole 64s; where[e] is the place of the first one of expert e.  position may be null.
// counts: [WAVES][groups] in LDS, zeroed.  Lanes with the same expert find each other bit by bit (a ballot for each bit of the number).
template <int WAVES>
__device__ __forceinline__ void sort_slots(const int* ids, int s0, int s1, int groups, int bits, int* counts, const int* where, int* order, int* position) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int run = ((s1 - s0 + WAVES - 1) / WAVES + 63) / 64 * 64;
    const int b = s0 + wave * run, e = b + run < s1 ? b + run : s1;
    int* mine = counts + wave * groups;
    for (int s = b + lane; s < e; s += 64) {
        const int id = ids[s];
        if ((unsigned)id < (unsigned)groups) atomicAdd(&mine[id], 1);         // (a count: the order of the additions does not matter)
    }
    __syncthreads();
    for (int g = threadIdx.x; g < groups; g += WAVES * 64) {
        int at = where[g];
#pragma unroll
        for (int w = 0; w < WAVES; w++) { const int c = counts[w * groups + g]; counts[w * groups + g] = at; at += c; }
    }
    __syncthreads();
    for (int s = b; s < e; s += 64) {
        const int slot = s + lane;
        const int id = slot < e ? ids[slot] : -1;
        const bool in = (unsigned)id < (unsigned)groups;
        unsigned long long same = __builtin_amdgcn_ballot_w64(in);
        for (int bit = 0; bit < bits; bit++) {
            const bool set = (id >> bit) & 1;
            const unsigned long long have = __builtin_amdgcn_ballot_w64(set);
            same &= set ? have : ~have;
        }
        const int before = __builtin_popcountll(same & ((1ull << lane) - 1));
        const int first = in ? mine[id] : 0;
        if (in) {
            const int place = first + before;
            order[place] = slot;
            if (position) position[slot] = place;
            if (before == 0) mine[id] = first + __builtin_popcountll(same);   // (one lane of each expert; the wave reads it in its next round)
        } else if (slot < e && position) {
            position[slot] = -1;
        }
        __builtin_amdgcn_wave_barrier();
    }
}

// Exclusive sums of totals[0 .. groups) by the workgroup, in place, and their total in totals[groups].
__device__ __forceinline__ void sum_totals(int* totals, int groups) {
    if (threadIdx.x < 64) {
        int before = 0;
        for (int g0 = 0; g0 < groups; g0 += 64) {
            const int g = g0 + (int)threadIdx.x;
            const int c = g < groups ? totals[g] : 0;
            const int upto = before + wave_prefix_sum(c, threadIdx.x);
            if (g < groups) totals[g] = upto - c;
            before = __builtin_amdgcn_readlane(upto, 63);
        }
        if (threadIdx.x == 0) totals[groups] = before;
    }
    __syncthreads();
}

constexpr int SORT_ONE_WAVES = 16;
// The whole sort in one workgroup; ids in LDS or in memory.  lds: (SORT_ONE_WAVES + 1) * groups + 1 ints.
__device__ __forceinline__ void sort_all(const int* ids, int count, int groups, int bits, int* lds, int* offsets, int* order, int* position) {
    int* counts = lds;
    int* totals = lds + SORT_ONE_WAVES * groups;
    for (int i = threadIdx.x; i < (SORT_ONE_WAVES + 1) * groups + 1; i += SORT_ONE_WAVES * 64) lds[i] = 0;
    __syncthreads();
    for (int s = threadIdx.x; s < count; s += SORT_ONE_WAVES * 64) {
        const int id = ids[s];
        if ((unsigned)id < (unsigned)groups) atomicAdd(&totals[id], 1);
    }
    __syncthreads();
    sum_totals(totals, groups);
    for (int g = threadIdx.x; g <= groups; g += SORT_ONE_WAVES * 64) offsets[g] = totals[g];
    sort_slots<SORT_ONE_WAVES>(ids, 0, count, groups, bits, counts, totals, order, position);
    for (int s = totals[groups] + threadIdx.x; s < count; s += SORT_ONE_WAVES * 64) order[s] = -1;
}

__global__ void __launch_bounds__(SORT_ONE_WAVES * 64) sort_one_kernel(const int* ids, int count, int groups, int bits, int* offsets, int* order, int* position) {
    extern __shared__ int sort_lds[];
    sort_all(ids, count, groups, bits, sort_lds, offsets, order, position);
}

// Longer lists in two launches: count each chunk's slots by expert, into counts [chunks][groups], then place each chunk's slots.  A workgroup of
// the second adds up the counts of all chunks by itself: 256 chunks of 128 experts are 128 KB out of the L2, which takes less than a launch
// between the two that adds them up once (16384 tokens, 8 of 128 experts: 13.8 us in three launches, 7.3 here, the counts coming from the selection).
__device__ __forceinline__ void count_ids(const int* ids, int s0, int s1, int groups, int* counts) {
    for (int s = s0 + threadIdx.x; s < s1; s += SORT_ONE_WAVES * 64) {
        const int id = ids[s];
        if ((unsigned)id < (unsigned)groups) atomicAdd(&counts[id], 1);
    }
}

__global__ void __launch_bounds__(SORT_ONE_WAVES * 64) sort_count_kernel(const int* ids, int count, int groups, int chunk, int* counts) {
    __shared__ int own[ROUTE_MAX_EXPERTS];
    for (int g = threadIdx.x; g < groups; g += SORT_ONE_WAVES * 64) own[g] = 0;
    __syncthreads();
    const int s0 = blockIdx.x * chunk, s1 = blockIdx.x + 1 == gridDim.x ? count : s0 + chunk;
    count_ids(ids, s0, s1, groups, own);
    __syncthreads();
    for (int g = threadIdx.x; g < groups; g += SORT_ONE_WAVES * 64) counts[(size_t)blockIdx.x * groups + g] = own[g];
}

// `parts` threads to an expert (their number a power of two, `width` experts), each a run of chunks
__global__ void __launch_bounds__(SORT_ONE_WAVES * 64) sort_place_kernel(const int* ids, int count, int groups, int bits, int chunk, int parts, const int* counts, int* offsets, int* order, int* position) {
    extern __shared__ int sort_lds[];                          // [SORT_ONE_WAVES][groups] counts, where [groups], totals [groups + 1], sums [2][1024]
    int* where = sort_lds + SORT_ONE_WAVES * groups;
    int* totals = where + groups;
    int* sums = totals + groups + 1;
    const int chunks = (int)gridDim.x, own = (int)blockIdx.x, width = SORT_ONE_WAVES * 64 / parts;
    for (int i = threadIdx.x; i < SORT_ONE_WAVES * groups; i += SORT_ONE_WAVES * 64) sort_lds[i] = 0;
    {
        const int g = threadIdx.x % width, part = threadIdx.x / width, per = (chunks + parts - 1) / parts;
        const int c0 = part * per < chunks ? part * per : chunks, c1 = c0 + per < chunks ? c0 + per : chunks;
        int before = 0, all = 0;
        if (g < groups) {
#pragma unroll 16
            for (int c = c0; c < c1; c++) {
                const int n = counts[(size_t)c * groups + g];
                all += n;
                before += c < own ? n : 0;
            }
        }
        sums[threadIdx.x] = before;
        sums[SORT_ONE_WAVES * 64 + threadIdx.x] = all;
    }
    __syncthreads();
    for (int g = threadIdx.x; g < groups; g += SORT_ONE_WAVES * 64) {
        int before = 0, all = 0;
        for (int p = 0; p < parts; p++) {
            before += sums[p * width + g];
            all += sums[SORT_ONE_WAVES * 64 + p * width + g];
        }
        where[g] = before;
        totals[g] = all;
    }
    __syncthreads();
    sum_totals(totals, groups);
    for (int g = threadIdx.x; g < groups; g += SORT_ONE_WAVES * 64) where[g] += totals[g];
    if (own == 0)
        for (int g = threadIdx.x; g <= groups; g += SORT_ONE_WAVES * 64) offsets[g] = totals[g];
    __syncthreads();
    const int s0 = own * chunk, s1 = own + 1 == chunks ? count : s0 + chunk;
    sort_slots<SORT_ONE_WAVES>(ids, s0, s1, groups, bits, sort_lds, where, order, position);
    for (long long s = (long long)totals[groups] + own * (SORT_ONE_WAVES * 64) + threadIdx.x; s < count; s += chunks * (SORT_ONE_WAVES * 64)) order[s] = -1;
}

// position from order, where the counts lay in position itself
__global__ void __launch_bounds__(256) sort_invert_kernel(const int* ids, const int* order, int* position, int count, int groups) {
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < count; i += (long long)gridDim.x * 256) {
        const int slot = order[i];
        if (slot >= 0) position[slot] = (int)i;
        if ((unsigned)ids[i] >= (unsigned)groups) position[i] = -1;
    }
}

// ---- routing: kernels ----
template <typename T> using weight_t = typename traits<T>::acc;        // routing weights: float32 (float64 for float64), not rounded to 16 bits

// A chunk of `per_block` tokens a workgroup, whose slots it counts by expert for the sort
template <typename T, int LANES, int V>
__global__ void __launch_bounds__(SORT_ONE_WAVES * 64) route_topk_kernel(weight_t<T>* weights, int* experts_out, int* counts, const T* logits, long long rs, int tokens, int experts, int k, int normalize,
                                                                        int per_block) {
    __shared__ int own[ROUTE_MAX_EXPERTS];
    for (int g = threadIdx.x; g < experts; g += SORT_ONE_WAVES * 64) own[g] = 0;
    __syncthreads();
    const int l = threadIdx.x % LANES, t0 = (int)blockIdx.x * per_block, t1 = blockIdx.x + 1 == gridDim.x ? tokens : t0 + per_block;
    for (int t = t0 + threadIdx.x / LANES; t - (int)threadIdx.x / LANES < t1; t += SORT_ONE_WAVES * 64 / LANES) {      // (whole waves together)
        const bool live = t < t1;
        int expert;
        weight_t<T> w;
        route_token<T, LANES, V>(logits + (long long)(live ? t : 0) * rs, live, experts, k, normalize != 0, l, expert, w);
        if (live && l < k) {
            weights[(size_t)t * k + l] = w;
            experts_out[(size_t)t * k + l] = expert;
            if (expert >= 0) atomicAdd(&own[expert], 1);
        }
    }
    if (!counts) return;
    __syncthreads();
    for (int g = threadIdx.x; g < experts; g += SORT_ONE_WAVES * 64) counts[(size_t)blockIdx.x * experts + g] = own[g];
}

// A few tokens: selection and sort in one workgroup and one launch
constexpr int ROUTE_ONE_THREADS = SORT_ONE_WAVES * 64;
template <typename T, int LANES, int V>
__global__ void __launch_bounds__(ROUTE_ONE_THREADS) route_one_kernel(weight_t<T>* weights, int* experts_out, int* offsets, int* order, int* position,
                                                                      const T* logits, long long rs, int tokens, int experts, int k, int normalize, int bits) {
    extern __shared__ int sort_lds[];
    int* ids = sort_lds + (SORT_ONE_WAVES + 1) * experts + 1;  // [tokens * k]
    const int l = threadIdx.x % LANES, t = threadIdx.x / LANES;
    const bool live = t < tokens;
    int expert;
    weight_t<T> w;
    route_token<T, LANES, V>(logits + (long long)(live ? t : 0) * rs, live, experts, k, normalize != 0, l, expert, w);
    if (live && l < k) { weights[(size_t)t * k + l] = w; experts_out[(size_t)t * k + l] = expert; ids[t * k + l] = expert; }
    __syncthreads();
    sort_all(ids, tokens * k, experts, bits, sort_lds, offsets, order, position);
}

// Gradient of the logits, bound by memory from about 10^5 tokens on (200000 of 128 in fp32 51 us, 4 TB/s; 16384 8.6 us).  With p the softmax over the experts that the weights were divided by, and g_j the weights' gradients,
//   dl_e = p_e (g_e - sum over j of w_j g_j),   g_e = 0 where e was not taken; with "normalize" p_e = w_j where taken and 0 elsewhere.
template <typename T, int LANES, int V>
__global__ void __launch_bounds__(256) route_backward_kernel(T* grad, const weight_t<T>* grad_weights, const weight_t<T>* weights, const int* taken, const T* logits, long long rs,
                                                             int tokens, int experts, int k, int normalize, long long first) {
    using A = typename traits<T>::acc;
    const int l = threadIdx.x % LANES;
    const long long t = (first + blockIdx.x) * (256 / LANES) + threadIdx.x / LANES;
    if (t >= tokens) return;                                   // (all lanes of a token)
    const int id_l = l < k ? taken[(size_t)t * k + l] : -1;
    const A w_l = id_l >= 0 ? weights[(size_t)t * k + l] : (A)0, g_l = id_l >= 0 ? grad_weights[(size_t)t * k + l] : (A)0;
    const A mean = reduce_lanes<LANES>(id_l >= 0 ? w_l * g_l : (A)0, [](A a, A b) { return a + b; });
    A p[V], d[V];
    if (!normalize) {
        A x[V], top = (A)-INFINITY, sum = 0;
#pragma unroll
        for (int v = 0; v < V; v++) {
            const int e = v * LANES + l;
            x[v] = e < experts ? widen(logits[t * rs + e]) : (A)-INFINITY;
            top = x[v] > top ? x[v] : top;
        }
        top = reduce_lanes<LANES>(top, [](A a, A b) { return a > b ? a : b; });
        if (top == (A)-INFINITY) top = 0;
#pragma unroll
        for (int v = 0; v < V; v++) { p[v] = x[v] == (A)-INFINITY ? (A)0 : exp(x[v] - top); sum += p[v]; }
        sum = reduce_lanes<LANES>(sum, [](A a, A b) { return a + b; });
        const A inv = sum == (A)0 ? (A)0 : (A)1 / sum;
#pragma unroll
        for (int v = 0; v < V; v++) { p[v] *= inv; d[v] = -p[v] * mean; }
    } else {
#pragma unroll
        for (int v = 0; v < V; v++) d[v] = 0;
    }
    const int base = (threadIdx.x & 63) / LANES * LANES;
    for (int j = 0; j < k; j++) {
        const int id = __shfl(id_l, base + j);
        const A w = __shfl(w_l, base + j), g = __shfl(g_l, base + j);
#pragma unroll
        for (int v = 0; v < V; v++)
            if (v * LANES + l == id) d[v] = (normalize ? w : p[v]) * (g - mean);
    }
#pragma unroll
    for (int v = 0; v < V; v++) {
        const int e = v * LANES + l;
        if (e < experts) grad[(size_t)t * experts + e] = round_to<T>(d[v]);
    }
}

// f(LANES, V): rows of 16 lanes hold up to 256 experts, 16 a lane; more take a wave.  (V = experts a lane, the next of 4, 8, 16.)
template <typename F>
static int pick_route_shape(int experts, F f) {
    using std::integral_constant;
    if (experts <= 64) return f(integral_constant<int, 16>{}, integral_constant<int, 4>{});
    if (experts <= 128) return f(integral_constant<int, 16>{}, integral_constant<int, 8>{});
    if (experts <= 256) return f(integral_constant<int, 16>{}, integral_constant<int, 16>{});
    return f(integral_constant<int, 64>{}, integral_constant<int, 16>{});
}

static int bits_of(int groups) {
    int bits = 0;
    while ((1 << bits) < groups) bits++;
    return bits;
}

// Lists up to this length are sorted by one workgroup in one launch
constexpr int SORT_ONE_MAX = 4096;

// Chunks of a list; a short last one is joined to the one before where the counts would otherwise be more than the slots
static int sort_chunks(int count, int chunk, int groups) {
    const int chunks = (count - 1) / chunk + 1;
    return (long long)chunks * groups > count ? chunks - 1 : chunks;
}

// The counts of a longer list lie in the null stream's own memory.  On other streams, whose calls would share a block of the pool, and in graphs they lie in `position`, which
// a third launch then fills; there are no more of them than slots.
struct SortCounts {
    NullStreamScratch lease;
    int* position;
    SortCounts(size_t ints, int* p) : lease(ints * sizeof(int)), position(p) {}
    bool in_place() const { return !lease.ptr; }
    int* ptr() const { return lease.ptr ? (int*)lease.ptr : position; }
};

static int launch_place(int* offsets, int* order, int* position, const int* ids, int count, int groups, int chunk, int chunks, const SortCounts& counts) {
    int width = 32;
    while (width < groups) width *= 2;
    const size_t lds = ((size_t)(SORT_ONE_WAVES + 2) * groups + 1 + 2 * SORT_ONE_WAVES * 64) * sizeof(int);
    if (lds > 64 * 1024 && !check_hip(hipFuncSetAttribute((const void*)sort_place_kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds), "hipFuncSetAttribute")) return -1;
    hipLaunchKernelGGL(sort_place_kernel, dim3(chunks), dim3(SORT_ONE_WAVES * 64), lds, current_stream(), ids, count, groups, bits_of(groups), chunk, SORT_ONE_WAVES * 64 / width, counts.ptr(), offsets, order,
                       counts.in_place() ? nullptr : position);
    if (!check_launch("sort_place_kernel")) return -1;
    if (!counts.in_place()) return 0;
    hipLaunchKernelGGL(sort_invert_kernel, dim3(count / 256 < 1024 ? count / 256 + 1 : 1024), dim3(256), 0, current_stream(), ids, order, position, count, groups);
    return check_launch("sort_invert_kernel") ? 0 : -1;
}

static int launch_sort_one(int* offsets, int* order, int* position, const int* ids, int count, int groups) {
    const size_t lds = ((size_t)(SORT_ONE_WAVES + 1) * groups + 1) * sizeof(int);
    if (lds > 64 * 1024 && !check_hip(hipFuncSetAttribute((const void*)sort_one_kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds), "hipFuncSetAttribute")) return -1;
    hipLaunchKernelGGL(sort_one_kernel, dim3(1), dim3(SORT_ONE_WAVES * 64), lds, current_stream(), ids, count, groups, bits_of(groups), offsets, order, position);
    return check_launch("sort_one_kernel") ? 0 : -1;
}

static int launch_sort(int* offsets, int* order, int* position, const int* ids, int count, int groups) {
    if (count <= SORT_ONE_MAX) return launch_sort_one(offsets, order, position, ids, count, groups);
    const int least = (count + SORT_CHUNKS - 1) / SORT_CHUNKS, chunk = ((least > groups ? least : groups) + 511) / 512 * 512, chunks = sort_chunks(count, chunk, groups);
    const SortCounts counts((size_t)chunks * groups, position);
    hipLaunchKernelGGL(sort_count_kernel, dim3(chunks), dim3(SORT_ONE_WAVES * 64), 0, current_stream(), ids, count, groups, chunk, counts.ptr());
    if (!check_launch("sort_count_kernel")) return -1;
    return launch_place(offsets, order, position, ids, count, groups, chunk, chunks, counts);
}

template <typename T>
static int launch_route(void* weights, int* experts_out, int* offsets, int* order, int* position, const void* logits, long long rs, int tokens, int experts, int k, int normalize) {
    return pick_route_shape(experts, [&](auto lanes_c, auto v_c) -> int {
        constexpr int LANES = decltype(lanes_c)::value, V = decltype(v_c)::value, PER = ROUTE_ONE_THREADS / LANES;
        if (tokens <= PER) {
            const size_t lds = ((size_t)(SORT_ONE_WAVES + 1) * experts + 1 + (size_t)tokens * k) * sizeof(int);
            auto kern = route_one_kernel<T, LANES, V>;
            if (lds > 64 * 1024 && !check_hip(hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds), "hipFuncSetAttribute")) return -1;
            hipLaunchKernelGGL(kern, dim3(1), dim3(ROUTE_ONE_THREADS), lds, current_stream(), (weight_t<T>*)weights, experts_out, offsets, order, position, (const T*)logits, rs,
                               tokens, experts, k, normalize, bits_of(experts));
            return check_launch("route_one_kernel") ? 0 : -1;
        }
        const int least = (tokens + SORT_CHUNKS - 1) / SORT_CHUNKS, whole = (experts + k - 1) / k, per_block = ((least > whole ? least : whole) + PER - 1) / PER * PER;
        if (tokens < 2 * per_block) {                          // too few for chunks that hold their counts
            hipLaunchKernelGGL((route_topk_kernel<T, LANES, V>), dim3((tokens + PER - 1) / PER), dim3(SORT_ONE_WAVES * 64), 0, current_stream(), (weight_t<T>*)weights, experts_out, nullptr,
                               (const T*)logits, rs, tokens, experts, k, normalize, PER);
            return check_launch("route_topk_kernel") ? launch_sort(offsets, order, position, experts_out, tokens * k, experts) : -1;
        }
        const int chunks = sort_chunks(tokens * k, per_block * k, experts);
        const SortCounts counts((size_t)chunks * experts, position);
        hipLaunchKernelGGL((route_topk_kernel<T, LANES, V>), dim3(chunks), dim3(SORT_ONE_WAVES * 64), 0, current_stream(), (weight_t<T>*)weights, experts_out, counts.ptr(), (const T*)logits, rs,
                           tokens, experts, k, normalize, per_block);
        if (!check_launch("route_topk_kernel")) return -1;
        return launch_place(offsets, order, position, experts_out, tokens * k, experts, per_block * k, chunks, counts);
    });
}

template <typename T>
static int launch_route_backward(void* grad, const void* grad_weights, const void* weights, const int* taken, const void* logits, long long rs, int tokens, int experts, int k, int normalize) {
    return pick_route_shape(experts, [&](auto lanes_c, auto v_c) -> int {
        constexpr int LANES = decltype(lanes_c)::value, V = decltype(v_c)::value, PER = 256 / LANES;
        return in_launches(((long long)tokens + PER - 1) / PER, 256, [&](unsigned blocks, long long first) -> int {
            hipLaunchKernelGGL((route_backward_kernel<T, LANES, V>), dim3(blocks), dim3(256), 0, current_stream(), (T*)grad, (const weight_t<T>*)grad_weights,
                               (const weight_t<T>*)weights, taken, (const T*)logits, rs, tokens, experts, k, normalize, first);
            return check_launch("route_backward_kernel") ? 0 : -1;
        });
    });
}

// ---- exchange: kernels ----
// All of them are bound by memory: a row is read and written once, in pieces of 16 bytes where rows allow it (VEC elements;
// otherwise element by element).  8192 tokens of 4096 in bf16, two rows each: dispatch 31 us (6.0 TB/s), combine 41 (4.6), its gradient 67 (4.5).
// (Stores that stream past the caches make combine 34 and its gradient 61, and whoever reads the rows next slower by more: dispatch and a kernel that reads its 134 MB
// take 66 us, 91 with them.)
typedef __attribute__((ext_vector_type(4))) unsigned int row_vec_t;
template <typename T, int VEC>
struct Piece {
    T e[VEC];
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (VEC == 1) e[0] = *p;
        else { const row_vec_t v = *(const row_vec_t*)p; __builtin_memcpy(e, &v, 16); }
    }
    __device__ __forceinline__ void store(T* p) const {
        if constexpr (VEC == 1) *p = e[0];
        else { row_vec_t v; __builtin_memcpy(&v, e, 16); *(row_vec_t*)p = v; }
    }
};

// A thread for each (token, piece): one load and k stores
template <typename T, int VEC>
__global__ void __launch_bounds__(256) dispatch_kernel(T* out, const T* x, const int* position, long long total, int pieces, int k, unsigned slots, long long x_rs, long long out_rs) {
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
        const long long t = i / pieces;
        const int c = (int)(i - t * pieces) * VEC;
        Piece<T, VEC> p;
        p.load(x + t * x_rs + c);
        for (int j = 0; j < k; j++) {
            const int at = position[t * k + j];
            if ((unsigned)at < slots) p.store(out + at * out_rs + c);
        }
    }
}

// A thread for each (token, piece): k loads, added up in the order of the slots in 32 bits (64 for float64), one rounding
template <typename T, int VEC>
__global__ void __launch_bounds__(256) combine_kernel(T* y, const T* z, const weight_t<T>* weights, const int* position, long long total, int pieces, int k, unsigned slots,
                                                      long long y_rs, long long z_rs) {
    using A = typename traits<T>::acc;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
        const long long t = i / pieces;
        const int c = (int)(i - t * pieces) * VEC;
        A sum[VEC];
#pragma unroll
        for (int v = 0; v < VEC; v++) sum[v] = 0;
        auto add = [&](const Piece<T, VEC>& p, bool in, A w) {
#pragma unroll
            for (int v = 0; v < VEC; v++) sum[v] = in ? sum[v] + w * widen(p.e[v]) : sum[v];
        };
        // two rows at a time, so that two loads are in flight (a slot without a row reads row 0 and is left out)
        for (int j = 0; j < k; j += 2) {
            const bool two = j + 1 < k;
            const int a0 = position[t * k + j], a1 = two ? position[t * k + j + 1] : -1;
            const bool in0 = (unsigned)a0 < slots, in1 = (unsigned)a1 < slots;
            const A w0 = weights ? weights[t * k + j] : (A)1, w1 = weights && two ? weights[t * k + j + 1] : (A)1;
            Piece<T, VEC> p0, p1;
            p0.load(z + (in0 ? a0 : 0) * z_rs + c);
            p1.load(z + (in1 ? a1 : 0) * z_rs + c);
            add(p0, in0, w0);
            add(p1, in1, w1);
        }
        Piece<T, VEC> o;
#pragma unroll
        for (int v = 0; v < VEC; v++) o.e[v] = round_to<T>(sum[v]);
        o.store(y + t * y_rs + c);
    }
}

// Rows behind the last group: a workgroup a row, and nothing to do for nearly all of them
__global__ void __launch_bounds__(256) zero_rows_behind_kernel(unsigned char* x, const int* offsets, int groups, int rows, long long row_bytes, long long width_bytes) {
    const int last = offsets[groups];
    for (long long r = (last < 0 ? 0 : last) + blockIdx.x; r < rows; r += gridDim.x)
        for (long long i = threadIdx.x; i < width_bytes / 2; i += 256) ((uint16_t*)(x + r * row_bytes))[i] = 0;
}

// A wave for each token: its gradient stays in registers (HELD pieces a lane; longer rows are read again for each slot), z is read once
// and dz written once.  The 64 lanes' partial dots are added in a fixed tree.
template <typename T, int VEC, int HELD>
__global__ void __launch_bounds__(256) combine_backward_kernel(T* dz, weight_t<T>* dw, const T* dy, const T* z, const weight_t<T>* weights, const int* position, int tokens, int k, int d,
                                                               unsigned slots, long long dy_rs, long long z_rs, long long dz_rs) {
    using A = typename traits<T>::acc;
    const int lane = threadIdx.x & 63;
    for (long long t = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); t < tokens; t += (long long)gridDim.x * 4) {
        const T* g = dy + t * dy_rs;
        Piece<T, VEC> held[HELD];
#pragma unroll
        for (int h = 0; h < HELD; h++) {
            const int c = (h * 64 + lane) * VEC;
            if (c < d) held[h].load(g + c);
        }
        for (int j = 0; j < k; j++) {
            const int at = position[t * k + j];
            if ((unsigned)at >= slots) {
                if (lane == 0) dw[t * k + j] = 0;
                continue;
            }
            const A w = weights[t * k + j];
            const T* zr = z + at * z_rs;
            T* o = dz + at * dz_rs;
            A dot = 0;
            auto piece = [&](const Piece<T, VEC>& gp, const Piece<T, VEC>& zp, int c) {
                Piece<T, VEC> op;
#pragma unroll
                for (int v = 0; v < VEC; v++) {
                    const A gv = widen(gp.e[v]);
                    dot += gv * widen(zp.e[v]);
                    op.e[v] = round_to<T>(w * gv);
                }
                op.store(o + c);
            };
            Piece<T, VEC> zp[HELD];
#pragma unroll
            for (int h = 0; h < HELD; h++) {
                const int c = (h * 64 + lane) * VEC;
                if (c < d) zp[h].load(zr + c);
            }
#pragma unroll
            for (int h = 0; h < HELD; h++) {
                const int c = (h * 64 + lane) * VEC;
                if (c < d) piece(held[h], zp[h], c);
            }
            for (int c = (HELD * 64 + lane) * VEC; c < d; c += 64 * VEC) {
                Piece<T, VEC> gp, zq;
                gp.load(g + c);
                zq.load(zr + c);
                piece(gp, zq, c);
            }
#pragma unroll
            for (int m = 32; m >= 1; m /= 2) dot += __shfl_xor(dot, m);
            if (lane == 0) dw[t * k + j] = dot;
        }
    }
}

static bool whole_vectors(int d, int elem, std::initializer_list<const void*> ptrs, std::initializer_list<long long> strides) {
    const int vec = 16 / elem;
    if (d % vec) return false;
    for (const void* p : ptrs) if ((uintptr_t)p & 15) return false;
    for (long long s : strides) if (s % vec) return false;
    return true;
}

static unsigned exchange_blocks(long long threads) {
    const long long blocks = (threads + 255) / 256, most = 1 << 20;
    return (unsigned)(blocks < most ? blocks : most);
}

static bool exchange_args_ok(const char* who, bool pointers, int tokens, int k, int d, std::initializer_list<long long> strides, int dtype) {
    if (!pointers || tokens <= 0 || k <= 0 || d <= 0) { set_error("%s: null operand or non-positive extent (tokens=%d k=%d d=%d)", who, tokens, k, d); return false; }
    if ((long long)tokens * k > ROUTE_MAX_SLOTS) { set_error("%s: more than %d slots (tokens * k)", who, ROUTE_MAX_SLOTS); return false; }
    for (long long s : strides)
        if (s < d) { set_error("%s: rows of %lld elements apart hold %d", who, s, d); return false; }
    if (!dtype_size(dtype)) { set_error("%s: unsupported dtype %d", who, dtype); return false; }
    return true;
}

static bool route_args_ok(const char* who, bool pointers, int tokens, int experts, int k, long long rs, int dtype) {
    if (!pointers || tokens <= 0 || experts <= 0 || k <= 0) { set_error("%s: null operand or non-positive extent (tokens=%d experts=%d k=%d)", who, tokens, experts, k); return false; }
    if (experts > ROUTE_MAX_EXPERTS || k > ROUTE_MAX_K || k > experts) {
        set_error("%s: at most %d experts, and k at most %d and no more than the experts (experts=%d k=%d)", who, ROUTE_MAX_EXPERTS, ROUTE_MAX_K, experts, k);
        return false;
    }
    if ((long long)tokens * k > ROUTE_MAX_SLOTS) { set_error("%s: more than %d slots (tokens * k)", who, ROUTE_MAX_SLOTS); return false; }
    if (rs < experts) { set_error("%s: logits rows of %lld elements apart hold %d", who, rs, experts); return false; }
    if (!dtype_size(dtype)) { set_error("%s: unsupported dtype %d", who, dtype); return false; }
    return true;
}

}  // namespace rp

using namespace rp;

extern "C" {

int rp_hip_route_forward(void* weights, int* experts, int* offsets, int* order, int* position, const void* logits, long long logits_rs,
                         int tokens, int num_experts, int k, int normalize, int dtype) {
    if (!route_args_ok("rp_hip_route_forward", weights && experts && offsets && order && position && logits, tokens, num_experts, k, logits_rs, dtype)) return -1;
    RP_DISPATCH_DTYPE(dtype, return launch_route<T>(weights, experts, offsets, order, position, logits, logits_rs, tokens, num_experts, k, normalize));
    return 0;
}

int rp_hip_route_backward(void* grad_logits, const void* grad_weights, const void* weights, const int* experts, const void* logits, long long logits_rs,
                          int tokens, int num_experts, int k, int normalize, int dtype) {
    if (!route_args_ok("rp_hip_route_backward", grad_logits && grad_weights && weights && experts && (logits || normalize), tokens, num_experts, k, logits ? logits_rs : num_experts, dtype)) return -1;
    RP_DISPATCH_DTYPE(dtype, return launch_route_backward<T>(grad_logits, grad_weights, weights, experts, logits, logits_rs, tokens, num_experts, k, normalize));
    return 0;
}

int rp_hip_group_rows(int* offsets, int* order, int* position, const int* ids, int count, int groups) {
    if (!offsets || !order || !position || !ids || count <= 0 || groups <= 0) { set_error("rp_hip_group_rows: null operand or non-positive extent (count=%d groups=%d)", count, groups); return -1; }
    if (groups > ROUTE_MAX_EXPERTS || count > ROUTE_MAX_SLOTS) { set_error("rp_hip_group_rows: at most %d groups and %d rows (%d, %d)", ROUTE_MAX_EXPERTS, ROUTE_MAX_SLOTS, groups, count); return -1; }
    return launch_sort(offsets, order, position, ids, count, groups);
}

int rp_hip_dispatch_rows(void* out, const void* x, const int* position, int tokens, int k, int d, long long x_rs, long long out_rs, int dtype) {
    if (!exchange_args_ok("rp_hip_dispatch_rows", out && x && position, tokens, k, d, {x_rs, out_rs}, dtype)) return -1;
    RP_DISPATCH_DTYPE(dtype, {
        constexpr int VEC = 16 / (int)sizeof(T);
        const unsigned slots = (unsigned)((long long)tokens * k);
        if (whole_vectors(d, sizeof(T), {out, x}, {x_rs, out_rs})) {
            const long long total = (long long)tokens * (d / VEC);
            hipLaunchKernelGGL((dispatch_kernel<T, VEC>), dim3(exchange_blocks(total)), dim3(256), 0, current_stream(), (T*)out, (const T*)x, position, total, d / VEC, k, slots, x_rs, out_rs);
        } else {
            const long long total = (long long)tokens * d;
            hipLaunchKernelGGL((dispatch_kernel<T, 1>), dim3(exchange_blocks(total)), dim3(256), 0, current_stream(), (T*)out, (const T*)x, position, total, d, k, slots, x_rs, out_rs);
        }
    });
    return check_launch("dispatch_kernel") ? 0 : -1;
}

int rp_hip_zero_rows_behind(void* x, const int* offsets, int groups, int rows, int width, long long x_rs, int dtype) {
    if (!x || !offsets || groups <= 0 || rows <= 0 || width <= 0) { set_error("rp_hip_zero_rows_behind: null operand or non-positive extent (groups=%d rows=%d width=%d)", groups, rows, width); return -1; }
    if (x_rs < width) { set_error("rp_hip_zero_rows_behind: rows of %lld elements apart hold %d", x_rs, width); return -1; }
    const long long es = (long long)dtype_size(dtype);
    if (!es) { set_error("rp_hip_zero_rows_behind: unsupported dtype %d", dtype); return -1; }
    hipLaunchKernelGGL(zero_rows_behind_kernel, dim3(rows < 1024 ? rows : 1024), dim3(256), 0, current_stream(), (unsigned char*)x, offsets, groups, rows, x_rs * es, width * es);
    return check_launch("zero_rows_behind_kernel") ? 0 : -1;
}

int rp_hip_combine_forward(void* y, const void* z, const void* weights, const int* position, int tokens, int k, int d, long long y_rs, long long z_rs, int dtype) {
    if (!exchange_args_ok("rp_hip_combine_forward", y && z && position, tokens, k, d, {y_rs, z_rs}, dtype)) return -1;
    RP_DISPATCH_DTYPE(dtype, {
        constexpr int VEC = 16 / (int)sizeof(T);
        const unsigned slots = (unsigned)((long long)tokens * k);
        if (whole_vectors(d, sizeof(T), {y, z}, {y_rs, z_rs})) {
            const long long total = (long long)tokens * (d / VEC);
            hipLaunchKernelGGL((combine_kernel<T, VEC>), dim3(exchange_blocks(total)), dim3(256), 0, current_stream(), (T*)y, (const T*)z, (const weight_t<T>*)weights, position, total, d / VEC, k,
                               slots, y_rs, z_rs);
        } else {
            const long long total = (long long)tokens * d;
            hipLaunchKernelGGL((combine_kernel<T, 1>), dim3(exchange_blocks(total)), dim3(256), 0, current_stream(), (T*)y, (const T*)z, (const weight_t<T>*)weights, position, total, d, k,
                               slots, y_rs, z_rs);
        }
    });
    return check_launch("combine_kernel") ? 0 : -1;
}

int rp_hip_combine_backward(void* grad_z, void* grad_weights, const void* grad_y, const void* z, const void* weights, const int* position, int tokens, int k, int d,
                            long long grad_y_rs, long long z_rs, long long grad_z_rs, int dtype) {
    if (!exchange_args_ok("rp_hip_combine_backward", grad_z && grad_weights && grad_y && z && weights && position, tokens, k, d, {grad_y_rs, z_rs, grad_z_rs}, dtype)) return -1;
    RP_DISPATCH_DTYPE(dtype, {
        constexpr int VEC = 16 / (int)sizeof(T);
        const unsigned slots = (unsigned)((long long)tokens * k);
        auto launch = [&](auto kern) {
            hipLaunchKernelGGL(kern, dim3(exchange_blocks((long long)tokens * 64)), dim3(256), 0, current_stream(), (T*)grad_z, (weight_t<T>*)grad_weights, (const T*)grad_y, (const T*)z,
                               (const weight_t<T>*)weights, position, tokens, k, d, slots, grad_y_rs, z_rs, grad_z_rs);
        };
        if (!whole_vectors(d, sizeof(T), {grad_z, grad_y, z}, {grad_y_rs, z_rs, grad_z_rs})) launch(combine_backward_kernel<T, 1, 8>);
        else if (d <= 64 * VEC * 2) launch(combine_backward_kernel<T, VEC, 2>);
        else launch(combine_backward_kernel<T, VEC, 8>);
    });
    return check_launch("combine_backward_kernel") ? 0 : -1;
}

}  // extern "C"
