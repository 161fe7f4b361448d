// bf16 / fp16 gradients of an adapter's factors: D_a = sum over the rows i of adapter a of low[i]^T . s[i], low [rows, rank] in float32, s [rows, width].
// With low = h and s = dy this is dB_a [rank, n]; with low = u and s = x it is dA_a^T, stored transposed.
//
// Bound by reading s, once per 32 of the rank: a workgroup owns one adapter, a strip of 128 columns of s and up to 32 of the rank, and its four
// waves share the rows of the adapter's segments, 32 at a time in turn.  s goes from memory to registers to v_mfma_f32_16x16x32 as a
// weight does in the kernel for few rows (rp_grouped_stream16.h): a lane transposes 8 rows x 8 columns with byte permutes.  low is
// rounded to two values of the tensors' type that add up to it to 2^-17 (float16: 2^-22, scaled by the largest value of the wave's rows, which it looks for first), a product each: h and u are
// sums in float32, and one rounding of theirs would be as large as the result's own.
// fp16, 2048 rows of 3 adapters, 1024 x 2048, rank 8: both 17 us, of which looking for the largest values takes 3, and beside dx's tiles 26 together.  (Eight waves a workgroup: 8192 rows of one adapter, 4096 x 4096, 48 us instead of
// 55 before its rows were shared out, 34 since, but 32 adapters and rank 64 144 instead of 93: a CU holds one such workgroup.)
#pragma once
#include "rp_adapter16.h"
#include "rp_grouped_stream16.h"

namespace rp {

constexpr int AG_WAVES = 4, AG_THREADS = AG_WAVES * 64, AG_COLS = 128, AG_PITCH = AG_COLS + 4;

struct AdapterGrad {
    void* out;                     // null: not asked for
    float* partials;               // null, or room for the shares' sums, each laid out as `out` (dense)
    const void* s;
    const float* low;
    int width, accumulate, strips, blocks;
    long long s_rs, out_ws, out_rs;
};

// NC: 16-row tiles of the rank; IN_TURN: a workgroup does one share of the rows after the other
template <typename T, int NC, bool TRANSPOSED, bool IN_TURN>
__device__ __forceinline__ void adapter_grad16_block(const AdapterGrad& ag, const RowGroups& gr, int rank, int rank_blocks, int shares, int block) {
    extern __shared__ __attribute__((aligned(16))) float gs_sums[];       // [AG_WAVES][16][AG_PITCH], and [16 NC][AG_COLS] of the shares before (IN_TURN)
    T* out = (T*)ag.out;
    const uint16_t* s = (const uint16_t*)ag.s;
    const float* low = ag.low;
    const int width = ag.width, accumulate = ag.accumulate;
    const long long s_rs = ag.s_rs, out_ws = ag.out_ws, out_rs = ag.out_rs;
    const int first_share = IN_TURN ? 0 : block % shares, id = IN_TURN ? block : block / shares, strip = id % ag.strips, rb = id / ag.strips % rank_blocks, w = id / ag.strips / rank_blocks;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), q = lane >> 4, j = lane & 15;
    const int n0 = strip * AG_COLS, r0 = rb * 16 * NC;
    const int left = width - n0 - 8 * j, by = pulled(left);
    const bool cut = n0 + AG_COLS > width && width % 8;
    uint32_t s_off[8];
#pragma unroll
    for (int e = 0; e < 8; e++) s_off[e] = left > 0 ? (uint32_t)(((8 * q + e) * s_rs + n0 + 8 * j - by) * 2) : BUFFER_OOB;
    constexpr int SLOTS = 2;
    u32x4_t raw[SLOTS][8];
    float lv[SLOTS][NC][8];
    int end = 0;                                              // of the segment in hand
    auto request_low = [&](float (&to)[NC][8], int row0) {
        const float* l = low + (long long)row0 * rank;
        const __amdgpu_buffer_rsrc_t l_rsrc = buffer_rsrc(l, row0 < end ? (long long)(end - row0) * rank * 4 : 0);
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int r = r0 + 16 * c + j;
                to[c][e] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(l_rsrc, r < rank ? ((8 * q + e) * rank + r) * 4 : (int)BUFFER_OOB, 0, 0));
            }
    };
    auto request = [&](auto slotc, int row0) {
        constexpr int SL = decltype(slotc)::value;
        const char* at = (const char*)(s + (long long)row0 * s_rs);       // (rows past the segment are another's: the descriptor ends with it)
        const __amdgpu_buffer_rsrc_t rsrc = buffer_rsrc(at, row0 < end ? ((long long)(end - 1 - row0) * s_rs + width) * 2 : 0);
#pragma unroll
        for (int e = 0; e < 8; e++) raw[SL][e] = __builtin_amdgcn_raw_buffer_load_b128(rsrc, (int)s_off[e], 0, 0);
        request_low(lv[SL], row0);
        __builtin_amdgcn_sched_barrier(0);
    };
    f32x4_t acc[NC][8];
    constexpr bool SCALED = std::is_same<T, f16_t>::value;
    uint32_t top[NC];                                         // of column 16 c + j of the rank: the largest value's bits, then its exponent
    auto multiply = [&](auto slotc) {
        constexpr int SL = decltype(slotc)::value;
        u32x4_t hi[NC], lo[NC];
#pragma unroll
        for (int c = 0; c < NC; c++) {
            if constexpr (SCALED) split_scaled<T>(lv[SL][c], low_up(top[c]), hi[c], lo[c]);
            else split_low<T>(lv[SL][c], hi[c], lo[c]);
        }
        if (cut) {
#pragma unroll
            for (int e = 0; e < 8; e++) raw[SL][e] = pull_into_place(raw[SL][e], by);
        }
#pragma unroll
        for (int f = 0; f < 8; f++) {
            u32x4_t b;
#pragma unroll
            for (int d = 0; d < 4; d++) b[d] = __builtin_amdgcn_perm(raw[SL][2 * d + 1][f / 2], raw[SL][2 * d][f / 2], (f & 1) ? 0x07060302u : 0x05040100u);
#pragma unroll
            for (int c = 0; c < NC; c++) {
                acc[c][f] = gs_ops<T>::mma(hi[c], b, acc[c][f]);
                acc[c][f] = gs_ops<T>::mma(lo[c], b, acc[c][f]);
            }
        }
    };
    // f(first row, rows from one round of the wave's to the next) for every segment that it has rounds of
    int share = first_share, rounds = 0;                      // of the segments before, so that short segments go to the waves in turn
    auto for_rounds = [&](auto f) {
        rounds = 0;
        for_groups_of(gr, w, [&](int begin, int stop) {
            end = stop;
            const int lag = (share * AG_WAVES + wave - rounds) % (AG_WAVES * shares);
            const int first = begin + (lag < 0 ? lag + AG_WAVES * shares : lag) * GS_ROUND;
            rounds += (end - begin + GS_ROUND - 1) / GS_ROUND;
            if (first < end) f(first, AG_WAVES * shares * GS_ROUND);
        });
    };
    while (true) {
#pragma unroll
        for (int c = 0; c < NC; c++) {
            top[c] = 0;
#pragma unroll
            for (int f = 0; f < 8; f++) acc[c][f] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        }
        if constexpr (SCALED)
            for_rounds([&](int first, int turn) {
                constexpr int AHEAD = 4;                      // rounds (the registers that the main loop's loads take are free here)
                for (int row0 = first; row0 < end; row0 += AHEAD * turn) {
                    float v[AHEAD][NC][8];
#pragma unroll
                    for (int i = 0; i < AHEAD; i++) request_low(v[i], row0 + i * turn);
#pragma unroll
                    for (int i = 0; i < AHEAD; i++)
#pragma unroll
                        for (int c = 0; c < NC; c++) largest_bits(top[c], v[i][c]);
                }
            });
        if constexpr (SCALED) {
#pragma unroll
            for (int c = 0; c < NC; c++) top[c] = low_exponent(top[c]);
        }
        for_rounds([&](int first, int turn) {
            static_for<0, SLOTS>([&](auto sc) { request(sc, first + decltype(sc)::value * turn); });
            for (int row0 = first; row0 < end; row0 += SLOTS * turn)
                static_for<0, SLOTS>([&](auto sc) {
                    multiply(sc);
                    request(sc, row0 + (SLOTS + decltype(sc)::value) * turn);
                });
        });
        if (rounds == 0) {                                        // an adapter without rows: zeros, or what is there
            for (int i = threadIdx.x; i < 16 * NC * AG_COLS && !accumulate && first_share == 0; i += AG_THREADS) {
                const int r = r0 + (TRANSPOSED ? i % (16 * NC) : i / AG_COLS), col = n0 + (TRANSPOSED ? i / (16 * NC) : i % AG_COLS);
                if (r < rank && col < width) out[w * out_ws + (TRANSPOSED ? col * out_rs + r : r * out_rs + col)] = round_to<T>(0.f);
            }
            return;
        }
        static_for<0, NC>([&](auto cc) {
            constexpr int c = decltype(cc)::value;
            if (c || (IN_TURN && share)) __syncthreads();
#pragma unroll
            for (int v = 0; v < 4; v++) {
                const float down = SCALED ? __shfl(low_down(top[c]), 4 * q + v) : 1.f;
#pragma unroll
                for (int f = 0; f < 8; f++) gs_sums[(wave * 16 + 4 * q + v) * AG_PITCH + 8 * j + f] = SCALED ? acc[c][f][v] * down : acc[c][f][v];
            }
            __syncthreads();
            // eight outputs a thread, neighbours along the output's rows
#pragma unroll
            for (int o = 0; o < 16 * AG_COLS / AG_THREADS; o++) {
                const int id = threadIdx.x + o * AG_THREADS, r = TRANSPOSED ? id & 15 : id / AG_COLS, col = TRANSPOSED ? id >> 4 : id % AG_COLS;
                if (r0 + 16 * c + r >= rank || n0 + col >= width) continue;
                float t = gs_sums[r * AG_PITCH + col];
#pragma unroll
                for (int p = 1; p < AG_WAVES; p++) t += gs_sums[(p * 16 + r) * AG_PITCH + col];
                const long long to = w * out_ws + (TRANSPOSED ? (n0 + col) * out_rs + r0 + 16 * c + r : (r0 + 16 * c + r) * out_rs + n0 + col);
                if (!IN_TURN && ag.partials) {
                    ag.partials[share * (out_ws * gr.weights) + to] = t;
                    continue;
                }
                if constexpr (IN_TURN) {                               // (in the order of the launch that adds them up; a thread's own values)
                    float* before = gs_sums + AG_WAVES * 16 * AG_PITCH + c * 16 * AG_COLS + id;
                    if (share) t = *before + t;
                    if (share + 1 < shares) { *before = t; continue; }
                }
                T* at = out + to;
                T y = round_to<T>(t);
                if (accumulate) y = round_to<T>(widen(*at) + widen(y));
                *at = y;
            }
        });
        if (!IN_TURN || ++share == shares) break;
    }
}

constexpr int AG_LDS = AG_WAVES * 16 * AG_PITCH * 4;

// dA's workgroups, then dB's: each alone leaves most of the chip waiting for loads.  Where few adapters have many rows each, several workgroups share the rows
// and a second launch adds their sums in order (adapter_grads16_join_kernel), or one workgroup does one share after the other where there is no memory for the sums.
struct AdapterGrads { AdapterGrad a, b; int rank, rank_blocks, shares; };
int launch_adapter_grads16_in_turn(const AdapterGrads& ag, const RowGroups& gr, int dtype);      // (rp_adapter16_grads.hip)
template <typename T, int NC, bool IN_TURN = false>
__device__ __forceinline__ void adapter_grads16_block(const AdapterGrads& ag, const RowGroups& gr, int id) {
    if (id < ag.a.blocks) adapter_grad16_block<T, NC, true, IN_TURN>(ag.a, gr, ag.rank, ag.rank_blocks, ag.shares, id);
    else if (id < ag.a.blocks + ag.b.blocks) adapter_grad16_block<T, NC, false, IN_TURN>(ag.b, gr, ag.rank, ag.rank_blocks, ag.shares, id - ag.a.blocks);
}

static inline int grads_rank_tiles(int rank) { return rank <= 16 ? 1 : 2; }
// Those gradients whose C is not null.  How many share an adapter's rows goes by the sizes alone, not by what is asked for.
static inline AdapterGrads plan_grads(const GroupedArgs& da, const GroupedArgs& db) {
    AdapterGrads ag;
    ag.a = AdapterGrad{da.C, nullptr, da.A, (const float*)da.B, da.k, da.accumulate, 0, 0, da.a_rs, da.c_ws, da.c_rs};
    ag.b = AdapterGrad{db.C, nullptr, db.B, (const float*)db.A, db.n, db.accumulate, 0, 0, db.b_rs, db.c_ws, db.c_rs};
    ag.rank = da.n;
    const int per = 16 * grads_rank_tiles(ag.rank);
    ag.rank_blocks = (ag.rank + per - 1) / per;
    ag.a.strips = (ag.a.width + AG_COLS - 1) / AG_COLS;
    ag.b.strips = (ag.b.width + AG_COLS - 1) / AG_COLS;
    // Shares of eight turns of 128 rows or more, as many as keep two workgroups on a CU (bf16, 7949 rows of one adapter, 384 x 1512, rank 32, forward and backward: 144 us, 118 with seven shares)
    const long long used = da.gr.groups < da.gr.weights ? da.gr.groups : da.gr.weights, blocks = used * (ag.a.strips + ag.b.strips) * ag.rank_blocks;
    const long long cus = device_cu_count() > 0 ? device_cu_count() : 256, turns = da.gr.rows / used / (AG_WAVES * GS_ROUND);
    const long long room = (long long)CallScratch::MOST / (((long long)ag.a.width + ag.b.width) * ag.rank * da.gr.weights * (long long)sizeof(float));
    long long shares = turns / 8 < 2 * cus / blocks ? turns / 8 : 2 * cus / blocks;
    shares = shares < room ? shares : room;
    ag.shares = shares > 1 ? (int)shares : 1;
    for (AdapterGrad* g : {&ag.a, &ag.b}) g->blocks = g->out ? g->strips * ag.rank_blocks * da.gr.weights : 0;
    return ag;
}

// out = the shares' sums in order, rounded once; adapters without rows have been seen to
template <typename T>
__global__ void __launch_bounds__(256) adapter_grads16_join_kernel(AdapterGrads ag, RowGroups gr, int a_blocks, int a_per, int b_per) {
    const bool first = (int)blockIdx.x < a_blocks;
    const AdapterGrad& g = first ? ag.a : ag.b;
    const int id = (int)blockIdx.x - (first ? 0 : a_blocks), per = first ? a_per : b_per, w = id / per, size = g.width * ag.rank, i = (id - w * per) * 256 + threadIdx.x;
    bool any = false;
    for_groups_of(gr, w, [&](int, int) { any = true; });
    if (!any || i >= size) return;
    const long long all = (long long)size * gr.weights, at = (long long)w * size + i;
    float t = g.partials[at];
#pragma unroll 4
    for (int s = 1; s < ag.shares; s++) t += g.partials[s * all + at];
    T* out = (T*)g.out + at;
    T y = round_to<T>(t);
    if (g.accumulate) y = round_to<T>(widen(*out) + widen(y));
    *out = y;
}

// Where shares of an adapter's rows are added up, `launch` leaves them in the call's memory for a launch of their own, or, without memory, `in_turn` has workgroups do one share after
// the other: the same bits (bf16, one adapter, backward, us: 7949 rows, 384 x 1512, rank 32 43 and 37; 8192 rows, 4096 x 4096, rank 16 261 and 320).
template <typename T, typename F, typename G>
static int with_joined_grads(AdapterGrads& ag, const RowGroups& gr, F launch, G in_turn) {
    if (ag.shares == 1) return launch();
    const size_t a_sums = ag.a.out ? (size_t)ag.shares * ag.a.width * ag.rank * gr.weights : 0, b_sums = ag.b.out ? (size_t)ag.shares * ag.b.width * ag.rank * gr.weights : 0;
    const CallScratch sums((a_sums + b_sums) * sizeof(float));
    if (!sums.ptr) return in_turn();
    ag.a.blocks *= ag.shares;
    ag.b.blocks *= ag.shares;
    ag.a.partials = (float*)sums.ptr;
    ag.b.partials = (float*)sums.ptr + a_sums;
    if (launch() != 0) return -1;
    const int a_per = (ag.a.width * ag.rank + 255) / 256, b_per = (ag.b.width * ag.rank + 255) / 256, a_blocks = ag.a.out ? a_per * gr.weights : 0, b_blocks = ag.b.out ? b_per * gr.weights : 0;
    hipLaunchKernelGGL(adapter_grads16_join_kernel<T>, dim3((unsigned)(a_blocks + b_blocks)), dim3(256), 0, current_stream(), ag, gr, a_blocks, a_per, b_per);
    return check_launch("adapter_grads16_join_kernel") ? 0 : -1;
}

}  // namespace rp
