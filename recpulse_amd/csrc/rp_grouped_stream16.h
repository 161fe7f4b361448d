// bf16 / fp16 rows in groups of a few rows each against row-major weights: decoding with experts, or the shared projection beside adapters.
//
// Bound by reading the weights: every weight that has a row is read once, in loads of 16 bytes a lane.  v_mfma_f32_16x16x32: lane
// (q, j) = (lane / 16, lane % 16) supplies k = 8q .. 8q + 7 of row j of x, one load, and of column j of the weight.
//   Strips of 128 columns go from memory to registers to the MFMAs, as in the few-row kernel for one matrix (rp_gemm_mfma16_stream128.hip):
//   a lane loads columns 8j .. 8j + 7 of eight rows of k and transposes the 8 x 8 block with byte permutes; residue c of the columns
//   becomes the operand of one MFMA, whose column j is column 8j + c of the strip.
//   Strips of 64 columns pass through LDS of the wave's own and come back with the transposing read (ds_read_b64_tr_b16), sixteen
//   adjacent columns an MFMA.
// A workgroup owns 16 * RB rows of one group and a strip; its eight waves share k, 32 rows of it at a time in turn, two to four rounds in flight
// each, and add their tiles through LDS in wave order.
//
// What a CU can fetch decides how the work is cut: some 40 GB/s from memory, however many bytes its waves have in flight (one weight of
// 4096 x 4096 by 32 strips of 128 columns 25.7 us, by 64 strips of 64 columns 19.2, by 128 strips of 32 columns, whose row pieces are
// half a cache line, 18.1), so all CUs have to fetch.  Where the strips of 128 columns are too few for that, k is cut up among workgroups
// too and a second launch adds their float32 sums in order (stream16_combine_kernel); where there is no memory for the sums that
// another stream's call cannot touch (CallScratch), strips are 64 columns instead.
#pragma once
#include "rp_grouped.h"

#include <type_traits>

namespace rp {

constexpr int GS_ROUND = 32, GS_WAVES = 8, GS_THREADS = GS_WAVES * 64;

template <typename T> struct gs_ops;
template <> struct gs_ops<bf16_t> {
    static __device__ __forceinline__ f32x4_t mma(u32x4_t a, u32x4_t b, f32x4_t c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    }
};
template <> struct gs_ops<f16_t> {
    static __device__ __forceinline__ f32x4_t mma(u32x4_t a, u32x4_t b, f32x4_t c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
    }
};
typedef uint16_t __attribute__((address_space(3))) gs_lds_u16;

// CPL: columns of a strip / 16 (8 or 4); RB: 16-row blocks.  Rounds a wave has in flight; LDS, the waves' sums of 16 rows over the staging
template <int CPL, int RB> constexpr int gs_slots() { return CPL == 8 || RB == 4 ? 2 : 4; }
template <int CPL> constexpr int gs_stage_pitch() { return 16 * CPL + 8; }      // 16-bit values; a transposing read's four rows start in different banks
template <int CPL> constexpr int gs_lds_bytes() {
    const int sums = GS_WAVES * 16 * (16 * CPL + 4) * 4, stage = CPL == 8 ? 0 : GS_WAVES * GS_ROUND * gs_stage_pitch<CPL>() * 2;
    return sums > stage ? sums : stage;
}

// How a launch's workgroups stand for (row tile, strip, share of k).  Workgroup b runs on XCD b % 8: all shares of k of a strip, and the two strips of a
// 256-byte piece of the rows, go to one XCD.
struct StreamGrid {
    int pieces;                    // 256-byte pieces of a row
    int nsplit;                    // shares of k
    float* partials;               // [nsplit][rows][n], or null: the outputs themselves
};

// TERM: `term` is added to the sums before they are rounded
template <typename T, int CPL, int RB, bool TERM = false>
__device__ __forceinline__ void stream16_block(const GroupedArgs& g, const StreamGrid& sg, long long block, const AdapterTerm* term = nullptr) {
    constexpr int SLOTS = gs_slots<CPL, RB>(), COLS = 16 * CPL, PITCH = COLS + 4, ROWS = 16 * RB, S = 8 / CPL;
    constexpr bool STAGED = CPL < 8;
    constexpr int LOADS = CPL, PPR = COLS / 8, STAGE_PITCH = gs_stage_pitch<CPL>();      // loads of a round; 16-byte pieces of a strip's row
    extern __shared__ __attribute__((aligned(16))) float gs_sums[];       // [GS_WAVES][16][PITCH]
    const unsigned slot = (unsigned)(block >> 3), within = slot % (S * sg.nsplit), piece = slot / (S * sg.nsplit) * 8 + (unsigned)(block & 7);
    const int split = (int)(within / S), n0 = ((int)(piece % sg.pieces) * S + (int)(within % S)) * COLS;
    if (n0 >= g.n) return;
    const RowTile rt = find_row_tile_number(g.gr, ROWS, (int)(piece / sg.pieces));
    if (rt.group < 0) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), q = lane >> 4, j = lane & 15;
    const int m = rt.end - rt.begin;
    const uint16_t* B = (const uint16_t*)g.B + rt.weight * g.b_ws + n0;
    const uint16_t* A = (const uint16_t*)g.A + rt.begin * g.a_rs;
    const char* b_end = (const char*)(B + ((long long)(g.k - 1) * g.b_rs + g.n - n0));
    const char* a_end = (const char*)(A + ((long long)(m - 1) * g.a_rs + g.k));
    uint32_t b_off[LOADS], a_off[RB];                                     // from a round's first row of the weight, and first k of the rows
#pragma unroll
    for (int e = 0; e < LOADS; e++) {                                     // (n is a multiple of 8)
        const int p = STAGED ? lane + 64 * e : 0, r = STAGED ? p / PPR : 8 * q + e, c = STAGED ? p % PPR * 8 : 8 * j;
        b_off[e] = n0 + c < g.n ? (uint32_t)((r * g.b_rs + c) * 2) : BUFFER_OOB;
    }
#pragma unroll
    for (int i = 0; i < RB; i++) a_off[i] = 16 * i + j < m ? (uint32_t)(((16 * i + j) * g.a_rs + 8 * q) * 2) : BUFFER_OOB;

    u32x4_t raw[SLOTS][LOADS], av[SLOTS][RB];
    // (Issued unconditionally, against descriptors that read zeros past k: behind a branch the compiler's waits count loads that may not have been issued.)
    auto request = [&](auto slotc, int k0) {
        constexpr int SL = decltype(slotc)::value;
        const char* bb = (const char*)(B + (long long)k0 * g.b_rs);
        const char* ab = (const char*)(A + k0);
        const __amdgpu_buffer_rsrc_t b_rsrc = buffer_rsrc(bb, k0 < g.k ? (long long)(b_end - bb) : 0), a_rsrc = buffer_rsrc(ab, k0 < g.k ? (long long)(a_end - ab) : 0);
        const bool k_in = k0 + 8 * q < g.k;                               // (k is a multiple of 8)
#pragma unroll
        for (int e = 0; e < LOADS; e++) raw[SL][e] = __builtin_amdgcn_raw_buffer_load_b128(b_rsrc, (int)b_off[e], 0, 2);       // (streamed: read once)
#pragma unroll
        for (int i = 0; i < RB; i++) av[SL][i] = __builtin_amdgcn_raw_buffer_load_b128(a_rsrc, (int)(k_in ? a_off[i] : BUFFER_OOB), 0, 0);
        __builtin_amdgcn_sched_barrier(0);
    };
    f32x4_t acc[RB][CPL];
#pragma unroll
    for (int i = 0; i < RB; i++)
#pragma unroll
        for (int c = 0; c < CPL; c++) acc[i][c] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    uint16_t* stage = (uint16_t*)gs_sums + wave * GS_ROUND * STAGE_PITCH;
    auto multiply = [&](auto slotc) {
        constexpr int SL = decltype(slotc)::value;
        if constexpr (STAGED) {
#pragma unroll
            for (int e = 0; e < LOADS; e++) *(u32x4_t*)(stage + (lane + 64 * e) / PPR * STAGE_PITCH + lane % PPR * 8) = raw[SL][e];      // (64 is a multiple of PPR)
            __builtin_amdgcn_wave_barrier();                              // (the wave's own LDS, whose instructions are executed in order)
        }
#pragma unroll
        for (int c = 0; c < CPL; c++) {
            u32x4_t b;
            if constexpr (STAGED) {
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const uint16_t* at = stage + (8 * q + 4 * h + (j >> 2)) * STAGE_PITCH + 16 * c + 4 * (j & 3);
                    const u32x2_t w = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((s16x4_t __attribute__((address_space(3)))*)(gs_lds_u16*)at));
                    b[2 * h] = w[0];
                    b[2 * h + 1] = w[1];
                }
            } else {
#pragma unroll
                for (int d = 0; d < 4; d++) b[d] = __builtin_amdgcn_perm(raw[SL][2 * d + 1][c / 2], raw[SL][2 * d][c / 2], (c & 1) ? 0x07060302u : 0x05040100u);
            }
#pragma unroll
            for (int i = 0; i < RB; i++) acc[i][c] = gs_ops<T>::mma(av[SL][i], b, acc[i][c]);
        }
        if constexpr (STAGED) __builtin_amdgcn_wave_barrier();
    };
    const int turn = GS_ROUND * GS_WAVES * sg.nsplit;                     // the shares of k are dealt round by round: the launch reads one window of the weights at a time
    const int first = (split * GS_WAVES + wave) * GS_ROUND;
    static_for<0, SLOTS>([&](auto sc) { request(sc, first + decltype(sc)::value * turn); });
    for (int k0 = first; k0 < g.k; k0 += SLOTS * turn)
        static_for<0, SLOTS>([&](auto sc) {
            multiply(sc);
            request(sc, k0 + (SLOTS + decltype(sc)::value) * turn);
        });

    // the waves' sums, 16 rows at a time, vectors of 8 columns a thread
    constexpr int VPR = COLS / 8, ITEMS = 16 * VPR;
    static_assert(ITEMS <= GS_THREADS, "a vector a thread");
    const int row16 = (int)threadIdx.x / VPR, cv = (int)threadIdx.x % VPR * 8;
    const bool in = (int)threadIdx.x < ITEMS && n0 + cv < g.n;
    static_for<0, RB>([&](auto ic) {
        constexpr int i = decltype(ic)::value;
        if (i || STAGED) __syncthreads();                                 // the rows before are added up; every wave is done with its staging
#pragma unroll
        for (int v = 0; v < 4; v++)
#pragma unroll
            for (int c = 0; c < CPL; c++) gs_sums[(wave * 16 + 4 * q + v) * PITCH + (STAGED ? 16 * c + j : 8 * j + c)] = acc[i][c][v];
        __syncthreads();
        const int row = rt.begin + 16 * i + row16;
        if (!in || row >= rt.end) return;
        float s[8];
#pragma unroll
        for (int v = 0; v < 8; v++) s[v] = 0.f;
#pragma unroll
        for (int w = 0; w < GS_WAVES; w++) {
            const float* at = gs_sums + (w * 16 + row16) * PITCH + cv;
            const f32x4_t lo = *(const f32x4_t*)at, hi = *(const f32x4_t*)(at + 4);
#pragma unroll
            for (int v = 0; v < 4; v++) { s[v] += lo[v]; s[4 + v] += hi[v]; }
        }
        if constexpr (TERM) {
            int a = -1;
            for (int t = 0; t < term->gr.groups; t++) a = row >= term->gr.begin(t) && row < term->gr.end(t) ? term->gr.weight(t) : a;
            const float* h = term->h + (long long)row * term->rank;
            const uint16_t* b = (const uint16_t*)term->b + a * term->b_ws + n0 + cv;
#pragma unroll 4
            for (int r = 0; r < (a < 0 ? 0 : term->rank); r++) {
                const float hr = h[r];
                T e[8];
                __builtin_memcpy(e, b + r * term->b_rs, 16);
#pragma unroll
                for (int v = 0; v < 8; v++) s[v] += hr * widen(e[v]);
            }
        }
        if (!TERM && sg.partials) {
            float* at = sg.partials + ((long long)split * g.gr.rows + row) * g.n + n0 + cv;
            *(f32x4_t*)at = f32x4_t{s[0], s[1], s[2], s[3]};
            *(f32x4_t*)(at + 4) = f32x4_t{s[4], s[5], s[6], s[7]};
            return;
        }
        uint16_t* out = (uint16_t*)g.C + row * g.c_rs + n0 + cv;
        T y[8], e[8];
        if (g.bias) __builtin_memcpy(e, (const uint16_t*)g.bias + (long long)rt.weight * g.n + n0 + cv, 16);
#pragma unroll
        for (int v = 0; v < 8; v++) y[v] = round_to<T>(g.bias ? s[v] + widen(e[v]) : s[v]);
        if (g.accumulate) {
            __builtin_memcpy(e, out, 16);
#pragma unroll
            for (int v = 0; v < 8; v++) y[v] = round_to<T>(widen(e[v]) + widen(y[v]));
        }
        __builtin_memcpy(out, y, 16);
    });
}

// Grid of the blocks above
static inline long long stream16_blocks(const GroupedArgs& g, int rows_of_tile, int cpl, int nsplit) {
    return (row_tile_numbers(g.gr.rows, g.gr.groups, rows_of_tile) * ((g.n + 127) / 128) + 7) / 8 * 8 * (8 / cpl) * nsplit;
}

// 16-row blocks of a row tile: enough for most groups of a draw around the mean
static inline int stream16_row_blocks(const RowGroups& gr) {
    const int mean = (gr.rows + gr.groups - 1) / gr.groups;
    if (gr.groups == 1) return mean <= 16 ? 1 : mean <= 32 ? 2 : 4;
    return mean <= 10 ? 1 : mean <= 20 ? 2 : 4;
}

// Shares of k that give each CU a workgroup: each at least two rounds a wave long, and their sums within `bytes`
static inline int stream16_splits(const GroupedArgs& g, size_t bytes) {
    const long long used = g.gr.groups < g.gr.rows ? g.gr.groups : g.gr.rows, tiles = used * ((g.n + 127) / 128);
    const int cus = device_cu_count() > 0 ? device_cu_count() : 256;
    long long n = tiles * 4 >= cus * 3ll ? 1 : (cus + tiles - 1) / tiles;
    const long long deep = g.k / (2 * GS_WAVES * GS_ROUND), room = (long long)(bytes / ((size_t)g.gr.rows * g.n * sizeof(float)));
    n = n < deep ? n : deep;
    n = n < room ? n : room;
    return n > 1 ? (int)n : 1;
}

}  // namespace rp
