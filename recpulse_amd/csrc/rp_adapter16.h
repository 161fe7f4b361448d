// bf16 / fp16 rows times an adapter's narrow factor: h[i] = scale x[i] . A_a (k x rank) in float32, and with B_a^T for A_a the gradient's
// u[i] = scale dy[i] . B_a^T.
//
// The product is bound by reading x (rows * k * 2 bytes) and, where every request has an adapter of its own, the adapters; its
// arithmetic is rank / 16 MFMAs per 16 rows and 32 of k.  A workgroup of sixteen (or eight) waves owns 16 or 32 rows of one segment and the
// whole rank; the waves share k, 32 at a time in turn, and add their sums in wave order: few rows still have 64 KB of loads in
// flight a CU, and there is one launch and no workspace.
//
// v_mfma_f32_16x16x32: lane (q, j) = (lane / 16, lane % 16) supplies k = 8q .. 8q + 7 of row j, one 16-byte load of x.  A factor that is
// contiguous along k (B^T) is read the same way.  One that is contiguous along the rank goes through LDS of the wave's own as it lies and
// comes back with the transposing read (ds_read_b64_tr_b16): 2-byte loads straight from memory would keep a CU's address unit busy for 8 us
// at 32 requests of k = 4096 and rank 16.
#pragma once
#include "rp_grouped.h"

#include <type_traits>

namespace rp {

// Ranks that have registers for their sums; wider factors go to the scalar kernel, where they would need their columns dealt to workgroups that each read x again (bf16, 2048 rows of 4096: rank
// 128 19 us here, rank 136 158 there)
constexpr int SH_STEP = 32, SH_MAX_RANK = 128;

typedef unsigned int u32x4_odd_t __attribute__((ext_vector_type(4), aligned(2)));       // a 16-byte vector at any element
typedef uint16_t __attribute__((address_space(3))) sh_lds_u16;

template <typename T> struct sh_ops;
template <> struct sh_ops<bf16_t> {
    static __device__ __forceinline__ f32x4_t mma(u32x4_t a, u32x4_t b, f32x4_t c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    }
};
template <> struct sh_ops<f16_t> {
    static __device__ __forceinline__ f32x4_t mma(u32x4_t a, u32x4_t b, f32x4_t c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
    }
};

// eight float32 values as two of T each: the nearest, and the nearest to what is left (nothing, where the first is not finite)
template <typename T>
__device__ __forceinline__ void split_low(const float* v, u32x4_t& hi, u32x4_t& lo) {
    T h[8], l[8];
#pragma unroll
    for (int e = 0; e < 8; e++) {
        h[e] = round_to<T>(v[e]);
        const float left = v[e] - widen(h[e]);
        l[e] = round_to<T>(__builtin_isfinite(left) ? left : 0.f);
    }
    __builtin_memcpy(&hi, h, 16);
    __builtin_memcpy(&lo, l, 16);
}

// float16 reaches from 2^-24 to 65504, and sums of small gradients lie below: before they are split, values that are multiplied together are brought to a largest one of
// 2^14 .. 2^15 by a power of two, and their product back.  Two values then add up to one to 2^-22 of it and 2^-39 of the largest.  (bfloat16 reaches as far as float32.)
__device__ __forceinline__ uint32_t finite_bits(float v) { const uint32_t b = __float_as_uint(v) & 0x7FFFFFFFu; return b < 0x7F800000u ? b : 0u; }
__device__ __forceinline__ void largest_bits(uint32_t& bits, const float* v) {
#pragma unroll
    for (int e = 0; e < 8; e++) { const uint32_t b = finite_bits(v[e]); bits = b > bits ? b : bits; }
}
// The biased exponent of the largest of the four lanes that share j = lane % 16, at least 15 (so that both powers are normal numbers)
__device__ __forceinline__ uint32_t low_exponent(uint32_t bits) {
#pragma unroll
    for (int d = 16; d < 64; d *= 2) { const uint32_t b = __shfl_xor(bits, d); bits = b > bits ? b : bits; }
    return bits >> 23 > 15u ? bits >> 23 : 15u;
}
__device__ __forceinline__ float low_up(uint32_t exponent) { return __uint_as_float((268u - exponent) << 23); }
__device__ __forceinline__ float low_down(uint32_t exponent) { return __uint_as_float((exponent - 14u) << 23); }
template <typename T>
__device__ __forceinline__ void split_scaled(const float* v, float up, u32x4_t& hi, u32x4_t& lo) {
    float w[8];
#pragma unroll
    for (int e = 0; e < 8; e++) w[e] = v[e] * up;
    split_low<T>(w, hi, lo);
}

// Which of a pair of 16-bit values are an infinity or NaN: their sign bits
template <typename T> __device__ __forceinline__ uint32_t not_finite(uint32_t v) {
    constexpr bool f16 = std::is_same<T, f16_t>::value;
    return ((v & (f16 ? 0x7C007C00u : 0x7F807F80u)) + (f16 ? 0x04000400u : 0x00800080u)) & 0x80008000u;       // (an exponent of ones carries)
}
template <typename T> __device__ __forceinline__ u32x4_t finite_only(u32x4_t v) {
#pragma unroll
    for (int d = 0; d < 4; d++) v[d] &= ~((not_finite<T>(v[d]) >> 15) * 0xFFFFu);
    return v;
}

// A vector of eight 16-bit values may straddle the end of its row, of which `left` are there: it is loaded `pulled(left)` values early, where it ends with the row (which
// holds eight at least), and shifted into place with zeros behind.  So every load is within its operand, none is behind a branch, and rows may start at any element.
__device__ __forceinline__ int pulled(int left) { return left > 0 && left < 8 ? 8 - left : 0; }
__device__ __forceinline__ u32x4_t pull_into_place(u32x4_t v, int by) { return __builtin_bit_cast(u32x4_t, __builtin_bit_cast(unsigned __int128, v) >> (16 * by)); }

// LDS of a wave's piece of the factor: 32 rows of k, 16 * NC columns and 8 more, so that the rows that a transposing read takes together start in different banks
template <int NC> constexpr int sh_pitch() { return 16 * NC + 8; }
// Waves: sixteen while their registers (128 a lane) hold two rounds of loads, eight for the wider factors
template <int NC, int PIECE> constexpr int sh_waves() { return NC <= 2 && (PIECE == 8 || NC == 1) ? 16 : 8; }
// Rounds in flight a wave: a narrow factor's are small, and with few rows nothing but loads takes time
template <int NC, int RT, int PIECE> constexpr int sh_slots() { return NC * RT <= 2 && (PIECE == 8 || NC == 1) ? 4 : 2; }
template <int NC, int RT, int SH_WAVES> constexpr int sh_lds_bytes(bool along_k) {
    const int stage = along_k ? 0 : SH_WAVES * SH_STEP * sh_pitch<NC>() * 2, sums = SH_WAVES * (SH_WAVES / 4) * 64 * 16;
    return stage > sums ? stage : sums;
}

// NC: 16-column tiles of the rank; RT: 16-row tiles; ALONG_K: the factor is contiguous along k; PIECE: values a load of the factor takes (8, or 1 where its
// rows are no whole vectors)
template <typename T, int NC, int RT, bool ALONG_K, int PIECE, int SH_WAVES>
__device__ __forceinline__ void adapter_shrink16_block(const GroupedArgs& g, int tile) {
    constexpr int PER_PASS = SH_WAVES / 4;      // waves; 16 x 16 tiles whose sums the threads add at a time, a value each
    extern __shared__ __attribute__((aligned(16))) unsigned char sh_lds[];
    const RowTile rt = find_row_tile_number(g.gr, 16 * RT, tile);
    if (rt.group < 0) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), q = lane >> 4, j = lane & 15;
    const int rank = g.n;
    const __amdgpu_buffer_rsrc_t x_rsrc = buffer_rsrc((const uint16_t*)g.A + rt.begin * g.a_rs, ((rt.end - 1 - rt.begin) * g.a_rs + g.k) * 2);
    uint32_t x_off[RT];
#pragma unroll
    for (int i = 0; i < RT; i++) {                               // (rows past the segment repeat its last: their sums are not stored)
        const int r = rt.begin + 16 * i + j;
        x_off[i] = (uint32_t)(((r < rt.end ? r : rt.end - 1) - rt.begin) * g.a_rs * 2);
    }
    const uint16_t* f = (const uint16_t*)g.B + rt.weight * g.b_ws;
    constexpr int PITCH = sh_pitch<NC>(), PER_ROW = 16 * NC / PIECE, PIECES = ALONG_K ? NC : SH_STEP * PER_ROW / 64;
    const __amdgpu_buffer_rsrc_t f_rsrc = buffer_rsrc(f, ALONG_K ? ((rank - 1) * g.b_cs + g.k) * 2 : (long long)g.k * g.b_rs * 2);
    uint16_t* stage = (uint16_t*)sh_lds + wave * SH_STEP * PITCH;
    if constexpr (!ALONG_K) {
        if (rank < 16 * NC)
            for (int i = lane; i < SH_STEP * PITCH / 2; i += 64) ((uint32_t*)stage)[i] = 0;       // columns past the rank
    }
    using piece_t = std::conditional_t<ALONG_K || PIECE == 8, u32x4_t, uint16_t>;
    constexpr int SLOTS = sh_slots<NC, RT, PIECE>();
    u32x4_t xv[SLOTS][RT];
    piece_t fv[SLOTS][PIECES];
    auto request = [&](auto slotc, int k0) {
        constexpr int S = decltype(slotc)::value;
        const int left = g.k - k0 - 8 * q, at = (k0 + 8 * q - pulled(left)) * 2;
#pragma unroll
        for (int i = 0; i < RT; i++) xv[S][i] = __builtin_amdgcn_raw_buffer_load_b128(x_rsrc, (int)(left > 0 ? x_off[i] + at : BUFFER_OOB), 0, 0);
#pragma unroll
        for (int p = 0; p < PIECES; p++) {
            if constexpr (ALONG_K) {
                const int c = 16 * p + j < rank ? 16 * p + j : rank - 1;
                fv[S][p] = __builtin_amdgcn_raw_buffer_load_b128(f_rsrc, (int)(left > 0 ? (uint32_t)(c * g.b_cs * 2) + at : BUFFER_OOB), 0, 0);
            } else {
                const int id = lane + 64 * p, r = k0 + id / PER_ROW, c = id % PER_ROW * PIECE;
                const int off = (int)(r < g.k && c < rank ? (uint32_t)((r * g.b_rs + c) * 2) : BUFFER_OOB);
                if constexpr (PIECE == 8) fv[S][p] = __builtin_amdgcn_raw_buffer_load_b128(f_rsrc, off, 0, 0);
                else fv[S][p] = __builtin_amdgcn_raw_buffer_load_b16(f_rsrc, off, 0, 0);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    f32x4_t acc[RT][NC];
#pragma unroll
    for (int i = 0; i < RT; i++)
#pragma unroll
        for (int c = 0; c < NC; c++) acc[i][c] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    auto multiply = [&](auto slotc, int k0) {
        constexpr int S = decltype(slotc)::value;
        const int by = pulled(g.k - k0 - 8 * q);
        const bool last = k0 + SH_STEP > g.k && g.k % 8;
        if (last) {
#pragma unroll
            for (int i = 0; i < RT; i++) xv[S][i] = pull_into_place(xv[S][i], by);
        }
        u32x4_t b[NC];
        if constexpr (ALONG_K) {
#pragma unroll
            for (int c = 0; c < NC; c++) b[c] = last ? pull_into_place(fv[S][c], by) : fv[S][c];
        } else {
#pragma unroll
            for (int p = 0; p < PIECES; p++) {
                const int id = lane + 64 * p;
                uint16_t* at = stage + id / PER_ROW * PITCH + id % PER_ROW * PIECE;
                if (id % PER_ROW * PIECE < rank) {
                    if constexpr (PIECE == 8) *(u32x4_t*)at = fv[S][p];
                    else *at = fv[S][p];
                }
            }
            // (the wave's own LDS, and its instructions are executed in order: no barrier)
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int c = 0; c < NC; c++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const uint16_t* at = stage + (8 * q + 4 * h + (j >> 2)) * PITCH + 16 * c + 4 * (j & 3);
                    const s16x4_t v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((s16x4_t __attribute__((address_space(3)))*)(sh_lds_u16*)at);
                    const u32x2_t w = __builtin_bit_cast(u32x2_t, v);
                    b[c][2 * h] = w[0];
                    b[c][2 * h + 1] = w[1];
                }
            __builtin_amdgcn_wave_barrier();
        }
#pragma unroll
        for (int i = 0; i < RT; i++)
#pragma unroll
            for (int c = 0; c < NC; c++) acc[i][c] = sh_ops<T>::mma(xv[S][i], b[c], acc[i][c]);
    };
    constexpr int TURN = SH_WAVES * SH_STEP;
    const int first = wave * SH_STEP;
    static_for<0, SLOTS>([&](auto sc) { request(sc, first + decltype(sc)::value * TURN); });       // (rounds past k load nothing and are zeros)
    for (int k0 = first; k0 < g.k; k0 += SLOTS * TURN)
        static_for<0, SLOTS>([&](auto sc) {
            multiply(sc, k0 + decltype(sc)::value * TURN);
            request(sc, k0 + (SLOTS + decltype(sc)::value) * TURN);
        });

    // the waves' sums
    float* sums = (float*)sh_lds;
    float* h = (float*)g.C;
    const float scale = g.scales ? g.scales[rt.weight] : 1.f;
    constexpr int TILES = RT * NC;
    static_for<0, (TILES + PER_PASS - 1) / PER_PASS>([&](auto passc) {
        constexpr int P0 = decltype(passc)::value * PER_PASS, P1 = P0 + PER_PASS < TILES ? P0 + PER_PASS : TILES;
        __syncthreads();
        static_for<P0, P1>([&](auto pc) {
            constexpr int p = decltype(pc)::value;
            *(f32x4_t*)(sums + ((wave * PER_PASS + p - P0) * 64 + lane) * 4) = acc[p / NC][p % NC];
        });
        __syncthreads();
        const int p = P0 + (int)(threadIdx.x >> 8), l = (threadIdx.x & 255) >> 2, v = threadIdx.x & 3;
        if (p < P1) {
            float s = 0;
#pragma unroll
            for (int w = 0; w < SH_WAVES; w++) s += sums[((w * PER_PASS + p - P0) * 64 + l) * 4 + v];
            const int row = rt.begin + 16 * (p / NC) + 4 * (l >> 4) + v, col = 16 * (p % NC) + (l & 15);
            if (row < rt.end && col < rank) h[(long long)row * g.c_rs + col] = scale * s;
        }
    });
}

}  // namespace rp
