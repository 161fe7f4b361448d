// bf16 / fp16 cross entropy of a large vocabulary on the tiles of the 16-bit MFMA kernel.
//
// Forward, a tile of logits z = x . W + b never leaves the registers: each row's largest value and sum of exponentials among the columns of a wave's patch are all that is written
// (8 bytes for 64 or 128 logits), and the target's logit by the lane that holds it.  Backward, the tile is made again and leaves as d = (exp(z - lse) - [v = t]) f, rounded to 16
// bits, a piece of the vocabulary at a time, which two more products take to dx and dW; db is summed from the same registers.
//
// d is stored over the largest |f| (times 2^14 in float16), and dx, dW and db are scaled back in their epilogues, before their one rounding.  As it is, the share of a rare class in a mean over thousands of
// rows would be zero in float16; and of rows with one f all targets' d, which is -f but for a small p, would be rounded alike: their common error, up to half a step, would be that of dx and dW (bf16 0.0030
// against 0.0024 where -1 is exact).  dx is a sum over all pieces: between two of them it stays in float32, a tile's sums in the order of its registers.
#pragma once
#include "rp_gemm_mfma16_kernel.h"
#include "rp_vocab.h"

namespace rp {

struct VocabPart { float top, sum; };

struct VocabTileArgs {
    GemmArgs g;                    // logits: C unused; dx, dw: as a product's
    int tiles_m, tiles_n, total;
    const int* targets;
    int v0, classes;               // first class of the piece; classes of the vocabulary
    // forward
    VocabPart* parts;              // [groups of columns][rows]
    float* hits;                   // [rows] logits of the targets
    // gradient of the logits
    uint16_t* d;                   // [rows][pitch]
    long long pitch;
    const float *lse, *f;          // [rows]; f null: every row with a target has the same (its rows are 2^most, and row_weight says what it is)
    float* db_parts;               // [groups of rows][pitch], or null
    void* db;                      // where one wave has all rows: db of the piece instead, or null
    int accumulate_db;
    // ... and of dx, dw
    const float* scale;            // what d has been multiplied by, inverted; null where f is
    const float *upstream, *count; // one element each, or null: 1
    int most;
    float* sums;                   // dx between pieces and sums of shares of k, tile by tile in the order of a tile's registers
    int first, last;
    // k in shares of k_share that workgroups of their own add up (their sums `share_stride` floats apart), where there are few tiles; 1: none
    int shares, k_share;
    long long share_stride;
};

// The value of v in the lane's other lanes of one row of accumulators (MT of them), joined by f
template <int MT, typename F> __device__ __forceinline__ float over_row(float v, F f) {
    auto dpp = [](float x, auto ctrl) { return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), decltype(ctrl)::value, 0xf, 0xf, false)); };
    v = f(v, dpp(v, std::integral_constant<int, 0x128>{}));       // rotated within 16 lanes by 8, 4, 2 and 1
    v = f(v, dpp(v, std::integral_constant<int, 0x124>{}));
    v = f(v, dpp(v, std::integral_constant<int, 0x122>{}));
    v = f(v, dpp(v, std::integral_constant<int, 0x121>{}));
    if constexpr (MT == 32) {                                     // the lane 16 away: both halves of 32 lanes, each in both
        const auto both = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = f(__uint_as_float(both[0]), __uint_as_float(both[1]));
    }
    return v;
}

// Where accumulator register v of row of tiles i lies in a wave's patch: row patch_step behind the lane's first one, 4 (lane / MT)
template <int MT> __device__ constexpr int patch_step(int i, int v) { return MT == 32 ? i * 32 + 8 * (v / 4) + v % 4 : i * 16 + v; }

// The thread's number, made anew where it is needed: what is computed from it would otherwise be kept over the main loop, which needs the registers
__device__ __forceinline__ int thread_again() {
    int t = threadIdx.x;
    asm volatile("" : "+v"(t));
    return t;
}

constexpr float LOG2_E = 1.44269504088896341f;
__device__ __forceinline__ float exp_less(float z, float base) { return __builtin_amdgcn_exp2f(__builtin_fmaf(z, LOG2_E, -base * LOG2_E)); }      // exp(z - base)

template <typename T, int TNI, int MT, int EDGE>
__device__ __forceinline__ void patch_bias(float (&bias)[TNI], bool (&in)[TNI], const void* from, int col0, int n, int lane) {
    static_for<0, TNI>([&](auto jc) {
        constexpr int j = decltype(jc)::value;
        const int col = col0 + j * MT + lane % MT;
        in[j] = !EDGE || col < n;
        bias[j] = from && in[j] ? widen(((const T*)from)[col]) : 0.f;
    });
}

// Logits to each row's share of the sum
struct VocabForward : M16Source {
    static constexpr bool ONCE = true, TAKES = true;
    const VocabTileArgs& a;
    __device__ __forceinline__ VocabForward(const VocabTileArgs& args) : a(args) {}
    template <typename T, int MT, int WGN, int TMI, int TNI, int EDGE, typename ACC>
    __device__ __forceinline__ bool take(ACC (&acc)[TMI][TNI], uint16_t* smem, int m0, int n0) {
        constexpr int NV = MT == 32 ? 16 : 4, WM = TMI * MT, WN = TNI * MT, BM = 4 / WGN * WM;
        const int t = thread_again(), lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), wm0 = wave / WGN * WM, wn0 = wave % WGN * WN;
        int* target = (int*)smem;                            // of the tile's rows, as columns of the piece
        __syncthreads();
        for (int r = t; r < BM; r += 256) target[r] = m0 + r < a.g.m ? a.targets[m0 + r] - a.v0 : -1;
        __syncthreads();
        float bias[TNI];
        bool in[TNI];
        patch_bias<T, TNI, MT, EDGE>(bias, in, a.g.bias, n0 + wn0, a.g.n, lane);
        const int row0 = wm0 + 4 * (lane / MT), column0 = n0 + wn0 + lane % MT;
        VocabPart* part = a.parts + (long long)(n0 / WN + wave % WGN) * a.g.m + m0 + row0;
        float* hits = a.hits + m0 + row0;
        const int* row_target = target + row0;
        const int left = a.g.m - m0 - row0;                  // rows behind the lane's first one
        constexpr int RB = MT == 16 ? 2 : 8;                  // rows at a time: what one waits for the others cover
        static_for<0, TMI * NV / RB>([&](auto qc) {
            constexpr int i = decltype(qc)::value / (NV / RB), v = decltype(qc)::value % (NV / RB) * RB;
            int at[RB];
            static_for<0, RB>([&](auto ec) { at[decltype(ec)::value] = row_target[patch_step<MT>(i, v + decltype(ec)::value)] - column0; });
            float z[RB][TNI], top[RB], base[RB], sum[RB];
            static_for<0, RB>([&](auto ec) {
                constexpr int e = decltype(ec)::value;
                static_for<0, TNI>([&](auto jc) {
                    constexpr int j = decltype(jc)::value;
                    z[e][j] = in[j] ? acc[i][j][v + e] + bias[j] : -INFINITY;
                    top[e] = j == 0 ? z[e][0] : fmaxf(top[e], z[e][j]);
                });
            });
            static_for<0, RB>([&](auto ec) {
                constexpr int e = decltype(ec)::value;
                top[e] = over_row<MT>(top[e], [](float x, float y) { return fmaxf(x, y); });
                base[e] = top[e] == -INFINITY ? 0.f : top[e];
            });
            static_for<0, RB>([&](auto ec) {
                constexpr int e = decltype(ec)::value;
                sum[e] = exp_less(z[e][0], base[e]);
                static_for<1, TNI>([&](auto jc) { sum[e] += exp_less(z[e][decltype(jc)::value], base[e]); });
            });
            static_for<0, RB>([&](auto ec) {
                constexpr int e = decltype(ec)::value;
                sum[e] = over_row<MT>(sum[e], [](float x, float y) { return x + y; });
            });
            static_for<0, RB>([&](auto ec) {
                constexpr int e = decltype(ec)::value, r = patch_step<MT>(i, v + e);
                if (lane % MT == 0 && r < left) part[r] = VocabPart{top[e], sum[e]};
            });
            bool any = false;
            static_for<0, RB>([&](auto ec) { const int c = at[decltype(ec)::value]; any = any || (c >= 0 && c < WN && c % MT == 0); });
            if (__builtin_amdgcn_ballot_w64(any)) {
                static_for<0, RB>([&](auto ec) {
                    constexpr int e = decltype(ec)::value, r = patch_step<MT>(i, v + e);
                    const int c = at[e];
                    static_for<0, TNI>([&](auto jc) {
                        constexpr int j = decltype(jc)::value;
                        if (c == j * MT && r < left && in[j]) hits[r] = z[e][j];
                    });
                });
            }
            __builtin_amdgcn_sched_barrier(0);               // (all rows mixed with each other take more registers than there are)
        });
        return true;
    }
};

// f of every row that has a target, where it is the same, and what d is multiplied by for it and dx, dw and db afterwards
__device__ __forceinline__ float row_weight(const VocabTileArgs& a) {
    const float u = a.upstream ? *a.upstream : 1.f;
    return a.count ? u / *a.count : u;
}
__device__ __forceinline__ float stored_weight(const VocabTileArgs& a) {
    const float u = row_weight(a);
    return __builtin_isfinite(u) ? ldexpf(1.f, a.most) : u;      // (an infinity belongs to the rows that have a target)
}
__device__ __forceinline__ float scale_back(const VocabTileArgs& a) {
    if (a.scale) return *a.scale;
    const float u = row_weight(a);
    return __builtin_isfinite(u) ? ldexpf(u, -a.most) : 1.f;
}

// Logits to their gradient
struct VocabGradient : M16Source {
    static constexpr bool ONCE = true, TAKES = true;
    const VocabTileArgs& a;
    __device__ __forceinline__ VocabGradient(const VocabTileArgs& args) : a(args) {}
    static constexpr size_t rows_at(int bm, int bn, int wgm) { return 4 * (size_t)(bm / wgm) * (bn / (4 / wgm) + 8) * 2; }      // bytes of the staged patches, which the rows' values lie behind
    template <typename T, int MT, int WGN, int TMI, int TNI, int EDGE, typename ACC>
    __device__ __forceinline__ bool take(ACC (&acc)[TMI][TNI], uint16_t* smem, int m0, int n0) {
        constexpr int NV = MT == 32 ? 16 : 4, WM = TMI * MT, WN = TNI * MT, BM = 4 / WGN * WM, EP = WN + 8;
        const int t = thread_again(), lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), wm0 = wave / WGN * WM, wn0 = wave % WGN * WN;
        uint16_t* region = smem + wave * (WM * EP);
        float* lse = (float*)(smem + 4 * WM * EP);
        float* f = lse + BM;
        int* target = (int*)(f + BM);
        const float same_f = a.f ? 0.f : stored_weight(a);
        __syncthreads();
        for (int r = t; r < BM; r += 256) {
            const bool there = m0 + r < a.g.m;
            lse[r] = there ? a.lse[m0 + r] * LOG2_E : 0.f;
            const int goal = there ? a.targets[m0 + r] : -1;
            f[r] = a.f ? there ? a.f[m0 + r] : 0.f : goal >= 0 && goal < a.classes ? same_f : 0.f;
            target[r] = there ? goal - a.v0 : -1;
        }
        __syncthreads();
        float bias[TNI], column[TNI];
        bool in[TNI];
        patch_bias<T, TNI, MT, EDGE>(bias, in, a.g.bias, n0 + wn0, a.g.n, lane);
        static_for<0, TNI>([&](auto jc) { column[decltype(jc)::value] = 0.f; });
        const int row0 = 4 * (lane / MT), column0 = n0 + wn0 + lane % MT;
        const float *row_lse = lse + wm0 + row0, *row_f = f + wm0 + row0;
        const int* row_target = target + wm0 + row0;
        uint16_t* staged = region + row0 * EP + lane % MT;
        constexpr int RB = 2;
        static_for<0, TMI * NV / RB>([&](auto qc) {
            constexpr int i = decltype(qc)::value / (NV / RB), v = decltype(qc)::value % (NV / RB) * RB;
            static_for<0, RB>([&](auto ec) {
                constexpr int e = decltype(ec)::value, r = patch_step<MT>(i, v + e);
                const float l = row_lse[r], fr = row_f[r];
                const int c = row_target[r] - column0;
                static_for<0, TNI>([&](auto jc) {
                    constexpr int j = decltype(jc)::value;
                    const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[i][j][v + e] + bias[j], LOG2_E, -l)) - (c == j * MT ? 1.f : 0.f);
                    const float d = in[j] && fr != 0.f ? p * fr : 0.f;      // (a row without a target has no gradient, whatever its logits are)
                    column[j] += d;
                    staged[r * EP + j * MT] = round_to<T>(d).bits;
                });
            });
            __builtin_amdgcn_sched_barrier(0);
        });
        if (a.db && wave / WGN == 0) {
            const float scale = scale_back(a);
            static_for<0, TNI>([&](auto jc) {
                constexpr int j = decltype(jc)::value;
                if constexpr (MT == 16) column[j] += __shfl_xor(column[j], 16);
                column[j] += __shfl_xor(column[j], 32);
                const int col = n0 + wn0 + j * MT + lane;
                if (lane < MT && col < a.g.n) {
                    T* to = (T*)a.db + col;
                    *to = round_to<T>(a.accumulate_db ? widen(*to) + column[j] * scale : column[j] * scale);
                }
            });
        }
        if (a.db_parts) {
            float* to = a.db_parts + (long long)(m0 / WM + wave / WGN) * a.pitch + n0 + wn0;
            static_for<0, TNI>([&](auto jc) {
                constexpr int j = decltype(jc)::value;
                if constexpr (MT == 16) column[j] += __shfl_xor(column[j], 16);
                column[j] += __shfl_xor(column[j], 32);
                if (lane < MT) to[j * MT + lane] = column[j];
            });
        }
        // (the wave's own rows: what its lanes staged is there when it reads)
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        constexpr int LPR = WN / 8, RPS = 64 / LPR;
        const int ecol = lane % LPR * 8;
#pragma unroll 4
        for (int r = lane / LPR; r < WM; r += RPS) {
            const int gm = m0 + wm0 + r;
            if (gm >= a.g.m) break;
            *(u32x4_t*)(a.d + gm * a.pitch + n0 + wn0 + ecol) = *(const u32x4_t*)(region + r * EP + ecol);
        }
        return true;
    }
};

// dx over the pieces, and dw
template <bool SUMS>
struct VocabGradProduct : M16Source {
    static constexpr bool ONCE = true, SCALED = true, TAKES = SUMS;
    const VocabTileArgs& a;
    __device__ __forceinline__ VocabGradProduct(const VocabTileArgs& args) : a(args) {}
    __device__ __forceinline__ float scale() const { return scale_back(a); }
    template <typename T, int MT, int WGN, int TMI, int TNI, int EDGE, typename ACC>
    __device__ __forceinline__ bool take(ACC (&acc)[TMI][TNI], uint16_t*, int m0, int n0) {
        constexpr int NV = MT == 32 ? 16 : 4, BM = 4 / WGN * TMI * MT, BN = WGN * TNI * MT;
        const int share = a.shares > 1 ? (int)blockIdx.x / a.total : 0;
        f32x4_t* own = (f32x4_t*)(a.sums + share * a.share_stride + ((long long)(m0 / BM) * a.tiles_n + n0 / BN) * (BM * BN)) + thread_again();
        if (!a.first) {
            static_for<0, TMI * TNI * NV / 4>([&](auto qc) {
                constexpr int q = decltype(qc)::value, i = q / (TNI * NV / 4), j = q / (NV / 4) % TNI, v = q % (NV / 4) * 4;
                const f32x4_t was = own[q * 256];
                static_for<0, 4>([&](auto ec) { acc[i][j][v + decltype(ec)::value] += was[decltype(ec)::value]; });
                if constexpr (MT == 16) held_in_place(acc[i][j]);      // (back where it was: the sums of both ways into the epilogue lie alike)
                if constexpr (q % 16 == 15) __builtin_amdgcn_sched_barrier(0);
            });
        }
        if (a.last && a.shares == 1) return false;
        static_for<0, TMI * TNI * NV / 4>([&](auto qc) {
            constexpr int q = decltype(qc)::value, i = q / (TNI * NV / 4), j = q / (NV / 4) % TNI, v = q % (NV / 4) * 4;
            own[q * 256] = f32x4_t{acc[i][j][v], acc[i][j][v + 1], acc[i][j][v + 2], acc[i][j][v + 3]};
        });
        return true;
    }
};

template <typename SRC, typename T, int BM, int BN, int WGM, bool A_MC, bool B_MC, int EDGE>
__global__ void __launch_bounds__(256, m16_blocks_per_cu(BM, BN, EDGE, 1)) vocab16_kernel(VocabTileArgs args) {
    SRC source(args);
    int slot = blockIdx.x, stride = gridDim.x;
    // (one plain matrix: the options that GemmArgs has beside are known to be unused here)
    GemmArgs g{args.g.C, args.g.A, args.g.B, args.g.bias, 1, args.g.m, args.g.k, args.g.n, 0, A_MC ? 1 : args.g.a_rs, A_MC ? args.g.a_cs : 1, 0, B_MC ? args.g.b_rs : 1, B_MC ? 1 : args.g.b_cs, 0, args.g.c_rs, 1, args.g.accumulate};
    if constexpr (std::is_same<SRC, VocabGradProduct<true>>::value && BM != 256) {
        if (args.shares > 1) {
            const int share = slot / args.total, k0 = share * args.k_share;
            slot -= share * args.total;
            stride = args.total;
            g.A = (const T*)g.A + k0 * g.a_cs;
            g.B = (const T*)g.B + k0 * g.b_rs;
            g.k = g.k - k0 < args.k_share ? g.k - k0 : args.k_share;
        }
    }
    gemm_mfma16_block<T, BM, BN, WGM, A_MC, B_MC, EDGE, false, 1, SRC>(g, args.tiles_m, args.tiles_n, nullptr, 0, args.total, slot, 0, stride, &source);
}

// What the shares of k add up to, in their order, scaled and rounded: a workgroup four quads of a tile's registers (tiles of 32 x 32 MFMAs, two by two waves)
template <typename T, int BM>
__global__ void __launch_bounds__(256) vocab16_join_kernel(VocabTileArgs a) {
    constexpr int TM = BM / 64, QUADS = TM * TM * 4;
    const int tile = blockIdx.x / (QUADS / 4), q0 = blockIdx.x % (QUADS / 4) * 4, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int m0 = tile / a.tiles_n * BM + wave / 2 * (BM / 2), n0 = tile % a.tiles_n * BM + wave % 2 * (BM / 2);
    const f32x4_t* own = (const f32x4_t*)(a.sums + (long long)tile * (BM * BM)) + threadIdx.x;
    f32x4_t sum[4] = {};
    for (int s = 0; s < a.shares; s++)
#pragma unroll
        for (int e = 0; e < 4; e++) sum[e] += *(const f32x4_t*)((const float*)(own + (q0 + e) * 256) + s * a.share_stride);
    const float scale = scale_back(a);
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const int i = (q0 + e) / (TM * 4), j = (q0 + e) / 4 % TM, col = n0 + j * 32 + (lane & 31), row = m0 + i * 32 + 8 * e + 4 * (lane >> 5);
        if (col >= a.g.n) continue;
#pragma unroll
        for (int u = 0; u < 4; u++) {
            if (row + u >= a.g.m) continue;
            T* to = (T*)a.g.C + (row + u) * a.g.c_rs + col;
            const T y = round_to<T>(sum[e][u] * scale);
            *to = a.g.accumulate ? round_to<T>(widen(*to) + widen(y)) : y;
        }
    }
}

template <typename SRC, typename T, int BM, int BN, int WGM, bool A_MC, bool B_MC, int EDGE>
static int launch_vocab16_tile(VocabTileArgs a) {
    a.tiles_m = (a.g.m + BM - 1) / BM;
    a.tiles_n = (a.g.n + BN - 1) / BN;
    a.total = scheduled_grid(a.tiles_m, a.tiles_n);
    size_t smem = m16_smem_bytes(BM, BN, WGM, A_MC, B_MC, 2, m16_mfma_tile(BM, BN));
    const size_t staged = VocabGradient::rows_at(BM, BN, WGM) + 12 * BM;
    if (std::is_same<SRC, VocabGradient>::value && staged > smem) smem = staged;
    const int cus = device_cu_count() / 8 * 8;
    int blocks = BM == 256 && BN == 256 && cus >= 8 && a.total > cus ? cus : a.total;      // one resident workgroup a CU, as for a product of its own
    if (a.shares > 1) blocks = a.total * a.shares;
    auto kern = vocab16_kernel<SRC, T, BM, BN, WGM, A_MC, B_MC, EDGE>;
    if (smem > 64 * 1024 && !check_hip(hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)smem), "hipFuncSetAttribute")) return -1;
    hipLaunchKernelGGL(kern, dim3(blocks), dim3(256), smem, current_stream(), a);
    if (!check_launch("vocab16_kernel")) return -1;
    if constexpr (std::is_same<SRC, VocabGradProduct<true>>::value && BM != 256) {
        if (a.shares > 1 && a.last) {
            constexpr int TM = BM / 64;
            hipLaunchKernelGGL((vocab16_join_kernel<T, BM>), dim3(a.tiles_m * a.tiles_n * TM * TM), dim3(256), 0, current_stream(), a);
            return check_launch("vocab16_join_kernel") ? 0 : -1;
        }
    }
    return 0;
}

// The launchers of a tile's translation unit.  logits: W row-major (b_mc) or its transpose; dx: likewise (b_mc where W is the transpose); dw: x^T . d or d^T . x.
enum VocabStep { VOCAB_FORWARD, VOCAB_GRADIENT, VOCAB_DX, VOCAB_DW };
template <typename T, int BM, int BN, int WGM, int EDGE>
static int launch_vocab16_logits(const VocabTileArgs& a, VocabStep step, bool b_mc) {
    if (step == VOCAB_FORWARD) return b_mc ? launch_vocab16_tile<VocabForward, T, BM, BN, WGM, false, true, EDGE>(a) : launch_vocab16_tile<VocabForward, T, BM, BN, WGM, false, false, EDGE>(a);
    return b_mc ? launch_vocab16_tile<VocabGradient, T, BM, BN, WGM, false, true, EDGE>(a) : launch_vocab16_tile<VocabGradient, T, BM, BN, WGM, false, false, EDGE>(a);
}
template <typename T, int BM, int BN, int WGM, int EDGE>
static int launch_vocab16_grads(const VocabTileArgs& a, VocabStep step, bool b_mc) {
    if (step == VOCAB_DW) return launch_vocab16_tile<VocabGradProduct<(BM < 256)>, T, BM, BN, WGM, true, true, EDGE>(a);
    return b_mc ? launch_vocab16_tile<VocabGradProduct<true>, T, BM, BN, WGM, false, true, EDGE>(a) : launch_vocab16_tile<VocabGradProduct<true>, T, BM, BN, WGM, false, false, EDGE>(a);
}

// edge: nothing, whole vectors, anything hangs over (M16_WHOLE, M16_EDGE, M16_RAGGED; the 256 x 256 tiles take the first two, the others the last two)
int launch_vocab16_logits_256_bf16(const VocabTileArgs& a, VocabStep step, bool b_mc, int edge);
int launch_vocab16_logits_256_f16(const VocabTileArgs& a, VocabStep step, bool b_mc, int edge);
int launch_vocab16_grads_256_bf16(const VocabTileArgs& a, VocabStep step, bool b_mc, int edge);
int launch_vocab16_grads_256_f16(const VocabTileArgs& a, VocabStep step, bool b_mc, int edge);
int launch_vocab16_logits_128(const VocabTileArgs& a, VocabStep step, bool b_mc, int edge, int dtype);
int launch_vocab16_logits_64x128(const VocabTileArgs& a, VocabStep step, bool b_mc, int edge, int dtype);
int launch_vocab16_grads_128(const VocabTileArgs& a, VocabStep step, bool b_mc, int edge, int dtype);
int launch_vocab16_grads_64(const VocabTileArgs& a, VocabStep step, bool b_mc, int edge, int dtype);

}  // namespace rp
