// bf16 / fp16 gated linear layer on the tiles of the 16-bit MFMA kernel: a tile holds the same columns of both halves of W, so that the gate and what it multiplies meet in one wave and neither is
// written and read again.
//
// The sums of a wave's patch go through LDS as float32, half a patch at a time: a lane then has eight neighbouring columns of both halves, stores h in 16 bytes and, where it is kept, z in whole cache
// lines, and the gate's code stands there twice and not once for each of 128 registers.  8192 rows, 4096 -> 8192 in bf16: see gated16_forward.
#pragma once
#include "rp_gated.h"
#include "rp_gemm_mfma16_kernel.h"

namespace rp {

struct GatedTileArgs {
    GemmArgs g;                    // A: x, B: W with n = both halves, C unused
    int tiles_m, tiles_n, total;
    GatedArgs l;
};

struct GatedTiles : M16Source {
    static constexpr bool ONCE = true, PAIRED = true, TAKES = true;
    const GatedTileArgs& a;
    const int pair;
    __device__ __forceinline__ GatedTiles(const GatedTileArgs& args) : a(args), pair(args.l.n) {}
    static constexpr size_t staged(int bm, int bn, int wgm) { return 4 * (size_t)(bm == 256 ? bm / wgm / 2 : bm / wgm) * (bn / (4 / wgm) + 4) * 4; }      // bytes of LDS

    template <typename T, int MT, int WGN, int TMI, int TNI, int EDGE, typename ACC>
    __device__ __forceinline__ bool take(ACC (&acc)[TMI][TNI], uint16_t* smem, int m0, int n0) {
        constexpr int NV = MT == 32 ? 16 : 4, WM = TMI * MT, WN = TNI * MT, HN = WN / 2, EP = WN + 4;
        constexpr int PASSES = MT == 16 ? 2 : 1, ROWS = WM / PASSES, LPR = HN / 8, RPS = 64 / LPR;       // rows of a pass; lanes to a row, rows to a step
        int t = threadIdx.x;
        asm volatile("" : "+v"(t));                          // (what is computed from it is not kept over the main loop)
        const int lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), wm0 = wave / WGN * WM;
        float* region = (float*)smem + wave * (ROWS * EP);
        const int n = a.l.n, ecol = lane % LPR * 8, col = n0 + wave % WGN * HN + ecol, left = n - col;      // the lane's eight columns, and how many there are from the first on
        float* put = region + 4 * (lane / MT) * EP + lane % MT;
        float bias[16];
#pragma unroll
        for (int u = 0; u < 8; u++) {
            const bool in = a.l.bias && (!EDGE || u < left);
            bias[u] = in ? widen(((const T*)a.l.bias)[col + u]) : 0.f;
            bias[8 + u] = in ? widen(((const T*)a.l.bias)[n + col + u]) : 0.f;
        }
        __syncthreads();                                     // every wave is done with the main loop's LDS
        static_for<0, PASSES>([&](auto pc) {
            constexpr int p = decltype(pc)::value, TI = TMI / PASSES;
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            static_for<0, TI * NV>([&](auto ivc) {
                constexpr int i = decltype(ivc)::value / NV, v = decltype(ivc)::value % NV, r = MT == 32 ? i * 32 + 8 * (v / 4) + v % 4 : i * 16 + v;
                static_for<0, TNI>([&](auto jc) {
                    constexpr int j = decltype(jc)::value;
                    put[r * EP + j * MT] = acc[p * TI + i][j][v];
                });
            });
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");      // (the wave's own rows: what its lanes staged is there when it reads)
            RP_DISPATCH_GATE(a.l.gate, rows<T, GATE, EDGE, EP, HN, RPS, ROWS>(region, bias, lane / LPR, ecol, m0 + wm0 + p * ROWS, col, left));
        });
        return true;
    }

    template <typename T, int GATE, int EDGE, int EP, int HN, int RPS, int ROWS>
    __device__ __forceinline__ void rows(const float* region, const float (&bias)[16], int first, int ecol, int m0, int col, int left) {
        const long long zn = 2ll * a.l.n;
        float* z = (float*)a.l.z;
        T* h = (T*)a.l.h;
        const bool whole = !EDGE || left >= 8;
        const bool z_vec = a.l.n % 4 == 0 && ((uintptr_t)z & 15) == 0;
#pragma unroll 1
        for (int r = first; r < ROWS; r += RPS) {
            const int gm = m0 + r;
            if (gm >= a.l.rows) break;
            float gate[8], up[8];
            *(f32x4_t*)gate = *(const f32x4_t*)(region + r * EP + ecol);
            *(f32x4_t*)(gate + 4) = *(const f32x4_t*)(region + r * EP + ecol + 4);
            *(f32x4_t*)up = *(const f32x4_t*)(region + r * EP + HN + ecol);
            *(f32x4_t*)(up + 4) = *(const f32x4_t*)(region + r * EP + HN + ecol + 4);
            T out[8];
#pragma unroll
            for (int u = 0; u < 8; u++) {
                gate[u] += bias[u];
                up[u] += bias[8 + u];
                out[u] = round_to<T>(gate_value<GATE>(gate[u]) * up[u]);
            }
            T* to = h + gm * a.l.h_rs + col;
            if (whole) {
                u32x4_t o;
                __builtin_memcpy(&o, out, 16);
                *(u32x4_any_t*)to = o;
            } else {
#pragma unroll
                for (int u = 0; u < 8; u++)
                    if (u < left) to[u] = out[u];
            }
            if (z) {
                float* zg = z + gm * zn + col;
                float* zu = zg + a.l.n;
                if (whole && z_vec) {
                    // (not read before the backward pass: out of the way of the operands in L2)
                    __builtin_nontemporal_store(*(const f32x4_t*)gate, (f32x4_t*)zg);
                    __builtin_nontemporal_store(*(const f32x4_t*)(gate + 4), (f32x4_t*)(zg + 4));
                    __builtin_nontemporal_store(*(const f32x4_t*)up, (f32x4_t*)zu);
                    __builtin_nontemporal_store(*(const f32x4_t*)(up + 4), (f32x4_t*)(zu + 4));
                } else {
#pragma unroll
                    for (int u = 0; u < 8; u++)
                        if (whole || u < left) { zg[u] = gate[u]; zu[u] = up[u]; }
                }
            }
        }
    }
};

template <typename T, int BM, int BN, int WGM, bool B_MC, int EDGE>
__global__ void __launch_bounds__(256, m16_blocks_per_cu(BM, BN, EDGE, 1)) gated16_kernel(GatedTileArgs args) {
    GatedTiles source(args);
    const GemmArgs g{nullptr, args.g.A, args.g.B, nullptr, 1, args.g.m, args.g.k, args.g.n, 0, args.g.a_rs, 1, 0, B_MC ? args.g.b_rs : 1, B_MC ? 1 : args.g.b_cs};
    gemm_mfma16_block<T, BM, BN, WGM, false, B_MC, EDGE, false, 1, GatedTiles>(g, args.tiles_m, args.tiles_n, nullptr, 0, args.total, (int)blockIdx.x, 0, (int)gridDim.x, &source);
}

template <typename T, int BM, int BN, int WGM, bool B_MC, int EDGE>
static int launch_gated16_tile(const GatedArgs& l) {
    GatedTileArgs a{};
    a.g = GemmArgs{nullptr, l.x, l.w, nullptr, 1, l.rows, l.k, 2 * l.n, 0, l.x_rs, 1, 0, l.w_rs, l.w_cs};
    a.l = l;
    a.tiles_m = (l.rows + BM - 1) / BM;
    a.tiles_n = (l.n + BN / 2 - 1) / (BN / 2);
    a.total = scheduled_grid(a.tiles_m, a.tiles_n);
    size_t smem = m16_smem_bytes(BM, BN, WGM, false, B_MC, 2, m16_mfma_tile(BM, BN));
    if (GatedTiles::staged(BM, BN, WGM) > smem) smem = GatedTiles::staged(BM, BN, WGM);
    const int cus = device_cu_count() / 8 * 8;
    const int blocks = BM == 256 && BN == 256 && cus >= 8 && a.total > cus ? cus : a.total;      // one resident workgroup a CU, as for a plain product
    auto kern = gated16_kernel<T, BM, BN, WGM, B_MC, EDGE>;
    if (smem > 64 * 1024 && !check_hip(hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)smem), "hipFuncSetAttribute")) return -1;
    hipLaunchKernelGGL(kern, dim3(blocks), dim3(256), smem, current_stream(), a);
    return check_launch("gated16_kernel") ? 0 : -1;
}
template <typename T, int BM, int BN, int WGM, int EDGE>
static int launch_gated16(const GatedArgs& l) {
    return l.w_cs == 1 ? launch_gated16_tile<T, BM, BN, WGM, true, EDGE>(l) : launch_gated16_tile<T, BM, BN, WGM, false, EDGE>(l);
}

// edge: nothing, whole vectors, anything hangs over (the 256 x 256 tiles take the first two, the others the last two)
int launch_gated16_256_bf16(const GatedArgs& l, int edge);
int launch_gated16_256_f16(const GatedArgs& l, int edge);
int launch_gated16_128(const GatedArgs& l, int edge, int dtype);
int launch_gated16_64x128(const GatedArgs& l, int edge, int dtype);

}  // namespace rp
