// bf16 / fp16 gated linear layer on the tiles of the 16-bit MFMA kernel: a tile holds the same columns of both halves of W, so that the gate and what it multiplies meet in one wave and neither is
// written and read again.
//
// The sums of a wave's patch go through LDS as float32, half a patch at a time: a lane then has eight neighbouring columns of both halves, stores h in 16 bytes and, where it is kept, z in whole cache
// lines, and the gate's code stands there twice and not once for each of 128 registers.  8192 rows, 4096 -> 8192 in bf16: see gated16_forward.
#pragma once
#include "rp_gated.h"
#include "rp_gemm_mfma16_kernel.h"

namespace rp {

typedef float f32x4_any_t __attribute__((ext_vector_type(4), aligned(4)));

struct GatedShares { int count, k; float* sums; };

struct GatedTileArgs {
    GemmArgs g;                    // A: x, B: W with n = both halves, C unused
    int tiles_m, tiles_n, total;
    GatedArgs l;
    // k in shares of k_share that workgroups of their own add up, where there are few tiles (1: none): their sums of g | u, [shares][rows][2 n], which a second launch joins
    int shares, k_share;
    float* sums;
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
        if constexpr (MT == 32) if (a.shares > 1) {
            const int n = a.l.n, share = (int)blockIdx.x / a.total, row0 = m0 + wm0 + 4 * (lane / MT), at0 = n0 + wave % WGN * HN + lane % MT;
            float* to = a.sums + ((long long)share * a.l.rows + row0) * 2 * n + at0;
            static_for<0, TMI * NV>([&](auto ivc) {
                constexpr int i = decltype(ivc)::value / NV, v = decltype(ivc)::value % NV, r = MT == 32 ? i * 32 + 8 * (v / 4) + v % 4 : i * 16 + v;
                static_for<0, TNI>([&](auto jc) {
                    constexpr int j = decltype(jc)::value, c = j * MT % HN, half = j * MT / HN;
                    if (row0 + r < a.l.rows && at0 + c < n) to[(long long)r * 2 * n + half * n + c] = acc[i][j][v];
                });
            });
            return true;
        }
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
            float value[8];
#pragma unroll
            for (int u = 0; u < 8; u++) {
                gate[u] += bias[u];
                up[u] += bias[8 + u];
                value[u] = gate_value<GATE>(gate[u]) * up[u];
            }
            round_vector<T>(out, value);
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
                if (whole) {
                    // (16 bytes at any element)
                    *(f32x4_any_t*)zg = *(const f32x4_t*)gate;
                    *(f32x4_any_t*)(zg + 4) = *(const f32x4_t*)(gate + 4);
                    *(f32x4_any_t*)zu = *(const f32x4_t*)up;
                    *(f32x4_any_t*)(zu + 4) = *(const f32x4_t*)(up + 4);
                } else {
#pragma unroll
                    for (int u = 0; u < 8; u++)
                        if (u < left) { zg[u] = gate[u]; zu[u] = up[u]; }
                }
            }
        }
    }
};

template <typename T, int BM, int BN, int WGM, bool B_MC, int EDGE>
__global__ void __launch_bounds__(256, m16_blocks_per_cu(BM, BN, EDGE, 1)) gated16_kernel(GatedTileArgs args) {
    GatedTiles source(args);
    int slot = blockIdx.x, stride = gridDim.x;
    GemmArgs g{nullptr, args.g.A, args.g.B, nullptr, 1, args.g.m, args.g.k, args.g.n, 0, args.g.a_rs, 1, 0, B_MC ? args.g.b_rs : 1, B_MC ? 1 : args.g.b_cs};
    if constexpr (BM != 256) {
        if (args.shares > 1) {
            const int share = slot / args.total, k0 = share * args.k_share;
            slot -= share * args.total;
            stride = args.total;
            g.A = (const T*)g.A + k0;
            g.B = (const T*)g.B + k0 * g.b_rs;
            g.k = g.k - k0 < args.k_share ? g.k - k0 : args.k_share;
        }
    }
    gemm_mfma16_block<T, BM, BN, WGM, false, B_MC, EDGE, false, 1, GatedTiles>(g, args.tiles_m, args.tiles_n, nullptr, 0, args.total, slot, 0, stride, &source);
}

// h, and z where it is kept, from the shares' sums, added in their order: a thread a column of both halves
template <typename T, int GATE>
__global__ void __launch_bounds__(256) gated16_join_kernel(GatedArgs l, const float* sums, int shares, int across) {
    const long long total = (long long)l.rows * across, one = 2ll * l.rows * l.n;
    for (long long id = blockIdx.x; id < total; id += gridDim.x) {
        const int row = (int)(id / across), c = (int)(id % across) * 256 + threadIdx.x;
        if (c >= l.n) continue;
        const float* at = sums + (long long)row * 2 * l.n + c;
        float gate = 0.f, up = 0.f;
#pragma unroll 4
        for (int s = 0; s < shares; s++) {
            gate += at[s * one];
            up += at[s * one + l.n];
        }
        if (l.bias) {
            gate += widen(((const T*)l.bias)[c]);
            up += widen(((const T*)l.bias)[l.n + c]);
        }
        if (l.z) {
            float* z = (float*)l.z + (long long)row * 2 * l.n + c;
            z[0] = gate;
            z[l.n] = up;
        }
        ((T*)l.h)[row * l.h_rs + c] = round_to<T>(gate_value<GATE>(gate) * up);
    }
}

template <typename T, int BM, int BN, int WGM, bool B_MC, int EDGE>
static int launch_gated16_tile(const GatedArgs& l, const GatedShares& shares) {
    GatedTileArgs a{};
    a.shares = shares.count;
    a.k_share = shares.k;
    a.sums = shares.sums;
    a.g = GemmArgs{nullptr, l.x, l.w, nullptr, 1, l.rows, l.k, 2 * l.n, 0, l.x_rs, 1, 0, l.w_rs, l.w_cs};
    a.l = l;
    a.tiles_m = (l.rows + BM - 1) / BM;
    a.tiles_n = (l.n + BN / 2 - 1) / (BN / 2);
    a.total = scheduled_grid(a.tiles_m, a.tiles_n);
    size_t smem = m16_smem_bytes(BM, BN, WGM, false, B_MC, 2, m16_mfma_tile(BM, BN));
    if (GatedTiles::staged(BM, BN, WGM) > smem) smem = GatedTiles::staged(BM, BN, WGM);
    const int cus = device_cu_count() / 8 * 8;
    int blocks = BM == 256 && BN == 256 && cus >= 8 && a.total > cus ? cus : a.total;      // one resident workgroup a CU, as for a plain product
    if (a.shares > 1) blocks = a.total * a.shares;
    auto kern = gated16_kernel<T, BM, BN, WGM, B_MC, EDGE>;
    if (smem > 64 * 1024 && !check_hip(hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)smem), "hipFuncSetAttribute")) return -1;
    hipLaunchKernelGGL(kern, dim3(blocks), dim3(256), smem, current_stream(), a);
    if (!check_launch("gated16_kernel")) return -1;
    if constexpr (BM != 256) if (a.shares > 1) {
        const int across = (l.n + 255) / 256;
        const long long joined = (long long)l.rows * across;
        RP_DISPATCH_GATE(l.gate, hipLaunchKernelGGL((gated16_join_kernel<T, GATE>), dim3((unsigned)(joined < (1 << 20) ? joined : 1 << 20)), dim3(256), 0, current_stream(), l, a.sums, a.shares, across));
        return check_launch("gated16_join_kernel") ? 0 : -1;
    }
    return 0;
}
template <typename T, int BM, int BN, int WGM, int EDGE>
static int launch_gated16(const GatedArgs& l, const GatedShares& shares = {1, 0, nullptr}) {
    return l.w_cs == 1 ? launch_gated16_tile<T, BM, BN, WGM, true, EDGE>(l, shares) : launch_gated16_tile<T, BM, BN, WGM, false, EDGE>(l, shares);
}

// edge: nothing, whole vectors, anything hangs over (the 256 x 256 tiles take the first two, the others the last two)
int launch_gated16_256_bf16(const GatedArgs& l, int edge);
int launch_gated16_256_f16(const GatedArgs& l, int edge);
int launch_gated16_128(const GatedArgs& l, int edge, int dtype);
int launch_gated16_64x128(const GatedArgs& l, const GatedShares& shares, int edge, int dtype);

}  // namespace rp
