// bf16 / fp16 shared projection with its rows' adapters, y[i] = x[i] . w + bias + h[i] . b_a, on the tiles of the 16-bit MFMA kernel: the adapters'
// term goes into a tile's accumulators between its last slab and its one rounding, so y is written once and never read.
//
// A wave adds the term of every segment that has rows in its patch: rank / 32 (or / 16) more k-steps with the other segments' rows zero.  h is
// float32 and is multiplied as two values of the tensors' type (split_low).  b comes straight from memory, 16 bytes a lane where it is
// contiguous along the rank (a_a^T, for dx) and else eight 2-byte loads: some 2 us a segment on a tile that takes 50 at k = 4096.
#pragma once
#include "rp_adapter16.h"
#include "rp_gemm_mfma16_kernel.h"

namespace rp {

struct AdapterTiles {
    static constexpr bool ONCE = true, TERM = true;
    AdapterTerm term;
    int tiles_m, tiles_n, m, n;
    __device__ __forceinline__ TileCoord tile(int id, GemmArgs&) const { return schedule_tile(id, tiles_m, tiles_n); }

    template <typename T, int MT, int TMI, int TNI, typename ACC>
    __device__ __forceinline__ void add_term(ACC (&acc)[TMI][TNI], int row0, int col0, int lane) const {
        constexpr int KSTEP = MT == 32 ? 16 : 32;
        const bool whole = term.rank % 4 == 0 && ((uintptr_t)term.h & 15) == 0;
        const int fr = lane % MT, oct = lane / MT, row_end = row0 + TMI * MT < m ? row0 + TMI * MT : m;
        for (int g0 = 0; g0 < term.gr.groups; g0 += 64) {
            int b = 0, e = 0, w = -1;
            if (g0 + lane < term.gr.groups) { b = term.gr.begin(g0 + lane); e = term.gr.end(g0 + lane); w = term.gr.weight(g0 + lane); }
            unsigned long long here = __builtin_amdgcn_ballot_w64(w >= 0 && b < row_end && e > row0);
            while (here) {
                const int l = __builtin_ctzll(here);
                here &= here - 1;
                const int sb = __builtin_amdgcn_readlane(b, l), se = __builtin_amdgcn_readlane(e, l), a = __builtin_amdgcn_readlane(w, l);
                const uint16_t* bp = (const uint16_t*)term.b + a * term.b_ws;
                for (int k0 = 0; k0 < term.rank; k0 += KSTEP) {
                    const int kk = k0 + 8 * oct, left = term.rank - kk;
                    s16x8_t hi[TMI], lo[TMI];
#pragma unroll
                    for (int i = 0; i < TMI; i++) {
                        const int row = row0 + i * MT + fr;
                        float v[8];
                        const float* h = term.h + (long long)row * term.rank + kk;
                        const bool in = row >= sb && row < se;
                        if (whole) {
                            const f32x4_t zero = {0.f, 0.f, 0.f, 0.f};
                            const f32x4_t p = in && left > 0 ? *(const f32x4_t*)h : zero, r = in && left > 4 ? *(const f32x4_t*)(h + 4) : zero;
#pragma unroll
                            for (int u = 0; u < 4; u++) { v[u] = p[u]; v[4 + u] = r[u]; }
                        } else {
#pragma unroll
                            for (int u = 0; u < 8; u++) v[u] = in && u < left ? h[u] : 0.f;
                        }
                        u32x4_t hv, lv;
                        split_low<T>(v, hv, lv);
                        hi[i] = __builtin_bit_cast(s16x8_t, hv);
                        lo[i] = __builtin_bit_cast(s16x8_t, lv);
                    }
                    static_for<0, TNI>([&](auto jc) {
                        constexpr int j = decltype(jc)::value;
                        const int col = col0 + j * MT + fr;
                        s16x8_t bf = {0, 0, 0, 0, 0, 0, 0, 0};
                        if (col < n) {
                            const uint16_t* p = bp + (long long)kk * term.b_rs + (long long)col * term.b_cs;
                            if (term.b_rs == 1) bf = __builtin_bit_cast(s16x8_t, load8(p, left));
                            else {
#pragma unroll
                                for (int u = 0; u < 8; u++) bf[u] = u < left ? (short)p[u * term.b_rs] : (short)0;
                            }
                        }
                        // (the in-place MFMAs are opaque to the compiler: what vector instructions wrote for them has to be there)
                        if constexpr (MT == 16) {
                            __builtin_amdgcn_sched_barrier(0);
                            asm volatile("s_nop 7" : "+v"(bf) : : "memory");
                            if constexpr (j == 0) {
#pragma unroll
                                for (int i = 0; i < TMI; i++) asm volatile("s_nop 7" : "+v"(hi[i]), "+v"(lo[i]) : : "memory");
                            }
                        }
                        static_for<0, TMI>([&](auto ic) {
                            constexpr int i = decltype(ic)::value;
                            if (row0 + i * MT >= se || row0 + (i + 1) * MT <= sb) return;
                            acc[i][j] = mfma16_ops<T>::mma(hi[i], bf, acc[i][j]);
                            acc[i][j] = mfma16_ops<T>::mma(lo[i], bf, acc[i][j]);
                        });
                    });
                }
            }
        }
    }
};

template <typename T, int BM, int BN, int WGM, bool B_MC, int EDGE>
__global__ void __launch_bounds__(256, m16_blocks_per_cu(BM, BN, EDGE, 1)) adapter_tiles16_kernel(GemmArgs args, AdapterTerm term, int tiles_m, int tiles_n, int total) {
    AdapterTiles source{term, tiles_m, tiles_n, args.m, args.n};
    GemmArgs g = args;
    gemm_mfma16_block<T, BM, BN, WGM, false, B_MC, EDGE, false, 1, AdapterTiles>(g, 0, 0, nullptr, 0, total, (int)blockIdx.x, 0, (int)gridDim.x, &source);
}

template <typename T, int BM, int BN, int WGM, bool B_MC, int EDGE>
static int launch_adapter_tiles16(const GroupedArgs& s, const AdapterTerm& term) {
    const int tiles_m = (s.gr.rows + BM - 1) / BM, tiles_n = (s.n + BN - 1) / BN, total = scheduled_grid(tiles_m, tiles_n);
    constexpr size_t smem = m16_smem_bytes(BM, BN, WGM, false, B_MC, 2, m16_mfma_tile(BM, BN));
    const GemmArgs g{s.C, s.A, s.B, s.bias, 1, s.gr.rows, s.k, s.n, 0, s.a_rs, s.a_cs, 0, s.b_rs, s.b_cs, 0, s.c_rs, 1, s.accumulate};
    const int cus = device_cu_count() / 8 * 8;
    const int blocks = BM == 256 && BN == 256 && cus >= 8 && total > cus ? cus : total;      // one resident workgroup a CU, as for a product of its own
    auto kern = adapter_tiles16_kernel<T, BM, BN, WGM, B_MC, EDGE>;
    if (smem > 64 * 1024 && !check_hip(hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)smem), "hipFuncSetAttribute")) return -1;
    hipLaunchKernelGGL(kern, dim3(blocks), dim3(256), smem, current_stream(), g, term, tiles_m, tiles_n, total);
    return check_launch("adapter_tiles16_kernel") ? 0 : -1;
}

template <typename T, int BM, int BN, int WGM, int EDGE>
static int launch_adapter_tiles16_layout(const GroupedArgs& s, const AdapterTerm& term) {
    return s.b_cs == 1 ? launch_adapter_tiles16<T, BM, BN, WGM, true, EDGE>(s, term) : launch_adapter_tiles16<T, BM, BN, WGM, false, EDGE>(s, term);
}

}  // namespace rp
