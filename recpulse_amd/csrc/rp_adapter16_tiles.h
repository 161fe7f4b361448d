// bf16 / fp16 shared projection with its rows' adapters, y[i] = x[i] . w + bias + h[i] . b_a, on the tiles of the 16-bit MFMA kernel: the adapters'
// term is what a tile's accumulators start from, so y is rounded once, written once and never read.
//
// For every segment that has rows in a wave's patch: rank / 32 (/ 16) k-steps of MFMAs, the other segments' rows zero.  h is float32 and is
// multiplied as two values of bfloat16; where the tensors are float16, which does not reach far enough for it, as three, and b, exactly, as two (five products).  b comes straight from memory, 16 bytes a lane where it is contiguous along
// the rank (a_a^T, for dx) and else in 2-byte loads.  4096 x 4096 x 4096 with seven segments in bf16: 119 us at rank 16 and 118 at rank 32 (float16 129), 107 without an adapter, beside 18
// and more for a pass over y.
// (Between the last slab and the epilogue the same code takes registers from the main loop of the 256 x 256 tile: a value or two reloaded
// from memory a slab, behind which all of its loads are waited for; 130.  In the epilogue, into registers of its own 16 rows at a
// time, it is unrolled eightfold and waits for its instructions: 134.)
#pragma once
#include "rp_adapter16.h"
#include "rp_gemm_mfma16_kernel.h"

namespace rp {

struct AdapterTileArgs {
    GemmArgs g;
    int tiles_m, tiles_n, total;
    AdapterTerm term;
};

struct AdapterTiles : M16Source {
    static constexpr bool MOVES = false, ONCE = true, TERM = true;
    bool odd = false;              // the wave met an infinity or NaN in b

    // The term's arguments are read from where the launch left them whenever they are needed: kept for the next tile they would take registers that the main loop needs.
    typedef const __attribute__((address_space(4))) AdapterTileArgs* args_t;       // (constant memory: scalar loads)
    static __device__ __forceinline__ args_t arguments() { return (args_t)__builtin_amdgcn_kernarg_segment_ptr(); }
    static __device__ __forceinline__ AdapterTerm term_of(args_t args) {
        const RowGroups gr{args->term.gr.offsets, args->term.gr.ids, args->term.gr.groups, args->term.gr.rows, args->term.gr.weights};
        return AdapterTerm{args->term.h, args->term.b, gr, args->term.rank, args->term.b_ws, args->term.b_rs, args->term.b_cs};
    }
    // f(begin, end, adapter) for every segment with an adapter that has some of the rows [row0, row_end); the wave looks at 64 segments at a time
    template <typename F> static __device__ __forceinline__ void for_segments(const RowGroups& gr, int row0, int row_end, int lane, F f) {
        for (int g0 = 0; g0 < gr.groups; g0 += 64) {
            int b = 0, e = 0, w = -1;
            if (g0 + lane < gr.groups) { b = gr.begin(g0 + lane); e = gr.end(g0 + lane); w = gr.weight(g0 + lane); }
            unsigned long long here = __builtin_amdgcn_ballot_w64(w >= 0 && b < row_end && e > row0);
            while (here) {
                const int l = __builtin_ctzll(here);
                here &= here - 1;
                f(__builtin_amdgcn_readlane(b, l), __builtin_amdgcn_readlane(e, l), __builtin_amdgcn_readlane(w, l));
            }
        }
    }

    // eight values as P of bfloat16 that add up to them: f(number, vector)
    template <int P, typename F> static __device__ __forceinline__ void parts(const float* v, F f) {
        float left[8];
#pragma unroll
        for (int u = 0; u < 8; u++) left[u] = v[u];
        static_for<0, P>([&](auto pc) {
            bf16_t part[8];
#pragma unroll
            for (int u = 0; u < 8; u++) {
                part[u] = round_to<bf16_t>(left[u]);
                left[u] -= widen(part[u]);
                left[u] = __builtin_isfinite(left[u]) ? left[u] : 0.f;
            }
            u32x4_t vec;
            __builtin_memcpy(&vec, part, 16);
            f(pc, vec);
        });
    }

    // acc: the sums of the calling wave's patch of the tile at (m0, n0), waves WGN to a row of patches
    template <typename T, int MT, int WGN, int TMI, int TNI, typename ACC>
    __device__ __forceinline__ void add_term(ACC (&acc)[TMI][TNI], int m0, int n0) {
        constexpr int KSTEP = MT == 32 ? 16 : 32, HP = std::is_same<T, f16_t>::value ? 3 : 2, BP = HP - 1;       // values that h and b are multiplied as
        args_t args = arguments();
        unsigned t = threadIdx.x;                             // (the lane's numbers are made anew, too)
        asm volatile("" : "+s"(args), "+v"(t));
        const AdapterTerm term = term_of(args);
        const int m = args->g.m, n = args->g.n;
        const int lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), fr = lane % MT, oct = lane / MT;
        const int row0 = m0 + wave / WGN * (TMI * MT), col0 = n0 + wave % WGN * (TNI * MT), row_end = row0 + TMI * MT < m ? row0 + TMI * MT : m;
        const bool whole = term.rank % 4 == 0 && ((uintptr_t)term.h & 15) == 0;
        for_segments(term.gr, row0, row_end, lane, [&](int sb, int se, int a) {
            const uint16_t* bp = (const uint16_t*)term.b + a * term.b_ws;
            for (int k0 = 0; k0 < term.rank; k0 += KSTEP) {
                const int kk = k0 + 8 * oct, left = term.rank - kk;
                // All loads first, and none behind a branch (out of range they read zeros): one round trip for them together.
                const __amdgpu_buffer_rsrc_t b_rsrc = buffer_rsrc(bp, ((long long)(term.rank - 1) * term.b_rs + (long long)(n - 1) * term.b_cs + 1) * 2);
                const __amdgpu_buffer_rsrc_t h_rsrc = buffer_rsrc(term.h + (long long)sb * term.rank, (long long)(se - sb) * term.rank * 4);
                s16x8_t bf[TNI];
                float hv[TMI][8];
#pragma unroll
                for (int i = 0; i < TMI; i++) {
                    const uint32_t at = (uint32_t)(((row0 + i * MT + fr - sb) * term.rank + kk) * 4);      // (rows before the segment wrap around, out of range)
                    if (whole) {
                        const u32x4_t p = __builtin_amdgcn_raw_buffer_load_b128(h_rsrc, (int)(left > 0 ? at : BUFFER_OOB), 0, 0);
                        const u32x4_t q = __builtin_amdgcn_raw_buffer_load_b128(h_rsrc, (int)(left > 4 ? at + 16 : BUFFER_OOB), 0, 0);
#pragma unroll
                        for (int u = 0; u < 4; u++) { hv[i][u] = __uint_as_float(p[u]); hv[i][4 + u] = __uint_as_float(q[u]); }
                    } else {
#pragma unroll
                        for (int u = 0; u < 8; u++) hv[i][u] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(h_rsrc, (int)(u < left ? at + 4 * u : BUFFER_OOB), 0, 0));
                    }
                }
                if (term.b_rs == 1 && term.rank % 8 == 0) {
#pragma unroll
                    for (int j = 0; j < TNI; j++) {
                        const int col = col0 + j * MT + fr;
                        bf[j] = __builtin_bit_cast(s16x8_t, __builtin_amdgcn_raw_buffer_load_b128(b_rsrc, (int)(col < n && left > 0 ? (uint32_t)((col * term.b_cs + kk) * 2) : BUFFER_OOB), 0, 0));
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < TNI; j++) {
                        const int col = col0 + j * MT + fr;
                        const uint32_t at = (uint32_t)((kk * term.b_rs + col * term.b_cs) * 2), step = (uint32_t)(term.b_rs * 2);
                        uint32_t x[8];
#pragma unroll
                        for (int u = 0; u < 8; u++) x[u] = __builtin_amdgcn_raw_buffer_load_b16(b_rsrc, (int)(col < n && u < left ? at + u * step : BUFFER_OOB), 0, 0);
                        u32x4_t y;
#pragma unroll
                        for (int d = 0; d < 4; d++) y[d] = x[2 * d] | x[2 * d + 1] << 16;
                        bf[j] = __builtin_bit_cast(s16x8_t, y);
                    }
                }
                // The patch's rows of other segments are zeros here: zero times an infinity or NaN of b would reach them, so that those are left to `finish`.
                uint32_t any = 0;
#pragma unroll
                for (int j = 0; j < TNI; j++) {
                    const u32x4_t v = __builtin_bit_cast(u32x4_t, bf[j]);
#pragma unroll
                    for (int d = 0; d < 4; d++) any |= not_finite<T>(v[d]);
                }
                if (__builtin_amdgcn_ballot_w64(any != 0)) {
                    odd = true;
#pragma unroll
                    for (int j = 0; j < TNI; j++) {
                        bf[j] = __builtin_bit_cast(s16x8_t, finite_only<T>(__builtin_bit_cast(u32x4_t, bf[j])));
                    }
                }
                u32x4_t hp[HP][TMI], bp16[BP][TNI];
#pragma unroll
                for (int i = 0; i < TMI; i++) parts<HP>(hv[i], [&](auto pc, u32x4_t v) { hp[decltype(pc)::value][i] = v; });
#pragma unroll
                for (int j = 0; j < TNI; j++) {
                    if constexpr (BP == 1) {
                        bp16[0][j] = __builtin_bit_cast(u32x4_t, bf[j]);
                    } else {
                        T b[8];
                        float wide[8];
                        __builtin_memcpy(b, &bf[j], 16);
#pragma unroll
                        for (int u = 0; u < 8; u++) wide[u] = widen(b[u]);
                        parts<BP>(wide, [&](auto pc, u32x4_t v) { bp16[decltype(pc)::value][j] = v; });
                    }
                }
                // (the in-place MFMAs are opaque to the compiler: what vector instructions wrote for them has to be there)
                if constexpr (MT == 16) {
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int j = 0; j < TNI; j++)
#pragma unroll
                        for (int p = 0; p < BP; p++) asm volatile("" : "+v"(bp16[p][j]) : : "memory");
#pragma unroll
                    for (int i = 0; i < TMI; i++)
#pragma unroll
                        for (int p = 0; p < HP; p++) asm volatile("" : "+v"(hp[p][i]) : : "memory");
                    asm volatile("s_nop 15" ::: "memory");
                    __builtin_amdgcn_sched_barrier(0);
                }
                static_for<0, TMI>([&](auto ic) {
                    constexpr int i = decltype(ic)::value;
                    static_for<0, HP * BP>([&](auto pc) {
                        constexpr int p = decltype(pc)::value % HP, q = decltype(pc)::value / HP;
                        if constexpr (p + q < HP) {           // (the rest is below 2^-24)
                            static_for<0, TNI>([&](auto jc) {
                                constexpr int j = decltype(jc)::value;
                                acc[i][j] = mfma16_ops<bf16_t>::mma(__builtin_bit_cast(s16x8_t, hp[p][i]), __builtin_bit_cast(s16x8_t, bp16[q][j]), acc[i][j]);
                            });
                        }
                    });
                });
            }
        });
    }

    // After the tile is stored: what h multiplies an infinity or NaN of b by is added to the rows of that segment alone
    template <typename T, int MT, int WGN, int TMI, int TNI>
    __device__ __forceinline__ void finish(int m0, int n0) {
        if (!odd) return;
        odd = false;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");           // (a wave adds to what its own lanes stored)
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        const args_t args = arguments();
        const AdapterTerm term = term_of(args);
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), m = args->g.m, n = args->g.n;
        const int row0 = m0 + wave / WGN * (TMI * MT), col0 = n0 + wave % WGN * (TNI * MT), row_end = row0 + TMI * MT < m ? row0 + TMI * MT : m, col_end = col0 + TNI * MT < n ? col0 + TNI * MT : n;
        T* y = (T*)args->g.C;
        const long long y_rs = args->g.c_rs;
        for_segments(term.gr, row0, row_end, lane, [&](int sb, int se, int a) {
            const int first = sb > row0 ? sb : row0, last = se < row_end ? se : row_end;
            for (int col = col0 + lane; col < col_end; col += 64)
            for (int r = 0; r < term.rank; r++) {
                const T b = ((const T*)term.b)[a * term.b_ws + r * term.b_rs + col * term.b_cs];
                if (!(not_finite<T>(b.bits) & 0x8000u)) continue;
                for (int row = first; row < last; row++) {
                    T* at = y + row * y_rs + col;
                    *at = round_to<T>(widen(*at) + term.h[(long long)row * term.rank + r] * widen(b));
                }
            }
        });
    }
};

template <typename T, int BM, int BN, int WGM, bool B_MC, int EDGE>
__global__ void __launch_bounds__(256, m16_blocks_per_cu(BM, BN, EDGE, 1)) adapter_tiles16_kernel(AdapterTileArgs args) {
    AdapterTiles source;
    // (one plain matrix: the options that GemmArgs has beside are known to be unused here)
    const GemmArgs g{args.g.C, args.g.A, args.g.B, args.g.bias, 1, args.g.m, args.g.k, args.g.n, 0, args.g.a_rs, 1, 0, B_MC ? args.g.b_rs : 1, B_MC ? 1 : args.g.b_cs, 0, args.g.c_rs, 1, args.g.accumulate};
    gemm_mfma16_block<T, BM, BN, WGM, false, B_MC, EDGE, false, 1, AdapterTiles>(g, args.tiles_m, args.tiles_n, nullptr, 0, args.total, (int)blockIdx.x, 0, (int)gridDim.x, &source);
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
    hipLaunchKernelGGL(kern, dim3(blocks), dim3(256), smem, current_stream(), AdapterTileArgs{g, tiles_m, tiles_n, total, term});
    return check_launch("adapter_tiles16_kernel") ? 0 : -1;
}

template <typename T, int BM, int BN, int WGM, int EDGE>
static int launch_adapter_tiles16_layout(const GroupedArgs& s, const AdapterTerm& term) {
    return s.b_cs == 1 ? launch_adapter_tiles16<T, BM, BN, WGM, true, EDGE>(s, term) : launch_adapter_tiles16<T, BM, BN, WGM, false, EDGE>(s, term);
}

}  // namespace rp
