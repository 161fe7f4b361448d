// The gradients of a 16-bit layer with adapters that come after u = scale dy . B^T, in one launch: workgroups for the factors' gradients beside the tiles of dx.
#pragma once
#include "rp_adapter16_grads.h"
#include "rp_adapter16_tiles.h"

namespace rp {

// (the tiles' arguments come first: add_term reads them from where the launch left them)
template <typename T, int B, int EDGE, int NC>
__global__ void __launch_bounds__(256, 2) adapter_backward16_kernel(AdapterTileArgs args, AdapterGrads ag, int grad_blocks) {
    const int id = (int)blockIdx.x;
    if (id < grad_blocks) {
        adapter_grads16_block<T, NC>(ag, args.term.gr, id);
        return;
    }
    AdapterTiles source;
    const GemmArgs g{args.g.C, args.g.A, args.g.B, nullptr, 1, args.g.m, args.g.k, args.g.n, 0, args.g.a_rs, 1, 0, 1, args.g.b_cs, 0, args.g.c_rs, 1, args.g.accumulate};
    gemm_mfma16_block<T, B, B, 2, false, false, EDGE, false, 1, AdapterTiles>(g, args.tiles_m, args.tiles_n, nullptr, 0, args.total, id - grad_blocks, 0, args.total, &source);
}

template <typename T, int B, int EDGE, int NC>
static int launch_adapter_backward16(const GroupedArgs& s, const AdapterTerm& term, AdapterGrads& ag) {
    const int tiles_m = (s.gr.rows + B - 1) / B, tiles_n = (s.n + B - 1) / B, total = scheduled_grid(tiles_m, tiles_n);
    constexpr size_t tile = m16_smem_bytes(B, B, 2, false, false, 2, 32), smem = tile > AG_LDS ? tile : AG_LDS;
    const GemmArgs g{s.C, s.A, s.B, nullptr, 1, s.gr.rows, s.k, s.n, 0, s.a_rs, s.a_cs, 0, s.b_rs, s.b_cs, 0, s.c_rs, 1, s.accumulate};
    auto kern = adapter_backward16_kernel<T, B, EDGE, NC>;
    if (smem > 64 * 1024 && !check_hip(hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)smem), "hipFuncSetAttribute")) return -1;
    auto apart = [&]() -> int {
        const int dtype = traits<T>::code;
        if ((B == 128 ? launch_adapter_tiles16_128(s, term, true, EDGE == M16_RAGGED, dtype) : launch_adapter_tiles16_64(s, term, EDGE == M16_RAGGED, dtype)) != 0) return -1;
        return launch_adapter_grads16_in_turn(ag, term.gr, dtype);
    };
    if ((long long)ag.a.blocks + ag.b.blocks + total > (1 << 23)) return apart();              // (more than a launch takes, or near it: the shares are few then)
    return with_joined_grads<T>(ag, term.gr, [&]() -> int {
        const int grad_blocks = (ag.a.blocks + ag.b.blocks + 7) / 8 * 8;        // (the tiles' schedule goes by workgroup modulo 8)
        hipLaunchKernelGGL(kern, dim3((unsigned)(grad_blocks + total)), dim3(256), smem, current_stream(), AdapterTileArgs{g, tiles_m, tiles_n, total, term}, ag, grad_blocks);
        return check_launch("adapter_backward16_kernel") ? 0 : -1;
    }, apart);
}

template <typename T, int B, int EDGE>
static int launch_adapter_backward16_rank(const GroupedArgs& s, const AdapterTerm& term, AdapterGrads& ag) {
    return grads_rank_tiles(ag.rank) == 1 ? launch_adapter_backward16<T, B, EDGE, 1>(s, term, ag) : launch_adapter_backward16<T, B, EDGE, 2>(s, term, ag);
}

template <typename T>
static int launch_adapter_backward16_tile(const GroupedArgs& s, const AdapterTerm& term, const GroupedArgs& da, const GroupedArgs& db, int tile, bool ragged) {
    AdapterGrads ag = plan_grads(da, db);
    if (tile == 128) return ragged ? launch_adapter_backward16_rank<T, 128, M16_RAGGED>(s, term, ag) : launch_adapter_backward16_rank<T, 128, M16_EDGE>(s, term, ag);
    return ragged ? launch_adapter_backward16_rank<T, 64, M16_RAGGED>(s, term, ag) : launch_adapter_backward16_rank<T, 64, M16_EDGE>(s, term, ag);
}

}  // namespace rp
