// Grouped products of bf16 / fp16 on the tiles of the 16-bit MFMA kernel: the same workgroups as one product's (gemm_mfma16_block),
// which take their tiles from the groups instead of from one matrix.  Bound as those are: large tiles by power (16384 rows of 16 groups, 4096 x 4096 in bf16: forward
// 557 us, dx 548, 1.0 PFLOP/s; dw 584, 16 slabs a tile and 537 MB of output), small ones by the chain of their slabs.
#pragma once
#include "rp_gemm_mfma16_kernel.h"
#include "rp_grouped.h"

namespace rp {

// By rows: row tiles never span two groups, and how many there are is known on the device only.  All groups' tiles are one list, group by group.
template <int BM>
struct GroupedRowTiles : M16Source {
    static constexpr bool MOVES = true, ONCE = true, TERM = false;
    GroupedArgs ga;
    RowTiles rows;
    int tiles_n, total;
    __device__ __forceinline__ GroupedRowTiles(const GroupedArgs& g, int tn) : ga(g), rows(g.gr, BM), tiles_n(tn), total(rows.total * tn) {}
    __device__ __forceinline__ int slots() const { return (total + 7) / 8 * 8; }
    __device__ __forceinline__ TileCoord tile(int id, GemmArgs& g) const {
        const int at = run_tile(id, total);
        if (at == total) return TileCoord{0, 0, false};
        const int row = at / tiles_n;
        const RowTile rt = rows.find(row);
        const TileCoord in = chunk_tile(at - rt.first * tiles_n, rt.tiles, tiles_n);
        const int begin = rt.begin + (in.tm - (row - rt.first)) * BM;
        g.A = (const uint16_t*)ga.A + begin * ga.a_rs;
        g.B = (const uint16_t*)ga.B + rt.weight * ga.b_ws;
        g.C = (uint16_t*)ga.C + begin * ga.c_rs;
        g.bias = ga.bias ? (const uint16_t*)ga.bias + (long long)rt.weight * ga.n : nullptr;
        g.m = begin + BM < rt.stop ? BM : rt.stop - begin;
        return TileCoord{0, in.tn, true};
    }
};

template <typename T, int BM, int BN, int WGM, bool B_MC, int EDGE>
__global__ void __launch_bounds__(256, m16_blocks_per_cu(BM, BN, EDGE, 1)) grouped_rows16_kernel(GroupedArgs ga, int tiles_n) {
    GroupedRowTiles<BM> source(ga, tiles_n);
    GemmArgs g{nullptr, nullptr, nullptr, nullptr, 1, 0, ga.k, ga.n, 0, ga.a_rs, ga.a_cs, 0, ga.b_rs, ga.b_cs, 0, ga.c_rs, 1, ga.accumulate};
    gemm_mfma16_block<T, BM, BN, WGM, false, B_MC, EDGE, false, 1, GroupedRowTiles<BM>>(g, 0, 0, nullptr, 0, source.slots(), (int)blockIdx.x, 0,
                                                                                       (int)gridDim.x, &source);
}

// By weights: tile for tile the same in every group, each group's tiles a run for each XCD, so that resident workgroups, each with one tile
// of every group in turn, all do the same work however uneven the groups are.  The reduction runs over the group's rows; an empty group leaves zeros.
struct GroupedWeightTiles : M16Source {
    static constexpr bool MOVES = true, ONCE = true, TERM = false;
    GroupedArgs ga;
    int tiles_k, tiles_n, slots;
    __device__ __forceinline__ TileCoord tile(int id, GemmArgs& g) const {
        const int w = id / slots;
        const int at = run_tile(id - w * slots, tiles_k * tiles_n);
        if (at == tiles_k * tiles_n) return TileCoord{0, 0, false};
        const int b = __builtin_amdgcn_readfirstlane(ga.gr.begin(w)), e = __builtin_amdgcn_readfirstlane(ga.gr.end(w));
        g.A = (const uint16_t*)ga.A + b * ga.a_rs;
        g.B = (const uint16_t*)ga.B + b * ga.b_rs;
        g.C = (uint16_t*)ga.C + w * ga.c_ws;
        g.k = e - b;
        return chunk_tile(at, tiles_k, tiles_n);
    }
};

template <typename T, int BM, int BN, int WGM, int EDGE>
__global__ void __launch_bounds__(256, m16_blocks_per_cu(BM, BN, EDGE, 1)) grouped_weights16_kernel(GroupedArgs ga, int tiles_k, int tiles_n, int slots, int total) {
    GroupedWeightTiles source{{}, ga, tiles_k, tiles_n, slots};
    GemmArgs g{nullptr, nullptr, nullptr, nullptr, 1, ga.k, 0, ga.n, 0, ga.a_cs, ga.a_rs, 0, ga.b_rs, ga.b_cs, 0, ga.c_rs, 1, ga.accumulate};
    gemm_mfma16_block<T, BM, BN, WGM, true, true, EDGE, false, 1, GroupedWeightTiles>(g, 0, 0, nullptr, 0, total, (int)blockIdx.x, 0, (int)gridDim.x, &source);
}

// A workgroup a tile, except for the 256 x 256 tile: one resident workgroup a CU, as for one product.
template <int BM, int BN>
static unsigned grouped16_blocks(long long tiles) {
    const long long most = BM == 256 && BN == 256 && device_cu_count() >= 8 ? device_cu_count() / 8 * 8 : (1 << 24) - 8;      // (fewer than 2^32 threads)
    tiles = (tiles + 7) / 8 * 8;
    return (unsigned)(tiles < most ? tiles : most);
}

template <typename T, int BM, int BN, int WGM, bool B_MC, int EDGE>
static int launch_grouped_rows16(const GroupedArgs& g) {
    const int tiles_n = (g.n + BN - 1) / BN;
    const long long tiles = max_row_tiles(g.gr.rows, g.gr.groups, BM) * tiles_n;
    if (tiles > 0x3fffffff) { set_error("grouped product: %lld tiles are more than a launch takes", tiles); return -1; }
    constexpr size_t smem = m16_smem_bytes(BM, BN, WGM, false, B_MC, 2, m16_mfma_tile(BM, BN));
    auto kern = grouped_rows16_kernel<T, BM, BN, WGM, B_MC, EDGE>;
    if (smem > 64 * 1024 && !check_hip(hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)smem), "hipFuncSetAttribute")) return -1;
    hipLaunchKernelGGL(kern, dim3(grouped16_blocks<BM, BN>(tiles)), dim3(256), smem, current_stream(), g, tiles_n);
    return check_launch("grouped_rows16_kernel") ? 0 : -1;
}

template <typename T, int BM, int BN, int WGM, int EDGE>
static int launch_grouped_weights16(const GroupedArgs& g) {
    const int tiles_k = (g.k + BM - 1) / BM, tiles_n = (g.n + BN - 1) / BN, slots = (int)(((long long)tiles_k * tiles_n + 7) / 8 * 8);
    const long long total = (long long)slots * g.gr.weights;
    if (total > 0x3fffffff) { set_error("grouped weight gradient: %lld tiles are more than a launch takes", total); return -1; }
    constexpr size_t smem = m16_smem_bytes(BM, BN, WGM, true, true, 2, m16_mfma_tile(BM, BN));
    auto kern = grouped_weights16_kernel<T, BM, BN, WGM, EDGE>;
    if (smem > 64 * 1024 && !check_hip(hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)smem), "hipFuncSetAttribute")) return -1;
    hipLaunchKernelGGL(kern, dim3(grouped16_blocks<BM, BN>(total)), dim3(256), smem, current_stream(), g, tiles_k, tiles_n, slots, (int)total);
    return check_launch("grouped_weights16_kernel") ? 0 : -1;
}

template <typename T, int BM, int BN, int WGM, int EDGE>
static int launch_grouped_rows16_layout(const GroupedArgs& g) {
    return g.b_cs == 1 ? launch_grouped_rows16<T, BM, BN, WGM, true, EDGE>(g) : launch_grouped_rows16<T, BM, BN, WGM, false, EDGE>(g);
}

}  // namespace rp
