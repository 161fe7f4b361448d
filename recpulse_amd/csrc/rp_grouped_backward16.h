// The three gradients of a grouped layer of bf16 / fp16 in one launch: workgroups for the columns' sums, for the tiles of the input's gradient and for
// those of the weights'.  Each of them alone leaves a small layer waiting for its loads, with a workgroup or two on a CU.
#pragma once
#include "rp_grouped_mfma16.h"
#include "rp_grouped_sums.h"

namespace rp {

struct BackwardGrid { int x_blocks, w_blocks, s_blocks, x_tiles_n, w_tiles_k, w_tiles_n, w_slots, w_total; };

template <typename T, int BX, int BW, int EDGE>
__global__ void __launch_bounds__(256, 2) grouped_backward16_kernel(GroupedArgs x, GroupedArgs w, GroupedSums sums, BackwardGrid bg) {
    extern __shared__ __attribute__((aligned(16))) uint16_t smem[];
    int id = (int)blockIdx.x;
    if (id < bg.s_blocks) {
        if (id < sums.gr.weights * ((sums.cols + 63) / 64)) grouped_sums_block<T, 4>(sums, id, (float*)smem);
        return;
    }
    id -= bg.s_blocks;
    if (id < bg.x_blocks) {
        GroupedRowTiles<BX> source(x, bg.x_tiles_n);
        GemmArgs g{nullptr, nullptr, nullptr, nullptr, 1, 0, x.k, x.n, 0, x.a_rs, x.a_cs, 0, x.b_rs, x.b_cs, 0, x.c_rs, 1, x.accumulate};
        gemm_mfma16_block<T, BX, BX, 2, false, false, EDGE, false, 1, GroupedRowTiles<BX>>(g, 0, 0, nullptr, 0, source.slots(), id, 0, bg.x_blocks, &source);
        return;
    }
    id -= bg.x_blocks;
    GroupedWeightTiles source{w, bg.w_tiles_k, bg.w_tiles_n, bg.w_slots};
    GemmArgs g{nullptr, nullptr, nullptr, nullptr, 1, w.k, 0, w.n, 0, w.a_cs, w.a_rs, 0, w.b_rs, w.b_cs, 0, w.c_rs, 1, w.accumulate};
    gemm_mfma16_block<T, BW, BW, 2, true, true, EDGE, false, 1, GroupedWeightTiles>(g, 0, 0, nullptr, 0, bg.w_total, id, 0, bg.w_blocks, &source);
}

template <typename T, int BX, int BW, int EDGE>
static int launch_grouped_backward16(const GroupedArgs& x, const GroupedArgs& w, const GroupedSums& sums) {
    constexpr size_t smem_x = m16_smem_bytes(BX, BX, 2, false, false, 2, 32), smem_w = m16_smem_bytes(BW, BW, 2, true, true, 2, 32), smem = smem_x > smem_w ? smem_x : smem_w;
    BackwardGrid bg;
    bg.x_tiles_n = (x.n + BX - 1) / BX;
    bg.w_tiles_k = (w.k + BW - 1) / BW;
    bg.w_tiles_n = (w.n + BW - 1) / BW;
    const long long slots = ((long long)bg.w_tiles_k * bg.w_tiles_n + 7) / 8 * 8, total = w.C ? slots * w.gr.weights : 0;
    const long long x_tiles = x.C ? max_row_tiles(x.gr.rows, x.gr.groups, BX) * bg.x_tiles_n : 0, s_blocks = sums.out ? sum_blocks(sums) : 0;
    if (total + x_tiles + s_blocks > GROUPED_BACKWARD16_MOST) { set_error("grouped backward: more tiles than a launch takes"); return -1; }
    bg.w_slots = (int)slots;
    bg.w_total = bg.w_blocks = (int)total;
    bg.x_blocks = (int)((x_tiles + 7) / 8 * 8);
    bg.s_blocks = (int)((s_blocks + 7) / 8 * 8);
    auto kern = grouped_backward16_kernel<T, BX, BW, EDGE>;
    if (smem > 64 * 1024 && !check_hip(hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)smem), "hipFuncSetAttribute")) return -1;
    hipLaunchKernelGGL(kern, dim3((unsigned)(bg.s_blocks + bg.x_blocks + bg.w_blocks)), dim3(256), smem, current_stream(), x, w, sums, bg);
    return check_launch("grouped_backward16_kernel") ? 0 : -1;
}

template <typename T, int EDGE>
static int launch_grouped_backward16_tiles(const GroupedArgs& x, int x_tile, const GroupedArgs& w, int w_tile, const GroupedSums& sums) {
    if (x_tile == 64) return launch_grouped_backward16<T, 64, 64, EDGE>(x, w, sums);
    return w_tile == 64 ? launch_grouped_backward16<T, 128, 64, EDGE>(x, w, sums) : launch_grouped_backward16<T, 128, 128, EDGE>(x, w, sums);
}

}  // namespace rp
