// The gradients of adapters' factors in a launch of their own, where dx is not asked for or goes on tiles of 256.
#include "rp_adapter16_grads.h"

namespace rp {

template <typename T, int NC>
__global__ void __launch_bounds__(AG_THREADS) adapter_grads16_kernel(AdapterGrads ag, RowGroups gr) { adapter_grads16_block<T, NC>(ag, gr, (int)blockIdx.x); }

template <typename T, int NC>
static int launch_grads(AdapterGrads& ag, const RowGroups& gr) {
    return with_joined_grads<T>(ag, gr, [&]() -> int {
        hipLaunchKernelGGL((adapter_grads16_kernel<T, NC>), dim3((unsigned)(ag.a.blocks + ag.b.blocks)), dim3(AG_THREADS), AG_LDS, current_stream(), ag, gr);
        return check_launch("adapter_grads16_kernel") ? 0 : -1;
    });
}

bool adapter_grad16_takes(const GroupedArgs& g, GroupedLow low) {
    const bool transposed = low == LOW_B;
    const long long s_rs = transposed ? g.a_rs : g.b_rs, s_cs = transposed ? g.a_cs : g.b_cs, l_rs = transposed ? g.b_rs : g.a_rs, l_cs = transposed ? g.b_cs : g.a_cs;
    const int width = transposed ? g.k : g.n, rank = transposed ? g.n : g.k;
    return width >= 8 && s_cs == 1 && s_rs >= width && s_rs < (1ll << 22) && l_rs == rank && (l_cs == 1 || rank == 1) && rank < (1 << 20) && !path_disabled("mfma");
}

int launch_adapter_grads16(const GroupedArgs& da, const GroupedArgs& db, int dtype) {
    AdapterGrads ag;
    if (!plan_grads(da, db, ag)) return -1;
    const bool one = grads_rank_tiles(ag.rank) == 1;
    if (dtype == RP_DTYPE_BFLOAT16) return one ? launch_grads<bf16_t, 1>(ag, da.gr) : launch_grads<bf16_t, 2>(ag, da.gr);
    return one ? launch_grads<f16_t, 1>(ag, da.gr) : launch_grads<f16_t, 2>(ag, da.gr);
}

}  // namespace rp
