// The gradients of adapters' factors in a launch of their own, where dx is not asked for or goes on tiles of 256.
#include "rp_adapter16_grads.h"

namespace rp {

template <typename T, int NC, bool IN_TURN>
__global__ void __launch_bounds__(AG_THREADS) adapter_grads16_kernel(AdapterGrads ag, RowGroups gr, int first) { adapter_grads16_block<T, NC, IN_TURN>(ag, gr, first + (int)blockIdx.x); }

template <typename T, int NC, bool IN_TURN>
static int launch_grads(const AdapterGrads& ag, const RowGroups& gr) {
    constexpr int lds = AG_LDS + (IN_TURN ? NC * 16 * AG_COLS * 4 : 0);
    static_assert(lds <= 64 * 1024, "no more than every launch may have");
    return in_launches((long long)ag.a.blocks + ag.b.blocks, AG_THREADS, [&](unsigned blocks, long long first) -> int {
        hipLaunchKernelGGL((adapter_grads16_kernel<T, NC, IN_TURN>), dim3(blocks), dim3(AG_THREADS), lds, current_stream(), ag, gr, (int)first);
        return check_launch("adapter_grads16_kernel") ? 0 : -1;
    });
}

template <typename T, bool IN_TURN>
static int launch_grads_rank(const AdapterGrads& ag, const RowGroups& gr) { return grads_rank_tiles(ag.rank) == 1 ? launch_grads<T, 1, IN_TURN>(ag, gr) : launch_grads<T, 2, IN_TURN>(ag, gr); }

int launch_adapter_grads16_in_turn(const AdapterGrads& ag, const RowGroups& gr, int dtype) {
    return dtype == RP_DTYPE_BFLOAT16 ? launch_grads_rank<bf16_t, true>(ag, gr) : launch_grads_rank<f16_t, true>(ag, gr);
}

template <typename T>
static int launch_joined(AdapterGrads& ag, const RowGroups& gr, int dtype) {
    return with_joined_grads<T>(ag, gr, [&] { return launch_grads_rank<T, false>(ag, gr); }, [&] { return launch_adapter_grads16_in_turn(ag, gr, dtype); });
}

bool adapter_grad16_takes(const GroupedArgs& g, GroupedLow low) {
    const bool transposed = low == LOW_B;
    const long long s_rs = transposed ? g.a_rs : g.b_rs, s_cs = transposed ? g.a_cs : g.b_cs, l_rs = transposed ? g.b_rs : g.a_rs, l_cs = transposed ? g.b_cs : g.a_cs;
    const int width = transposed ? g.k : g.n, rank = transposed ? g.n : g.k;
    return width >= 8 && s_cs == 1 && s_rs >= width && s_rs < (1ll << 22) && l_rs == rank && (l_cs == 1 || rank == 1) && rank < (1 << 20) && !path_disabled("mfma");
}

int launch_adapter_grads16(const GroupedArgs& da, const GroupedArgs& db, int dtype) {
    AdapterGrads ag = plan_grads(da, db);
    return dtype == RP_DTYPE_BFLOAT16 ? launch_joined<bf16_t>(ag, da.gr, dtype) : launch_joined<f16_t>(ag, da.gr, dtype);
}

}  // namespace rp
