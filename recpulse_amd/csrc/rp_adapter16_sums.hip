// A shared projection as float32 sums on 128 x 128 tiles, for layers whose adapters' term is added by a launch of its own.
#include "rp_gemm_mfma16_kernel.h"
#include "rp_grouped.h"

namespace rp {

template <typename T, int EDGE>
static int sums128(const GemmArgs& g, bool b_mc, float* sums) {
    const int k_per_split = (g.k + M16_BK - 1) / M16_BK * M16_BK;
    return b_mc ? m16_launch<T, 128, 128, 2, false, true, EDGE, true>(g, sums, 1, k_per_split) : m16_launch<T, 128, 128, 2, false, false, EDGE, true>(g, sums, 1, k_per_split);
}

int launch_sums16_128(const GemmArgs& g, bool b_mc, bool ragged, float* sums, int dtype) {
    if (dtype == RP_DTYPE_BFLOAT16) return ragged ? sums128<bf16_t, M16_RAGGED>(g, b_mc, sums) : sums128<bf16_t, M16_EDGE>(g, b_mc, sums);
    return ragged ? sums128<f16_t, M16_RAGGED>(g, b_mc, sums) : sums128<f16_t, M16_EDGE>(g, b_mc, sums);
}

}  // namespace rp
