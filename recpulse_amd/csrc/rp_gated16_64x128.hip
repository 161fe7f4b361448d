// bf16 / fp16 gated linear layer on 64 x 128 tiles: 64 rows, 64 columns of each half of W.
#include "rp_gated16.h"

namespace rp {

int launch_gated16_64x128(const GatedArgs& l, const GatedShares& shares, int edge, int dtype) {
    if (dtype == RP_DTYPE_BFLOAT16) return edge == M16_RAGGED ? launch_gated16<bf16_t, 64, 128, 2, M16_RAGGED>(l, shares) : launch_gated16<bf16_t, 64, 128, 2, M16_EDGE>(l, shares);
    return edge == M16_RAGGED ? launch_gated16<f16_t, 64, 128, 2, M16_RAGGED>(l, shares) : launch_gated16<f16_t, 64, 128, 2, M16_EDGE>(l, shares);
}

}  // namespace rp
