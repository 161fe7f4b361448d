// bf16 gated linear layer on 256 x 256 tiles: 256 rows, 128 columns of each half of W.
#include "rp_gated16.h"

namespace rp {

int launch_gated16_256_bf16(const GatedArgs& l, int edge) { return edge == M16_WHOLE ? launch_gated16<bf16_t, 256, 256, 2, M16_WHOLE>(l) : launch_gated16<bf16_t, 256, 256, 2, M16_EDGE>(l); }

}  // namespace rp
