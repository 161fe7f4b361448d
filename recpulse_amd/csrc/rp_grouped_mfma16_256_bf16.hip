// Grouped bf16 products on 256 x 256 tiles (a unit of its own: one takes a minute to compile).
#include "rp_grouped_mfma16.h"

namespace rp {

int launch_grouped_rows16_256_bf16(const GroupedArgs& g) { return launch_grouped_rows16_layout<bf16_t, 256, 256, 2, M16_EDGE>(g); }
int launch_grouped_weights16_256_bf16(const GroupedArgs& g) { return launch_grouped_weights16<bf16_t, 256, 256, 2, M16_EDGE>(g); }

}  // namespace rp
