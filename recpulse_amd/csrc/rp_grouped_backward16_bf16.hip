// The gradients of a grouped layer in one launch, bf16.
#include "rp_grouped_backward16.h"

namespace rp {

int launch_grouped_backward16_bf16(const GroupedArgs& x, const GroupedArgs& w, int edge, const GroupedSums& sums, bool ragged) {
    if (edge == 128) return ragged ? launch_grouped_backward16<bf16_t, 128, M16_RAGGED>(x, w, sums) : launch_grouped_backward16<bf16_t, 128, M16_EDGE>(x, w, sums);
    return ragged ? launch_grouped_backward16<bf16_t, 64, M16_RAGGED>(x, w, sums) : launch_grouped_backward16<bf16_t, 64, M16_EDGE>(x, w, sums);
}

}  // namespace rp
