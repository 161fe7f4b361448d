// The gradients of a grouped layer in one launch, fp16.
#include "rp_grouped_backward16.h"

namespace rp {

int launch_grouped_backward16_f16(const GroupedArgs& x, int x_tile, const GroupedArgs& w, int w_tile, const GroupedSums& sums, bool ragged) {
    return ragged ? launch_grouped_backward16_tiles<f16_t, M16_RAGGED>(x, x_tile, w, w_tile, sums) : launch_grouped_backward16_tiles<f16_t, M16_EDGE>(x, x_tile, w, w_tile, sums);
}

}  // namespace rp
