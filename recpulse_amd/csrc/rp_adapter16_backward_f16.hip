// The gradients of a layer with adapters in one launch, fp16.
#include "rp_adapter16_backward.h"

namespace rp {

int launch_adapter_backward16_f16(const GroupedArgs& shared, const AdapterTerm& term, const GroupedArgs& da, const GroupedArgs& db, int tile, bool ragged) {
    return launch_adapter_backward16_tile<f16_t>(shared, term, da, db, tile, ragged);
}

}  // namespace rp
