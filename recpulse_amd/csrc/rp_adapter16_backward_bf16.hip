// The gradients of a layer with adapters in one launch, bf16.
#include "rp_adapter16_backward.h"

namespace rp {

int launch_adapter_backward16_bf16(const GroupedArgs& shared, const AdapterTerm& term, const GroupedArgs& da, const GroupedArgs& db, int tile, bool ragged) {
    return launch_adapter_backward16_tile<bf16_t>(shared, term, da, db, tile, ragged);
}

}  // namespace rp
