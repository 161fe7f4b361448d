// f16 shared projections with adapters on 256 x 256 tiles.
#include "rp_adapter16_tiles.h"

namespace rp {

int launch_adapter_tiles16_256_f16(const GroupedArgs& s, const AdapterTerm& term, bool edge) {
    return edge ? launch_adapter_tiles16_layout<f16_t, 256, 256, 2, M16_EDGE>(s, term) : launch_adapter_tiles16_layout<f16_t, 256, 256, 2, M16_WHOLE>(s, term);
}

}  // namespace rp
