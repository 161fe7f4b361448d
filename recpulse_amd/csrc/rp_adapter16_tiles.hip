// bf16 / fp16 shared projections with adapters on 128 x 128 and 64 x 64 tiles.
#include "rp_adapter16_tiles.h"

namespace rp {

template <typename T>
static int tiles128(const GroupedArgs& s, const AdapterTerm& term, bool edge, bool ragged) {
    if (ragged) return launch_adapter_tiles16_layout<T, 128, 128, 2, M16_RAGGED>(s, term);
    return edge ? launch_adapter_tiles16_layout<T, 128, 128, 2, M16_EDGE>(s, term) : launch_adapter_tiles16_layout<T, 128, 128, 2, M16_WHOLE>(s, term);
}

template <typename T>
static int tiles64(const GroupedArgs& s, const AdapterTerm& term, bool ragged) {
    return ragged ? launch_adapter_tiles16_layout<T, 64, 64, 2, M16_RAGGED>(s, term) : launch_adapter_tiles16_layout<T, 64, 64, 2, M16_EDGE>(s, term);
}

int launch_adapter_tiles16_128(const GroupedArgs& s, const AdapterTerm& term, bool edge, bool ragged, int dtype) {
    return dtype == RP_DTYPE_BFLOAT16 ? tiles128<bf16_t>(s, term, edge, ragged) : tiles128<f16_t>(s, term, edge, ragged);
}

int launch_adapter_tiles16_64(const GroupedArgs& s, const AdapterTerm& term, bool ragged, int dtype) {
    return dtype == RP_DTYPE_BFLOAT16 ? tiles64<bf16_t>(s, term, ragged) : tiles64<f16_t>(s, term, ragged);
}

}  // namespace rp
