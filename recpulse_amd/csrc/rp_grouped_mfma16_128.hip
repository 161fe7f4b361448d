// Grouped bf16 / fp16 products on 128 x 128 tiles.
#include "rp_grouped_mfma16.h"

namespace rp {

template <typename T>
static int rows(const GroupedArgs& g, bool ragged) {
    return ragged ? launch_grouped_rows16_layout<T, 128, 128, 2, M16_RAGGED>(g) : launch_grouped_rows16_layout<T, 128, 128, 2, M16_EDGE>(g);
}

template <typename T>
static int weights(const GroupedArgs& g, bool ragged) {
    return ragged ? launch_grouped_weights16<T, 128, 128, 2, M16_RAGGED>(g) : launch_grouped_weights16<T, 128, 128, 2, M16_EDGE>(g);
}

int launch_grouped_rows16_128(const GroupedArgs& g, bool ragged, int dtype) { return dtype == RP_DTYPE_BFLOAT16 ? rows<bf16_t>(g, ragged) : rows<f16_t>(g, ragged); }
int launch_grouped_weights16_128(const GroupedArgs& g, bool ragged, int dtype) { return dtype == RP_DTYPE_BFLOAT16 ? weights<bf16_t>(g, ragged) : weights<f16_t>(g, ragged); }

}  // namespace rp
