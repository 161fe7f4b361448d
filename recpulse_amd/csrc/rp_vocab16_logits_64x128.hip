// bf16 / fp16 cross entropy of a large vocabulary: logits on 64 x 128 tiles.
#include "rp_vocab16.h"

namespace rp {

int launch_vocab16_logits_64x128(const VocabTileArgs& a, VocabStep step, bool b_mc, int edge, int dtype) {
    if (dtype == RP_DTYPE_BFLOAT16) return edge == M16_RAGGED ? launch_vocab16_logits<bf16_t, 64, 128, 2, M16_RAGGED>(a, step, b_mc) : launch_vocab16_logits<bf16_t, 64, 128, 2, M16_EDGE>(a, step, b_mc);
    return edge == M16_RAGGED ? launch_vocab16_logits<f16_t, 64, 128, 2, M16_RAGGED>(a, step, b_mc) : launch_vocab16_logits<f16_t, 64, 128, 2, M16_EDGE>(a, step, b_mc);
}

}  // namespace rp
