// bf16 / fp16 cross entropy of a large vocabulary: dx and dW on 64 x 64 tiles.
#include "rp_vocab16.h"

namespace rp {

int launch_vocab16_grads_64(const VocabTileArgs& a, VocabStep step, bool b_mc, int edge, int dtype) {
    if (dtype == RP_DTYPE_BFLOAT16) return edge == M16_RAGGED ? launch_vocab16_grads<bf16_t, 64, 64, 2, M16_RAGGED>(a, step, b_mc) : launch_vocab16_grads<bf16_t, 64, 64, 2, M16_EDGE>(a, step, b_mc);
    return edge == M16_RAGGED ? launch_vocab16_grads<f16_t, 64, 64, 2, M16_RAGGED>(a, step, b_mc) : launch_vocab16_grads<f16_t, 64, 64, 2, M16_EDGE>(a, step, b_mc);
}

}  // namespace rp
