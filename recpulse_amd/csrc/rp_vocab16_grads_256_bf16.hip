// bf16 cross entropy of a large vocabulary: dx and dW on 256 x 256 tiles.
#include "rp_vocab16.h"

namespace rp {

int launch_vocab16_grads_256_bf16(const VocabTileArgs& a, VocabStep step, bool b_mc, int edge) {
    return edge == M16_WHOLE ? launch_vocab16_grads<bf16_t, 256, 256, 2, M16_WHOLE>(a, step, b_mc) : launch_vocab16_grads<bf16_t, 256, 256, 2, M16_EDGE>(a, step, b_mc);
}

}  // namespace rp
