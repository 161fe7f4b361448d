// Cross entropy of a large vocabulary straight from the rows before it: z = x . W + b, loss_i = log sum_v exp(z_iv) - z_it.
#pragma once
#include "rp_grouped.h"
#include "rp_teams.h"

namespace rp {

struct VocabArgs {
    const void *x, *w, *bias;
    const int* targets;
    int rows, k, classes, reduction;
    long long x_rs, x_cs, w_rs, w_cs;
};
struct VocabGrads {
    void *dx, *dw, *db;
    long long dx_rs, dw_rs, dw_cs;
    int accumulate_dx, accumulate_dw, accumulate_db;
};

// A workspace in pieces of whole 256 bytes: counted with a null base, handed out with the caller's
class VocabRoom {
public:
    explicit VocabRoom(void* base) : base_((char*)base) {}
    template <typename P> P* take(long long count) {
        P* at = (P*)(base_ + used_);
        used_ += (count * (long long)sizeof(P) + 255) / 256 * 256;
        return at;
    }
    long long used() const { return used_; }
private:
    char* base_;
    long long used_ = 0;
};

// The result from the rows' losses in stats, and how many rows have a target (rp_vocab.hip)
int vocab_result_f32(float* loss_out, float* stats, const VocabArgs& g);
// bf16 / fp16 on MFMA tiles (rp_vocab16.hip): operands with a unit stride and rows of at least a 16-byte vector
bool vocab16_takes(const VocabArgs& g, int dtype);
long long vocab16_room(int rows, int k, int classes, bool backward);      // bytes of its workspace
int vocab16_forward(float* loss_out, float* stats, const VocabArgs& g, void* workspace, int dtype);
int vocab16_backward(const VocabGrads& o, const VocabArgs& g, const float* stats, const float* upstream, void* workspace, int dtype);

}  // namespace rp
