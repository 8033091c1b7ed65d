// What stands behind the vocabulary head: log probabilities of given tokens and the distillation loss.
// Both give the gradient of the logits to the caller, which starts the backward pass with it:
//
//     DistillTop d = distill_top(logits, teacher.top_ids, teacher.top_log_probs, 2.0f, &weight);
//     logits.backward(d.grad_logits);
//
// logits are [..., vocab], f32 or f16; the results have the leading dimensions.  See motifcl_amd.h for the
// definitions, also of masked and empty rows.
#pragma once

#include <motifcl/tensor/tensor.hpp>

namespace motifcl {

struct TokenLogProbs {
    Tensor log_prob, entropy, lse;  // F32 [...]
    Tensor top_ids, top_log_probs;  // I32, F32 [..., top]; invalid without alternatives
};
// tokens: I32 [...], outside [0, vocab) for an ignored position
TokenLogProbs token_log_probs(const Tensor& logits, const Tensor& tokens, int top = 0, float temperature = 1.0f);

// Gradient of the logits for the gradients of log_prob and, if not null, of entropy (F32 [...]).
Tensor token_log_probs_backward(const Tensor& logits, const Tensor& tokens, const TokenLogProbs& forward,
                                const Tensor& grad_log_prob, const Tensor* grad_entropy = nullptr, float temperature = 1.0f);

struct DistillTop {
    Tensor loss;         // F32 [...]: temperature^2 KL(teacher || student) of each row
    Tensor grad_logits;  // gradient of the weighted sum of the losses
};
// teacher_ids I32 and teacher_logits F32 [..., entries]; weight F32 [...] or null
DistillTop distill_top(const Tensor& logits, const Tensor& teacher_ids, const Tensor& teacher_logits,
                       float temperature = 1.0f, const Tensor* weight = nullptr);

}  // namespace motifcl
