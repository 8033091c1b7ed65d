// Log probabilities and the distillation loss on the HIP library.
#include <motifcl/ops/loss.hpp>

#include <string>

#include <motifcl/runtime/backend.hpp>

#include "rows.hpp"

namespace motifcl {
namespace {

Shape with(Shape lead, int64_t last) {
    lead.dims.push_back(last);
    return lead;
}

}  // namespace

TokenLogProbs token_log_probs(const Tensor& logits, const Tensor& tokens, int top, float temperature) {
    const int element = rows::element_of(logits, "token_log_probs");
    const Shape lead = rows::leading(logits, "token_log_probs");
    rows::check_numbers(tokens, logits, DType::I32, lead, "token_log_probs tokens");
    MCL_CHECK(top >= 0 && top <= MCC_MOST_TOP, "token_log_probs gives at most 128 alternatives");
    Backend& backend = logits.backend();
    const std::size_t n = static_cast<std::size_t>(lead.numel()), vocab = rows::length(logits);
    TokenLogProbs r;
    r.log_prob = Tensor::empty(backend, lead);
    r.entropy = Tensor::empty(backend, lead);
    r.lse = Tensor::empty(backend, lead);
    if (top > 0) {
        r.top_ids = Tensor::empty(backend, with(lead, top), DType::I32);
        r.top_log_probs = Tensor::empty(backend, with(lead, top));
    }
    const std::size_t k = static_cast<std::size_t>(top);
    const std::size_t ws = mcc_token_log_probs_workspace_nbytes(n, vocab, k, element);
    const int rc = mcc_token_log_probs(
        backend.hip_stream(), logits.data(), logits.nbytes(), vocab, static_cast<const std::int32_t*>(tokens.data()),
        tokens.nbytes(), rows::f32(r.log_prob), r.log_prob.nbytes(), rows::f32(r.entropy), r.entropy.nbytes(),
        rows::f32(r.lse), r.lse.nbytes(), top ? static_cast<std::int32_t*>(r.top_ids.data()) : nullptr, 4 * n * k,
        top ? rows::f32(r.top_log_probs) : nullptr, 4 * n * k, ws ? backend.workspace(ws) : nullptr, ws, n, vocab, k,
        element, temperature);
    MCL_CHECK(rc == MCC_OK, std::string("hip token_log_probs failed: ") + mcc_last_error());
    return r;
}

Tensor token_log_probs_backward(const Tensor& logits, const Tensor& tokens, const TokenLogProbs& forward,
                                const Tensor& grad_log_prob, const Tensor* grad_entropy, float temperature) {
    const int element = rows::element_of(logits, "token_log_probs_backward");
    const Shape lead = rows::leading(logits, "token_log_probs_backward");
    rows::check_numbers(tokens, logits, DType::I32, lead, "token_log_probs_backward tokens");
    rows::check_numbers(forward.lse, logits, DType::F32, lead, "token_log_probs_backward lse");
    rows::check_numbers(forward.entropy, logits, DType::F32, lead, "token_log_probs_backward entropy");
    rows::check_numbers(grad_log_prob, logits, DType::F32, lead, "token_log_probs_backward grad_log_prob");
    if (grad_entropy)
        rows::check_numbers(*grad_entropy, logits, DType::F32, lead, "token_log_probs_backward grad_entropy");
    Backend& backend = logits.backend();
    const std::size_t n = static_cast<std::size_t>(lead.numel()), vocab = rows::length(logits);
    Tensor grad = Tensor::empty(backend, logits.shape(), logits.dtype());
    const int rc = mcc_token_log_probs_backward(
        backend.hip_stream(), logits.data(), logits.nbytes(), vocab, static_cast<const std::int32_t*>(tokens.data()),
        tokens.nbytes(), rows::f32(forward.lse), forward.lse.nbytes(), rows::f32(forward.entropy), forward.entropy.nbytes(),
        rows::f32(grad_log_prob), grad_log_prob.nbytes(), grad_entropy ? rows::f32(*grad_entropy) : nullptr,
        grad_entropy ? grad_entropy->nbytes() : 0, grad.data(), grad.nbytes(), vocab, n, vocab, element, temperature);
    MCL_CHECK(rc == MCC_OK, std::string("hip token_log_probs_backward failed: ") + mcc_last_error());
    return grad;
}

DistillTop distill_top(const Tensor& logits, const Tensor& teacher_ids, const Tensor& teacher_logits, float temperature,
                       const Tensor* weight) {
    const int element = rows::element_of(logits, "distill_top");
    const Shape lead = rows::leading(logits, "distill_top");
    MCL_CHECK(teacher_ids.ndim() >= 1, "distill_top teacher_ids requires at least one dimension");
    const std::size_t k = rows::length(teacher_ids);
    rows::check_numbers(teacher_ids, logits, DType::I32, with(lead, teacher_ids.shape()[-1]), "distill_top teacher_ids");
    rows::check_numbers(teacher_logits, logits, DType::F32, teacher_ids.shape(), "distill_top teacher_logits");
    if (weight) rows::check_numbers(*weight, logits, DType::F32, lead, "distill_top weight");
    Backend& backend = logits.backend();
    const std::size_t n = static_cast<std::size_t>(lead.numel()), vocab = rows::length(logits);
    DistillTop r;
    r.loss = Tensor::empty(backend, lead);
    r.grad_logits = Tensor::empty(backend, logits.shape(), logits.dtype());
    const int rc = mcc_distill_top(
        backend.hip_stream(), logits.data(), logits.nbytes(), vocab, static_cast<const std::int32_t*>(teacher_ids.data()),
        teacher_ids.nbytes(), rows::f32(teacher_logits), teacher_logits.nbytes(), weight ? rows::f32(*weight) : nullptr,
        weight ? weight->nbytes() : 0, rows::f32(r.loss), r.loss.nbytes(), r.grad_logits.data(), r.grad_logits.nbytes(),
        vocab, n, vocab, k, element, temperature);
    MCL_CHECK(rc == MCC_OK, std::string("hip distill_top failed: ") + mcc_last_error());
    return r;
}

}  // namespace motifcl
