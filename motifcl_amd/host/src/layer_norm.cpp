// nn::LayerNorm on the HIP library.
#include <motifcl/nn/layer_norm.hpp>

#include <memory>
#include <string>
#include <utility>
#include <vector>

#include <motifcl/autograd/node.hpp>

#include "rows.hpp"

namespace motifcl::nn {
namespace {

// The gain the forward pass used is kept as a handle: the parameters are updated after the backward pass.
struct LayerNormBackwardNode : autograd::Node {
    LayerNormBackwardNode(Tensor input, Tensor gain, Tensor bias, Tensor mean, Tensor rstd)
        : input_(std::move(input)), gain_(std::move(gain)), bias_(std::move(bias)), mean_(std::move(mean)),
          rstd_(std::move(rstd)) {}

    std::vector<Tensor> inputs() const override { return {input_, gain_, bias_}; }

    void backward(const Tensor& grad_out) override {
        MCL_CHECK(grad_out.dtype() == input_.dtype() && grad_out.backend_ptr() == input_.backend_ptr(),
                  "LayerNorm backward expects a gradient of the output's type on its backend");
        Backend& backend = input_.backend();
        const std::size_t cols = rows::length(input_), n = static_cast<std::size_t>(mean_.numel());
        const int element = rows::element_of(input_, "LayerNorm");
        Tensor grad_input, grad_gain, grad_bias;
        if (input_.requires_grad()) grad_input = Tensor::empty(backend, input_.shape(), input_.dtype());
        if (gain_.requires_grad()) grad_gain = Tensor::empty(backend, gain_.shape());
        if (bias_.requires_grad()) grad_bias = Tensor::empty(backend, bias_.shape());
        if (!grad_input.valid() && !grad_gain.valid() && !grad_bias.valid()) return;
        const std::size_t ws = mcc_layer_norm_backward_workspace_nbytes(n, cols, element);
        const int rc = mcc_layer_norm_backward(
            backend.hip_stream(), grad_out.data(), grad_out.nbytes(), cols, input_.data(), input_.nbytes(), cols,
            rows::f32(mean_), mean_.nbytes(), rows::f32(rstd_), rstd_.nbytes(), rows::f32(gain_), gain_.nbytes(),
            grad_input.valid() ? grad_input.data() : nullptr, grad_input.valid() ? grad_input.nbytes() : 0, cols,
            grad_gain.valid() ? rows::f32(grad_gain) : nullptr, gain_.nbytes(),
            grad_bias.valid() ? rows::f32(grad_bias) : nullptr, bias_.nbytes(), ws ? backend.workspace(ws) : nullptr, ws, n,
            cols, element);
        MCL_CHECK(rc == MCC_OK, std::string("hip layer_norm backward failed: ") + mcc_last_error());
        if (grad_gain.valid()) gain_._accumulate_grad(grad_gain);
        if (grad_bias.valid()) bias_._accumulate_grad(grad_bias);
        if (grad_input.valid()) input_.backward(grad_input);
    }

private:
    Tensor input_, gain_, bias_, mean_, rstd_;
};

}  // namespace

LayerNorm::LayerNorm(Backend& backend, int features, float eps) : backend_(&backend), features_(features), eps_(eps) {
    MCL_CHECK(features_ > 0, "LayerNorm requires positive dimensions");
    const std::vector<float> ones(static_cast<std::size_t>(features_), 1.0f);
    gain.value = Tensor::from_cpu(*backend_, {features_}, DType::F32, ones.data());
    bias.value = Tensor::zeros(*backend_, {features_});
    gain.value.set_requires_grad(true);
    bias.value.set_requires_grad(true);
}

void LayerNorm::zero_grad() {
    gain.value.zero_grad();
    bias.value.zero_grad();
}

Tensor LayerNorm::forward(const Tensor& x) {
    const int element = rows::element_of(x, "LayerNorm");
    const Shape lead = rows::leading(x, "LayerNorm");
    MCL_CHECK(x.shape()[-1] == features_, "LayerNorm input feature mismatch");
    MCL_CHECK(x.backend_ptr() == backend_, "LayerNorm backend mismatch");
    Tensor y = Tensor::empty(*backend_, x.shape(), x.dtype());
    Tensor mean = Tensor::empty(*backend_, lead), rstd = Tensor::empty(*backend_, lead);
    const std::size_t cols = static_cast<std::size_t>(features_);
    const int rc = mcc_layer_norm(backend_->hip_stream(), x.data(), x.nbytes(), cols, rows::f32(gain.value),
                                  gain.value.nbytes(), rows::f32(bias.value), bias.value.nbytes(), y.data(), y.nbytes(),
                                  cols, rows::f32(mean), mean.nbytes(), rows::f32(rstd), rstd.nbytes(),
                                  static_cast<std::size_t>(lead.numel()), cols, element, eps_);
    MCL_CHECK(rc == MCC_OK, std::string("hip layer_norm failed: ") + mcc_last_error());
    if (autograd::is_enabled() && training_) {
        y.set_requires_grad(true);
        y._set_grad_fn(std::make_shared<LayerNormBackwardNode>(x, gain.value, bias.value, mean, rstd));
    }
    return y;
}

}  // namespace motifcl::nn
