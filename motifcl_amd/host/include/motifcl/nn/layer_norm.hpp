// Layer norm in front of counter layers, on the HIP library: a Module whose gain and bias are ordinary
// parameters (their gradients go to adam_update_fast / sgd_update) and whose autograd node passes the
// input's gradient on, as CounterStateLinear's does.  The norm of MotifCL itself (src/ops/norm.cpp) is
// another one, without a mean.
#pragma once

#include <vector>

#include <motifcl/nn/module.hpp>
#include <motifcl/runtime/backend.hpp>

namespace motifcl::nn {

class LayerNorm : public Module {
public:
    LayerNorm(Backend& backend, int features, float eps = 1e-5f);

    // x [..., features], f32 or f16; while training the node is attached whether or not x wants a gradient,
    // because gain and bias do.
    Tensor forward(const Tensor& x) override;
    std::vector<Parameter*> parameters() override { return {&gain, &bias}; }
    void zero_grad() override;

    void set_training(bool t) { training_ = t; }
    bool training() const { return training_; }
    int features() const { return features_; }
    float eps() const { return eps_; }

    Parameter gain;  // F32 [features], ones
    Parameter bias;  // F32 [features], zeros

private:
    Backend* backend_ = nullptr;
    int features_ = 0;
    float eps_ = 1e-5f;
    bool training_ = true;
};

}  // namespace motifcl::nn
