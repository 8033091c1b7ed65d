// A student of LayerNorm and CounterStateLinear learns from a teacher's top log probabilities: the losses,
// the gradients that reach the norm's parameters and the state's update, against plain loops in double
// precision; and what the three operators refuse.
#include "test_util.hpp"

#include <algorithm>
#include <numeric>

using namespace motifcl;

namespace {

using Vec = std::vector<double>;

Vec wide(const std::vector<float>& v) { return Vec(v.begin(), v.end()); }

Vec log_softmax(const double* z, int n, double t) {
    const double m = *std::max_element(z, z + n);
    double s = 0.0;
    for (int i = 0; i < n; ++i) s += std::exp((z[i] - m) / t);
    Vec out(static_cast<std::size_t>(n));
    for (int i = 0; i < n; ++i) out[static_cast<std::size_t>(i)] = (z[i] - m) / t - std::log(s);
    return out;
}

void near(const std::vector<float>& got, const Vec& want, double tol, const std::string& label) {
    if (got.size() != want.size()) throw std::runtime_error(label + " size mismatch");
    double worst = 0.0;
    for (std::size_t i = 0; i < got.size(); ++i) worst = std::max(worst, std::fabs(got[i] - want[i]));
    if (!(worst <= tol)) throw std::runtime_error(label + " off by " + std::to_string(worst));
}

template <typename F>
void expect_error(F body, const std::string& needle) {
    try {
        body();
    } catch (const Error& e) {
        if (std::string(e.what()).find(needle) != std::string::npos) return;
        throw std::runtime_error(std::string("wrong message: ") + e.what());
    }
    throw std::runtime_error("no Error for: " + needle);
}

}  // namespace

int main() {
    return host_test::run("test_distillation", [](Backend& backend) {
        const int rows = 20, width = 32, vocab = 100, top = 8;
        const double t = 2.0, eps = 1e-5;
        std::vector<float> xh(rows * width), teacher_h(rows * vocab), weight_h(rows, 1.0f / rows);
        host_test::fill_normal(xh, 1, 1.0f);
        host_test::fill_normal(teacher_h, 2, 2.0f);
        std::vector<std::int32_t> tokens_h(rows);
        for (int r = 0; r < rows; ++r) tokens_h[r] = (7 * r) % vocab;
        tokens_h[3] = -100;  // ignored
        auto x = Tensor::from_cpu(backend, {rows, width}, DType::F32, xh.data());
        auto teacher_logits = Tensor::from_cpu(backend, {rows, vocab}, DType::F32, teacher_h.data());
        auto tokens = Tensor::from_cpu(backend, {rows}, DType::I32, tokens_h.data());
        auto weight = Tensor::from_cpu(backend, {rows}, DType::F32, weight_h.data());
        x.set_requires_grad(true);

        TokenLogProbs teacher = token_log_probs(teacher_logits, tokens, top);
        const auto ids = teacher.top_ids.to_vector<std::int32_t>();
        const Vec tz = wide(teacher_h);
        Vec want_lp(rows), want_top(rows * top), want_entropy(rows);
        for (int r = 0; r < rows; ++r) {
            const Vec lp = log_softmax(&tz[r * vocab], vocab, 1.0);
            std::vector<int> order(vocab);
            std::iota(order.begin(), order.end(), 0);
            std::stable_sort(order.begin(), order.end(), [&](int a, int b) { return lp[a] > lp[b]; });
            for (int k = 0; k < top; ++k) {
                if (ids[r * top + k] != order[k]) throw std::runtime_error("top_ids differ");
                want_top[r * top + k] = lp[order[k]];
            }
            want_lp[r] = tokens_h[r] < 0 ? 0.0 : lp[tokens_h[r]];
            for (double l : lp) want_entropy[r] -= std::exp(l) * l;
        }
        // |z| < 10: every log probability within 300 half steps of binary32 of 1
        near(teacher.log_prob.to_vector<float>(), want_lp, 2e-5, "log_prob");
        near(teacher.top_log_probs.to_vector<float>(), want_top, 2e-5, "top_log_probs");
        near(teacher.entropy.to_vector<float>(), want_entropy, 1e-4, "entropy");

        nn::LayerNorm norm(backend, width);
        nn::CounterStateLinear head(backend, width, vocab);
        const Vec w = wide(head.decode_weight().to_vector<float>());
        const auto state = head.state.to_vector<std::uint8_t>();
        Tensor h = norm.forward(x);
        Tensor logits = head.forward(h);
        DistillTop d = distill_top(logits, teacher.top_ids, teacher.top_log_probs, static_cast<float>(t), &weight);
        logits.backward(d.grad_logits);

        // the same in double precision
        const Vec y = wide(teacher.top_log_probs.to_vector<float>());
        Vec want_loss(rows), want_gz(rows * vocab), want_gx(rows * width), want_gain(width), want_bias(width);
        for (int r = 0; r < rows; ++r) {
            const float* xr = &xh[r * width];
            double mean = 0.0, var = 0.0;
            for (int c = 0; c < width; ++c) mean += xr[c] / double(width);
            for (int c = 0; c < width; ++c) var += (xr[c] - mean) * (xr[c] - mean) / width;
            const double rstd = 1.0 / std::sqrt(var + eps);
            Vec z(vocab), gh(width);
            for (int o = 0; o < vocab; ++o)
                for (int c = 0; c < width; ++c) z[o] += w[o * width + c] * (xr[c] - mean) * rstd;
            const Vec lp = log_softmax(z.data(), vocab, t), lq = log_softmax(&y[r * top], top, t);
            for (int o = 0; o < vocab; ++o) want_gz[r * vocab + o] = t / rows * std::exp(lp[o]);
            for (int k = 0; k < top; ++k) {
                const double q = std::exp(lq[k]);
                want_loss[r] += t * t * q * (lq[k] - lp[ids[r * top + k]]);
                want_gz[r * vocab + ids[r * top + k]] -= t / rows * q;
            }
            for (int o = 0; o < vocab; ++o)
                for (int c = 0; c < width; ++c) gh[c] += want_gz[r * vocab + o] * w[o * width + c];
            double a = 0.0, b = 0.0;
            for (int c = 0; c < width; ++c) {
                const double xhat = (xr[c] - mean) * rstd;
                a += gh[c] / width;
                b += gh[c] * xhat / width;
                want_gain[c] += gh[c] * xhat;
                want_bias[c] += gh[c];
            }
            for (int c = 0; c < width; ++c) want_gx[r * width + c] = rstd * (gh[c] - a - (xr[c] - mean) * rstd * b);
        }
        near(d.loss.to_vector<float>(), want_loss, 1e-4, "loss");
        near(d.grad_logits.to_vector<float>(), want_gz, 1e-6, "grad_logits");
        if (!x.grad() || !norm.gain.value.grad() || !norm.bias.value.grad()) throw std::runtime_error("a gradient is missing");
        near(x.grad()->to_vector<float>(), want_gx, 1e-5, "grad_x");
        near(norm.gain.value.grad()->to_vector<float>(), want_gain, 1e-5, "grad_gain");
        near(norm.bias.value.grad()->to_vector<float>(), want_bias, 1e-5, "grad_bias");
        if (head.state.to_vector<std::uint8_t>() == state) throw std::runtime_error("the head's state did not move");

        // the side optimizer takes the parameters' gradients; then the next step can run
        for (nn::Parameter* p : norm.parameters()) {
            auto m = Tensor::zeros(backend, {width}), v = Tensor::zeros(backend, {width});
            const auto before = p->value.to_vector<float>();
            adam_update_fast(p->value, *p->value.grad(), m, v, 1e-2f, 0.9f, 0.999f, 1e-8f, 1);
            if (p->value.to_vector<float>() == before) throw std::runtime_error("adam left a parameter as it was");
        }
        expect_error([&] { norm.forward(x).backward(h); }, "gradient accumulation");
        norm.zero_grad();
        x.zero_grad();
        norm.forward(x).backward(h);
        if (!norm.gain.value.grad()) throw std::runtime_error("the second step has no gradient");

        // cross entropy: the gradient of -mean log p, rows of ignored positions left out
        std::vector<float> up(rows, -1.0f / rows);
        auto grad_lp = Tensor::from_cpu(backend, {rows}, DType::F32, up.data());
        const auto g = token_log_probs_backward(teacher_logits, tokens, teacher, grad_lp).to_vector<float>();
        Vec want_g(rows * vocab);
        for (int r = 0; r < rows; ++r) {
            if (tokens_h[r] < 0) continue;
            const Vec lp = log_softmax(&tz[r * vocab], vocab, 1.0);
            for (int o = 0; o < vocab; ++o) want_g[r * vocab + o] = (std::exp(lp[o]) - (o == tokens_h[r])) / rows;
        }
        near(g, want_g, 1e-6, "cross entropy gradient");

        {  // without training, and under a guard, no node is attached
            autograd::NoGradGuard guard;
            if (norm.forward(x).requires_grad()) throw std::runtime_error("a node was attached under NoGradGuard");
        }
        norm.set_training(false);
        if (norm.forward(x)._grad_fn()) throw std::runtime_error("a node was attached without training");

        auto narrow = Tensor::zeros(backend, {rows, width - 1});
        auto bytes = Tensor::zeros(backend, {rows, width}, DType::U8);
        expect_error([&] { norm.forward(narrow); }, "feature mismatch");
        expect_error([&] { norm.forward(bytes); }, "f32 and f16 only");
        expect_error([&] { nn::LayerNorm(backend, 0); }, "positive dimensions");
        expect_error([&] { token_log_probs(teacher_logits, weight); }, "tokens has the wrong type");
        expect_error([&] { token_log_probs(narrow, teacher.top_ids); }, "tokens shape mismatch");
        expect_error([&] { token_log_probs(teacher_logits, tokens, 129); }, "at most 128");
        expect_error([&] { token_log_probs(teacher_logits, tokens, 101); }, "at most vocab alternatives");
        expect_error([&] { token_log_probs(teacher_logits, tokens, 4, 0.0f); }, "temperature");
        expect_error([&] { token_log_probs_backward(teacher_logits, tokens, teacher, tokens); }, "grad_log_prob has the wrong type");
        expect_error([&] { distill_top(logits, teacher.top_ids, weight); }, "teacher_logits shape mismatch");
        expect_error([&] { distill_top(logits, tokens, weight); }, "teacher_ids shape mismatch");
        expect_error([&] { distill_top(logits, teacher.top_ids, teacher.top_log_probs, 1.0f, &narrow); }, "weight shape mismatch");
    });
}
