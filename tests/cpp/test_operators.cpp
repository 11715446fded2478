// test_operators.cpp — the fine-tuning operators through ttp::Store's methods, against their
// formulas in double on the host.  Also built with host-side AddressSanitizer/UBSan (make asan).
//
// The operators' device memory is the weights of further tensors of the same store, so the test
// needs only the drop-in header.  Tolerances: logits are of order 1 and there are 7 of them, so a
// float32 log-probability and what is made of it is a few 2^-24 off; 1e-5 is asked.
#include <cmath>
#include <cstring>
#include <limits>
#include <stdexcept>
#include <vector>

#include "common.hpp"
#include "ttperf/ttperf.hpp"

namespace {

constexpr uint64_t kRows = 8, kCols = 7, kOuts = 5, kPairs = 2;
constexpr double kBeta = 0.5, kLow = 0.2, kHigh = 0.3, kKl = 0.1, kScale = 8.0;

// tensors: the layer's weight and bias, then memory
enum : uint32_t { W, B, Z, Y, STARTS, REF, ADV, LOGPS, MARGINS, SCALARS, GRAD, KEPT, SCALES, OUT,
                  DY, DX, kTensors };

std::vector<ttp::TensorSpec> specs() {
    std::vector<ttp::TensorSpec> s(kTensors);
    const auto set = [&](uint32_t i, uint64_t n) { s[i].shape = {n}; };
    for (uint32_t i = 0; i < kTensors; ++i) set(i, kRows * kCols);
    set(W, kCols * kOuts);
    set(B, kOuts);
    set(Y, 2 * kRows);                  // int64
    set(STARTS, 2 * (2 * kPairs + 1));  // int64
    for (uint32_t i : {(uint32_t)REF, (uint32_t)ADV, (uint32_t)LOGPS}) set(i, kRows);
    set(MARGINS, kPairs);
    set(SCALARS, 2);
    set(KEPT, kRows * 32 / 4);  // bytes
    set(SCALES, kRows / 4);
    set(DY, kRows * kOuts);
    return s;
}

struct Memory {
    ttp::Store& store;
    float* at(uint32_t i) { return (float*)store.device_ptr(TTP_BUF_PARAM, i); }
    void put(uint32_t i, const void* p, size_t bytes) {
        std::vector<float> v(store.numel(i));
        test::check(bytes == v.size() * 4, "memory of tensor " + std::to_string(i));
        std::memcpy(v.data(), p, bytes);
        store.set_weights(i, v);
    }
    std::vector<float> get(uint32_t i) { return store.weights(i); }
    ttp_matrix matrix(uint32_t i, uint64_t cols = kCols) {
        return {at(i), kRows, cols, cols, TTP_DTYPE_F32, 0};
    }
};

void near(const std::vector<float>& got, const std::vector<double>& want, const std::string& what) {
    test::check(got.size() == want.size(), what + ": size");
    for (size_t i = 0; i < want.size(); ++i)
        if (!(std::fabs(got[i] - want[i]) <= 1e-5 * (1 + std::fabs(want[i])))) {
            test::check(false, what + "[" + std::to_string(i) + "] = " + std::to_string(got[i]) +
                                   ", expected " + std::to_string(want[i]));
            return;
        }
}

template <class F>
void refused(F&& f, const std::string& what) {
    try {
        f();
    } catch (const std::exception&) {
        return;
    }
    test::check(false, what + " was not refused");
}

double sigmoid(double x) { return 1 / (1 + std::exp(-x)); }

}  // namespace

int main() {
    test::DeviceGuard guard;
    ttp::Store store(specs(), ttp::Mode::FP32);
    Memory mem{store};
    store.configure_scaler(kScale);

    std::vector<float> z(kRows * kCols), ref(kRows), adv(kRows);
    for (size_t i = 0; i < z.size(); ++i) z[i] = std::sin(1.3f * (float)i) * 2.0f;
    const std::vector<int64_t> y = {0, 6, -1, 3, 2, 5, 1, 4}, starts = {0, 2, 4, 6, 8};
    std::vector<double> logp(kRows);
    std::vector<std::vector<double>> p(kRows, std::vector<double>(kCols));
    for (size_t t = 0; t < kRows; ++t) {
        double s = 0;
        for (size_t v = 0; v < kCols; ++v) s += std::exp((double)z[t * kCols + v]);
        for (size_t v = 0; v < kCols; ++v) p[t][v] = std::exp((double)z[t * kCols + v]) / s;
        logp[t] = y[t] < 0 ? 0.0 : std::log(p[t][(size_t)y[t]]);
        ref[t] = (float)(logp[t] + 0.2 * std::cos(3.0 * (double)t));
        adv[t] = t % 2 ? -0.7f : 1.1f;
    }
    mem.put(Z, z.data(), z.size() * 4);
    mem.put(Y, y.data(), y.size() * 8);
    mem.put(STARTS, starts.data(), starts.size() * 8);
    mem.put(REF, ref.data(), ref.size() * 4);
    mem.put(ADV, adv.data(), adv.size() * 4);
    const auto* dy_y = (const int64_t*)mem.at(Y);
    const ttp_matrix logits = mem.matrix(Z), grad = mem.matrix(GRAD);
    const auto want_grad = [&](const std::vector<double>& c) {
        std::vector<double> g(kRows * kCols);
        for (size_t t = 0; t < kRows; ++t)
            for (size_t v = 0; v < kCols; ++v)
                g[t * kCols + v] = y[t] < 0 ? 0.0 : c[t] * (((int64_t)v == y[t]) - p[t][v]);
        return g;
    };

    store.token_logprobs(logits, dy_y, mem.at(LOGPS));
    near(mem.get(LOGPS), logp, "token_logprobs");

    {
        std::vector<double> d(2 * kPairs), h(kPairs), c(kRows);
        for (size_t t = 0; t < kRows; ++t) d[t / 2] += y[t] < 0 ? 0.0 : logp[t] - ref[t];
        double loss = 0;
        for (size_t k = 0; k < kPairs; ++k) {
            h[k] = kBeta * (d[k] - d[k + kPairs]);
            loss += std::log1p(std::exp(-h[k])) / kPairs;
            const double dh = kScale * -sigmoid(-h[k]) * kBeta / kPairs;
            for (size_t t = 0; t < kRows; ++t) {
                if (t / 2 == k) c[t] = dh;
                if (t / 2 == k + kPairs) c[t] = -dh;
            }
        }
        ttp_preference_args a{};
        a.logits = &logits;
        a.targets = dy_y;
        a.starts = (const int64_t*)mem.at(STARTS);
        a.ref_logps = mem.at(REF);
        a.pairs = kPairs;
        a.beta = kBeta;
        a.grad = &grad;
        a.logps = mem.at(LOGPS);
        a.margins = mem.at(MARGINS);
        a.loss = mem.at(SCALARS);
        store.preference_loss(a);
        near(mem.get(MARGINS), h, "margins");
        near({mem.get(SCALARS)[0]}, {loss}, "preference loss");
        near(mem.get(GRAD), want_grad(c), "preference gradient");
        a.beta = 0.0;
        refused([&] { store.preference_loss(a); }, "beta 0");
    }
    {
        std::vector<double> c(kRows);
        double loss = 0, kl = 0;
        for (size_t t = 0; t < kRows; ++t) {
            if (y[t] < 0) continue;
            const double r = std::exp(logp[t] - ref[t]), g = ref[t] - logp[t];
            const double held = std::min(std::max(r, 1 - kLow), 1 + kHigh);
            const double plain = r * adv[t], clipped = held * adv[t], k = std::expm1(g) - g;
            loss += -std::min(plain, clipped) + kKl * k;
            kl += k;
            c[t] = kScale * ((plain <= clipped ? -plain : 0.0) - kKl * std::expm1(g)) / 7;
        }
        ttp_policy_args a{};
        a.logits = &logits;
        a.targets = dy_y;
        a.old_logps = a.ref_logps = mem.at(REF);
        a.advantages = mem.at(ADV);
        a.clip_low = kLow;
        a.clip_high = kHigh;
        a.kl_coef = kKl;
        a.grad = &grad;
        a.logps = mem.at(LOGPS);
        a.loss = mem.at(SCALARS);
        a.kl = mem.at(SCALARS) + 1;
        store.policy_loss(a);
        near(mem.get(SCALARS), {loss / 7, kl / 7}, "policy loss and kl");
        near(mem.get(GRAD), want_grad(c), "policy gradient");
        a.loss = a.kl;
        refused([&] { store.policy_loss(a); }, "one place for two results");
    }

    // the logits as an activation: values and GELU from the kept ones, gradients into W and B
    const ttp_checkpoint8 kept{mem.at(KEPT), mem.at(SCALES), kRows, kCols, TTP_CHECKPOINT_INT8, 0};
    const ttp_matrix out = mem.matrix(OUT), dx = mem.matrix(DX), dy = mem.matrix(DY, kOuts);
    store.checkpoint8(logits, kept);
    store.restore8(kept, out);
    const std::vector<float> x = mem.get(OUT);
    for (size_t i = 0; i < x.size(); ++i)  // half a step, 2^-5 for magnitudes up to 2
        test::check(std::fabs(x[i] - z[i]) <= 1.0 / 64, "restore8");
    const std::vector<float> before = mem.get(KEPT);
    store.gelu_checkpoint8(logits, TTP_GELU_ERF, out, kept);
    test::assert_bits(mem.get(KEPT), before, "gelu_checkpoint8's kept values");
    store.gelu_backward8(kept, TTP_GELU_ERF, logits, dx);
    std::vector<double> y64(z.size()), dx64(z.size());
    for (size_t i = 0; i < z.size(); ++i) {
        const auto phi = [](double v) { return 0.5 * std::erfc(-v / std::sqrt(2.0)); };
        y64[i] = z[i] * phi(z[i]);
        dx64[i] = z[i] * (phi(x[i]) + x[i] * std::exp(-0.5 * x[i] * x[i]) / std::sqrt(2 * M_PI));
    }
    near(mem.get(OUT), y64, "gelu");
    near(mem.get(DX), dx64, "gelu's gradient");

    std::vector<float> d(kRows * kOuts);
    for (size_t i = 0; i < d.size(); ++i) d[i] = std::cos(0.7f * (float)i);
    mem.put(DY, d.data(), d.size() * 4);
    std::vector<double> dw(kCols * kOuts), dwt(kCols * kOuts), db(kOuts);
    for (size_t t = 0; t < kRows; ++t)
        for (size_t o = 0; o < kOuts; ++o) {
            db[o] += d[t * kOuts + o];
            for (size_t i = 0; i < kCols; ++i) {
                dw[i * kOuts + o] += (double)x[t * kCols + i] * d[t * kOuts + o];
                dwt[o * kCols + i] = dw[i * kOuts + o];
            }
        }
    store.accumulate_linear_grad8(W, kept, dy, B);
    near(store.grad(W), dw, "the weight's gradient");
    near(store.grad(B), db, "the bias's gradient");
    store.accumulate_linear_grad8(W, kept, dy);  // a second micro-batch, without the bias
    for (double& v : dw) v *= 2;
    near(store.grad(W), dw, "the weight's gradient, twice");
    near(store.grad(B), db, "the bias's gradient, once");
    store.zero_grad();
    store.accumulate_linear_grad8(W, kept, dy, TTP_NO_TENSOR, true);
    near(store.grad(W), dwt, "the transposed weight's gradient");
    test::check(!store.has_grad(B), "no bias was asked for");
    refused([&] { store.accumulate_linear_grad8(B, kept, dy); }, "another tensor's size");
    return test::finish("test_operators");
}
