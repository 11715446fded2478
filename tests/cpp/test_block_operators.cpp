// test_block_operators.cpp — a block's operators through ttp::Store's methods, against their formulas
// in double on the host.  Also built with host-side AddressSanitizer/UBSan (make asan).
//
// The operators' device memory is the weights of further tensors of the same store, so the test
// needs only the drop-in header.  Tolerances: numbers of order 1 and sums of at most 9 of them, so
// a float32 result is a few 2^-24 off; 1e-5 is asked.
#include <cmath>
#include <cstring>
#include <stdexcept>
#include <vector>

#include "common.hpp"
#include "ttperf/ttperf.hpp"

namespace {

constexpr uint64_t kRows = 6, kCols = 9, kOuts = 5, kVocab = 7;
constexpr double kEps = 1e-4;

// tensors: the weights, then memory
enum : uint32_t { TABLE, PLACES, NORM_W, NORM_B, W, B, X, Y, DY, DX, MEAN, RSTD, TOKENS, AT, OUT, RES,
                  SEED, kTensors };

std::vector<ttp::TensorSpec> specs() {
    std::vector<ttp::TensorSpec> s(kTensors);
    const auto set = [&](uint32_t i, uint64_t n) { s[i].shape = {n}; };
    for (uint32_t i = 0; i < kTensors; ++i) set(i, kRows * kCols);
    set(TABLE, kVocab * kCols);
    set(PLACES, 3 * kCols);
    set(NORM_W, kCols);
    set(NORM_B, kCols);
    set(W, kCols * kOuts);
    set(B, kOuts);
    for (uint32_t i : {(uint32_t)MEAN, (uint32_t)RSTD}) set(i, kRows);
    for (uint32_t i : {(uint32_t)TOKENS, (uint32_t)AT}) set(i, 2 * kRows);  // int64
    for (uint32_t i : {(uint32_t)OUT, (uint32_t)RES}) set(i, kRows * kOuts);
    set(SEED, 2);
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
    std::vector<double> waves(uint32_t i, double step) {
        std::vector<float> v(store.numel(i));
        for (size_t k = 0; k < v.size(); ++k) v[k] = (float)std::sin(step * (double)(k + 1));
        store.set_weights(i, v);
        return std::vector<double>(v.begin(), v.end());
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

// element j of a group (Philox 4x32 of ten rounds, 16 bits each)
uint32_t half(uint64_t seed, uint64_t stream, uint64_t group, int j) {
    uint32_t c[4] = {(uint32_t)group, (uint32_t)(group >> 32), (uint32_t)stream,
                     (uint32_t)(stream >> 32)};
    uint32_t k[2] = {(uint32_t)seed, (uint32_t)(seed >> 32)};
    for (int r = 0; r < 10; ++r) {
        const uint64_t a = (uint64_t)c[0] * 0xD2511F53u, b = (uint64_t)c[2] * 0xCD9E8D57u;
        const uint32_t n[4] = {(uint32_t)(b >> 32) ^ c[1] ^ k[0], (uint32_t)b,
                               (uint32_t)(a >> 32) ^ c[3] ^ k[1], (uint32_t)a};
        std::memcpy(c, n, sizeof c);
        k[0] += 0x9E3779B9u;
        k[1] += 0xBB67AE85u;
    }
    return c[j / 2] >> (16 * (j % 2)) & 0xFFFFu;
}
bool kept(const ttp_dropout& d, uint64_t row, uint64_t col, uint64_t cols) {
    return half(d.seed, d.stream, row * ((cols + 7) / 8) + col / 8, (int)(col % 8)) >=
           (uint32_t)std::lround(d.p * 65536);
}
double factor(const ttp_dropout& d) { return 65536.0 / (65536 - std::lround(d.p * 65536)); }

}  // namespace

int main() {
    test::DeviceGuard guard;
    ttp::Store store(specs(), ttp::Mode::FP32);
    Memory mem{store};
    const std::vector<double> table = mem.waves(TABLE, 0.7), places = mem.waves(PLACES, 1.1);
    const std::vector<double> nw = mem.waves(NORM_W, 0.4), nb = mem.waves(NORM_B, 0.9);
    const std::vector<double> w = mem.waves(W, 1.7), b = mem.waves(B, 0.3);
    const std::vector<double> dy = mem.waves(DY, 2.3), res = mem.waves(RES, 0.6);
    const std::vector<int64_t> tokens = {3, 0, 3, -1, 6, 3}, at = {0, 1, 2, 0, 1, 2};
    mem.put(TOKENS, tokens.data(), tokens.size() * 8);
    mem.put(AT, at.data(), at.size() * 8);

    // lookup
    ttp_matrix x = mem.matrix(X), y = mem.matrix(Y);
    store.embedding(TABLE, (const int64_t*)mem.at(TOKENS), x, 1.5, PLACES,
                    (const int64_t*)mem.at(AT));
    std::vector<double> xs(kRows * kCols);
    for (uint64_t r = 0; r < kRows; ++r)
        for (uint64_t c = 0; c < kCols; ++c)
            xs[r * kCols + c] = (tokens[r] < 0 ? 0.0 : 1.5 * table[tokens[r] * kCols + c]) +
                                places[at[r] * kCols + c];
    near(mem.get(X), xs, "embedding");

    // its gradient, twice: assigned, then added
    const ttp_matrix g = mem.matrix(DY);
    std::vector<double> dt(kVocab * kCols);
    for (int pass = 0; pass < 2; ++pass) {
        store.accumulate_embedding_grad(TABLE, (const int64_t*)mem.at(TOKENS), g, 0.5);
        for (uint64_t r = 0; r < kRows; ++r)
            for (uint64_t c = 0; c < kCols && tokens[r] >= 0; ++c)
                dt[tokens[r] * kCols + c] += 0.5 * dy[r * kCols + c];
        near(store.grad(TABLE), dt, "embedding gradient");
    }

    // layer norm and its gradients
    store.layer_norm(NORM_W, NORM_B, x, y, mem.at(MEAN), mem.at(RSTD), kEps);
    std::vector<double> ys(xs.size()), h(xs.size()), dx(xs.size()), dw(kCols), db(kCols);
    for (uint64_t r = 0; r < kRows; ++r) {
        double m = 0, v = 0, gm = 0, ghm = 0;
        for (uint64_t c = 0; c < kCols; ++c) m += xs[r * kCols + c] / kCols;
        for (uint64_t c = 0; c < kCols; ++c) v += std::pow(xs[r * kCols + c] - m, 2) / kCols;
        const double s = 1 / std::sqrt(v + kEps);
        for (uint64_t c = 0; c < kCols; ++c) {
            const uint64_t i = r * kCols + c;
            h[i] = (xs[i] - m) * s;
            ys[i] = h[i] * nw[c] + nb[c];
            gm += dy[i] * nw[c] / kCols;
            ghm += dy[i] * nw[c] * h[i] / kCols;
            dw[c] += dy[i] * h[i];
            db[c] += dy[i];
        }
        for (uint64_t c = 0; c < kCols; ++c) {
            const uint64_t i = r * kCols + c;
            dx[i] = xs[i] + s * (dy[i] * nw[c] - gm - h[i] * ghm);
        }
    }
    near(mem.get(Y), ys, "layer norm");
    store.layer_norm_backward(NORM_W, NORM_B, x, g, mem.at(MEAN), mem.at(RSTD), mem.matrix(DX), &x);
    near(mem.get(DX), dx, "layer norm's input gradient");
    near(store.grad(NORM_W), dw, "layer norm's weight gradient");
    near(store.grad(NORM_B), db, "layer norm's bias gradient");

    // dropout, its seed on the host and on the device
    ttp_dropout d{0.25, 0x123456789ABCDEFull, 1ull << 33, nullptr};
    mem.put(SEED, &d.seed, 8);
    for (int pass = 0; pass < 2; ++pass) {
        store.dropout(d, x, y);
        std::vector<double> want(xs.size());
        for (uint64_t i = 0; i < xs.size(); ++i)
            want[i] = kept(d, i / kCols, i % kCols, kCols) ? xs[i] * factor(d) : 0.0;
        near(mem.get(Y), want, "dropout");
        d.device_seed = (const uint64_t*)mem.at(SEED);
    }

    // a linear product with all that may follow it, either way round
    for (int transposed = 0; transposed < 2; ++transposed) {
        const ttp_matrix out = mem.matrix(OUT, kOuts), r = mem.matrix(RES, kOuts);
        store.linear({&x, &r, &out, &d, W, B, transposed, TTP_ACTIVATION_GELU_ERF});
        std::vector<double> want(kRows * kOuts);
        for (uint64_t i = 0; i < kRows; ++i)
            for (uint64_t o = 0; o < kOuts; ++o) {
                double z = b[o];
                for (uint64_t c = 0; c < kCols; ++c)
                    z += xs[i * kCols + c] * w[transposed ? o * kCols + c : c * kOuts + o];
                z *= 0.5 * std::erfc(-z / std::sqrt(2.0));
                want[i * kOuts + o] =
                    res[i * kOuts + o] + (kept(d, i, o, kOuts) ? z * factor(d) : 0.0);
            }
        near(mem.get(OUT), want, "linear");
    }

    // refusals: shapes, tensors, values, overlaps
    ttp_matrix out = mem.matrix(OUT, kOuts), narrow = mem.matrix(X, kCols - 1);
    refused([&] { store.linear({&narrow, nullptr, &out, nullptr, W, B, 0, 0}); }, "a narrow input");
    refused([&] { store.linear({&x, nullptr, &out, nullptr, kTensors, B, 0, 0}); }, "no such weight");
    refused([&] { store.linear({&x, nullptr, &out, nullptr, W, W, 0, 0}); }, "a weight for a bias");
    refused([&] { store.linear({&x, nullptr, &out, nullptr, W, B, 0, 4}); }, "an activation");
    refused([&] { store.linear({&x, nullptr, nullptr, nullptr, W, B, 0, 0}); }, "no output");
    refused([&] { store.linear({nullptr, nullptr, &out, nullptr, W, B, 0, 0}); }, "no input");
    const ttp_matrix weight{mem.at(W), 1, kOuts, kOuts, TTP_DTYPE_F32, 0};
    const ttp_matrix one{mem.at(X), 1, kCols, kCols, TTP_DTYPE_F32, 0};
    refused([&] { store.linear({&one, nullptr, &weight, nullptr, W, B, 0, 0}); },
            "an output in the weight");
    d.p = 1.0;
    refused([&] { store.dropout(d, x, y); }, "p = 1");
    refused([&] { store.layer_norm(W, NORM_B, x, y, mem.at(MEAN), mem.at(RSTD)); }, "a long weight");
    refused([&] { store.layer_norm(NORM_W, NORM_B, x, y, mem.at(MEAN), mem.at(RSTD), -1.0); },
            "a negative eps");
    refused([&] { store.layer_norm(NORM_W, NORM_B, x, y, mem.at(MEAN), mem.at(MEAN)); },
            "one array twice");
    refused([&] {
        store.layer_norm_backward(NORM_W, NORM_W, x, g, mem.at(MEAN), mem.at(RSTD), mem.matrix(DX));
    }, "a weight that is the bias");
    refused([&] { store.embedding(TABLE, nullptr, x); }, "no tokens");
    refused([&] { store.embedding(B, (const int64_t*)mem.at(TOKENS), x); }, "a short table");
    refused([&] { store.accumulate_embedding_grad(TABLE, nullptr, g); }, "no tokens");
    near(mem.get(X), xs, "the input, unchanged");
    return test::finish("test_block_operators");
}
