// RmsNorm, Linear and AdamW of the autograd graph (cortex_hip_graph.hpp) on the
// GPU: the gradients of a residual block's loss against central differences of
// the same loss in double on the host, a tensor used twice, and AdamW's
// parameters against its formula on those gradients.
#include <cmath>
#include <cstdio>
#include <vector>

#include "cortex_hip_graph.hpp"

namespace hip = cortex::_fw::hip;

static int failures = 0;
#define EXPECT(cond, ...)                   \
    do {                                    \
        if (!(cond)) {                      \
            ++failures;                     \
            std::printf("FAIL: " __VA_ARGS__); \
            std::printf("\n");              \
        }                                   \
    } while (0)

static std::vector<float> rnd(size_t n, unsigned seed, float scale, float mean = 0.0f) {
    std::vector<float> v(n);
    unsigned x = seed * 2654435761u + 12345u;
    for (auto &e : v) {
        x = x * 1664525u + 1013904223u;
        e = mean + scale * (static_cast<float>(x >> 8) / 8388608.0f - 1.0f);
    }
    return v;
}

constexpr size_t B = 12, D = 20, F = 28;
using Params = std::vector<std::vector<double>>;  // x, g, w1, b1, w2, b2

static double act(double z) { return z * 0.5 * std::erfc(-z / std::sqrt(2.0)); }

// The block's loss: softmax cross-entropy of gelu(norm(x) g W1 + b1) W2 + b2 + x.
static double loss_of(const Params &p, const std::vector<int32_t> &labels) {
    double total = 0;
    for (size_t r = 0; r < B; ++r) {
        const double *x = &p[0][r * D];
        double ss = 0;
        for (size_t i = 0; i < D; ++i) ss += x[i] * x[i];
        const double rs = 1 / std::sqrt(ss / D + 1e-5);
        std::vector<double> u(F), y(D);
        for (size_t j = 0; j < F; ++j) {
            double z = p[3][j];
            for (size_t i = 0; i < D; ++i) z += x[i] * rs * p[1][i] * p[2][i * F + j];
            u[j] = act(z);
        }
        double top = -1e300, sum = 0;
        for (size_t i = 0; i < D; ++i) {
            y[i] = p[5][i] + x[i];
            for (size_t j = 0; j < F; ++j) y[i] += u[j] * p[4][j * D + i];
            top = std::fmax(top, y[i]);
        }
        for (double v : y) sum += std::exp(v - top);
        total += top + std::log(sum) - y[labels[r]];
    }
    return total / B;
}

int main() {
    const std::vector<std::vector<int64_t>> shapes = {{(int64_t)B, (int64_t)D}, {(int64_t)D}, {(int64_t)D, (int64_t)F},
                                                      {(int64_t)F}, {(int64_t)F, (int64_t)D}, {(int64_t)D}};
    const std::vector<std::vector<float>> init = {rnd(B * D, 1, 1.5f), rnd(D, 2, 0.2f, 1.0f), rnd(D * F, 3, 0.4f),
                                                  rnd(F, 4, 0.2f),     rnd(F * D, 5, 0.4f),   rnd(D, 6, 0.2f)};
    Params host;
    std::vector<hip::TensorPtr> t;
    for (size_t i = 0; i < init.size(); ++i) {
        host.emplace_back(init[i].begin(), init[i].end());
        t.push_back(std::make_shared<hip::Tensor>(hip::Tensor::from_host(shapes[i], init[i].data(), true)));
    }
    std::vector<int32_t> labels(B);
    for (size_t r = 0; r < B; ++r) labels[r] = static_cast<int32_t>((5 * r) % D);
    int32_t *dlab = nullptr;
    hip::check(cxm_dev_malloc(reinterpret_cast<void **>(&dlab), B * sizeof(int32_t)), "labels");
    hip::check(cxm_memcpy_h2d(dlab, labels.data(), B * sizeof(int32_t), hip::stream()), "labels");

    const std::vector<hip::TensorPtr> params = {t[1], t[2], t[3], t[4], t[5]};
    hip::AdamW opt(params, 0.1f);
    opt.set_decay(0, 0.0f);
    std::vector<std::vector<double>> m(params.size()), v(params.size());
    for (int step = 1; step <= 3; ++step) {
        auto n = hip::rms_norm(t[0], t[1]);
        auto u = hip::linear(n, t[2], t[3], CXM_ACT_GELU);
        auto y = hip::linear(u, t[4], t[5], CXM_ACT_NONE, t[0]);
        auto loss = hip::softmax_cross_entropy(y, dlab);
        for (size_t i = 1; i < t.size(); ++i) {
            const auto h = t[i]->host();
            host[i].assign(h.begin(), h.end());
        }
        EXPECT(std::fabs(loss->host()[0] - loss_of(host, labels)) < 1e-5, "step %d loss", step);
        t[0]->grad_ptr().reset();
        hip::backward(loss);
        std::vector<std::vector<float>> g;
        for (const auto &p : t) g.push_back(p->grad().host());
        // central differences in double: truncation and rounding about 1e-9 each, the
        // fp32 gradients' sums of up to 28 products about 1e-6
        for (size_t i = 0; i < t.size(); ++i)
            for (size_t k = 0; k < host[i].size(); k += host[i].size() / 5) {
                Params q = host;
                q[i][k] += 1e-5;
                const double up = loss_of(q, labels);
                q[i][k] -= 2e-5;
                const double num = (up - loss_of(q, labels)) / 2e-5;
                EXPECT(std::fabs(num - g[i][k]) < 5e-6, "step %d tensor %zu [%zu]: %g against %g", step, i, k, (double)g[i][k],
                       num);
            }
        opt.step(1e-2);
        for (size_t i = 0; i < params.size(); ++i) {
            EXPECT(!params[i]->has_grad(), "the gradients are dropped");
            const auto now = params[i]->host();
            m[i].resize(now.size());
            v[i].resize(now.size());
            bool ok = true;
            for (size_t k = 0; k < now.size(); ++k) {
                const double gr = g[i + 1][k];
                m[i][k] = 0.9 * m[i][k] + 0.1 * gr;
                v[i][k] = 0.999 * v[i][k] + 0.001 * gr * gr;
                const double mh = m[i][k] / (1 - std::pow(0.9, step)), vh = v[i][k] / (1 - std::pow(0.999, step));
                const double want = host[i + 1][k] * (1 - 1e-2 * (i == 0 ? 0.0 : 0.1f)) - 1e-2 * mh / (std::sqrt(vh) + 1e-8);
                // a few fp32 roundings of the parameter and 1e-6 of an update of 1e-2
                ok = ok && std::fabs(now[k] - want) <= 4 * 6e-8 * std::fabs(want) + 1e-7;
            }
            EXPECT(ok, "step %d: parameter %zu", step, i);
        }
    }
    {  // the same tensor as input and residual twice over: contributions add
        auto w = std::make_shared<hip::Tensor>(hip::Tensor::from_host({(int64_t)D, (int64_t)D}, rnd(D * D, 9, 0.3f).data(), true));
        auto x = std::make_shared<hip::Tensor>(hip::Tensor::from_host(shapes[0], init[0].data(), true));
        hip::backward(hip::linear(x, w, nullptr, CXM_ACT_NONE, x));
        const auto gx = x->grad().host();
        const auto wh = w->host();
        bool ok = true;
        for (size_t r = 0; r < B; ++r)
            for (size_t i = 0; i < D; ++i) {
                double want = 1, size = 1;
                for (size_t j = 0; j < D; ++j) want += wh[i * D + j], size += std::fabs(wh[i * D + j]);
                ok = ok && std::fabs(gx[r * D + i] - want) <= 24 * 6e-8 * size;
            }
        EXPECT(ok, "x as input and residual");
    }
    cxm_dev_free(dlab);
    hip::check(cxm_device_sync(), "sync");
    if (failures == 0) std::printf("ALL OK\n");
    return failures == 0 ? 0 : 1;
}
