// More of the autograd graph's layers and AdamW (cortex_hip_graph.hpp) on the GPU:
// parameters that do not all have a gradient at every step, and layers whose inputs
// take none.
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

static std::vector<float> rnd(size_t n, unsigned seed, float scale) {
    std::vector<float> v(n);
    unsigned x = seed * 2654435761u + 12345u;
    for (auto &e : v) {
        x = x * 1664525u + 1013904223u;
        e = scale * (static_cast<float>(x >> 8) / 8388608.0f - 1.0f);
    }
    return v;
}
static hip::TensorPtr leaf(std::vector<int64_t> shape, unsigned seed, bool grad = true) {
    size_t n = 1;
    for (auto d : shape) n *= static_cast<size_t>(d);
    return std::make_shared<hip::Tensor>(hip::Tensor::from_host(shape, rnd(n, seed, 0.4f).data(), grad));
}

// One parameter and its moments in double.  Of eight steps in fp32, each adds at
// most 4 roundings of |m|'s parts and 5 of v to the moments (half of it to the
// root); the update has 12 roundings more and the parameter 3.
struct Exact {
    std::vector<double> m, v, size;
    int t = 0;
    bool step(const std::vector<float> &before, const std::vector<float> &g, const std::vector<float> &after) {
        const double lr = 1e-2, u32 = std::ldexp(1.0, -24);
        m.resize(g.size()), v.resize(g.size()), size.resize(g.size());
        ++t;
        bool ok = true;
        for (size_t k = 0; k < g.size(); ++k) {
            m[k] = 0.9 * m[k] + 0.1 * g[k];
            size[k] = 0.9 * size[k] + 0.1 * std::fabs(g[k]);
            v[k] = 0.999 * v[k] + 0.001 * g[k] * static_cast<double>(g[k]);
            const double c = lr / (1 - std::pow(0.9, t)) / (std::sqrt(v[k] / (1 - std::pow(0.999, t))) + 1e-8);
            const double want = before[k] - c * m[k];
            const double tol = u32 * (3 * (std::fabs(before[k]) + c * size[k]) + (12 + 8 * 7) * c * size[k]);
            ok = ok && std::fabs(after[k] - want) <= tol;
        }
        return ok;
    }
};

// `late` has its first gradient at the third step, `some` one at every other step:
// their bias corrections go by their own steps.
static void own_step_numbers() {
    auto x = leaf({12, 20}, 1, false), w = leaf({20, 28}, 2), late = leaf({28, 28}, 3), some = leaf({28, 10}, 4);
    const std::vector<hip::TensorPtr> params = {w, late, some};
    std::vector<Exact> exact(3);
    hip::AdamW opt(params);
    opt.step(1e-2);
    for (int s = 1; s <= 8; ++s) {
        auto y = hip::linear(x, w, nullptr, CXM_ACT_TANH);
        if (s >= 3) y = hip::linear(y, late, nullptr, CXM_ACT_SILU);
        if (s % 2 == 0) y = hip::linear(y, some);
        hip::backward(y);
        std::vector<std::vector<float>> before, g;
        for (const auto &p : params) {
            before.push_back(p->host());
            g.push_back(p->has_grad() ? p->grad().host() : std::vector<float>{});
        }
        opt.step(1e-2);
        for (size_t i = 0; i < params.size(); ++i) {
            const auto now = params[i]->host();
            if (g[i].empty()) EXPECT(now == before[i], "step %d: parameter %zu has no gradient and moved", s, i);
            else EXPECT(exact[i].step(before[i], g[i], now), "step %d: parameter %zu", s, i);
        }
    }
    EXPECT(exact[0].t == 8 && exact[1].t == 6 && exact[2].t == 4, "steps");
}

// A layer gives the same bits whether or not its backward pass will come.
static void without_gradients() {
    for (int act : {CXM_ACT_NONE, CXM_ACT_RELU, CXM_ACT_SIGMOID, CXM_ACT_TANH, CXM_ACT_GELU, CXM_ACT_SILU})
        for (int with : {0, 1, 2, 3}) {
            std::vector<float> y[2];
            for (int grad : {0, 1}) {
                auto x = leaf({37, 20}, 5, grad), w = leaf({20, 53}, 6, grad), g = leaf({20}, 7, grad);
                auto b = with & 1 ? leaf({53}, 8, grad) : nullptr, r = with & 2 ? leaf({37, 53}, 9, grad) : nullptr;
                auto t = hip::linear(hip::rms_norm(x, g), w, b, act, r);
                EXPECT((t->flow() != nullptr) == (grad != 0), "act %d: the flow", act);
                y[grad] = t->host();
            }
            EXPECT(y[0] == y[1], "act %d, bias and residual %d: other bits without gradients", act, with);
        }
    auto x = leaf({37, 20}, 5, false), w = leaf({20, 53}, 6, false), r = leaf({37, 53}, 9, true);
    hip::backward(hip::linear(x, w, nullptr, CXM_ACT_GELU, r));
    EXPECT(r->grad().host() == std::vector<float>(37 * 53, 1.0f), "the gradient of the residual alone");
}

int main() {
    own_step_numbers();
    without_gradients();
    hip::check(cxm_device_sync(), "sync");
    if (failures == 0) std::printf("ALL OK\n");
    return failures == 0 ? 0 : 1;
}
