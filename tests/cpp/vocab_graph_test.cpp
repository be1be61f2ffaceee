// The autograd graph (cortex_hip_graph.hpp) from tokens to losses over a
// vocabulary on the GPU: a table looked up twice, layer norm, a dense layer, log
// probabilities of given tokens and a distilled teacher, against central
// differences of the same loss in double.
#include <cmath>
#include <cstdio>
#include <cstring>
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

using Vec = std::vector<float>;
using Exact = std::vector<double>;

static Vec rnd(size_t n, unsigned seed, float scale, float mean = 0.0f) {
    Vec v(n);
    unsigned x = seed * 2654435761u + 12345u;
    for (auto &e : v) {
        x = x * 1664525u + 1013904223u;
        e = mean + scale * (static_cast<float>(x >> 8) / 8388608.0f - 1.0f);
    }
    return v;
}
static hip::TensorPtr leaf(std::vector<int64_t> shape, const Vec &v, bool grad = true) {
    return std::make_shared<hip::Tensor>(hip::Tensor::from_host(shape, v.data(), grad));
}
// The graph's ids are device int32: the bits in an fp32 tensor.
static hip::TensorPtr ids_of(const std::vector<int32_t> &ids) {
    Vec bits(ids.size());
    std::memcpy(bits.data(), ids.data(), ids.size() * 4);
    return leaf({static_cast<int64_t>(ids.size())}, bits, false);
}
static const int32_t *ints(const hip::TensorPtr &t) { return reinterpret_cast<const int32_t *>(t->data()); }

constexpr int T = 12, V = 37, D = 20, K = 4;
constexpr float TEMP = 0.8f;
struct Problem {
    std::vector<int32_t> first, second, answers, teacher_ids;
    Vec table, w, b, out, teacher, seed;
};

static Problem problem() {
    Problem p;
    for (int t = 0; t < T; ++t) {
        p.first.push_back(t % 5 == 4 ? -1 : (7 * t) % V);
        p.second.push_back(t < 6 ? 3 : (5 * t) % V);
        p.answers.push_back(t == 2 ? -1 : (11 * t + 1) % V);
        for (int j = 0; j < K; ++j) p.teacher_ids.push_back(t == 7 || (t == 3 && j == 1) ? -1 : (13 * t + 9 * j) % V);
    }
    p.table = rnd(V * D, 1, 1.0f), p.w = rnd(D, 2, 0.3f, 1.0f), p.b = rnd(D, 3, 0.3f), p.out = rnd(D * V, 4, 0.4f);
    p.teacher = rnd(T * K, 5, 2.0f), p.seed = rnd(T, 6, 1.0f);
    return p;
}

// The sum over rows of seed (log probability + divergence) in double; `size`: the
// largest sum of |y out| of a logit.
static double loss(const Problem &p, const Exact &table, const Exact &w, const Exact &b, const Exact &out,
                   double *size = nullptr) {
    const double temp = TEMP;
    double sum = 0;
    for (int t = 0; t < T; ++t) {
        double h[D], z[V], mean = 0, var = 0, s1 = 0, s2 = 0, q = 0;
        for (int d = 0; d < D; ++d) {
            h[d] = (p.first[t] < 0 ? 0.0 : 1.5 * table[p.first[t] * D + d]) + table[p.second[t] * D + d];
            mean += h[d] / D;
        }
        for (double v : h) var += (v - mean) * (v - mean) / D;
        for (int v = 0; v < V; ++v) {
            double mag = 0;
            z[v] = 0;
            for (int d = 0; d < D; ++d) {
                const double term = ((h[d] - mean) / std::sqrt(var + 1e-5) * w[d] + b[d]) * out[d * V + v];
                z[v] += term, mag += std::fabs(term);
            }
            if (size && mag > *size) *size = mag;
            s1 += std::exp(z[v]), s2 += std::exp(temp * z[v]);
        }
        if (p.answers[t] >= 0) sum += p.seed[t] * (z[p.answers[t]] - std::log(s1));
        for (int j = 0; j < K; ++j)
            if (p.teacher_ids[t * K + j] >= 0) q += std::exp(temp * p.teacher[t * K + j]);
        for (int j = 0; j < K; ++j) {
            const int id = p.teacher_ids[t * K + j];
            if (id < 0) continue;
            const double lq = temp * p.teacher[t * K + j] - std::log(q);
            sum += p.seed[t] * std::exp(lq) * (lq - (temp * z[id] - std::log(s2)));
        }
    }
    return sum;
}

int main() {
    const Problem p = problem();
    auto table = leaf({V, D}, p.table), w = leaf({D}, p.w), b = leaf({D}, p.b), out = leaf({D, V}, p.out);
    auto first = ids_of(p.first), second = ids_of(p.second), answers = ids_of(p.answers), tids = ids_of(p.teacher_ids);
    auto teacher = leaf({T, K}, p.teacher, false), seed = leaf({T}, p.seed, false);
    auto forward = [&] {
        auto x = hip::add(hip::embedding(table, ints(first), T, 1.5f), hip::embedding(table, ints(second), T));
        auto z = hip::linear(hip::layer_norm(x, w, b), out);
        return hip::add(hip::log_prob(z, ints(answers)), hip::distill(z, ints(tids), teacher->data(), K, TEMP));
    };
    auto root = forward();
    hip::backward(root, *seed);

    const std::vector<hip::TensorPtr> params = {table, w, b, out};
    std::vector<Exact> at;
    std::vector<Vec> grads;
    for (const auto &q : params) {
        const Vec v = q->host();
        at.emplace_back(v.begin(), v.end());
        grads.push_back(q->grad().host());
    }
    // A logit is off by the roundings of a sum of D and of the norm's two, a probability by twice that and by its
    // row's sum's; then sums over V, D, T: 8 of them, of magnitudes that meet the result's norm.
    double a = 0, value = 0;
    const double want = loss(p, at[0], at[1], at[2], at[3], &a);
    const double rel = std::ldexp(1.0, -24) * 8 * (2 * ((2 * D + 8) * a + 2 * a) + 128 + 6 * a + 4 + V + 2 * D + T);
    const Vec rows = root->host();
    for (int t = 0; t < T; ++t) value += static_cast<double>(rows[t]) * p.seed[t];
    EXPECT(std::fabs(value - want) <= rel * (1 + a) * T, "losses %g, in double %g", value, want);
    const char *names[] = {"table", "w", "b", "out"};
    for (size_t i = 0; i < at.size(); ++i) {
        const Vec dir = rnd(at[i].size(), 11 + static_cast<unsigned>(i), 1.0f);
        double len = 0, norm = 0, got = 0;
        for (float v : dir) len += static_cast<double>(v) * v;
        len = std::sqrt(len);
        for (size_t k = 0; k < dir.size(); ++k) {
            got += dir[k] / len * grads[i][k];
            norm += static_cast<double>(grads[i][k]) * grads[i][k];
        }
        auto moved = [&](double h) {
            std::vector<Exact> m = at;
            for (size_t k = 0; k < dir.size(); ++k) m[i][k] += h * dir[k] / len;
            return loss(p, m[0], m[1], m[2], m[3]);
        };
        const double slope = (moved(1e-4) - moved(-1e-4)) / 2e-4;  // (third derivatives times 2e-9: below 1e-6)
        EXPECT(std::fabs(slope - got) <= rel * std::sqrt(norm) + 1e-6, "%s: slope %g, gradient's %g", names[i], slope, got);
    }
    // once more: added to the gradients that the leaves have (twice as much, exactly, but for the order of two
    // contributions to the table: one rounding)
    hip::backward(forward(), *seed);
    for (size_t i = 0; i < params.size(); ++i) {
        const Vec g = params[i]->grad().host();
        for (size_t k = 0; k < g.size(); ++k)
            if (std::fabs(g[k] - 2.0 * grads[i][k]) > rel * std::fabs(grads[i][k]) + 1e-6) {
                EXPECT(false, "%s: the second pass", names[i]);
                break;
            }
    }
    // without gradients: the same bits
    auto plain = [](const hip::TensorPtr &t) { return leaf(t->shape(), t->host(), false); };
    table = plain(table), w = plain(w), b = plain(b), out = plain(out);
    auto again = forward();
    EXPECT(!again->flow() && again->host() == rows, "other bits without gradients");
    hip::check(cxm_device_sync(), "sync");
    if (failures == 0) std::printf("ALL OK\n");
    return failures == 0 ? 0 : 1;
}
