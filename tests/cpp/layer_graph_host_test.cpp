// Host test of the autograd graph's optimizer and layers
// (include/cortex_hip_graph.hpp): the caching pool itself over host memory,
// every kernel entry a stand-in that only notes what it was called with.
// Checks what the graph asks the library for: how often AdamW makes its list
// of tensors, which step number each parameter gets, and that layers keep nothing
// for a backward pass that does not come.  Prints ALL OK and returns 0 when every check passes.
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <vector>

#include "../../cortexmind_amd/csrc/pool.hpp"
#include "cortex_hip_graph.hpp"

namespace hip = cortex::_fw::hip;

namespace {

struct HostBackend {
    static int alloc(void **p, size_t bytes) { return (*p = std::malloc(bytes)) ? 0 : 2; }
    static void release(void *p) { std::free(p); }
    static int sync() { return 0; }
};
cxm::CachingPool<HostBackend> &pool() {
    static cxm::CachingPool<HostBackend> p;
    return p;
}

int creates = 0, live = 0;
std::vector<std::pair<const void *, size_t>> steps;  // (parameter, step number) of every step
size_t step_of(const hip::TensorPtr &p) {            // the last one, 0 for none
    for (auto it = steps.rbegin(); it != steps.rend(); ++it)
        if (it->first == p->data()) return it->second;
    return 0;
}

// of the last forward call, and the backward calls
const void *saved_z = nullptr, *saved_rstd = nullptr;
int backwards = 0;

int failures = 0;
#define EXPECT(c, ...)                          \
    do {                                        \
        if (!(c)) {                             \
            std::printf("FAIL %d: ", __LINE__); \
            std::printf(__VA_ARGS__);           \
            std::printf("\n");                  \
            ++failures;                         \
        }                                       \
    } while (0)

}  // namespace

struct cxm_adamw {
    std::vector<cxm_adamw_tensor_t> list;
};

extern "C" {

const char *cxm_error_string(int) { return "stand-in"; }
int cxm_pool_alloc(void **p, size_t bytes, cxm_stream_t s) { return pool().allocate(p, bytes, 0, s); }
int cxm_pool_free(void *p) { return pool().deallocate(p); }
int cxm_memcpy_h2d(void *d, const void *s, size_t n, cxm_stream_t) { return std::memcpy(d, s, n), CXM_OK; }
int cxm_memcpy_d2h(void *d, const void *s, size_t n, cxm_stream_t) { return std::memcpy(d, s, n), CXM_OK; }
int cxm_memcpy_d2d(void *d, const void *s, size_t n, cxm_stream_t) { return std::memcpy(d, s, n), CXM_OK; }
int cxm_memset(void *d, int v, size_t n, cxm_stream_t) { return std::memset(d, v, n), CXM_OK; }
int cxm_stream_sync(cxm_stream_t) { return CXM_OK; }
int cxm_binary_f32(const float *, const float *, float *, size_t, int, cxm_stream_t) { return CXM_OK; }
int cxm_bcast_col_f32(const float *, const float *, float *, size_t, size_t, int, cxm_stream_t) { return CXM_OK; }
int cxm_softmax_xent_f32(const float *, const int32_t *, float *, float *, size_t, size_t, cxm_stream_t) { return CXM_OK; }
int cxm_rmsnorm_fwd_t(const void *, const void *, const void *, float, void *, void *, uint8_t *, float *, float *rstd,
                      size_t, size_t, int, cxm_stream_t) {
    saved_rstd = rstd;
    return CXM_OK;
}
int cxm_rmsnorm_bwd_t(const void *, const float *, const void *, const void *, const void *, void *, void *, size_t,
                      size_t, int, cxm_stream_t) {
    return CXM_OK;
}
int cxm_linear_fwd_t(const void *, const void *, const void *, const void *, void *z, void *, size_t, size_t, size_t, int,
                     int, int, cxm_stream_t) {
    saved_z = z;
    return CXM_OK;
}
int cxm_linear_bwd_t(const void *, const void *, const void *, const void *, void *, void *, void *, void *, size_t,
                     size_t, size_t, int, int, int, cxm_stream_t) {
    ++backwards;
    return CXM_OK;
}
int cxm_adamw_create(cxm_adamw **h, const cxm_adamw_tensor_t *t, size_t n, int, int, int) {
    ++creates, ++live;
    *h = new cxm_adamw{std::vector<cxm_adamw_tensor_t>(t, t + n)};
    return CXM_OK;
}
int cxm_adamw_step(cxm_adamw *h, double, double, double, double, size_t t, const float *, uint64_t, cxm_stream_t) {
    for (const auto &e : h->list) steps.emplace_back(e.p, t);
    return CXM_OK;
}
int cxm_adamw_destroy(cxm_adamw *h) {
    --live;
    delete h;
    return CXM_OK;
}

}  // extern "C"

namespace {

hip::TensorPtr leaf(size_t rows, size_t cols) {
    std::vector<int64_t> shape;
    if (rows) shape.push_back(static_cast<int64_t>(rows));
    shape.push_back(static_cast<int64_t>(cols));
    return hip::make_tensor(shape, true);
}

// Steps of a normalised residual block: the gradients are dropped after each, and
// yet the list of tensors is made once.
void lists_made(size_t B, size_t D, size_t F) {
    auto X = hip::make_tensor({static_cast<int64_t>(B), static_cast<int64_t>(D)});
    auto gain = leaf(0, D), W1 = leaf(D, F), b1 = leaf(0, F), W2 = leaf(F, D), b2 = leaf(0, D);
    hip::AdamW opt({gain, W1, b1, W2, b2}, 0.01f);
    creates = 0;
    for (int s = 0; s < 20; ++s) {
        auto h = hip::linear(hip::rms_norm(X, gain), W1, b1, CXM_ACT_GELU);
        auto y = hip::linear(h, W2, b2, CXM_ACT_NONE, X);
        hip::backward(hip::softmax_cross_entropy(y, nullptr));
        opt.step(1e-3);
        EXPECT(!W1->has_grad() && !gain->has_grad(), "the gradients are dropped");
    }
    EXPECT(creates == 1, "%zux%zux%zu: the list was made %d times in 20 steps", B, D, F, creates);
}

// A gradient that the caller keeps is not written by the next backward pass.
void kept_gradient() {
    auto x = leaf(4, 6), w = leaf(6, 8);
    hip::AdamW opt({x, w});
    auto run = [&] { hip::backward(hip::linear(x, w, nullptr, CXM_ACT_NONE, nullptr)); };
    run();
    const hip::TensorPtr handle = x->grad_ptr();
    const hip::Tensor copy = w->grad();
    opt.step(1e-3);
    run();
    EXPECT(x->grad().data() != handle->data(), "a gradient held by its handle is written again");
    EXPECT(w->grad().data() != copy.data(), "a gradient held by its storage is written again");
}

// A parameter's step number counts its own steps: one that joins late begins at
// 1, one that misses steps does not count them, and a step without gradients is none.
void own_step_numbers() {
    auto x = hip::make_tensor({4, 6});
    auto w = leaf(6, 8), late = leaf(8, 8), some = leaf(8, 5);
    hip::AdamW opt({w, late, some});
    steps.clear();
    creates = 0;
    opt.step(1e-3);
    EXPECT(steps.empty() && creates == 0, "a step without gradients");
    size_t nl = 0, ns = 0;
    int made = 0;
    for (size_t s = 1; s <= 12; ++s) {
        auto y = hip::linear(x, w);
        if (s >= 3) y = hip::linear(y, late), ++nl;
        if (s % 2 == 0) y = hip::linear(y, some), ++ns;
        const size_t before = steps.size();
        hip::backward(y);
        opt.step(1e-3);
        opt.step(1e-3);  // none has a gradient now
        EXPECT(step_of(w) == s && step_of(late) == nl && step_of(some) == ns, "step %zu: %zu %zu %zu for %zu %zu %zu", s,
               step_of(w), step_of(late), step_of(some), s, nl, ns);
        EXPECT(steps.size() - before == size_t(1) + (s >= 3) + (s % 2 == 0), "step %zu: %zu parameters", s, steps.size() - before);
        if (s == 6) made = creates;
    }
    // {w}, {some} and {late} are of different numbers from step 5 on: their lists stay
    EXPECT(made == creates, "%d lists were made after step 6", creates - made);
}

// What the backward reads (z, 1 / rms) is asked for only where it will be read.
void nothing_kept_without_gradients() {
    auto x = hip::make_tensor({4, 6}), w = hip::make_tensor({6, 8}), b = hip::make_tensor({8}), g = hip::make_tensor({6}),
         r = hip::make_tensor({4, 8});
    auto wg = leaf(6, 8), bg = leaf(0, 8), gg = leaf(0, 6), rg = leaf(4, 8), xg = leaf(4, 6);
    for (int act : {CXM_ACT_RELU, CXM_ACT_GELU}) {
        EXPECT(!hip::linear(x, w, b, act, r)->flow() && !saved_z, "act %d: z without a gradient", act);
        EXPECT(hip::linear(x, wg, b, act, r)->flow() && saved_z, "act %d: z for the weight", act);
        EXPECT(hip::linear(xg, w, b, act, r)->flow() && saved_z, "act %d: z for x", act);
        EXPECT(hip::linear(x, w, bg, act, r)->flow() && saved_z, "act %d: z for the bias", act);
        auto y = hip::linear(x, w, b, act, rg);  // dY is the residual's gradient
        EXPECT(y->flow() && !saved_z, "act %d: z for the residual alone", act);
        backwards = 0;
        hip::backward(y);
        EXPECT(backwards == 0 && rg->has_grad(), "act %d: the residual's gradient alone", act);
        rg->grad_ptr().reset();
    }
    EXPECT(!hip::rms_norm(x, g)->flow() && !saved_rstd, "1 / rms without a gradient");
    EXPECT(hip::rms_norm(x, gg)->flow() && saved_rstd, "1 / rms for the gain");
    EXPECT(hip::rms_norm(xg, g)->flow() && saved_rstd, "1 / rms for x");
}

}  // namespace

int main() {
    const size_t sizes[][3] = {{12, 20, 28},     {64, 64, 64},      {128, 128, 512},    {256, 256, 256},
                               {512, 256, 1024}, {32, 784, 1024},   {1, 1, 1},          {100, 333, 77},
                               {64, 1024, 4096}, {1024, 1024, 1024}};
    for (const auto &s : sizes) lists_made(s[0], s[1], s[2]);
    kept_gradient();
    own_step_numbers();
    nothing_kept_without_gradients();
    EXPECT(live == 0, "%d lists are left", live);
    pool().release_cached();
    if (failures == 0) std::printf("ALL OK\n");
    return failures == 0 ? 0 : 1;
}
