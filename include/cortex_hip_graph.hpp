// cortex_hip_graph.hpp -- reverse-mode autograd over the gfx950 backend:
// the concrete GradientFlows the reference declares but never implements,
// a backward driver and SGD.
//
// The reference's autograd is the abstract meta::GradientFlow with
// `virtual void backward(const Tensor& _grad) = 0` and a name
// (source/CortexMind/framework/Graph/flow.hpp:15-24); GradientLink attaches a
// flow to a tensor (Graph/link.cpp:11-13).  No subclass, no driver and no
// optimizer exist there.  This header keeps that interface (GradientFlow,
// backward(const Tensor&), ToString()) and adds flows for every operator on
// the path -- MatMul, AddBias, Add, MulRow (Broadcast::row::mul), MulScalar
// (ScalarOp::mul), ReLU / Sigmoid / Tanh, the fused AffineAct, Softmax and
// LogSoftmax, Sum and Mean over an axis, SoftmaxCrossEntropy, RmsNorm and
// Linear (a dense layer with bias, activation and residual) -- each
// running the library's kernels through the C ABI on hip::stream(), plus
// backward(root[, seed]), sgd() and AdamW.  Tensors are shared handles (TensorPtr)
// so that a flow can reach its inputs' gradients.
//
// Gradients accumulate: the first contribution to a tensor's gradient is
// written directly, later ones are added (matrix_t::add in place).
// Flows that need a forward output keep its storage, not the tensor: the
// output owns the flow, and a handle back would make a reference cycle.
// Header-only; link with -lcxm_hip.
#ifndef CORTEX_HIP_GRAPH_HPP
#define CORTEX_HIP_GRAPH_HPP

#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <functional>
#include <initializer_list>
#include <map>
#include <memory>
#include <string>
#include <string_view>
#include <unordered_set>
#include <utility>
#include <vector>

#include "cortex_hip.hpp"

namespace cortex::_fw::hip {

using TensorPtr = std::shared_ptr<Tensor>;

// An fp32 tensor on the HIP device.
inline TensorPtr make_tensor(std::vector<std::int64_t> shape, bool requires_grad = false) {
    return std::make_shared<Tensor>(std::move(shape), DType::Float32, DeviceType::HIP, requires_grad);
}
inline Tensor device_tensor(std::vector<std::int64_t> shape) {
    return Tensor(std::move(shape), DType::Float32, DeviceType::HIP);
}

// meta::GradientFlow (Graph/flow.hpp:15-24).  `inputs` are the tensors the
// flow sends gradients to; the driver walks them to order the flows.
struct GradientFlow {
    explicit GradientFlow(std::string name) : name_(std::move(name)) {}
    virtual ~GradientFlow() = default;
    virtual void backward(const Tensor &grad) = 0;
    std::string_view ToString() const noexcept { return name_; }
    std::vector<TensorPtr> inputs;

private:
    std::string name_;
};

// A tensor takes part in the backward pass when it asks for a gradient or
// was produced by a flow.
inline bool needs_grad(const TensorPtr &t) { return t->isRequired() || t->flow() != nullptr; }

// Gives t a gradient that the caller then fills: in the buffer of its last one
// where an optimizer left that and nobody else holds it, else in a new one.
inline void new_grad(const TensorPtr &t) {
    TensorPtr spare = std::move(t->spare_grad_ptr());
    // (storage() is a handle of its own, beside the tensor's)
    const bool free = spare && spare.use_count() == 1 && spare->storage().use_count() == 2 && spare->shape() == t->shape();
    t->grad_ptr() = free ? std::move(spare) : make_tensor(t->shape());
}

// Adds a gradient contribution to t: `write(dst)` fills a buffer of t's
// shape; the first contribution writes t's gradient directly.
inline void accumulate(const TensorPtr &t, const std::function<void(float *)> &write) {
    if (!t->has_grad()) {
        new_grad(t);
        write(t->grad().data());
        return;
    }
    Tensor tmp = device_tensor(t->shape());
    write(tmp.data());
    matrix_t::add(t->grad().data(), tmp.data(), t->grad().len());
}

// Where a kernel that forms several gradients at once writes t's
// contribution: t's gradient itself when it has none yet, else `tmp`, which
// grad_done then adds in; a scratch buffer when t takes no gradient.
inline float *grad_dst(const TensorPtr &t, Tensor &tmp) {
    if (needs_grad(t) && !t->has_grad()) {
        new_grad(t);
        return t->grad().data();
    }
    tmp = device_tensor(t->shape());
    return tmp.data();
}
inline void grad_done(const TensorPtr &t, Tensor &tmp) {
    if (needs_grad(t) && !tmp.empty()) matrix_t::add(t->grad().data(), tmp.data(), t->len());
}

// GradientLink (Graph/link.cpp:11-13): attach a flow to the tensor it produced.
inline void link(const TensorPtr &out, std::shared_ptr<GradientFlow> flow) { out->flow() = std::move(flow); }

// The graph's ops run device kernels on their operands' storage: a tensor
// that is not fp32 HIP memory is refused on the host (CXM_ASSERT's exit)
// before any launch could touch it.
inline void on_device(std::initializer_list<const Tensor *> ts, const char *what) {
    for (const Tensor *t : ts)
        if (t->device() != DeviceType::HIP || t->dtype() != DType::Float32) {
            std::fprintf(stderr, "[ERROR] %s: operand is not an fp32 HIP tensor\n", what);
            std::exit(1);
        }
}

// Rows and columns of a 2-D tensor.
inline std::size_t rows_of(const Tensor &t) { return static_cast<std::size_t>(t.dim(0)); }
inline std::size_t cols_of(const Tensor &t) { return static_cast<std::size_t>(t.dim(1)); }

// ------------------------------------------------------------------ flows

// C[M,N] = A[M,K] B[K,N]: dA = dC B^T, dB = A^T dC (cxm_gemm_f32 with the
// transposed operand forms).
struct MatMulFlow : GradientFlow {
    TensorPtr a, b;
    MatMulFlow(TensorPtr a_, TensorPtr b_) : GradientFlow("MatMul"), a(std::move(a_)), b(std::move(b_)) {
        inputs = {a, b};
    }
    void backward(const Tensor &dc) override {
        const std::size_t M = rows_of(*a), K = cols_of(*a), N = cols_of(*b);
        if (needs_grad(a))
            accumulate(a, [&](float *da) {
                check(cxm_gemm_f32(dc.data(), b->data(), da, M, N, K, 0, 1, nullptr, CXM_ACT_NONE, nullptr, stream()),
                      "MatMulFlow: dA");
            });
        if (needs_grad(b))
            accumulate(b, [&](float *db) {
                check(cxm_gemm_f32(a->data(), dc.data(), db, K, M, N, 1, 0, nullptr, CXM_ACT_NONE, nullptr, stream()),
                      "MatMulFlow: dB");
            });
    }
};

// Y[M,N] = X + b[N] (Broadcast::row::add): dX = dY, db = sum over rows of dY.
struct AddBiasFlow : GradientFlow {
    TensorPtr x, bias;
    AddBiasFlow(TensorPtr x_, TensorPtr b_) : GradientFlow("AddBias"), x(std::move(x_)), bias(std::move(b_)) {
        inputs = {x, bias};
    }
    void backward(const Tensor &dy) override {
        const std::size_t M = rows_of(*x), N = cols_of(*x);
        if (needs_grad(x))
            accumulate(x, [&](float *dx) {
                check(cxm_memcpy_d2d(dx, dy.data(), M * N * sizeof(float), stream()), "AddBiasFlow: dX");
            });
        if (needs_grad(bias))
            accumulate(bias, [&](float *db) { reduce::sum(dy.data(), db, 1, M, N); });
    }
};

// Y = A + B (same shape, matrix_t::add): dA = dY, dB = dY.
struct AddFlow : GradientFlow {
    TensorPtr a, b;
    AddFlow(TensorPtr a_, TensorPtr b_) : GradientFlow("Add"), a(std::move(a_)), b(std::move(b_)) { inputs = {a, b}; }
    void backward(const Tensor &dy) override {
        for (const TensorPtr &t : {a, b})
            if (needs_grad(t))
                accumulate(t, [&](float *d) {
                    check(cxm_memcpy_d2d(d, dy.data(), dy.len() * sizeof(float), stream()), "AddFlow");
                });
    }
};

// Y[M,N] = X * s[N] (Broadcast::row::mul): dX = dY * s, ds = sum over rows
// of dY * X.  One pass of the fused affine backward with no activation
// (cxm_affine_act_bwd_f32, ACT_NONE) forms both; its bias sum is dropped.
struct MulRowFlow : GradientFlow {
    TensorPtr x, scale;
    MulRowFlow(TensorPtr x_, TensorPtr s_) : GradientFlow("MulRow"), x(std::move(x_)), scale(std::move(s_)) {
        inputs = {x, scale};
    }
    void backward(const Tensor &dy) override {
        const std::size_t M = rows_of(*x), N = cols_of(*x);
        Tensor tx, ts, db = device_tensor({static_cast<std::int64_t>(N)});
        float *dx = grad_dst(x, tx), *ds = grad_dst(scale, ts);
        check(cxm_affine_act_bwd_f32(x->data(), scale->data(), x->data(), dy.data(), dx, ds, db.data(), M, N,
                                     CXM_ACT_NONE, stream()),
              "MulRowFlow");
        grad_done(x, tx);
        grad_done(scale, ts);
    }
};

// Y = X * c (ScalarOp::mul): dX = dY * c.
struct MulScalarFlow : GradientFlow {
    TensorPtr x;
    float c;
    MulScalarFlow(TensorPtr x_, float c_) : GradientFlow("MulScalar"), x(std::move(x_)), c(c_) { inputs = {x}; }
    void backward(const Tensor &dy) override {
        if (!needs_grad(x)) return;
        accumulate(x, [&](float *dx) { ScalarOp::mul(dy.data(), c, dx, dy.len()); });
    }
};

// Y = act(X) for act in RELU, SIGMOID, TANH: dX = dY * act'(Y) from the
// saved output (relu' = [Y > 0], sigmoid' = Y (1 - Y), tanh' = 1 - Y^2).
struct ActFlow : GradientFlow {
    TensorPtr x;
    std::shared_ptr<Storage> y;
    int act;
    static const char *name_of(int a) { return a == CXM_ACT_RELU ? "ReLU" : a == CXM_ACT_SIGMOID ? "Sigmoid" : "Tanh"; }
    ActFlow(TensorPtr x_, std::shared_ptr<Storage> y_, int a)
        : GradientFlow(name_of(a)), x(std::move(x_)), y(std::move(y_)), act(a) {
        inputs = {x};
    }
    void backward(const Tensor &dy) override {
        if (!needs_grad(x)) return;
        accumulate(x, [&](float *dx) {
            check(cxm_act_bwd_f32(y->as<float>(), dy.data(), dx, dy.len(), act, stream()), "ActFlow");
        });
    }
};

// Y = act(X * s[N] + b[N]) in one pass (cxm_affine_act_fwd_f32): the
// backward forms dX, ds and db in one pass too (cxm_affine_act_bwd_f32)
// from X, s, the saved Y and dY.
struct AffineActFlow : GradientFlow {
    TensorPtr x, scale, bias;
    std::shared_ptr<Storage> y;
    int act;
    AffineActFlow(TensorPtr x_, TensorPtr s_, TensorPtr b_, std::shared_ptr<Storage> y_, int a)
        : GradientFlow("AffineAct"), x(std::move(x_)), scale(std::move(s_)), bias(std::move(b_)), y(std::move(y_)),
          act(a) {
        inputs = {x, scale, bias};
    }
    void backward(const Tensor &dy) override {
        const std::size_t M = rows_of(*x), N = cols_of(*x);
        Tensor tx, ts, tb;
        float *dx = grad_dst(x, tx), *ds = grad_dst(scale, ts), *db = grad_dst(bias, tb);
        check(cxm_affine_act_bwd_f32(x->data(), scale->data(), y->as<float>(), dy.data(), dx, ds, db, M, N, act,
                                     stream()),
              "AffineActFlow");
        grad_done(x, tx);
        grad_done(scale, ts);
        grad_done(bias, tb);
    }
};

// Row softmax (log_mode 0) or log-softmax (1) over the last axis of
// [rows, cols]: dX from the saved output (cxm_softmax_bwd_f32).
struct SoftmaxFlow : GradientFlow {
    TensorPtr x;
    std::shared_ptr<Storage> y;
    int log_mode;
    SoftmaxFlow(TensorPtr x_, std::shared_ptr<Storage> y_, int log)
        : GradientFlow(log ? "LogSoftmax" : "Softmax"), x(std::move(x_)), y(std::move(y_)), log_mode(log) {
        inputs = {x};
    }
    void backward(const Tensor &dy) override {
        if (!needs_grad(x)) return;
        accumulate(x, [&](float *dx) {
            check(cxm_softmax_bwd_f32(y->as<float>(), dy.data(), dx, rows_of(*x), cols_of(*x), log_mode, stream()),
                  "SoftmaxFlow");
        });
    }
};

// Z[outer, inner] = reduce::sum / reduce::mean of X[outer, dim, inner] over
// dim: dX[o, d, i] = dZ[o, i] (/ dim for the mean).
struct SumFlow : GradientFlow {
    TensorPtr x;
    std::size_t outer, dim, inner;
    int mean;
    SumFlow(TensorPtr x_, std::size_t o, std::size_t d, std::size_t i, int m)
        : GradientFlow(m ? "Mean" : "Sum"), x(std::move(x_)), outer(o), dim(d), inner(i), mean(m) {
        inputs = {x};
    }
    void backward(const Tensor &dz) override {
        if (!needs_grad(x)) return;
        accumulate(x, [&](float *dx) {
            check(cxm_reduce_sum_bwd_f32(dz.data(), dx, outer, dim, inner, mean, stream()), "SumFlow");
        });
    }
};

// loss = mean over rows of -log_softmax(logits)[r, label_r]; the forward
// kernel also writes dloss/dlogits = (softmax - onehot) / rows, which the
// backward scales by the incoming gradient (a one-element device tensor,
// read on the device: dlogits * g[0], one rounding; exact for the seed 1).
struct SoftmaxCrossEntropyFlow : GradientFlow {
    TensorPtr logits;
    Tensor dlogits;
    SoftmaxCrossEntropyFlow(TensorPtr l, Tensor d)
        : GradientFlow("SoftmaxCrossEntropy"), logits(std::move(l)), dlogits(std::move(d)) {
        inputs = {logits};
    }
    void backward(const Tensor &g) override {
        if (!needs_grad(logits)) return;
        if (g.len() != 1) check(CXM_E_INVALID, "SoftmaxCrossEntropyFlow: the loss gradient is not a scalar");
        accumulate(logits, [&](float *dl) {
            // column broadcast over one row: dl[0, j] = dlogits[0, j] * g[0]
            check(cxm_bcast_col_f32(dlogits.data(), g.data(), dl, 1, dlogits.len(), CXM_OP_MUL, stream()),
                  "SoftmaxCrossEntropyFlow");
        });
    }
};

// ---------------------------------------------------------------- ops

inline TensorPtr matmul(const TensorPtr &a, const TensorPtr &b) {
    on_device({a.get(), b.get()}, "matmul");
    auto c = make_tensor({a->dim(0), b->dim(1)});
    matrix_t::matmul(a->data(), b->data(), c->data(), rows_of(*a), cols_of(*a), cols_of(*b));
    if (needs_grad(a) || needs_grad(b)) link(c, std::make_shared<MatMulFlow>(a, b));
    return c;
}

inline TensorPtr add_bias(const TensorPtr &x, const TensorPtr &b) {
    on_device({x.get(), b.get()}, "add_bias");
    auto y = make_tensor(x->shape());
    Broadcast::row::add(x->data(), b->data(), y->data(), rows_of(*x), cols_of(*x));
    if (needs_grad(x) || needs_grad(b)) link(y, std::make_shared<AddBiasFlow>(x, b));
    return y;
}

inline TensorPtr add(const TensorPtr &a, const TensorPtr &b) {
    on_device({a.get(), b.get()}, "add");
    auto y = make_tensor(a->shape());
    matrix_t::add(a->data(), b->data(), y->data(), a->len());
    if (needs_grad(a) || needs_grad(b)) link(y, std::make_shared<AddFlow>(a, b));
    return y;
}

// X[M,N] * s[N] (Broadcast::row::mul)
inline TensorPtr mul_row(const TensorPtr &x, const TensorPtr &s) {
    on_device({x.get(), s.get()}, "mul_row");
    auto y = make_tensor(x->shape());
    Broadcast::row::mul(x->data(), s->data(), y->data(), rows_of(*x), cols_of(*x));
    if (needs_grad(x) || needs_grad(s)) link(y, std::make_shared<MulRowFlow>(x, s));
    return y;
}

// X * c (ScalarOp::mul)
inline TensorPtr mul_scalar(const TensorPtr &x, float c) {
    on_device({x.get()}, "mul_scalar");
    auto y = make_tensor(x->shape());
    ScalarOp::mul(x->data(), c, y->data(), x->len());
    if (needs_grad(x)) link(y, std::make_shared<MulScalarFlow>(x, c));
    return y;
}

inline TensorPtr activate(const TensorPtr &x, int act) {
    on_device({x.get()}, "activation");
    auto y = make_tensor(x->shape());
    check(cxm_unary_f32(x->data(), y->data(), x->len(), act, stream()), "activation");
    if (needs_grad(x)) link(y, std::make_shared<ActFlow>(x, y->storage(), act));
    return y;
}
inline TensorPtr relu(const TensorPtr &x) { return activate(x, CXM_ACT_RELU); }
inline TensorPtr sigmoid(const TensorPtr &x) { return activate(x, CXM_ACT_SIGMOID); }
inline TensorPtr tanh(const TensorPtr &x) { return activate(x, CXM_ACT_TANH); }

// act(X * s + b) as one kernel each way; act in NONE, RELU, SIGMOID, TANH.
inline TensorPtr affine_act(const TensorPtr &x, const TensorPtr &s, const TensorPtr &b, int act) {
    on_device({x.get(), s.get(), b.get()}, "affine_act");
    auto y = make_tensor(x->shape());
    check(cxm_affine_act_fwd_f32(x->data(), s->data(), b->data(), y->data(), rows_of(*x), cols_of(*x), act, stream()),
          "affine_act");
    if (needs_grad(x) || needs_grad(s) || needs_grad(b))
        link(y, std::make_shared<AffineActFlow>(x, s, b, y->storage(), act));
    return y;
}

inline TensorPtr softmax_rows(const TensorPtr &x, int log_mode) {
    on_device({x.get()}, "softmax");
    auto y = make_tensor(x->shape());
    check(cxm_softmax_fwd_f32(x->data(), y->data(), rows_of(*x), cols_of(*x), log_mode, stream()), "softmax");
    if (needs_grad(x)) link(y, std::make_shared<SoftmaxFlow>(x, y->storage(), log_mode));
    return y;
}
inline TensorPtr softmax(const TensorPtr &x) { return softmax_rows(x, 0); }
inline TensorPtr log_softmax(const TensorPtr &x) { return softmax_rows(x, 1); }

// reduce::sum / reduce::mean over the middle axis of X viewed as
// [outer, dim, inner] (X's element count must be outer * dim * inner);
// the result has shape [outer, inner].
inline TensorPtr reduce_axis(const TensorPtr &x, std::size_t outer, std::size_t dim, std::size_t inner, int mean) {
    on_device({x.get()}, "reduce");
    if (outer * dim * inner != x->len()) check(CXM_E_INVALID, "reduce: outer * dim * inner != element count");
    auto z = make_tensor({static_cast<std::int64_t>(outer), static_cast<std::int64_t>(inner)});
    if (mean) reduce::mean(x->data(), z->data(), outer, dim, inner);
    else reduce::sum(x->data(), z->data(), outer, dim, inner);
    if (needs_grad(x)) link(z, std::make_shared<SumFlow>(x, outer, dim, inner, mean));
    return z;
}
inline TensorPtr sum(const TensorPtr &x, std::size_t outer, std::size_t dim, std::size_t inner) {
    return reduce_axis(x, outer, dim, inner, 0);
}
inline TensorPtr mean(const TensorPtr &x, std::size_t outer, std::size_t dim, std::size_t inner) {
    return reduce_axis(x, outer, dim, inner, 1);
}

// Y = X / rms(X) * w over the rows of X [rows, cols] (cxm_rmsnorm_fwd_t):
// dX and dw from X and the saved 1 / rms (cxm_rmsnorm_bwd_t).
struct RmsNormFlow : GradientFlow {
    TensorPtr x, w;
    Tensor rstd;
    RmsNormFlow(TensorPtr x_, TensorPtr w_, Tensor rstd_)
        : GradientFlow("RmsNorm"), x(std::move(x_)), w(std::move(w_)), rstd(std::move(rstd_)) {
        inputs = {x, w};
    }
    void backward(const Tensor &dy) override {
        Tensor tx, tw;
        float *dx = grad_dst(x, tx), *dw = grad_dst(w, tw);
        check(cxm_rmsnorm_bwd_t(x->data(), rstd.data(), w->data(), dy.data(), nullptr, dx, dw, rows_of(*x), cols_of(*x),
                                CXM_DT_F32, stream()),
              "RmsNormFlow");
        grad_done(x, tx);
        grad_done(w, tw);
    }
};
inline TensorPtr rms_norm(const TensorPtr &x, const TensorPtr &w, float eps = 1e-5f) {
    on_device({x.get(), w.get()}, "rms_norm");
    if (w->len() != cols_of(*x)) check(CXM_E_INVALID, "rms_norm: one weight per column");
    auto y = make_tensor(x->shape());
    const bool grad = needs_grad(x) || needs_grad(w);
    Tensor rstd;
    if (grad) rstd = device_tensor({x->dim(0)});
    check(cxm_rmsnorm_fwd_t(x->data(), nullptr, w->data(), eps, nullptr, y->data(), nullptr, nullptr,
                            grad ? rstd.data() : nullptr, rows_of(*x), cols_of(*x), CXM_DT_F32, stream()),
          "rms_norm");
    if (grad) link(y, std::make_shared<RmsNormFlow>(x, w, std::move(rstd)));
    return y;
}

// Y = act(X W + bias) + residual (cxm_linear_fwd_t), bias and residual
// optional: the gradients of X, W and the bias from the saved X W + bias
// (cxm_linear_bwd_t); the residual's is dY.  X W + bias is saved only where one
// of those three takes a gradient (without it the fp32 product applies a ReLU
// itself).
struct LinearFlow : GradientFlow {
    TensorPtr x, w, bias, res;
    Tensor z;
    int act;
    LinearFlow(TensorPtr x_, TensorPtr w_, TensorPtr b_, TensorPtr r_, Tensor z_, int act_)
        : GradientFlow("Linear"), x(std::move(x_)), w(std::move(w_)), bias(std::move(b_)), res(std::move(r_)),
          z(std::move(z_)), act(act_) {
        inputs = {x, w};
        if (bias) inputs.push_back(bias);
        if (res) inputs.push_back(res);
    }
    void backward(const Tensor &dy) override {
        const std::size_t M = rows_of(*x), K = cols_of(*x), N = cols_of(*w);
        Tensor tx, tw, tb, dz;
        const bool products = needs_grad(x) || needs_grad(w) || (bias && needs_grad(bias));
        if (products && act != CXM_ACT_NONE) dz = device_tensor(dy.shape());
        float *dx = needs_grad(x) ? grad_dst(x, tx) : nullptr;
        // a tensor that is an input twice already has its first contribution when the second is made
        float *dw = needs_grad(w) ? grad_dst(w, tw) : nullptr;
        float *db = bias && needs_grad(bias) ? grad_dst(bias, tb) : nullptr;
        if (products)
            check(cxm_linear_bwd_t(x->data(), w->data(), z.empty() ? nullptr : z.data(), dy.data(),
                                   dz.empty() ? nullptr : dz.data(), dx, dw, db, M, K, N, 0, act, CXM_DT_F32, stream()),
                  "LinearFlow");
        grad_done(x, tx);
        grad_done(w, tw);
        if (db) grad_done(bias, tb);
        if (res && needs_grad(res))
            accumulate(res, [&](float *d) {
                check(cxm_memcpy_d2d(d, dy.data(), dy.len() * sizeof(float), stream()), "LinearFlow: residual");
            });
    }
};
// act: CXM_ACT_NONE, RELU, SIGMOID, TANH, GELU or SILU.
inline TensorPtr linear(const TensorPtr &x, const TensorPtr &w, const TensorPtr &bias = nullptr, int act = CXM_ACT_NONE,
                        const TensorPtr &res = nullptr) {
    on_device({x.get(), w.get()}, "linear");
    if (bias) on_device({bias.get()}, "linear");
    if (res) on_device({res.get()}, "linear");
    const std::size_t M = rows_of(*x), K = cols_of(*x), N = cols_of(*w);
    if (rows_of(*w) != K || (bias && bias->len() != N) || (res && res->len() != M * N))
        check(CXM_E_INVALID, "linear: sizes do not match");
    auto y = make_tensor({x->dim(0), w->dim(1)});
    const bool products = needs_grad(x) || needs_grad(w) || (bias && needs_grad(bias));
    Tensor z;
    if (products && act != CXM_ACT_NONE) z = device_tensor(y->shape());
    check(cxm_linear_fwd_t(x->data(), w->data(), bias ? bias->data() : nullptr, res ? res->data() : nullptr,
                           z.empty() ? nullptr : z.data(), y->data(), M, K, N, 0, act, CXM_DT_F32, stream()),
          "linear");
    if (products || (res && needs_grad(res)))
        link(y, std::make_shared<LinearFlow>(x, w, bias, res, std::move(z), act));
    return y;
}

// labels: device int32 [rows].
inline TensorPtr softmax_cross_entropy(const TensorPtr &logits, const std::int32_t *labels) {
    on_device({logits.get()}, "softmax_cross_entropy");
    auto loss = make_tensor({1});
    Tensor dl = device_tensor(logits->shape());
    check(cxm_softmax_xent_f32(logits->data(), labels, loss->data(), dl.data(), rows_of(*logits), cols_of(*logits),
                               stream()),
          "softmax_cross_entropy");
    if (needs_grad(logits)) link(loss, std::make_shared<SoftmaxCrossEntropyFlow>(logits, std::move(dl)));
    return loss;
}

// ------------------------------------------------------------ backward

// Runs every flow reachable from `root` once, each after all flows that
// consume its output: reverse topological order of the graph.  The root's
// gradient is `seed` (a device fp32 tensor of the root's element count),
// or ones when the root has no gradient yet and no seed is given.
inline void backward(const TensorPtr &root, const Tensor *seed = nullptr) {
    std::vector<TensorPtr> order;
    std::unordered_set<const Tensor *> seen;
    std::function<void(const TensorPtr &)> visit = [&](const TensorPtr &t) {
        if (!t->flow() || !seen.insert(t.get()).second) return;
        for (const auto &in : t->flow()->inputs) visit(in);
        order.push_back(t);
    };
    visit(root);
    if (seed) {
        if (seed->len() != root->len() || seed->device() != DeviceType::HIP)
            check(CXM_E_INVALID, "backward: seed does not match the root");
        root->grad_ptr() = make_tensor(root->shape());
        check(cxm_memcpy_d2d(root->grad().data(), seed->data(), seed->len() * sizeof(float), stream()), "backward: seed");
    } else if (!root->has_grad()) {  // d root / d root = 1
        root->grad_ptr() = make_tensor(root->shape());
        const std::vector<float> ones(root->len(), 1.0f);
        check(cxm_memcpy_h2d(root->grad().data(), ones.data(), ones.size() * sizeof(float), stream()), "backward: seed");
        check(cxm_stream_sync(stream()), "backward: seed");
    }
    for (auto it = order.rbegin(); it != order.rend(); ++it) {
        const TensorPtr &t = *it;
        if (t->has_grad()) t->flow()->backward(t->grad());
    }
}
inline void backward(const TensorPtr &root, const Tensor &seed) { backward(root, &seed); }

// W -= lr * dW for every parameter with a gradient (matrix_t::sub of
// ScalarOp::mul: two roundings), then the gradients are dropped.
inline void sgd(const std::vector<TensorPtr> &params, float lr) {
    for (const auto &p : params) {
        if (!p->has_grad()) continue;
        on_device({p.get(), &p->grad()}, "sgd");
        check(cxm_sgd_f32(p->data(), p->grad().data(), lr, p->len(), stream()), "sgd");
        p->grad_ptr().reset();
    }
}

// AdamW over the parameters that have a gradient (cxm_adamw_step), after which
// the gradients are dropped, as by sgd(), but their buffers stay with the
// parameters for the next backward pass: the pool would hand them out in another
// order, and the list of pointers, which is kept on the device (making it
// blocks), would not hold for the next step.  Owns the fp32 moments and counts
// each parameter's own steps, which the bias corrections go by: a parameter
// whose first gradient comes late begins at 1.  Parameters of one count are one
// list and one launch, all of them where every step gives each a gradient; a list
// is made again only when other parameters than before are at one count or a
// storage has moved.
class AdamW {
public:
    explicit AdamW(std::vector<TensorPtr> params, float decay = 0.0f) : params_(std::move(params)) {
        for (const auto &p : params_) {
            on_device({p.get()}, "AdamW");
            m_.push_back(zeros(p->shape()));
            v_.push_back(zeros(p->shape()));
            decay_.push_back(decay);
            steps_.push_back(0);
        }
    }
    AdamW(const AdamW &) = delete;
    AdamW &operator=(const AdamW &) = delete;
    ~AdamW() {
        drop([](const List &) { return true; });
        for (const auto &p : params_) p->spare_grad_ptr().reset();
    }
    // Weight decay of parameter i alone.
    void set_decay(std::size_t i, float decay) {
        decay_.at(i) = decay;
        drop([&](const List &l) { return has(l, m_[i].data()); });
    }
    void step(double lr, double beta1 = 0.9, double beta2 = 0.999, double eps = 1e-8) {
        std::map<std::size_t, std::vector<cxm_adamw_tensor_t>> by;  // step number -> its tensors
        for (std::size_t i = 0; i < params_.size(); ++i) {
            if (!params_[i]->has_grad() || params_[i]->len() == 0) continue;
            on_device({params_[i].get(), &params_[i]->grad()}, "AdamW");
            cxm_adamw_tensor_t t{};
            t.p = params_[i]->data();
            t.g = params_[i]->grad().data();
            t.m = m_[i].data();
            t.v = v_[i].data();
            t.n = params_[i]->len();
            t.decay = decay_[i];
            by[steps_[i] + 1].push_back(t);
        }
        for (const auto &[t, tensors] : by)
            check(cxm_adamw_step(list_of(tensors), lr, beta1, beta2, eps, t, nullptr, 0, stream()), "AdamW");
        for (std::size_t i = 0; i < params_.size(); ++i) {
            if (!params_[i]->has_grad()) continue;
            ++steps_[i];
            params_[i]->spare_grad_ptr() = std::move(params_[i]->grad_ptr());
        }
    }

private:
    struct List {
        std::vector<cxm_adamw_tensor_t> tensors;
        cxm_adamw *handle;
    };
    static Tensor zeros(const std::vector<std::int64_t> &shape) {
        Tensor t = device_tensor(shape);
        check(cxm_memset(t.data(), 0, t.len() * sizeof(float), stream()), "AdamW");
        return t;
    }
    static bool same(const List &l, const std::vector<cxm_adamw_tensor_t> &tensors) {
        bool eq = l.tensors.size() == tensors.size();
        for (std::size_t i = 0; eq && i < tensors.size(); ++i)
            eq = l.tensors[i].p == tensors[i].p && l.tensors[i].g == tensors[i].g && l.tensors[i].m == tensors[i].m;
        return eq;
    }
    // Whether the parameter of moments m is in the list.
    static bool has(const List &l, const void *m) {
        for (const auto &t : l.tensors)
            if (t.m == m) return true;
        return false;
    }
    // The handle for these tensors; lists that one of them was in before go.
    cxm_adamw *list_of(const std::vector<cxm_adamw_tensor_t> &tensors) {
        for (const List &l : lists_)
            if (same(l, tensors)) return l.handle;
        drop([&](const List &l) {
            for (const auto &t : tensors)
                if (has(l, t.m)) return true;
            return false;
        });
        cxm_adamw *h = nullptr;
        check(cxm_adamw_create(&h, tensors.data(), tensors.size(), CXM_DT_F32, CXM_DT_F32, CXM_DT_F32), "AdamW");
        lists_.push_back({tensors, h});
        return h;
    }
    template <class F>
    void drop(const F &which) {
        std::vector<List> keep;
        for (List &l : lists_) {
            if (which(l)) (void)cxm_adamw_destroy(l.handle);
            else keep.push_back(std::move(l));
        }
        lists_ = std::move(keep);
    }
    std::vector<TensorPtr> params_;
    std::vector<Tensor> m_, v_;
    std::vector<float> decay_;
    std::vector<std::size_t> steps_;
    std::vector<List> lists_;
};

}  // namespace cortex::_fw::hip

#endif  // CORTEX_HIP_GRAPH_HPP
