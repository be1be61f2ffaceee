"""The training and serving operators of a normalised, residual layer: timed
and compared cases.

Every case is a dict of plain values; ``kind`` names the operator and the
other fields its sizes and options:

* ``norm``: h = x + residual, the root-mean-square norm of h's rows, and its
  output in the type of the input or in 8 bits (e4m3) with a scale per row;
* ``norm_bwd``: its backward: the gradient of the rows, joined with the one
  that reaches h past the norm, and the gradient of the weight;
* ``linear``: act(x W + bias) + residual, optionally with x W + bias kept for
  the backward;
* ``linear_bwd``: its backward: dz = dy act'(z), the gradients of x, W and
  the bias;
* ``linear_q8``: the same product of 8-bit operands with a scale per row of x
  and per column of the result;
* ``adamw``: one AdamW step over all tensors of a model, with its moments in
  32 bits, or in 8 bits with a scale per block of 256 values.

``own`` is false: ``run`` computes the operators from elementary torch
operations, in 32 bits, rounded once at the end.  ``own`` is true: ``run``
makes the library's calls.

Definitions shared by both:

* an 8-bit value is an e4m3 float (3 mantissa bits, largest 448); a row or
  block holds value / scale with scale = (largest magnitude) / 448, or zeros
  with scale 0 where that scale is below the smallest normal float;
* h is rounded to its type, and the norm reads the rounded h, as the backward
  does;
* the optimizer's 8-bit moments are m and the square root of v, rounded
  stochastically (a root above zero never to zero): the 16 random bits of
  each come from `noise` of the step's seed and the value's number, where
  tensors are numbered in blocks of 256.
"""
import math

import torch

own = False

EPS = 1e-5
BLOCK = 256
_TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_F8 = torch.float8_e4m3fn
_TINY = torch.finfo(torch.float32).tiny
_BETA1, _BETA2, _ADAM_EPS, _LR, _DECAY, _SEED = 0.9, 0.999, 1e-8, 1e-3, 0.1, 20261


class Buffer:
    """A GPU tensor as the engine's calls take their operands."""

    def __init__(self, tensor):
        self.tensor = tensor
        self.ptr = tensor.data_ptr()
        self.size = tensor.numel()


# ------------------------------------------------------------------ cases


def listed():
    return [
        # the smallest call: one new token's activations before a layer, where latency counts
        {"name": "norm_1x4096", "kind": "norm", "rows": 1, "cols": 4096, "dtype": "bf16", "residual": True, "q8": False},
        # a batch of sequences normalised and stored in 8 bits for the product that follows
        {"name": "norm_q8_4096x4096", "kind": "norm", "rows": 4096, "cols": 4096, "dtype": "bf16", "residual": True,
         "q8": True},
        # an ordinary fp32 activation whose sizes are multiples of nothing
        {"name": "norm_5000x1003_f32", "kind": "norm", "rows": 5000, "cols": 1003, "dtype": "f32", "residual": False,
         "q8": False},
        # the norm's backward in a training step
        {"name": "norm_bwd_8192x2048", "kind": "norm_bwd", "rows": 8192, "cols": 2048, "dtype": "bf16", "residual": True},
        # a wide layer's forward in training: bias, GELU, the pre-activation kept
        {"name": "linear_4096x1024x4096", "kind": "linear", "m": 4096, "k": 1024, "n": 4096, "dtype": "bf16",
         "trans_w": False, "act": "gelu", "bias": True, "residual": False, "save": True},
        # a layer that ends a residual block, of sizes that are multiples of nothing
        {"name": "linear_2500x1003x1499", "kind": "linear", "m": 2500, "k": 1003, "n": 1499, "dtype": "f16",
         "trans_w": False, "act": "none", "bias": True, "residual": True, "save": False},
        # serving one new token: the weight is read once
        {"name": "linear_1x4096x8192", "kind": "linear", "m": 1, "k": 4096, "n": 8192, "dtype": "bf16", "trans_w": True,
         "act": "silu", "bias": False, "residual": False, "save": False},
        # the backward of a wide layer
        {"name": "linear_bwd_4096x1024x4096", "kind": "linear_bwd", "m": 4096, "k": 1024, "n": 4096, "dtype": "bf16",
         "trans_w": False, "act": "gelu"},
        # a prompt's tokens through an 8-bit layer
        {"name": "linear_q8_4096x4096x4096", "kind": "linear_q8", "m": 4096, "k": 4096, "n": 4096, "dtype": "bf16",
         "act": "none", "bias": False, "residual": True},
        # sixteen sequences' new tokens through an 8-bit layer
        {"name": "linear_q8_16x8192x8192", "kind": "linear_q8", "m": 16, "k": 8192, "n": 8192, "dtype": "bf16",
         "act": "relu", "bias": True, "residual": False},
        # the optimizer step of a small fp32 network
        {"name": "adamw_small_f32", "kind": "adamw", "layers": 3, "width": 784, "inner": 1024, "dtype": "f32",
         "master": False, "q8": False},
        # the largest: a model of 200 million parameters, bf16 with fp32 masters and 8-bit moments
        {"name": "adamw_200m_q8", "kind": "adamw", "layers": 24, "width": 1024, "inner": 4096, "dtype": "bf16",
         "master": True, "q8": True},
    ]


def _size(rng, low, high):
    """A size spread over the logarithm of [low, high]; about half of the
    larger ones are multiples of 64, as layer widths often are."""
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if v >= 128 and rng.random() < 0.5:
        v = v // 64 * 64
    return max(low, min(high, v))


def draw(rng):
    kind = rng.choice(["norm", "norm_bwd", "linear", "linear", "linear_bwd", "linear_q8", "adamw"])
    dtype = rng.choice(["bf16", "f16", "f32"])
    if kind in ("norm", "norm_bwd"):
        while True:
            r, c = _size(rng, 1, 65536), _size(rng, 8, 65536)
            if r * c <= 1 << 25:
                break
        case = {"kind": kind, "rows": r, "cols": c, "dtype": dtype, "residual": rng.random() < 0.6}
        if kind == "norm":
            case["q8"] = rng.random() < 0.4
        return case
    if kind == "adamw":
        q8 = rng.random() < 0.6
        return {"kind": kind, "layers": rng.randint(1, 16), "width": _size(rng, 16, 1024), "inner": _size(rng, 16, 4096),
                "dtype": dtype, "master": dtype != "f32" and rng.random() < 0.5, "q8": q8}
    while True:  # one to a few rows when serving, many in training
        m = _size(rng, 1, 64) if kind != "linear_bwd" and rng.random() < 0.4 else _size(rng, 64, 8192)
        k, n = _size(rng, 32, 8192), _size(rng, 32, 8192)
        if m * k * n <= (1 << 34 if dtype == "f32" or kind == "linear_bwd" else 1 << 35):
            break
    act = rng.choice(["none", "relu", "sigmoid", "tanh", "gelu", "silu"])
    case = {"kind": kind, "m": m, "k": k, "n": n, "dtype": dtype, "act": act}
    if kind == "linear_q8":
        case["dtype"] = rng.choice(["bf16", "f16"])
    else:
        case["trans_w"] = rng.random() < 0.5
    if kind != "linear_bwd":
        case.update({"bias": rng.random() < 0.5, "residual": rng.random() < 0.5})
    if kind == "linear":
        case["save"] = rng.random() < 0.5
    return case


# ----------------------------------------------------------------- inputs


def _normal(g, shape, dtype=torch.float32, std=1.0, mean=0.0):
    return torch.empty(shape, dtype=torch.float32, device="cuda").normal_(mean, std, generator=g).to(dtype)


def _rows_to_8_bits(x):
    """(codes, scales) of the rows of x."""
    x = x.float()
    scale = x.abs().amax(1) / 448.0
    scale = torch.where(scale < _TINY, torch.zeros_like(scale), scale)
    inv = torch.where(scale == 0, torch.zeros_like(scale), 1.0 / scale)
    return (x * inv[:, None]).to(_F8), scale


def _adamw_sizes(case):
    """Tensors of the model: per layer two weights, their biases and a norm's weight."""
    w, f = case["width"], case["inner"]
    return [w * f, f, f * w, w, w] * case["layers"]


def _inputs(case, seed):
    """The tensors a program holds before the call."""
    g, kind = torch.Generator(device="cuda").manual_seed(int(seed)), case["kind"]
    t = _TORCH[case["dtype"]]
    if kind == "norm":
        r, c = case["rows"], case["cols"]
        v = {"x": _normal(g, (r, c), t), "w": _normal(g, (c,), t, 0.1, 1.0)}
        if case["residual"]:
            v["res"] = _normal(g, (r, c), t, 2.0)
        return v
    if kind == "norm_bwd":
        r, c = case["rows"], case["cols"]
        v = {"h": _normal(g, (r, c), t, 2.0), "w": _normal(g, (c,), t, 0.1, 1.0), "dy": _normal(g, (r, c), t)}
        v["rstd"] = torch.rsqrt(v["h"].float().square().mean(1) + EPS)
        if case["residual"]:
            v["dh"] = _normal(g, (r, c), t)
        return v
    if kind == "adamw":
        blocks = [(s + BLOCK - 1) // BLOCK for s in _adamw_sizes(case)]
        total = sum(blocks) * BLOCK
        v = {"grad": _normal(g, (total,), t, 1e-3), "master": _normal(g, (total,), torch.float32, 0.02),
             "m": _normal(g, (total,), torch.float32, 3e-4),
             "r": _normal(g, (total,), torch.float32, 1e-3).abs_().add_(1e-5)}
        # every tensor starts on a block; what lies between two of them stays zero
        at = 0
        for size, nb in zip(_adamw_sizes(case), blocks):
            for name in v:
                v[name][at + size:at + nb * BLOCK] = 0
            at += nb * BLOCK
        v["p"] = v["master"].to(t)
        if not case["master"]:
            del v["master"]
        return v
    m, k, n = case["m"], case["k"], case["n"]
    if kind == "linear_q8":
        v = {}
        v["x"], v["x_scale"] = _rows_to_8_bits(_normal(g, (m, k)))
        v["w"], v["w_scale"] = _rows_to_8_bits(_normal(g, (n, k), std=1.0 / math.sqrt(k)))
    else:
        v = {"x": _normal(g, (m, k), t),
             "w": _normal(g, (n, k) if case["trans_w"] else (k, n), t, 1.0 / math.sqrt(k))}
    if kind == "linear_bwd":
        v.update({"z": _normal(g, (m, n), t), "dy": _normal(g, (m, n), t)})
        return v
    if case["bias"]:
        v["bias"] = _normal(g, (n,), t, 0.1)
    if case["residual"]:
        v["res"] = _normal(g, (m, n), t)
    return v


def prepare(case, seed):
    """Inputs, output buffers and the optimizer that a program keeps."""
    v, kind, t = _inputs(case, seed), case["kind"], _TORCH[case["dtype"]]

    def new(*shape, dtype=t):
        return torch.empty(shape, dtype=dtype, device="cuda")

    out = {}
    if kind == "norm":
        r, c = case["rows"], case["cols"]
        if case["residual"]:
            out["h"] = new(r, c)
        if case["q8"]:
            out.update({"q": new(r, c, dtype=_F8), "scale": new(r, dtype=torch.float32)})
        else:
            out["y"] = new(r, c)
        out["rstd"] = new(r, dtype=torch.float32)
    elif kind == "norm_bwd":
        out = {"dx": torch.empty_like(v["h"]), "dw": torch.empty_like(v["w"])}
    elif kind == "linear_bwd":
        out = {"dz": torch.empty_like(v["z"]), "dx": torch.empty_like(v["x"]), "dw": torch.empty_like(v["w"]),
               "db": new(case["n"])}
    elif kind == "adamw":
        out["p"] = v["p"]
        if case["master"]:
            out["master"] = v["master"]
        if case["q8"]:
            for name in ("m", "r"):
                q, scale = _rows_to_8_bits(v.pop(name).view(-1, BLOCK))
                out[name], out[name + "_scale"] = q, scale
        else:
            out["m"], out["v"] = v.pop("m"), v.pop("r").square_()
    else:
        out["y"] = new(case["m"], case["n"])
        if case.get("save"):
            out["z"] = new(case["m"], case["n"])
    state = {"case": case, "in": v, "out": out, "step": 100, "opt": None}
    for names in (v, out):
        state.update({name: Buffer(x) for name, x in names.items()})
    if kind == "adamw":
        blocks = [(s + BLOCK - 1) // BLOCK for s in _adamw_sizes(case)]
        # weights decay, biases and norm weights do not
        decay = [_DECAY if i % 5 in (0, 2) else 0.0 for i in range(len(blocks))]
        state["decay"] = torch.tensor(decay, device="cuda").repeat_interleave(torch.tensor(blocks, device="cuda"))[:, None]
        if own:  # the optimizer object, which holds the list of tensors
            state["opt"] = _optimizer(case, state, decay)
    return state


def _optimizer(case, state, decay):
    from cortexmind_amd import engine

    tensors, at = [], 0
    for size, wd in zip(_adamw_sizes(case), decay):
        nb = (size + BLOCK - 1) // BLOCK

        def part(name, step=1):
            t = state[name].tensor.view(-1)
            return Buffer(t[at // step:(at + size + step - 1) // step])

        entry = {"p": part("p"), "g": part("grad"), "n": size, "decay": wd, "m": part("m")}
        if case["master"]:
            entry["master"] = part("master")
        if case["q8"]:
            entry.update({"v": part("r"), "m_scale": part("m_scale", BLOCK), "v_scale": part("r_scale", BLOCK)})
        else:
            entry["v"] = part("v")
        tensors.append(entry)
        at += nb * BLOCK
    dt = _dtype(case)
    return engine.AdamW(tensors, dt, dt, state_8bit=case["q8"])


# -------------------------------------------------------------- one pass


def run(state):
    case = state["case"]
    if own:
        _OWN[case["kind"]](state, case)
    else:
        _PLAIN[case["kind"]](state["in"], state["out"], case, state)
    return state["out"]


def _dtype(case):
    from cortexmind_amd import _lib

    return {"f32": _lib.DT_F32, "bf16": _lib.DT_BF16, "f16": _lib.DT_F16}[case["dtype"]]


def _act_code(case):
    from cortexmind_amd import engine

    return {"none": engine.ACT_NONE, "relu": engine.ACT_RELU, "sigmoid": engine.ACT_SIGMOID, "tanh": engine.ACT_TANH,
            "gelu": engine.ACT_GELU, "silu": engine.ACT_SILU}[case["act"]]


def _own_norm(s, case):
    from cortexmind_amd import engine

    engine.rmsnorm.forward(s["x"], s["w"], s.get("y"), case["rows"], case["cols"], _dtype(case), eps=EPS,
                           residual=s.get("res"), H=s.get("h"), Q=s.get("q"), scale=s.get("scale"), rstd=s["rstd"])


def _own_norm_bwd(s, case):
    from cortexmind_amd import engine

    engine.rmsnorm.backward(s["h"], s["rstd"], s["w"], s["dy"], s["dx"], s["dw"], case["rows"], case["cols"],
                            _dtype(case), dH=s.get("dh"))


def _own_linear(s, case):
    from cortexmind_amd import engine

    engine.linear.forward(s["x"], s["w"], s["y"], case["m"], case["k"], case["n"], _dtype(case), bias=s.get("bias"),
                          act=_act_code(case), residual=s.get("res"), Z=s.get("z"), trans_w=case["trans_w"])


def _own_linear_bwd(s, case):
    from cortexmind_amd import engine

    engine.linear.backward(s["x"], s["w"], s["z"], s["dy"], s["dz"], s["dx"], s["dw"], s["db"], case["m"], case["k"],
                           case["n"], _dtype(case), act=_act_code(case), trans_w=case["trans_w"])


def _own_linear_q8(s, case):
    from cortexmind_amd import engine

    engine.linear.forward_q8(s["x"], s["x_scale"], s["w"], s["w_scale"], s["y"], case["m"], case["k"], case["n"],
                             _dtype(case), bias=s.get("bias"), act=_act_code(case), residual=s.get("res"))


def _own_adamw(s, case):
    s["opt"].step(_LR, s["step"], beta1=_BETA1, beta2=_BETA2, eps=_ADAM_EPS, seed=_SEED + s["step"])
    s["step"] += 1


_OWN = {"norm": _own_norm, "norm_bwd": _own_norm_bwd, "linear": _own_linear, "linear_bwd": _own_linear_bwd,
        "linear_q8": _own_linear_q8, "adamw": _own_adamw}


# --------------------------------------------- the operators in plain form


def _plain_norm(v, out, case, _):
    h = v["x"]
    if case["residual"]:
        h = (v["x"].float() + v["res"].float()).to(h.dtype)
        out["h"] = h
    h = h.float()
    rstd = 1.0 / torch.sqrt((h * h).mean(1) + EPS)
    y = h * rstd[:, None] * v["w"].float()
    out["rstd"] = rstd
    if case["q8"]:
        out["q"], out["scale"] = _rows_to_8_bits(y)
    else:
        out["y"] = y.to(v["x"].dtype)


def _plain_norm_bwd(v, out, case, _):
    dy, xhat = v["dy"].float(), v["h"].float() * v["rstd"][:, None]
    g = dy * v["w"].float()
    dx = v["rstd"][:, None] * (g - xhat * (g * xhat).mean(1, keepdim=True))
    if case["residual"]:
        dx = dx + v["dh"].float()
    out["dx"] = dx.to(v["h"].dtype)
    out["dw"] = (dy * xhat).sum(0).to(v["w"].dtype)


def _act(name, z):
    if name == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if name == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-z))
    if name == "tanh":
        return torch.tanh(z)
    if name == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    if name == "silu":
        return z / (1.0 + torch.exp(-z))
    return z


def _slope(name, z):
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "sigmoid":
        y = 1.0 / (1.0 + torch.exp(-z))
        return y * (1.0 - y)
    if name == "tanh":
        y = torch.tanh(z)
        return 1.0 - y * y
    if name == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))
    if name == "silu":
        y = 1.0 / (1.0 + torch.exp(-z))
        return y * (1.0 + z * (1.0 - y))
    return torch.ones_like(z)


def _finish(z, v, out, case):
    """Bias, activation and residual of a product."""
    if case["bias"]:
        z = z + v["bias"].float()
    y = _act(case["act"], z)
    if case["residual"]:
        y = y + v["res"].float()
    t = out["y"].dtype
    if case.get("save"):
        out["z"] = z.to(t)
    out["y"] = y.to(t)


def _plain_linear(v, out, case, _):
    w = v["w"].float()
    _finish(v["x"].float() @ (w.t() if case["trans_w"] else w), v, out, case)


def _plain_linear_q8(v, out, case, _):
    z = (v["x"].float() @ v["w"].float().t()) * v["x_scale"][:, None] * v["w_scale"][None, :]
    _finish(z, v, out, case)


def _plain_linear_bwd(v, out, case, _):
    t = v["x"].dtype
    dz = v["dy"].float() * _slope(case["act"], v["z"].float())
    x, w = v["x"].float(), v["w"].float()
    out["dz"] = dz.to(t)
    out["db"] = dz.sum(0).to(t)
    out["dx"] = (dz @ (w if case["trans_w"] else w.t())).to(t)
    out["dw"] = (dz.t() @ x if case["trans_w"] else x.t() @ dz).to(t)


def noise(seed, n, device):
    """32 random bits (as int64) of the values numbered 0 .. n - 1, n below
    2^32, in a step of this seed: two multiply-and-shift rounds over the
    number and the seed."""
    c = torch.arange(n, device=device, dtype=torch.int64)
    c = c ^ (seed * 0x9E3779B1 & 0xFFFFFFFF)
    for mul in (0x85EBCA6B, 0xC2B2AE35):
        c = c ^ (c >> 16)
        c = (c * mul) & 0xFFFFFFFF
    return c ^ (c >> 16)


def _rounded(a, bits):
    """a >= 0, at most 448, rounded to e4m3 up or down: up with the probability
    of the distance, decided by 16 random bits."""
    low = a < 2.0 ** -6  # there the steps are even: adding 2^-6 makes them so
    a = torch.where(low, a + 2.0 ** -6, a)
    a = ((a.view(torch.int32) + (bits << 4).to(torch.int32)) & ~0xFFFFF).view(torch.float32)
    return torch.where(low, a - 2.0 ** -6, a)


def _moment_8_bits(x, bits, root):
    """Blocks of a moment as codes and scales."""
    scale = x.abs().amax(1, keepdim=True) / 448.0
    scale = torch.where(scale < _TINY, torch.zeros_like(scale), scale)
    inv = torch.where(scale == 0, torch.zeros_like(scale), 1.0 / scale)
    a = (x.abs() * inv).clamp(max=448.0)
    q = _rounded(a, bits)
    if root:
        q = torch.where((a > 0) & (q == 0), torch.full_like(q, 2.0 ** -9), q)
    else:
        q = torch.copysign(q, x)
    return q.to(_F8), scale[:, 0]


def _plain_adamw(v, out, case, state):
    t = state["step"]
    state["step"] += 1
    p = (out["master"] if case["master"] else out["p"]).float().view(-1, BLOCK)
    g = v["grad"].float().view(-1, BLOCK)
    if case["q8"]:
        m = out["m"].float() * out["m_scale"][:, None]
        r = out["r"].float() * out["r_scale"][:, None]
        w = r * r
    else:
        m, w = out["m"].view(-1, BLOCK), out["v"].view(-1, BLOCK)
    m = _BETA1 * m + (1.0 - _BETA1) * g
    w = _BETA2 * w + (1.0 - _BETA2) * (g * g)
    r = torch.sqrt(w)
    p = p * (1.0 - _LR * state["decay"])
    p = p - (_LR / (1.0 - _BETA1 ** t)) * m / (r / math.sqrt(1.0 - _BETA2 ** t) + _ADAM_EPS)
    if case["master"]:
        out["master"].copy_(p.view(-1))
    out["p"].copy_(p.view(-1))
    if case["q8"]:
        bits = noise(_SEED + t, p.numel(), p.device).view(-1, BLOCK)
        q, scale = _moment_8_bits(m, bits & 0xFFFF, False)
        out["m"].copy_(q)
        out["m_scale"].copy_(scale)
        q, scale = _moment_8_bits(r, bits >> 16, True)
        out["r"].copy_(q)
        out["r_scale"].copy_(scale)
    else:
        out["m"].copy_(m.view(-1))
        out["v"].copy_(w.view(-1))


_PLAIN = {"norm": _plain_norm, "norm_bwd": _plain_norm_bwd, "linear": _plain_linear, "linear_bwd": _plain_linear_bwd,
          "linear_q8": _plain_linear_q8, "adamw": _plain_adamw}


# ------------------------------------------------------------------- work


def work(case):
    """Compulsory traffic (each input read once, each output written once)
    and the operations of the products."""
    kind, e = case["kind"], 4 if case["dtype"] == "f32" else 2
    if kind == "norm":
        r, c = case["rows"], case["cols"]
        streams = e * (3 if case["residual"] else 1) + (1 if case["q8"] else e)
        return {"bytes": r * c * streams + e * c + 4 * r * (2 if case["q8"] else 1), "flops": 0}
    if kind == "norm_bwd":
        r, c = case["rows"], case["cols"]
        return {"bytes": r * c * e * (4 if case["residual"] else 3) + 2 * e * c + 4 * r, "flops": 0}
    if kind == "adamw":
        n = sum(_adamw_sizes(case))
        each = e + (8 + e if case["master"] else 2 * e) + (4 + 16 / BLOCK if case["q8"] else 16)
        return {"bytes": n * each, "flops": 0}
    m, k, n = case["m"], case["k"], case["n"]
    if kind == "linear_bwd":
        return {"bytes": e * (2 * m * k + 2 * k * n + 3 * m * n + n), "flops": 4 * m * k * n}
    io = 1 if kind == "linear_q8" else e
    bytes_ = io * (m * k + k * n) + e * m * n * (1 + case["residual"] + case.get("save", False)) + e * n * case["bias"]
    if kind == "linear_q8":
        bytes_ += 4 * (m + n)
    return {"bytes": bytes_, "flops": 2 * m * k * n}


# ------------------------------------------------------------ in 64 bits


def exact(case, seed):
    """The definitions in float64.  An 8-bit value has none: it is one of the
    two representable values beside the exact one."""
    v, kind = _inputs(case, seed), case["kind"]
    d = {name: x.double() for name, x in v.items()}
    if kind == "norm":
        h, out = d["x"], {}
        if case["residual"]:
            out["h"] = d["x"] + d["res"]
            h = out["h"].to(v["x"].dtype).double()
        out["rstd"] = (h.pow(2).sum(1) / case["cols"] + EPS).pow(-0.5)
        y = h * out["rstd"][:, None] * d["w"]
        if case["q8"]:
            out["q"], out["scale"] = None, y.abs().max(1).values / 448.0
        else:
            out["y"] = y
        return out
    if kind == "norm_bwd":
        n = d["h"] * d["rstd"][:, None]
        wdy = d["dy"] * d["w"]
        along = (wdy * n).sum(1, keepdim=True) / case["cols"]
        return {"dx": (wdy - along * n) * d["rstd"][:, None] + d.get("dh", 0.0), "dw": (d["dy"] * n).sum(0)}
    if kind == "adamw":
        return _exact_adamw(case, d, v["p"].dtype)
    if kind == "linear_bwd":
        z = d["z"].requires_grad_()
        (slope,) = torch.autograd.grad(_exact_act(case["act"], z).sum(), z)
        dz = d["dy"] * slope
        w = d["w"].t().contiguous() if case["trans_w"] else d["w"]
        dw = d["x"].t().contiguous() @ dz
        return {"dz": dz, "db": dz.sum(0), "dx": dz @ w.t().contiguous(),
                "dw": dw.t().contiguous() if case["trans_w"] else dw}
    x, w = d["x"], d["w"]
    if kind == "linear_q8":
        x, w = x * d["x_scale"][:, None], (w * d["w_scale"][:, None]).t().contiguous()
    elif case["trans_w"]:
        w = w.t().contiguous()
    z = x @ w + d.get("bias", 0.0)
    out = {"y": _exact_act(case["act"], z) + d.get("res", 0.0)}
    if case.get("save"):
        out["z"] = z
    return out


def _exact_act(name, z):
    if name == "relu":
        return z.clamp(min=0.0)
    if name == "sigmoid":
        return torch.sigmoid(z)
    if name == "tanh":
        return torch.tanh(z)
    if name == "gelu":
        return z * torch.special.ndtr(z)
    if name == "silu":
        return z * torch.sigmoid(z)
    return z * 1.0


def _exact_adamw(case, d, dtype):
    def held(name):  # what the 8-bit state stands for
        q, scale = _rows_to_8_bits(d[name].float().view(-1, BLOCK))
        return (q.double() * scale.double()[:, None]).view(-1)

    blocks = [(s + BLOCK - 1) // BLOCK for s in _adamw_sizes(case)]
    decay = torch.cat([torch.full((nb * BLOCK,), _DECAY if i % 5 in (0, 2) else 0.0, dtype=torch.float64, device="cuda")
                       for i, nb in enumerate(blocks)])
    m = held("m") if case["q8"] else d["m"]
    v = held("r") ** 2 if case["q8"] else d["r"].float().square().double()
    m = _BETA1 * m + (1 - _BETA1) * d["grad"]
    v = _BETA2 * v + (1 - _BETA2) * d["grad"] ** 2
    p = d["master"] if case["master"] else d["p"]
    mhat, vhat = m / (1 - _BETA1 ** 100), v / (1 - _BETA2 ** 100)
    p = p - _LR * (decay * p + mhat / (vhat.sqrt() + _ADAM_EPS))
    out = {"p": p}
    if case["master"]:
        out["master"] = p
    if case["q8"]:
        out.update({"m": None, "r": None, "m_scale": m.view(-1, BLOCK).abs().amax(1) / 448,
                    "r_scale": v.view(-1, BLOCK).sqrt().amax(1) / 448})
    else:
        out.update({"m": m, "v": v})
    return out
