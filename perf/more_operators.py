"""The two ends of a model over its vocabulary, in training and serving:
timed and compared cases.

Every case is a dict of plain values; ``kind`` names the operator and the
other fields its sizes and options:

* ``embed``: rows of a table looked up by token and scaled;
* ``embed_bwd``: the table's gradient: the sum of the rows of dy that share a
  token, in the table's type or in fp32;
* ``norm``: h = x + residual and the layer norm of h's rows with weight and
  bias;
* ``norm_bwd``: its backward: the gradient of the rows, joined with the one
  that reaches h past the norm, and those of weight and bias;
* ``logprob``: log probabilities of given tokens under softmax(scale * logits),
  the distribution's entropy, the log of its sum of exponentials, and the
  ``top`` most likely tokens (ties: the lowest id) with their log
  probabilities;
* ``logprob_bwd``: the gradient of the logits from those of the log
  probabilities and the entropies;
* ``distill``: the divergence of softmax(scale * logits) from a teacher's
  distribution over its ``top`` tokens, softmax(scale * teacher);
* ``distill_bwd``: the gradient of the logits.

``own`` is false: ``run`` computes the operators from elementary torch
operations, in 32 bits, rounded once at the end.  ``own`` is true: ``run``
makes the library's calls.

Logits are rows ``ld`` elements apart, of which the first ``vocab`` count.  A
negative token is padding: a row of zeros when looked up, no part of a
gradient, log probability 0; a negative teacher id is no entry.
"""
import math

import numpy as np
import torch

own = False

EPS = 1e-5
_TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BANNED, _EVERY = 5, 16  # token ids that a mask bans: id % 16 == 5


class Buffer:
    """A GPU tensor as the engine's calls take their operands."""

    def __init__(self, tensor):
        self.tensor = tensor
        self.ptr = tensor.data_ptr()
        self.size = tensor.numel()


# ------------------------------------------------------------------ cases


def listed():
    return [
        # the smallest call: one new token's row, where latency counts
        {"name": "embed_1x4096", "kind": "embed", "tokens": 1, "vocab": 32768, "cols": 4096, "dtype": "bf16"},
        # a batch of sequences looked up in an fp32 table whose sizes are multiples of nothing
        {"name": "embed_20001x1003_f32", "kind": "embed", "tokens": 20001, "vocab": 50001, "cols": 1003, "dtype": "f32"},
        # the table's gradient in a training step; a few tokens make up a large part of the text
        {"name": "embed_bwd_32768x2048", "kind": "embed_bwd", "tokens": 32768, "vocab": 65536, "cols": 2048,
         "dtype": "bf16", "grad": "bf16"},
        # a small batch's gradient in fp32 from fp16 rows, of sizes that are multiples of nothing
        {"name": "embed_bwd_5003x771_f16", "kind": "embed_bwd", "tokens": 5003, "vocab": 10007, "cols": 771,
         "dtype": "f16", "grad": "f32"},
        # sixteen sequences' new tokens before a layer
        {"name": "norm_16x4096", "kind": "norm", "rows": 16, "cols": 4096, "dtype": "bf16", "residual": True},
        # a batch of rows whose sizes are multiples of nothing
        {"name": "norm_20001x1003_f16", "kind": "norm", "rows": 20001, "cols": 1003, "dtype": "f16", "residual": False},
        # the norm's backward in a training step
        {"name": "norm_bwd_8192x2048", "kind": "norm_bwd", "rows": 8192, "cols": 2048, "dtype": "bf16", "residual": True},
        # sixteen sequences' next tokens with their alternatives, as a server reports them
        {"name": "logprob_16x131072", "kind": "logprob", "rows": 16, "vocab": 131072, "ld": 131072, "dtype": "bf16",
         "top": 20, "scale": 1.0, "masked": True},
        # scoring a batch of texts: rows of an odd length, a few alternatives, a temperature of 0.8
        {"name": "logprob_2500x50001_f16", "kind": "logprob", "rows": 2500, "vocab": 50001, "ld": 50001, "dtype": "f16",
         "top": 5, "scale": 1.25, "masked": False},
        # the policy step of a model trained by reward, with a bonus for entropy; a vocabulary padded for its product
        {"name": "logprob_bwd_2048x65500", "kind": "logprob_bwd", "rows": 2048, "vocab": 65500, "ld": 65536,
         "dtype": "bf16", "scale": 1.0, "masked": False, "entropy": True},
        # the largest: a training step's loss against a teacher's 64 likeliest tokens, at a temperature of 2
        {"name": "distill_2048x131072", "kind": "distill", "rows": 2048, "vocab": 131072, "ld": 131072, "dtype": "bf16",
         "top": 64, "scale": 0.5, "masked": False},
        # its gradient in fp32, rows of an odd length
        {"name": "distill_bwd_1000x30011_f32", "kind": "distill_bwd", "rows": 1000, "vocab": 30011, "ld": 30011,
         "dtype": "f32", "top": 17, "scale": 1.0, "masked": False},
    ]


def _size(rng, low, high):
    """A size spread over the logarithm of [low, high]; about half of the
    larger ones are multiples of 64, as widths and vocabularies often are."""
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if v >= 128 and rng.random() < 0.5:
        v = v // 64 * 64
    return max(low, min(high, v))


def draw(rng):
    kind = rng.choice(["embed", "embed_bwd", "norm", "norm_bwd", "logprob", "logprob_bwd", "distill", "distill_bwd"])
    dtype = rng.choice(["bf16", "f16", "f32"])
    most = 1 << (26 if dtype == "f32" else 27)  # elements of the largest operand
    if kind in ("norm", "norm_bwd"):
        while True:
            r, c = _size(rng, 1, 65536), _size(rng, 8, 65536)
            if r * c <= most // 4:
                break
        return {"kind": kind, "rows": r, "cols": c, "dtype": dtype, "residual": rng.random() < 0.6}
    if kind in ("embed", "embed_bwd"):
        while True:
            t, v, c = _size(rng, 1, 131072), _size(rng, 16, 262144), _size(rng, 8, 8192)
            if t * c <= most // 2 and v * c <= most:
                break
        case = {"kind": kind, "tokens": t, "vocab": v, "cols": c, "dtype": dtype}
        if kind == "embed_bwd":
            case["grad"] = dtype if rng.random() < 0.5 else "f32"
        return case
    while True:
        r, v = _size(rng, 1, 16384), _size(rng, 16, 262144)
        if r * v <= most:
            break
    case = {"kind": kind, "rows": r, "vocab": v, "ld": (v + 63) // 64 * 64 if rng.random() < 0.3 else v, "dtype": dtype,
            "scale": rng.choice([0.5, 1.0, 1.0, 1.25, 2.0]), "masked": rng.random() < 0.3}
    if kind == "logprob":
        case["top"] = min(rng.choice([0, 1, 5, 20, 64]), v // 2)
    elif kind == "logprob_bwd":
        case["entropy"] = rng.random() < 0.5
    else:
        case["top"] = min(_size(rng, 1, 256), v // 2)
    return case


# ----------------------------------------------------------------- inputs


def _normal(g, shape, dtype=torch.float32, std=1.0, mean=0.0):
    return torch.empty(shape, dtype=torch.float32, device="cuda").normal_(mean, std, generator=g).to(dtype)


def _tokens(g, n, vocab):
    """Token ids as a text has them, id i in proportion to 1 / (i + 1); one in
    64 is padding."""
    u = torch.rand(n, device="cuda", generator=g, dtype=torch.float64)
    ids = (torch.exp(u * math.log(vocab + 1.0)) - 1.0).long().clamp(0, vocab - 1)
    pad = torch.rand(n, device="cuda", generator=g) < 1.0 / 64.0
    return torch.where(pad, -1, ids).to(torch.int32)


def _scale(case):
    """A lookup's scale: the root of the row's length."""
    return float(np.float32(math.sqrt(case["cols"])))


def _allowed(ids):
    return torch.where(ids % _EVERY == _BANNED, ids - 1, ids)


def _lse(x, scale):
    """log sum exp of the scaled rows, in 64 bits, a slice at a time."""
    step = max(1, (1 << 25) // x.shape[1])
    return torch.cat([torch.logsumexp(x[i:i + step].double() * scale, 1) for i in range(0, x.shape[0], step)])


def _inputs(case, seed):
    """The tensors a program holds before the call."""
    g, kind = torch.Generator(device="cuda").manual_seed(int(seed)), case["kind"]
    t = _TORCH[case["dtype"]]
    if kind == "embed":
        return {"table": _normal(g, (case["vocab"], case["cols"]), t, 0.02), "ids": _tokens(g, case["tokens"], case["vocab"])}
    if kind == "embed_bwd":
        return {"ids": _tokens(g, case["tokens"], case["vocab"]), "dy": _normal(g, (case["tokens"], case["cols"]), t, 0.01)}
    if kind in ("norm", "norm_bwd"):
        r, c = case["rows"], case["cols"]
        # rows whose mean is not zero, as after a few residual layers
        off = _normal(g, (r, 1))
        v = {"x": (_normal(g, (r, c), std=2.0) + off).to(t), "w": _normal(g, (c,), t, 0.1, 1.0)}
        if kind == "norm":
            v["bias"] = _normal(g, (c,), t, 0.1)
            if case["residual"]:
                v["res"] = _normal(g, (r, c), t)
            return v
        v["h"] = v.pop("x")
        d = v["h"].double()
        mean = d.mean(1)
        v["mean"] = mean.float()
        v["rstd"] = ((d - mean[:, None]).square().mean(1) + EPS).rsqrt().float()
        v["dy"] = _normal(g, (r, c), t)
        if case["residual"]:
            v["dh"] = _normal(g, (r, c), t)
        return v
    r, n, ld = case["rows"], case["vocab"], case["ld"]
    x = _normal(g, (r, ld), t, 3.0)
    if case["masked"]:
        x[:, _BANNED::_EVERY] = -math.inf
    v = {"logits": x}
    if kind in ("logprob", "logprob_bwd"):
        ids = torch.randint(n, (r,), device="cuda", generator=g)
        ids = _allowed(ids) if case["masked"] else ids
        v["tokens"] = torch.where(torch.rand(r, device="cuda", generator=g) < 1.0 / 64.0, -1, ids).to(torch.int32)
    else:
        k = case["top"]
        # the teacher's distinct tokens: k steps of an odd stride round the vocabulary, from a place of the row's own
        first = torch.randint(n, (r, 1), device="cuda", generator=g)
        ids = (first + torch.arange(k, device="cuda") * max(1, n // k)) % n
        # two banned neighbours may become one token twice
        v["ids"] = (_allowed(ids) if case["masked"] else ids).to(torch.int32)
        v["teacher"] = _normal(g, (r, k), std=2.0, mean=5.0)
    if kind == "logprob_bwd":
        v["dlogp"] = _normal(g, (r,))
        if case["entropy"]:
            v["dentropy"] = _normal(g, (r,), std=0.1)
    if kind == "distill_bwd":
        v["dloss"] = torch.rand(r, device="cuda", generator=g) + 0.5
    if kind in ("logprob_bwd", "distill_bwd"):
        lse = _lse(x[:, :n], case["scale"])
        v["lse"] = lse.float()
        if case.get("entropy"):
            v["entropy"] = _entropy64(x[:, :n], case["scale"], lse).float()
    return v


def _entropy64(x, scale, lse):
    step = max(1, (1 << 25) // x.shape[1])
    out = []
    for i in range(0, x.shape[0], step):
        logp = x[i:i + step].double() * scale - lse[i:i + step, None]
        out.append(-(logp.exp() * torch.where(logp == -math.inf, 0.0, logp)).sum(1))
    return torch.cat(out)


def prepare(case, seed):
    """Inputs and output buffers."""
    v, kind, t = _inputs(case, seed), case["kind"], _TORCH[case["dtype"]]

    def new(*shape, dtype=t):
        return torch.empty(shape, dtype=dtype, device="cuda")

    f32 = torch.float32
    if kind == "embed":
        out = {"y": new(case["tokens"], case["cols"])}
    elif kind == "embed_bwd":
        out = {"dw": new(case["vocab"], case["cols"], dtype=_TORCH[case["grad"]])}
    elif kind == "norm":
        r, c = case["rows"], case["cols"]
        out = {"y": new(r, c), "mean": new(r, dtype=f32), "rstd": new(r, dtype=f32)}
        if case["residual"]:
            out["h"] = new(r, c)
    elif kind == "norm_bwd":
        out = {"dx": torch.empty_like(v["h"]), "dw": torch.empty_like(v["w"]), "db": torch.empty_like(v["w"])}
    elif kind == "logprob":
        r, k = case["rows"], case["top"]
        out = {name: new(r, dtype=f32) for name in ("logp", "entropy", "lse")}
        if k:
            out.update({"top_logp": new(r, k, dtype=f32), "top_ids": new(r, k, dtype=torch.int32)})
    elif kind == "distill":
        out = {name: new(case["rows"], dtype=f32) for name in ("loss", "lse")}
    else:
        out = {"dlogits": new(case["rows"], case["vocab"])}
    state = {"case": case, "in": v, "out": out}
    for names in (v, out):
        state.update({name: Buffer(x) for name, x in names.items()})
    return state


# -------------------------------------------------------------- one pass


def run(state):
    case = state["case"]
    if own:
        _OWN[case["kind"]](state, case)
    else:
        _PLAIN[case["kind"]](state["in"], state["out"], case)
    return state["out"]


def _code(name):
    from cortexmind_amd import _lib

    return {"f32": _lib.DT_F32, "bf16": _lib.DT_BF16, "f16": _lib.DT_F16}[name]


def _own_embed(s, case):
    from cortexmind_amd import engine

    engine.embedding.forward(s["table"], s["ids"], s["y"], case["tokens"], case["vocab"], case["cols"],
                             _code(case["dtype"]), scale=_scale(case))


def _own_embed_bwd(s, case):
    from cortexmind_amd import engine

    engine.embedding.backward(s["ids"], s["dy"], s["dw"], case["tokens"], case["vocab"], case["cols"],
                              _code(case["dtype"]), scale=_scale(case), g_dtype=_code(case["grad"]))


def _own_norm(s, case):
    from cortexmind_amd import engine

    engine.layernorm.forward(s["x"], s["w"], s["y"], case["rows"], case["cols"], _code(case["dtype"]), bias=s["bias"],
                             eps=EPS, residual=s.get("res"), H=s.get("h"), mean=s["mean"], rstd=s["rstd"])


def _own_norm_bwd(s, case):
    from cortexmind_amd import engine

    engine.layernorm.backward(s["h"], s["mean"], s["rstd"], s["w"], s["dy"], s["dx"], s["dw"], case["rows"],
                              case["cols"], _code(case["dtype"]), db=s["db"], dH=s.get("dh"))


def _own_logprob(s, case):
    from cortexmind_amd import engine

    engine.logprob.forward(s["logits"], s["tokens"], s["logp"], case["rows"], case["vocab"], _code(case["dtype"]),
                           scale=case["scale"], ld=case["ld"], entropy=s["entropy"], lse=s["lse"], top=case["top"],
                           top_logp=s.get("top_logp"), top_ids=s.get("top_ids"))


def _own_logprob_bwd(s, case):
    from cortexmind_amd import engine

    engine.logprob.backward(s["logits"], s["tokens"], s["lse"], s["dlogp"], s["dlogits"], case["rows"], case["vocab"],
                            _code(case["dtype"]), scale=case["scale"], ld=case["ld"], entropy=s.get("entropy"),
                            dentropy=s.get("dentropy"))


def _own_distill(s, case):
    from cortexmind_amd import engine

    engine.distill.forward(s["logits"], s["ids"], s["teacher"], s["loss"], s["lse"], case["rows"], case["vocab"],
                           case["top"], _code(case["dtype"]), scale=case["scale"], ld=case["ld"])


def _own_distill_bwd(s, case):
    from cortexmind_amd import engine

    engine.distill.backward(s["logits"], s["ids"], s["teacher"], s["lse"], s["dloss"], s["dlogits"], case["rows"],
                            case["vocab"], case["top"], _code(case["dtype"]), scale=case["scale"], ld=case["ld"])


_OWN = {"embed": _own_embed, "embed_bwd": _own_embed_bwd, "norm": _own_norm, "norm_bwd": _own_norm_bwd,
        "logprob": _own_logprob, "logprob_bwd": _own_logprob_bwd, "distill": _own_distill,
        "distill_bwd": _own_distill_bwd}


# --------------------------------------------- the operators in plain form


def _plain_embed(v, out, case):
    ids = v["ids"].long()
    y = v["table"][ids.clamp(min=0)].float() * _scale(case)
    out["y"] = torch.where(ids[:, None] < 0, 0.0, y).to(v["table"].dtype)


def _plain_embed_bwd(v, out, case):
    ids = v["ids"].long()
    # one row more, for the padding
    dw = torch.zeros((case["vocab"] + 1, case["cols"]), dtype=torch.float32, device=ids.device)
    dw.index_add_(0, torch.where(ids < 0, case["vocab"], ids), v["dy"].float())
    out["dw"] = (dw[:-1] * _scale(case)).to(out["dw"].dtype)


def _plain_norm(v, out, case):
    h = v["x"]
    if case["residual"]:
        h = (v["x"].float() + v["res"].float()).to(h.dtype)
        out["h"] = h
    h = h.float()
    mean = h.mean(1)
    c = h - mean[:, None]
    rstd = 1.0 / torch.sqrt((c * c).mean(1) + EPS)
    out["mean"], out["rstd"] = mean, rstd
    out["y"] = (c * rstd[:, None] * v["w"].float() + v["bias"].float()).to(v["x"].dtype)


def _plain_norm_bwd(v, out, case):
    dy, n = v["dy"].float(), (v["h"].float() - v["mean"][:, None]) * v["rstd"][:, None]
    g = dy * v["w"].float()
    dx = v["rstd"][:, None] * (g - g.mean(1, keepdim=True) - n * (g * n).mean(1, keepdim=True))
    if case["residual"]:
        dx = dx + v["dh"].float()
    out["dx"] = dx.to(v["h"].dtype)
    out["dw"] = (dy * n).sum(0).to(v["w"].dtype)
    out["db"] = dy.sum(0).to(v["w"].dtype)


def _log_sum(z):
    top = z.max(1, keepdim=True).values
    return top[:, 0] + torch.log(torch.exp(z - top).sum(1))


def _plain_logprob(v, out, case):
    x, ids = v["logits"][:, :case["vocab"]].float(), v["tokens"].long()
    z = x * case["scale"]
    lse = _log_sum(z)
    logp = z - lse[:, None]
    given = torch.gather(logp, 1, ids.clamp(min=0)[:, None])[:, 0]
    out["logp"] = torch.where(ids < 0, 0.0, given)
    out["entropy"] = -(torch.exp(logp) * torch.where(logp == -math.inf, 0.0, logp)).sum(1)
    out["lse"] = lse
    if case["top"]:
        # one number per value and place: larger values first, of equal ones the lower place
        bits = (x + 0.0).view(torch.int32).long()
        key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits) * (1 << 32) - torch.arange(case["vocab"], device=x.device)
        best = torch.topk(key, case["top"], dim=1).values
        place = torch.remainder(-best, 1 << 32)
        out["top_ids"] = place.to(torch.int32)
        out["top_logp"] = torch.gather(logp, 1, place)


def _plain_logprob_bwd(v, out, case):
    ids = v["tokens"].long()
    logp = v["logits"][:, :case["vocab"]].float() * case["scale"] - v["lse"][:, None]
    p = torch.exp(logp)
    g = torch.where(ids < 0, 0.0, v["dlogp"])
    d = -g[:, None] * p
    if case["entropy"]:
        inner = torch.where(logp == -math.inf, 0.0, logp) + v["entropy"][:, None]
        d = d - v["dentropy"][:, None] * p * inner
    d.scatter_add_(1, ids.clamp(min=0)[:, None], g[:, None])
    out["dlogits"] = (d * case["scale"]).to(v["logits"].dtype)


def _teacher(v, case):
    """The teacher's probabilities and their logarithms."""
    z = v["teacher"] * case["scale"]
    logq = z - _log_sum(z)[:, None]
    return torch.exp(logq), logq


def _plain_distill(v, out, case):
    z = v["logits"][:, :case["vocab"]].float() * case["scale"]
    lse = _log_sum(z)
    q, logq = _teacher(v, case)
    out["loss"] = (q * (logq - torch.gather(z, 1, v["ids"].long()) + lse[:, None])).sum(1)
    out["lse"] = lse


def _plain_distill_bwd(v, out, case):
    p = torch.exp(v["logits"][:, :case["vocab"]].float() * case["scale"] - v["lse"][:, None])
    q, _ = _teacher(v, case)
    p.scatter_add_(1, v["ids"].long(), -q)
    out["dlogits"] = (p * (v["dloss"] * case["scale"])[:, None]).to(v["logits"].dtype)


_PLAIN = {"embed": _plain_embed, "embed_bwd": _plain_embed_bwd, "norm": _plain_norm, "norm_bwd": _plain_norm_bwd,
          "logprob": _plain_logprob, "logprob_bwd": _plain_logprob_bwd, "distill": _plain_distill,
          "distill_bwd": _plain_distill_bwd}


# ------------------------------------------------------------------- work


def _distinct(tokens, vocab):
    """How many different tokens a text of `_tokens` holds on average."""
    i = np.arange(vocab, dtype=np.float64)
    p = np.log((i + 2.0) / (i + 1.0)) / math.log(vocab + 1.0) * (63.0 / 64.0)
    return float((1.0 - np.exp(tokens * np.log1p(-p))).sum())


def work(case):
    """Compulsory traffic: each input read once (of a table the rows that the
    tokens name), each output written once; and the operations of the norms and
    the exponentials' sums (three an element at least)."""
    kind, e = case["kind"], 4 if case["dtype"] == "f32" else 2
    if kind == "embed":
        t, c = case["tokens"], case["cols"]
        return {"bytes": e * c * (t + _distinct(t, case["vocab"])) + 4 * t, "flops": t * c}
    if kind == "embed_bwd":
        t, c = case["tokens"], case["cols"]
        eg = 4 if case["grad"] == "f32" else 2
        return {"bytes": e * t * c + eg * case["vocab"] * c + 4 * t, "flops": t * c}
    if kind == "norm":
        r, c = case["rows"], case["cols"]
        return {"bytes": e * r * c * (4 if case["residual"] else 2) + 2 * e * c + 8 * r, "flops": 7 * r * c}
    if kind == "norm_bwd":
        r, c = case["rows"], case["cols"]
        return {"bytes": e * r * c * (4 if case["residual"] else 3) + 3 * e * c + 8 * r, "flops": 12 * r * c}
    r, n, k = case["rows"], case["vocab"], case.get("top", 0)
    if kind == "logprob":
        return {"bytes": e * r * n + r * (16 + 8 * k), "flops": 5 * r * n}
    if kind == "logprob_bwd":
        return {"bytes": 2 * e * r * n + r * (20 if case["entropy"] else 12), "flops": (7 if case["entropy"] else 4) * r * n}
    if kind == "distill":
        return {"bytes": e * r * n + r * (8 + 8 * k), "flops": 3 * r * n}
    return {"bytes": 2 * e * r * n + r * (8 + 8 * k), "flops": 4 * r * n}


# ------------------------------------------------------------ in 64 bits


def exact(case, seed):
    """The definitions in float64; whole numbers have no such value."""
    v, kind = _inputs(case, seed), case["kind"]
    d = {name: x.double() for name, x in v.items() if x.is_floating_point()}
    if kind == "embed":
        rows = d["table"].index_select(0, v["ids"].relu().long())
        return {"y": rows * (_scale(case) * (v["ids"] >= 0).double()[:, None])}
    if kind == "embed_bwd":
        dw = torch.zeros(case["vocab"], case["cols"], dtype=torch.float64, device="cuda")
        keep = v["ids"] >= 0
        dw.index_put_((v["ids"][keep].long(),), d["dy"][keep], accumulate=True)
        return {"dw": dw.mul_(_scale(case))}
    if kind == "norm":
        h, out = d["x"], {}
        if case["residual"]:
            out["h"] = d["x"] + d["res"]
            h = out["h"].to(v["x"].dtype).double()
        var, mean = torch.var_mean(h, 1, correction=0)
        out["mean"], out["rstd"] = mean, (var + EPS).pow(-0.5)
        out["y"] = torch.addcmul(d["bias"], (h - mean[:, None]) * out["rstd"][:, None], d["w"])
        return out
    if kind == "norm_bwd":
        n = (d["h"] - d["mean"][:, None]) * d["rstd"][:, None]
        wdy = d["dy"] * d["w"]
        cols = case["cols"]
        along, flat = (wdy * n).sum(1, keepdim=True) / cols, wdy.sum(1, keepdim=True) / cols
        return {"dx": (wdy - flat - along * n) * d["rstd"][:, None] + d.get("dh", 0.0),
                "dw": (d["dy"] * n).sum(0), "db": d["dy"].sum(0)}
    if kind.startswith("logprob"):
        return _exact_logprob(case, v, d)
    return _exact_distill(case, v, d)


def _exact_logprob(case, v, d):
    z = d["logits"][:, :case["vocab"]] * case["scale"]
    rows, ids = torch.arange(case["rows"], device="cuda"), v["tokens"].long()
    if case["kind"] == "logprob":
        lse = torch.logsumexp(z, 1)
        out = {"lse": lse, "logp": (z[rows, ids.relu()] - lse) * (ids >= 0),
               "entropy": _entropy64(d["logits"][:, :case["vocab"]], case["scale"], lse)}
        if case["top"]:
            out["top_ids"] = None
            out["top_logp"] = z.sort(1, descending=True).values[:, :case["top"]] - lse[:, None]
        return out
    # the lse and entropy that came with the inputs, not those of the logits
    logp = z - d["lse"][:, None]
    slope = -d["dlogp"] * (ids >= 0)
    p = logp.exp()
    grad = p * slope[:, None]
    if case["entropy"]:
        grad -= torch.nan_to_num(p * (logp + d["entropy"][:, None]), nan=0.0) * d["dentropy"][:, None]
    grad[rows, ids.relu()] -= slope
    return {"dlogits": grad * case["scale"]}


def _exact_distill(case, v, d):
    z = d["logits"][:, :case["vocab"]] * case["scale"]
    logq = torch.log_softmax(d["teacher"] * case["scale"], 1)
    q, ids = logq.exp(), v["ids"].long()
    if case["kind"] == "distill":
        lse = torch.logsumexp(z, 1)
        cross = (q * z.gather(1, ids)).sum(1)
        return {"lse": lse, "loss": (q * logq).sum(1) - cross + lse}
    target = torch.zeros_like(z).scatter_add_(1, ids, q)
    return {"dlogits": ((z - d["lse"][:, None]).exp() - target) * (d["dloss"] * case["scale"])[:, None]}
