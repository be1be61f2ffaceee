"""The operators as a program uses them together: a residual block
  h1 = x, n1 = norm(h1), u = gelu(n1 W1 + b1), y = u W2 + b2 + h1
trained with AdamW, fp32 and bf16, against the same block in float64; its
gradients against differences; the block served from 8-bit operands; and a
whole step captured into a HIP graph and replayed beside eager work."""
import math

import numpy as np
import pytest
import torch

from cortexmind_amd import engine
from cortexmind_amd._lib import ACT_GELU, ACT_NONE, DT_BF16, DT_F32, E_CAPTURE, CxmError
from cortexmind_amd.data import SplitMix64
from cortexmind_amd.device import DeviceArray, Stream
from gpu_util import dev
from layer_util import E4M3, HALF, U32, close, from_bits, get, rounded, up
from test_graph_capture_gpu import capture, hip_rt

pytestmark = pytest.mark.gpu
EPS = 1e-5
NAMES = ("g", "w1", "b1", "w2", "b2")


def cdf(v):
    return 0.5 * torch.special.erfc(v * -math.sqrt(0.5))


class Block:
    """The block's parameters, activations and gradients on the device."""

    def __init__(self, rows, width, inner, dt, seed=1, master=False):
        self.rows, self.width, self.inner, self.dt = rows, width, inner, dt
        r = SplitMix64(seed)
        shapes = {"g": (width,), "w1": (width, inner), "b1": (inner,), "w2": (inner, width), "b2": (width,)}
        stds = {"g": 0.1, "w1": width ** -0.5, "b1": 0.1, "w2": inner ** -0.5, "b2": 0.1}
        self.host = {k: rounded(r.normal(s, 1.0 if k == "g" else 0.0, stds[k]), dt) for k, s in shapes.items()}
        self.x = rounded(r.normal((rows, width)), dt)
        self.dy = rounded(r.normal((rows, width)), dt)
        self.p = {k: up(v, dt) for k, v in self.host.items()}
        zero = lambda *s: up(np.zeros(s), dt)  # noqa: E731
        self.d = {"x": up(self.x, dt), "dy": up(self.dy, dt), "n": zero(rows, width), "u": zero(rows, inner),
                  "z": zero(rows, inner), "y": zero(rows, width), "dz": zero(rows, inner), "du": zero(rows, inner),
                  "dn": zero(rows, width), "dx": zero(rows, width), "rstd": DeviceArray((rows,), np.float32)}
        self.grad = {k: zero(*s) for k, s in shapes.items()}
        f = lambda k: dev(np.zeros(shapes[k], np.float32))  # noqa: E731
        self.state = [{"p": self.p[k], "g": self.grad[k], "m": f(k), "v": f(k), "decay": 0.1 if k[0] == "w" else 0.0}
                      for k in NAMES]
        if master:
            for s, k in zip(self.state, NAMES):
                s["master"] = dev(self.host[k].astype(np.float32))
        self.opt = engine.AdamW(self.state, dt, dt)

    def forward(self, stream=None):
        p, d, kw = self.p, self.d, {"stream": stream}
        engine.rmsnorm.forward(d["x"], p["g"], d["n"], self.rows, self.width, self.dt, eps=EPS, rstd=d["rstd"], **kw)
        engine.linear.forward(d["n"], p["w1"], d["u"], self.rows, self.width, self.inner, self.dt, bias=p["b1"],
                              act=ACT_GELU, Z=d["z"], **kw)
        # in fp32 the sum without an activation needs a place of its own only for the residual
        engine.linear.forward(d["u"], p["w2"], d["y"], self.rows, self.inner, self.width, self.dt, bias=p["b2"],
                              residual=d["x"], **kw)

    def backward(self, stream=None):
        p, d, g, kw = self.p, self.d, self.grad, {"stream": stream}
        engine.linear.backward(d["u"], p["w2"], None, d["dy"], None, d["du"], g["w2"], g["b2"], self.rows, self.inner,
                               self.width, self.dt, act=ACT_NONE, **kw)
        engine.linear.backward(d["n"], p["w1"], d["z"], d["du"], d["dz"], d["dn"], g["w1"], g["b1"], self.rows, self.width,
                               self.inner, self.dt, act=ACT_GELU, **kw)
        engine.rmsnorm.backward(d["x"], d["rstd"], p["g"], d["dn"], d["dx"], g["g"], self.rows, self.width, self.dt,
                                dH=d["dy"], **kw)

    def step(self, t, stream=None, **kw):
        self.forward(stream)
        self.backward(stream)
        self.opt.step(1e-3, t, stream=stream, **kw)


def block64(p, x, dy):
    """(y, gradients) in float64."""
    t = {k: torch.from_numpy(np.asarray(v, np.float64)).requires_grad_() for k, v in {**p, "x": x}.items()}
    h = t["x"]
    n = h / torch.sqrt((h * h).mean(1, keepdim=True) + EPS) * t["g"]
    z = n @ t["w1"] + t["b1"]
    y = (z * cdf(z)) @ t["w2"] + t["b2"] + h
    grads = torch.autograd.grad((y * torch.from_numpy(dy)).sum(), list(t.values()))
    return y.detach().numpy(), dict(zip(t, (g.numpy() for g in grads)))


def rel(got, want):
    return np.linalg.norm(got - want) / np.linalg.norm(want)


@pytest.mark.parametrize("dt,sizes", [(DT_F32, (48, 40, 104)), (DT_F32, (300, 129, 250)), (DT_BF16, (48, 40, 104)),
                                      (DT_BF16, (300, 129, 250)), (DT_BF16, (1024, 256, 1024))])
def test_step_matches_float64(hip, dt, sizes):
    """Norms of the differences: fp32 within 2e-6 of each norm (sums of up to
    1024 fp32 products, three products deep); bf16 within 4 roundings of 2^-8
    (an activation, dz, the gradient and the value itself round)."""
    b = Block(*sizes, dt)
    b.step(1)
    y, g = block64(b.host, b.x, b.dy)
    bar = 2e-6 if dt == DT_F32 else 4 * HALF[dt]
    assert rel(get(b.d["y"], dt), y) <= bar
    assert rel(get(b.d["dx"], dt), g["x"]) <= bar
    for k in NAMES:
        assert rel(get(b.grad[k], dt), g[k]) <= bar, k
    for s, k in zip(b.state, NAMES):  # the optimizer reads the device's gradients
        got, grad = get(b.p[k], dt), get(b.grad[k], dt)
        want = b.host[k] * (1 - 1e-3 * s["decay"]) - 1e-3 * grad / (np.abs(grad) + 1e-8)
        close(got, want, (HALF[dt] + 4 * U32) * np.abs(want) + 1e-3 * 1e-5, k)


def test_gradients_match_differences(hip):
    """fp32 gradients against central differences of the float64 block."""
    b = Block(6, 20, 28, DT_F32, 3)
    b.forward()
    b.backward()
    step = 1e-5
    for k, i in (("g", (3,)), ("w1", (4, 5)), ("b1", (7,)), ("w2", (9, 2)), ("b2", (0,))):
        e = np.zeros_like(b.host[k])
        e[i] = step
        up_, down = ({**b.host, k: b.host[k] + s * e} for s in (1, -1))
        num = ((block64(up_, b.x, b.dy)[0] - block64(down, b.x, b.dy)[0]) * b.dy).sum() / (2 * step)
        assert abs(num - get(b.grad[k], DT_F32)[i]) <= 1e-4, k


def test_served_from_8_bits(hip):
    """norm to 8 bits -> 8-bit layer: against float64 on the very codes the norm wrote."""
    for rows in (1, 5, 70, 600):
        b = Block(rows, 200, 328, DT_BF16, 5)
        q, s = DeviceArray((rows, 200), np.uint8), DeviceArray((rows,), np.float32)
        wq, ws = DeviceArray((328, 200), np.uint8), DeviceArray((328,), np.float32)
        wt = up(b.host["w1"].T, DT_BF16)
        engine.quant.rows(wt, wq, ws, 328, 200, DT_BF16)
        engine.rmsnorm.forward(b.d["x"], b.p["g"], None, rows, 200, DT_BF16, eps=EPS, Q=q, scale=s)
        engine.linear.forward_q8(q, s, wq, ws, b.d["u"], rows, 200, 328, DT_BF16, bias=b.p["b1"], act=ACT_GELU)
        xs, wv = E4M3[q.numpy()] * s.numpy()[:, None].astype(np.float64), E4M3[wq.numpy()] * ws.numpy()[:, None].astype(np.float64)
        z = xs @ wv.T + b.host["b1"]
        want = z * cdf(torch.from_numpy(z)).numpy()
        size = np.abs(xs) @ np.abs(wv.T) + np.abs(b.host["b1"])
        # what 8-bit products lose (see test_linear_gpu), times GELU's largest slope
        lost = 1.13 * 6 * math.sqrt(200 / 12) * 2.0 ** -13 * np.abs(xs).max(1)[:, None] * np.abs(wv).max(1)[None, :]
        close(get(b.d["u"], DT_BF16), want, (HALF[DT_BF16] + 1.1e-5) * np.abs(want) + 1.2e-5 * size + lost)


@pytest.mark.parametrize("dt,sizes", [(DT_BF16, (96, 72, 200)), (DT_F32, (64, 40, 100)), (DT_BF16, (3, 512, 1003))])
def test_captured_step_replays(hip, dt, sizes):
    """The whole step as a graph, its learning rate, step number and factor
    on the device: every replay gives the eager run's bits, with eager work
    of other sizes on the same stream and synchronizations between replays."""
    h, s = hip_rt(), Stream()
    a, b, other = Block(*sizes, dt, 7, dt != DT_F32), Block(*sizes, dt, 7, dt != DT_F32), Block(130, 300, 64, dt, 8)
    scal = DeviceArray((3,), np.float32)
    for blk in (other, Block(*sizes, dt, 9)):
        blk.step(1, s)  # the stream's scratch exists, at its largest, before capture
    s.sync()
    graph, exe = capture(h, s, lambda: a.step(1, s, scalars=scal))
    try:
        for t in range(1, 7):
            scal.upload(np.array([1e-3 / t, t, 1.0], np.float32), s)
            assert h.hipGraphLaunch(exe, s.handle) == 0
            s.sync()
            b.step(t, s, scalars=scal)
            other.step(t, s)
            s.sync()
            for k in NAMES:
                assert np.array_equal(a.p[k].numpy(), b.p[k].numpy()), (t, k)
                assert np.array_equal(a.grad[k].numpy(), b.grad[k].numpy()), (t, k)
            assert np.array_equal(a.d["y"].numpy(), b.d["y"].numpy()), t
    finally:
        h.hipGraphExecDestroy(exe)
        h.hipGraphDestroy(graph)
        s.close()


def test_capture_without_scratch_is_refused(hip):
    """A new stream has no scratch: calls that need it are CXM_E_CAPTURE and
    record nothing; those that need none are recorded."""
    h, s = hip_rt(), Stream()
    b = Block(130, 1003, 300, DT_BF16, 11)

    def body():
        for fn in (lambda: engine.rmsnorm.backward(b.d["x"], b.d["rstd"], b.p["g"], b.d["dn"], b.d["dx"], b.grad["g"], 130,
                                                   1003, DT_BF16, stream=s),
                   lambda: engine.linear.forward(b.d["n"], b.p["w1"], b.d["u"], 130, 1003, 300, DT_BF16, stream=s),
                   lambda: engine.linear.backward(b.d["n"], b.p["w1"], b.d["z"], b.d["du"], b.d["dz"], b.d["dn"],
                                                  b.grad["w1"], b.grad["b1"], 130, 1003, 300, DT_BF16, act=ACT_GELU,
                                                  stream=s)):
            with pytest.raises(CxmError) as e:
                fn()
            assert e.value.status == E_CAPTURE
        engine.rmsnorm.forward(b.d["x"], b.p["g"], b.d["n"], 130, 1003, DT_BF16, stream=s)

    graph, exe = capture(h, s, body)
    try:
        assert h.hipGraphLaunch(exe, s.handle) == 0
        s.sync()
        got = from_bits(b.d["n"].numpy(), DT_BF16)
        want = b.x / np.sqrt((b.x ** 2).mean(1, keepdims=True) + EPS) * b.host["g"]
        close(got, want, (HALF[DT_BF16] + 128 * U32) * np.abs(want))
    finally:
        h.hipGraphExecDestroy(exe)
        h.hipGraphDestroy(graph)
        s.close()


def test_two_streams_at_once(hip):
    """The same work queued on two streams without waiting in between (split
    products, column sums and their scratch among it) gives each its own result."""
    a, b = Block(130, 512, 300, DT_BF16, 13), Block(130, 512, 300, DT_BF16, 14)
    wa, wb = Block(130, 512, 300, DT_BF16, 13), Block(130, 512, 300, DT_BF16, 14)
    s, u = Stream(), Stream()
    for blk, st in ((a, s), (b, u)):  # each stream's scratch
        Block(130, 512, 300, DT_BF16, 15).step(1, st)
    s.sync()
    u.sync()
    for t in range(1, 6):
        a.step(t, s)
        b.step(t, u)
    for t in range(1, 6):
        wa.step(t)
        wb.step(t)
    for x in (s, u):
        x.sync()
    for got, want in ((a, wa), (b, wb)):
        for k in NAMES:
            assert np.array_equal(got.p[k].numpy(), want.p[k].numpy()), k
            assert np.array_equal(got.grad[k].numpy(), want.grad[k].numpy()), k
    s.close()
    u.close()
