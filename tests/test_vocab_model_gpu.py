"""The two ends of a language model together, through the C ABI: tokens looked
up in a table and added to positions, layer norm, logits by the same table,
log probabilities of the given answers (with an entropy bonus), a teacher's top
tokens distilled, and all of it backward into the one table's gradient.  Against
float64, on its own, captured and replayed, two graphs of one stream in turn,
and on two streams at once.

Tolerance of the fp32 gradients, relative to a gradient's norm.  A logit is a sum
of D = 40 products of a normed row (its own sums of D, and 8 roundings) and the
table: off by (2 D + 8) U32 sum |y E|, at most A of them; a probability is off by
twice that, of itself, and by the 128 + 3 gap + 4 roundings of its row's sum, with
gaps below 2 A.  What goes back adds sums over the V = 301 logits, D columns and
T = 48 tokens.  Each is relative to a sum of magnitudes; K = 8 such sums meet
their result's norm, which cancellation makes smaller.  16-bit types round the
rows four times on the way in (looked up, h, y, logits), of which the logits' own
is HALF A absolute and so 2 HALF A of a probability, and four times on the way
back (dlogits, dy, dh, the table's gradient, twice)."""
import ctypes

import numpy as np
import pytest

from cortexmind_amd import engine
from cortexmind_amd._lib import DT_BF16, DT_F32, E_CAPTURE, call, lib
from cortexmind_amd.data import SplitMix64
from cortexmind_amd.device import DeviceArray, Stream
from gpu_util import dev
from layer_util import HALF, NAMES, U32, get, out, rounded, up
from test_graph_capture_gpu import CAPTURE_RELAXED, capture, hip_rt

pytestmark = pytest.mark.gpu

T, V, D, TOP, SCALE, BONUS = 48, 301, 40, 6, 0.7, 0.05
ANSWERED = 30  # rows with an answer; the others are distilled


def parameters(dt, seed):
    g = SplitMix64(seed)
    return {"E": rounded(g.normal((V, D), 0.0, 0.3), dt), "w": rounded(g.normal((D,), 1.0, 0.2), dt),
            "b": rounded(g.normal((D,), 0.0, 0.2), dt)}


def batch(dt, seed):
    r = np.random.default_rng(seed)
    ids = r.integers(0, V, T).astype(np.int32)
    ids[::11] = -1   # padding
    ids[5:9] = 17    # the same token again
    answers = r.integers(0, V, ANSWERED).astype(np.int32)
    answers[::7] = -1
    return {"ids": ids, "answers": answers, "P": rounded(SplitMix64(seed + 99).normal((T, D)), dt)}


class Model:
    """The device's buffers of one model, and its step."""

    def __init__(self, p, teacher, dt):
        self.dt = dt
        self.p = {k: up(v, dt) for k, v in p.items()}
        self.t = {k: up(v, dt) for k, v in teacher.items()}
        self.x = {"ids": dev(np.zeros(T, np.int32)), "answers": dev(np.zeros(ANSWERED, np.int32)), "P": out((T, D), dt)}
        f32 = lambda *s: dev(np.zeros(s, np.float32))  # noqa: E731
        self.emb, self.h, self.y, self.dy, self.dh = (out((T, D), dt) for _ in range(5))
        self.logits, self.dlogits = out((T, V), dt), out((T, V), dt)
        self.th, self.ty, self.tl = out((T, D), dt), out((T, D), dt), out((T, V), dt)
        self.mean, self.rstd, self.lse, self.logp, self.entropy = f32(T), f32(T), f32(T), f32(T), f32(T)
        self.top_logp, self.top_ids = f32(T, TOP), dev(np.zeros((T, TOP), np.int32))
        self.loss = f32(T - ANSWERED)
        self.g = {k: out(v.shape, dt) for k, v in p.items()}
        # of each answer -1 / count, of each entropy -BONUS / count; of each distilled row 1 / count
        self.dlogp = dev(np.full(ANSWERED, -1.0 / ANSWERED, np.float32))
        self.dent = dev(np.full(ANSWERED, -BONUS / ANSWERED, np.float32))
        self.dloss = dev(np.full(T - ANSWERED, 1.0 / (T - ANSWERED), np.float32))

    def take(self, b):
        self.x["ids"].upload(b["ids"])
        self.x["answers"].upload(b["answers"])
        fresh = up(b["P"], self.dt)
        call("cxm_memcpy_d2d", self.x["P"].ptr, fresh.ptr, T * D * (4 if self.dt == DT_F32 else 2), None)
        call("cxm_device_sync")

    def forward(self, p, emb, h, y, logits, mean, rstd, s):
        dt = self.dt
        engine.embedding.forward(p["E"], self.x["ids"], emb, T, V, D, dt, scale=2.0, stream=s)
        engine.layernorm.forward(emb, p["w"], y, T, D, dt, bias=p["b"], residual=self.x["P"], H=h, mean=mean, rstd=rstd,
                                 stream=s)
        engine.linear.forward(y, p["E"], logits, T, D, V, dt, trans_w=True, stream=s)

    def step(self, s=None):
        dt, n, e = self.dt, ANSWERED, 4 if self.dt == DT_F32 else 2
        self.forward(self.t, self.emb, self.th, self.ty, self.tl, None, None, s)
        call("cxm_logprob_fwd_t", self.tl.ptr, V, None, SCALE, None, None, None, self.top_logp.ptr, self.top_ids.ptr,
             TOP, T, V, dt, s and s.handle)
        self.forward(self.p, self.emb, self.h, self.y, self.logits, self.mean, self.rstd, s)
        engine.logprob.forward(self.logits, self.x["answers"], self.logp, n, V, dt, entropy=self.entropy, lse=self.lse,
                               stream=s)
        engine.logprob.backward(self.logits, self.x["answers"], self.lse, self.dlogp, self.dlogits, n, V, dt,
                                entropy=self.entropy, dentropy=self.dent, stream=s)
        # the distilled rows; the teacher's log probabilities, of softmax(SCALE z), are logits of that distribution
        at, ti, tt = n * V * e, n * TOP * 4, n * TOP * 4
        h = s and s.handle
        call("cxm_distill_fwd_t", self.logits.ptr + at, V, self.top_ids.ptr + ti, self.top_logp.ptr + tt, TOP, 1.0,
             self.loss.ptr, self.lse.ptr + 4 * n, T - n, V, dt, h)
        call("cxm_distill_bwd_t", self.logits.ptr + at, V, self.top_ids.ptr + ti, self.top_logp.ptr + tt, TOP, 1.0,
             self.lse.ptr + 4 * n, self.dloss.ptr, self.dlogits.ptr + at, V, T - n, V, dt, h)
        engine.linear.backward(self.y, self.p["E"], None, self.dlogits, None, self.dy, self.g["E"], None, T, D, V, dt,
                               trans_w=True, stream=s)
        engine.layernorm.backward(self.h, self.mean, self.rstd, self.p["w"], self.dy, self.dh, self.g["w"], T, D, dt,
                                  db=self.g["b"], stream=s)
        engine.embedding.backward(self.x["ids"], self.dh, self.g["E"], T, V, D, dt, scale=2.0, accumulate=True, stream=s)

    def results(self):
        call("cxm_device_sync")
        r = {k: v.numpy() for k, v in self.g.items()}
        r.update(logp=self.logp.numpy()[:ANSWERED], entropy=self.entropy.numpy()[:ANSWERED], loss=self.loss.numpy(),
                 top_ids=self.top_ids.numpy(), top_logp=self.top_logp.numpy(), dP=self.dh.numpy())
        return r


def softmax(z):
    e = np.exp(z - z.max(axis=1, keepdims=True))
    return e / e.sum(axis=1, keepdims=True)


def definition(p, x, dt, top_ids, top_logp, grad=True):
    """Loss and gradients in float64, the teacher's tokens given."""
    keep = (x["ids"] >= 0)[:, None]
    h = np.where(keep, 2.0 * p["E"][np.maximum(x["ids"], 0)], 0.0) + x["P"]
    mean, var = h.mean(axis=1, keepdims=True), h.var(axis=1, keepdims=True)
    rstd = 1.0 / np.sqrt(var + 1e-5)
    n = (h - mean) * rstd
    y = n * p["w"] + p["b"]
    z = y @ p["E"].T
    q = softmax(z)
    logq = np.log(q)
    a = x["answers"]
    live = (a >= 0).astype(float)
    rows = np.arange(ANSWERED)
    logp = np.where(a >= 0, logq[rows, np.maximum(a, 0)], 0.0)
    entropy = -(q * logq).sum(axis=1)[:ANSWERED]  # of rows without an answer too
    t = np.zeros((T - ANSWERED, V))
    np.put_along_axis(t, top_ids[ANSWERED:].astype(np.int64), softmax(top_logp[ANSWERED:].astype(np.float64)), axis=1)
    with np.errstate(divide="ignore", invalid="ignore"):
        kl = np.where(t > 0, t * (np.log(t) - logq[ANSWERED:]), 0.0).sum(axis=1)
    loss = -logp.sum() / ANSWERED - BONUS * entropy.sum() / ANSWERED + kl.mean()
    values = {"logp": logp, "entropy": entropy, "loss": kl}
    if not grad:
        return loss, values, None, z
    dz = np.zeros_like(z)
    one = np.zeros((ANSWERED, V))
    one[rows, np.maximum(a, 0)] = 1.0
    qa = q[:ANSWERED]
    dz[:ANSWERED] = (-live[:, None] * (one - qa) + BONUS * qa * (logq[:ANSWERED] + entropy[:, None])) / ANSWERED
    dz[ANSWERED:] = (q[ANSWERED:] - t) / (T - ANSWERED)
    dy = dz @ p["E"]
    g = dy * p["w"]
    dh = rstd * (g - g.mean(axis=1, keepdims=True) - n * (g * n).mean(axis=1, keepdims=True))
    dE = dz.T @ y
    np.add.at(dE, x["ids"][x["ids"] >= 0], 2.0 * dh[x["ids"] >= 0])
    return loss, values, {"E": dE, "w": (dy * n).sum(axis=0), "b": dy.sum(axis=0), "dP": dh}, z


def tolerance(p, x, dt, y_bound):
    """Of the gradients, relative to their norms; A: the largest sum |y E| there can be."""
    a = y_bound
    rel = U32 * (2 * ((2 * D + 8) * a + 2 * a) + 128 + 6 * a + 4 + V + 2 * D + T) * 8
    if dt != DT_F32:
        rel += HALF[dt] * (2 * a + 2 * (3 * a) + 9)
    return rel


def sum_bound(p, x):
    h = np.where((x["ids"] >= 0)[:, None], 2.0 * p["E"][np.maximum(x["ids"], 0)], 0.0) + x["P"]
    n = (h - h.mean(axis=1, keepdims=True)) / h.std(axis=1, keepdims=True)
    return (np.abs(n * p["w"] + p["b"]) @ np.abs(p["E"]).T).max()


@pytest.mark.parametrize("dt", [DT_F32, DT_BF16], ids=NAMES.get)
def test_step(hip, dt):
    p, teacher, x = parameters(dt, 3), parameters(dt, 4), batch(dt, 5)
    m = Model(p, teacher, dt)
    m.take(x)
    m.step()
    got = m.results()
    loss, values, grads, z = definition(p, x, dt, got["top_ids"], got["top_logp"])
    rel = tolerance(p, x, dt, sum_bound(p, x))
    # logits off by half of that at most, so log probabilities too; an entropy by its gap's share of it
    for k, v in values.items():
        assert np.abs(got[k] - v).max() <= rel * (1.0 + np.abs(z).max()), k
    for k, v in grads.items():
        d = get(m.g[k] if k in m.g else m.dh, dt) - v
        assert np.linalg.norm(d) <= rel * np.linalg.norm(v), (k, np.linalg.norm(d) / np.linalg.norm(v), rel)


def test_gradients_match_differences(hip):
    """fp32 gradients against central differences of the float64 loss along random directions."""
    dt = DT_F32
    p, teacher, x = parameters(dt, 13), parameters(dt, 14), batch(dt, 15)
    m = Model(p, teacher, dt)
    m.take(x)
    m.step()
    got = m.results()
    rel = tolerance(p, x, dt, sum_bound(p, x))
    r = np.random.default_rng(1)
    for k in ("E", "w", "b"):
        v = r.standard_normal(p[k].shape)
        v /= np.linalg.norm(v)
        at = lambda t: definition({**p, k: p[k] + t * v}, x, dt, got["top_ids"], got["top_logp"], False)[0]  # noqa: E731
        # (third derivatives times 1e-4^2 / 6, and 1e-16 / 1e-4 of the losses' roundings: below 1e-7)
        slope, g = (at(1e-4) - at(-1e-4)) / 2e-4, got[k].astype(np.float64)
        assert abs(slope - (g * v).sum()) <= rel * np.linalg.norm(g) + 1e-7, k


def same(a, b):
    return [k for k in a if not np.array_equal(a[k], b[k])]


@pytest.mark.parametrize("dt", [DT_F32, DT_BF16], ids=NAMES.get)
def test_captured_steps_in_turn(hip, dt):
    """Two captured steps of one stream, whose workspaces they share, replayed in turn on new data with eager work
    between: each replay's bits are the eager step's."""
    h, s = hip_rt(), Stream()
    p, teacher = parameters(dt, 23), parameters(dt, 24)
    one, two, plain = Model(p, teacher, dt), Model(teacher, p, dt), {}
    try:
        for m in (one, two):
            m.take(batch(dt, 1))
            m.step(s)  # the stream's workspaces
        s.sync()
        exes = [capture(h, s, lambda m=m: m.step(s)) for m in (one, two)]
        other = Model(parameters(dt, 25), teacher, dt)
        other.take(batch(dt, 77))
        for i in range(3):
            for j, m in enumerate((one, two)):
                m.take(batch(dt, 30 + 2 * i + j))
                assert h.hipGraphLaunch(exes[j][1], s.handle) == 0
                other.step(s)
                s.sync()
                got = m.results()
                plain = Model(p, teacher, dt) if j == 0 else Model(teacher, p, dt)
                plain.take(batch(dt, 30 + 2 * i + j))
                plain.step()
                assert not same(got, plain.results()), (i, j)
        for g, e in exes:
            h.hipGraphExecDestroy(e)
            h.hipGraphDestroy(g)
    finally:
        s.close()


def test_two_streams_at_once(hip):
    dt = DT_BF16
    p, teacher = parameters(dt, 43), parameters(dt, 44)
    want = []
    for i in range(2):
        m = Model(p, teacher, dt)
        m.take(batch(dt, 50 + i))
        m.step()
        want.append(m.results())
    streams = [Stream(), Stream()]
    try:
        ms = [Model(p, teacher, dt) for _ in streams]
        for i, m in enumerate(ms):
            m.take(batch(dt, 50 + i))
        for _ in range(20):
            for m, s in zip(ms, streams):
                m.step(s)
        for s in streams:
            s.sync()
        for m, w in zip(ms, want):
            assert not same(m.results(), w)
    finally:
        for s in streams:
            s.close()


def test_capture_without_scratch_is_refused(hip):
    """Calls that need a workspace which their stream does not have yet, under capture: refused, nothing recorded."""
    h, s, L = hip_rt(), Stream(), lib()
    x, f = DeviceArray((4 * 60000,), np.uint16), dev(np.zeros(8 * 60000, np.float32))
    ids = dev(np.zeros(64, np.int32))
    dt, st = DT_BF16, s.handle
    try:
        assert h.hipStreamBeginCapture(s.handle, CAPTURE_RELAXED) == 0
        got = [
            L.cxm_layernorm_bwd_t(x.ptr, f.ptr, f.ptr, x.ptr + 2000, x.ptr + 4000, None, x.ptr + 6000, x.ptr + 8000, None, 8,
                                  64, dt, st),
            L.cxm_embedding_bwd_t(ids.ptr, x.ptr, 1.0, f.ptr, 0, 64, 100, 64, dt, DT_F32, st),
            L.cxm_logprob_fwd_t(x.ptr, 60000, ids.ptr, 1.0, f.ptr, None, None, f.ptr + 4000, f.ptr + 8000, 5, 2, 60000, dt, st),
            L.cxm_distill_fwd_t(x.ptr, 60000, ids.ptr, f.ptr, 5, 1.0, f.ptr + 4000, f.ptr + 8000, 2, 60000, dt, st),
        ]
        graph, n = ctypes.c_void_p(), ctypes.c_size_t(99)
        assert h.hipStreamEndCapture(s.handle, ctypes.byref(graph)) == 0
        h.hipGraphGetNodes.argtypes = [ctypes.c_void_p, ctypes.c_void_p, ctypes.POINTER(ctypes.c_size_t)]
        h.hipGraphGetNodes.restype = ctypes.c_int
        assert h.hipGraphGetNodes(graph, None, ctypes.byref(n)) == 0
        h.hipGraphDestroy(graph)
        assert got == [E_CAPTURE] * 4 and n.value == 0, (got, n.value)
    finally:
        s.close()


def test_table_past_2_31_elements(hip):
    """Offsets that 32 bits do not hold: the last rows of a table of 2^31 + elements, looked up and their gradient."""
    vocab, cols, dt = (1 << 22) + 3, 516, DT_BF16
    table = DeviceArray((vocab * cols,), np.uint16)
    t = np.array([vocab - 1, 0, vocab - 1, -1, vocab // 2, vocab - 2], np.int32)
    rows = rounded(SplitMix64(61).normal((len(t), cols)), dt)
    bits, ids, y = up(rows, dt), dev(t), out((len(t), cols), dt)
    for i in (0, 1, 4, 5):
        call("cxm_memcpy_d2d", table.ptr + 2 * int(t[i]) * cols, bits.ptr + 2 * i * cols, 2 * cols, None)
    engine.embedding.forward(table, ids, y, len(t), vocab, cols, dt)
    want = rows[[0, 1, 0, 3, 4, 5]]
    want[3] = 0.0
    assert np.array_equal(get(y, dt), want)
    whole = rounded(np.arange(len(t) * cols).reshape(len(t), cols) % 9 - 4.0, dt)  # whole numbers: exact sums
    dy = up(whole, dt)
    engine.embedding.backward(ids, dy, table, len(t), vocab, cols, dt)
    got = out((5, cols), dt)
    for i, v in enumerate((vocab - 1, 0, vocab // 2, vocab - 2, vocab - 3)):
        call("cxm_memcpy_d2d", got.ptr + 2 * i * cols, table.ptr + 2 * v * cols, 2 * cols, None)
    assert np.array_equal(get(got, dt), [whole[0] + whole[2], whole[1], whole[4], whole[5], np.zeros(cols)])
