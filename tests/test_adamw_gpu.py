"""The AdamW step over many tensors, through engine.AdamW, against float64.

Tolerances: m and v are two products and a sum (3 fp32 roundings of parts no
larger than |b m| + |c g|); the update is four operations on them and a
square root, 8 roundings; p's own product and sum two more.  8-bit moments:
the stored value is one of the two neighbours of (exact value) / scale, and
the upper one exactly when the value's random bits say so, except where the
distance is within 1e-3 of a step of the border."""
import numpy as np
import pytest

from cortexmind_amd import engine
from cortexmind_amd._lib import DT_BF16, DT_F16, DT_F32, E_INVALID, CxmError
from cortexmind_amd.data import SplitMix64
from cortexmind_amd.device import Stream
from gpu_util import dev
from layer_util import E4M3, HALF, NAMES, TINY, U32, close, e4m3_below, get, rounded, up

pytestmark = pytest.mark.gpu
LR, B1, B2, EPS = 1e-3, 0.9, 0.999, 1e-8
SIZES = [1, 7, 255, 256, 257, 2048, 2049, 5000, 100003]


def noise(number, seed):
    key = np.uint32((seed * 0x9E3779B1 & 0xFFFFFFFF) ^ (seed >> 32))
    x = number.astype(np.uint32) ^ key ^ ((number >> np.uint64(32)).astype(np.uint32) * np.uint32(0xC2B2AE35))
    with np.errstate(over="ignore"):
        for mul in (0x85EBCA6B, 0xC2B2AE35):
            x = (x ^ (x >> np.uint32(16))) * np.uint32(mul)
    return x ^ (x >> np.uint32(16))


class Model:
    """Tensors with random parameters, gradients and moments, on both sides."""

    def __init__(self, sizes, pd, gd, master, q8, seed=1, off=0, decays=(0.1, 0.0)):
        g = SplitMix64(seed)
        self.pd, self.gd, self.master, self.q8 = pd, gd, master, q8
        self.host, self.dev = [], []
        first = 0
        for i, n in enumerate(sizes):
            w = g.normal((n,), 0.0, 0.05)
            h = {"p": rounded(w, pd), "master": w.astype(np.float64), "g": rounded(g.normal((n,), 0.0, 1e-2), gd), "n": n,
                 "decay": decays[i % len(decays)], "first": first}
            nb = (n + 255) // 256
            first += 256 * nb
            d = {"p": up(h["p"], pd, off), "g": up(h["g"], gd, off), "n": n, "decay": h["decay"]}
            if master:
                d["master"] = dev(w.astype(np.float32), off)
            if q8:
                h["m"] = (g.next_u64(n) % np.uint64(127)).astype(np.uint8) | ((g.next_u64(n) & np.uint64(128)).astype(np.uint8))
                h["v"] = (g.next_u64(n) % np.uint64(127)).astype(np.uint8)
                h["m_scale"] = g.uniform((nb,), 1e-6, 1e-5)
                h["v_scale"] = g.uniform((nb,), 1e-6, 1e-4)
                d.update(m=dev(h["m"], off), v=dev(h["v"], off), m_scale=dev(h["m_scale"]), v_scale=dev(h["v_scale"]))
            else:
                h["m"] = g.normal((n,), 0.0, 1e-3)
                h["v"] = (g.normal((n,), 0.0, 1e-2) ** 2).astype(np.float32)
                d.update(m=dev(h["m"], off), v=dev(h["v"], off))
            self.host.append(h)
            self.dev.append(d)
        self.opt = engine.AdamW(self.dev, pd, gd, state_8bit=q8)

    def exact(self, h, t, lr=LR, factor=1.0):
        n = h["n"]
        p = h["master"] if self.master else h["p"]
        g = h["g"] * factor
        if self.q8:
            at = np.arange(n) // 256
            m0 = E4M3[h["m"]] * h["m_scale"].astype(np.float64)[at]
            v0 = (E4M3[h["v"]] * h["v_scale"].astype(np.float64)[at]) ** 2
        else:
            m0, v0 = h["m"].astype(np.float64), h["v"].astype(np.float64)
        m, v = B1 * m0 + (1 - B1) * g, B2 * v0 + (1 - B2) * g * g
        size = B1 * np.abs(m0) + (1 - B1) * np.abs(g)
        d = np.sqrt(v / (1 - B2 ** t)) + EPS
        u = lr / (1 - B1 ** t) * m / d
        us = lr / (1 - B1 ** t) * size / d
        return p * (1 - lr * h["decay"]) - u, np.abs(p) + us, us, m, size, v

    def check(self, t, lr=LR, factor=1.0, seed=0):
        for h, d in zip(self.host, self.dev):
            p, psize, us, m, msize, v = self.exact(h, t, lr, factor)
            tol = 3 * U32 * psize + 12 * U32 * us
            if self.master:
                close(get(d["master"], DT_F32), p, tol, "master")
                # the copy is the master, rounded
                assert np.array_equal(get(d["p"], self.pd), rounded(d["master"].numpy(), self.pd))
            else:
                close(get(d["p"], self.pd), p, tol + HALF[self.pd] * np.abs(p) + TINY[self.pd], "p")
            if not self.q8:
                close(get(d["m"], DT_F32), m, 4 * U32 * msize + 1e-44, "m")
                close(get(d["v"], DT_F32), v, 5 * U32 * v + 1e-44, "v")
                continue
            bits = noise(np.arange(h["n"], dtype=np.uint64) + np.uint64(h["first"]), seed)
            at = np.arange(h["n"]) // 256
            for name, want, rnd in (("m", m, bits & np.uint32(0xFFFF)), ("v", np.sqrt(v), bits >> np.uint32(16))):
                scale = d[name + "_scale"].numpy().astype(np.float64)
                code = d[name].numpy()
                amax = np.array([np.abs(want[at == b]).max() for b in range(scale.size)])
                close(scale, amax / 448.0, 8 * U32 * amax / 448.0, name + "_scale")
                s = scale[at]
                a = np.minimum(np.abs(want) / np.where(s > 0, s, 1.0), 448.0)
                lo, share = e4m3_below(a)
                pick = (share + rnd / 65536.0 >= 1.0).astype(int)
                expect = lo + pick
                if name == "v":
                    expect = np.where((a > 0) & (expect == 0), 1, expect)
                else:
                    nz = (E4M3[code] != 0)
                    assert np.array_equal(np.signbit(E4M3[code])[nz], np.signbit(want)[nz])
                got = (code & 127).astype(int)
                near = np.abs(share + rnd / 65536.0 - 1.0) < 1e-3
                # (a share that rounding carries past 0 or 1 gives the same code, but for those near the border)
                assert np.all((got == expect) | (near & (np.abs(got - expect) <= 1))), name
                assert np.mean(near) < 0.01 or h["n"] < 3000


KINDS = [(DT_F32, DT_F32, False), (DT_BF16, DT_BF16, False), (DT_BF16, DT_BF16, True), (DT_BF16, DT_F32, True),
         (DT_BF16, DT_F32, False), (DT_F16, DT_F16, False), (DT_F16, DT_F16, True), (DT_F16, DT_F32, True),
         (DT_F16, DT_F32, False)]
kind_id = lambda k: f"{NAMES[k[0]]}-{NAMES[k[1]]}{'-master' if k[2] else ''}"  # noqa: E731


@pytest.mark.parametrize("q8", [False, True], ids=["m32", "m8"])
@pytest.mark.parametrize("kind", KINDS, ids=kind_id)
def test_step(hip, kind, q8):
    m = Model(SIZES, *kind, q8)
    m.opt.step(LR, 3, seed=77)
    m.check(3, seed=77)


@pytest.mark.parametrize("q8", [False, True], ids=["m32", "m8"])
@pytest.mark.parametrize("t", [1, 2, 1000, 10 ** 6])
def test_steps_corrections(hip, t, q8):
    m = Model([3000], DT_F32, DT_F32, False, q8, 5)
    m.opt.step(LR, t, seed=t)
    m.check(t, seed=t)


@pytest.mark.parametrize("off", [1, 3])
@pytest.mark.parametrize("q8", [False, True], ids=["m32", "m8"])
@pytest.mark.parametrize("kind", [KINDS[0], KINDS[2]], ids=kind_id)
def test_misaligned(hip, kind, q8, off):
    m = Model([1, 600, 5000], *kind, q8, 9, off)
    m.opt.step(LR, 10, seed=123456789123)
    m.check(10, seed=123456789123)


def test_scalars_on_the_device(hip):
    """Learning rate, step and gradient factor read from the device: the
    corrections in fp32 instead of fp64, 4 roundings more."""
    for q8 in (False, True):
        m = Model([4000, 77], DT_F32, DT_F32, False, q8, 11)
        s = dev(np.array([2e-3, 5.0, 0.25], np.float32))
        m.opt.step(123.0, 0, scalars=s, seed=5)
        for h, d in zip(m.host, m.dev):
            p, psize, us, *_ = m.exact(h, 5, float(np.float32(2e-3)), 0.25)
            close(get(d["p"], DT_F32), p, 3 * U32 * psize + 24 * U32 * us, "p")


def test_zero_states_first_step(hip):
    """From zero moments: the first update is lr * sign(g), and a zero gradient
    leaves everything as it is."""
    n = 1000
    g = np.where(np.arange(n) % 3 == 0, 0.0, np.where(np.arange(n) % 2, 0.01, -0.02))
    p = np.linspace(-1, 1, n).astype(np.float32)
    for q8 in (False, True):
        d = {"p": dev(p), "g": dev(g.astype(np.float32)), "n": n}
        if q8:
            d.update(m=dev(np.zeros(n, np.uint8)), v=dev(np.zeros(n, np.uint8)), m_scale=dev(np.zeros(4, np.float32)),
                     v_scale=dev(np.zeros(4, np.float32)))
        else:
            d.update(m=dev(np.zeros(n, np.float32)), v=dev(np.zeros(n, np.float32)))
        opt = engine.AdamW([d], state_8bit=q8)
        opt.step(LR, 1)
        close(d["p"].numpy(), p - LR * np.sign(g), 4 * U32 * (np.abs(p) + LR) + LR * 2e-6)
        assert np.all(d["m"].numpy()[g == 0] == 0) and np.all(d["v"].numpy()[g == 0] == 0)
        opt.close()


def test_non_finite_gradients_stay_alone(hip):
    """A NaN or an infinite gradient reaches its own value only."""
    for q8 in (False, True):
        a, b = Model([1000], DT_F32, DT_F32, False, q8, 13), Model([1000], DT_F32, DT_F32, False, q8, 13)
        g = a.host[0]["g"].astype(np.float32)
        keep = b.host[0]["g"].astype(np.float32)
        g[[5, 300]] = [np.nan, np.inf]
        keep[[5, 300]] = 0.0
        a.dev[0]["g"].upload(g)
        b.dev[0]["g"].upload(keep)
        a.opt.step(LR, 2, seed=1)
        b.opt.step(LR, 2, seed=1)
        rest = np.delete(np.arange(1000), [5, 300])
        assert np.array_equal(a.dev[0]["p"].numpy()[rest], b.dev[0]["p"].numpy()[rest])
        assert np.all(np.isnan(a.dev[0]["p"].numpy()[[5]]))
        if q8:
            assert np.all(a.dev[0]["m"].numpy()[[5, 300]] & 127 == 127)
            assert np.all(np.isfinite(a.dev[0]["m_scale"].numpy()))
            assert np.all(np.isfinite(E4M3[a.dev[0]["m"].numpy()[rest]]))


def test_stochastic_rounding_is_unbiased(hip):
    """One value stored many times: its mean is within 5 standard deviations
    (each rounding's is at most half a step, 14 at 224 to 448 ... here 16 / 2)."""
    n = 1 << 16
    g = np.full(n, 0.3, np.float32)
    g[::256] = 1.0  # each block's largest
    z8, zs = np.zeros(n, np.uint8), np.zeros(n // 256, np.float32)
    d = {"p": dev(np.zeros(n, np.float32)), "g": dev(g), "m": dev(z8), "v": dev(z8), "m_scale": dev(zs), "v_scale": dev(zs)}
    opt = engine.AdamW([d], state_8bit=True)
    opt.step(LR, 1, seed=42)
    for name in ("m", "v"):
        v = E4M3[d[name].numpy()]
        mean = np.delete(v, np.arange(0, n, 256)).mean()
        assert abs(mean - 0.3 * 448) <= 5 * 8 / np.sqrt(n) + 1e-3, (name, mean)
        assert len(np.unique(v)) == 3


def test_list_refused(hip):
    """A tensor listed twice, and gradients shared by two tensors (allowed)."""
    m = Model([100], DT_F32, DT_F32, False, False)
    with pytest.raises(CxmError) as e:
        engine.AdamW([m.dev[0], m.dev[0]])
    assert e.value.status == E_INVALID
    k = Model([100, 100], DT_F32, DT_F32, False, False, 3)
    k.dev[1]["g"] = k.dev[0]["g"]
    k.host[1]["g"] = k.host[0]["g"]
    k.opt = engine.AdamW(k.dev)
    k.opt.step(LR, 2)
    k.check(2)


def test_other_stream_and_repeat(hip):
    s = Stream()
    a, b = Model(SIZES, DT_BF16, DT_BF16, True, True, 17), Model(SIZES, DT_BF16, DT_BF16, True, True, 17)
    for t in (1, 2, 3):
        a.opt.step(LR, t, seed=t)
        b.opt.step(LR, t, seed=t, stream=s)
    s.sync()
    for x, y in zip(a.dev, b.dev):
        for name in ("p", "master", "m", "v", "m_scale", "v_scale"):
            assert np.array_equal(x[name].numpy(), y[name].numpy()), name
    s.close()
