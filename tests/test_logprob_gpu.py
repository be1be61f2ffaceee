"""Log probabilities of given tokens, the entropy, the top tokens and the
logits' gradient, through the C ABI, against float64 (tolerances: vocab_util)."""
import numpy as np
import pytest

from cortexmind_amd._lib import DT_BF16, DT_F16, DT_F32, call
from cortexmind_amd.device import DeviceArray
from gpu_util import dev
from layer_util import DTYPES, HALF, NAMES, TINY, U32, close, from_bits, get, out, ptr, rounded, up
from vocab_util import LOWEST, Rows, logits, top_of, upload

pytestmark = pytest.mark.gpu
# a wave or a workgroup per row, rows cut in two to many segments, ends of segments and chunks
SHAPES = [(1, 1), (3, 2), (5, 7), (2, 8), (3, 9), (70, 33), (5, 64), (9, 515), (1030, 130), (1100, 2049), (3, 4096), (2, 4099),
          (1029, 4103), (2, 16384), (1, 16388), (5, 20001), (3, 65537), (1, 131075)]


def forward(x, tok, dt, scale=1.0, top=0, ld=None, off=0, want=("logp", "entropy", "lse"), stream=None):
    rows, vocab = x.shape
    ld = vocab if ld is None else ld
    dx, dtok = upload(x, dt, ld, off), dev(tok) if tok is not None else None
    o = {k: dev(np.full(rows, -99.0, np.float32)) for k in want}
    if top:
        o["top_logp"], o["top_ids"] = dev(np.full((rows, top), -99.0, np.float32)), dev(np.full((rows, top), -99, np.int32))
    call("cxm_logprob_fwd_t", dx.ptr, ld, ptr(dtok), scale, ptr(o.get("logp")), ptr(o.get("entropy")), ptr(o.get("lse")),
         ptr(o.get("top_logp")), ptr(o.get("top_ids")), top, rows, vocab, dt, stream)
    return {k: v.numpy() for k, v in o.items()}


def check(x, tok, got, scale, top):
    r = Rows(x, scale)
    rows = np.arange(len(x))
    if "lse" in got:
        close(got["lse"], r.lse[:, 0], r.lse_err[:, 0], "lse")
    if "entropy" in got:
        close(got["entropy"], r.entropy[:, 0], r.entropy_err[:, 0], "entropy")
        assert np.all(got["entropy"] >= 0)
    if "logp" in got:
        want, gap = (a[rows, np.maximum(tok, 0)] for a in (r.logp, r.gap))
        given = tok >= 0
        dead = given & np.isinf(want)
        assert np.all(got["logp"][dead] == -np.inf) and np.all(got["logp"][~given] == 0)
        live = given & ~dead
        close(got["logp"][live], want[live], r.logp_err(gap, want)[live], "logp")
    if top:
        best = top_of(x, top)
        assert np.array_equal(got["top_ids"], best)
        for j in range(top):
            want, gap = (a[rows, best[:, j]] for a in (r.logp, r.gap))
            live = ~np.isinf(want)
            assert np.all(got["top_logp"][~live, j] == -np.inf)
            close(got["top_logp"][live, j], want[live], r.logp_err(gap, want)[live], f"top {j}")


def given(rows, vocab, seed):
    t = np.random.default_rng(seed).integers(0, vocab, rows).astype(np.int32)
    t[::7] = -1 if rows > 3 else t[::7]
    return t


@pytest.mark.parametrize("dt", DTYPES, ids=NAMES.get)
@pytest.mark.parametrize("rows,vocab", SHAPES)
def test_forward(hip, rows, vocab, dt):
    x, tok = logits(rows, vocab, dt, 1), given(rows, vocab, rows)
    for top, scale, ld, off, want in ((min(5, vocab), 1.0, vocab, 0, ("logp", "entropy", "lse")),
                                      (0, 0.5, vocab + 3, 1, ("logp", "entropy")),
                                      (min(64, vocab), 1.25, vocab + 64, 3, ("lse",)), (0, 2.0, vocab, 0, ("logp",)),
                                      (1, 1.0, vocab, 0, ())):
        got = forward(x, tok if "logp" in want else None, dt, scale, top, ld, off, want)
        check(x, tok, got, scale, top)


@pytest.mark.parametrize("dt", DTYPES, ids=NAMES.get)
@pytest.mark.parametrize("vocab", [70, 3000, 16384, 40001])
@pytest.mark.parametrize("rows", [2, 1100])
def test_ties(hip, rows, vocab, dt):
    """Equal logits: the lowest ids, within a lane, a segment and over segments."""
    if rows * vocab > 5e6:
        rows = 100
    x = np.zeros((rows, vocab))
    x[0] = np.arange(vocab) % 3  # many of the largest
    x[1, vocab // 2:] = 1.0      # the second half, after all
    if rows > 2:
        x[2] = np.where(np.arange(vocab) % 2, 0.0, -0.0)  # equal zeros
        x[3] = np.arange(vocab) // (vocab // 13) % 5       # steps
        x[4] = -np.inf
        x[4, [vocab - 1, 3]] = -1.0                        # fewer than asked for: the rest by id
        x[5] = np.linspace(-8, 8, vocab)
        x[6] = x[5, ::-1]
    x = rounded(x, dt)
    for top in (1, 7, 64):
        got = forward(x, None, dt, 1.0, top, want=("lse",))
        check(x, None, got, 1.0, top)


@pytest.mark.parametrize("dt", DTYPES, ids=NAMES.get)
@pytest.mark.parametrize("vocab", [5, 200, 9000, 50000])
def test_masks(hip, vocab, dt):
    """Masked logits of -inf and of the type's lowest value, all of a row's among them."""
    x = logits(6, vocab, dt, 11)
    x[0, ::2] = -np.inf
    x[1, 1:] = -np.inf
    x[2, ::2] = LOWEST[dt]
    x[3] = LOWEST[dt]
    x[4, :vocab // 2 + 1] = -np.inf
    tok = np.array([1 % vocab, 0, 1 % vocab, vocab - 1, 0, 0], np.int32)
    top = min(vocab, 6)
    got = forward(x, tok, dt, 1.0, top)
    check(x, tok, got, 1.0, top)
    assert got["logp"][1] == 0 and got["entropy"][1] == 0 and got["logp"][4] == -np.inf
    # all of a row equal, and lowest: a distribution like any other
    assert abs(got["entropy"][3] - np.log(vocab)) <= 200 * U32 * (1 + np.log(vocab))


@pytest.mark.parametrize("dt", DTYPES, ids=NAMES.get)
@pytest.mark.parametrize("vocab", [5, 200, 9000, 50000])
def test_rows_without_a_distribution(hip, vocab, dt):
    """All -inf, a NaN, +inf, tokens outside the vocabulary; other rows are as without them."""
    x = logits(6, vocab, dt, 12)
    x[1] = -np.inf
    x[2, vocab // 3] = np.nan
    x[3, vocab - 1] = np.inf
    tok = np.array([0, 1, 2, 3, vocab, 2 ** 31 - 1], np.int32)
    top = min(vocab, 4)
    got = forward(x, tok, dt, 1.0, top)
    assert got["lse"][1] == -np.inf and np.isnan(got["logp"][1]) and np.isnan(got["entropy"][1])
    assert np.array_equal(got["top_ids"][1], np.arange(top)) and np.all(np.isnan(got["top_logp"][1]))
    for k in ("lse", "logp", "entropy"):
        assert np.all(np.isnan(got[k][2:4])), k
    assert np.all(got["top_ids"][2] == -1) and np.all(np.isnan(got["top_logp"][2:4]))
    assert got["top_ids"][3, 0] == vocab - 1 and np.all(np.isnan(got["logp"][4:]))
    # as many rows, so that they are cut alike (how many there are decides the segments, and so the sums' order)
    keep = [0, 4, 5]
    x[1:4] = x[0]
    without = forward(x, np.zeros(6, np.int32), dt, 1.0, top)
    for k in ("lse", "entropy", "top_ids", "top_logp"):
        assert np.array_equal(got[k][keep], without[k][keep]), k


def test_large_and_small_values(hip):
    """Logits far from zero lose nothing by it."""
    for dt, mean in ((DT_F32, 3e5), (DT_F32, -3e5), (DT_F16, 2e4)):
        x, tok = logits(4, 5000, dt, 13, 8.0, mean), given(4, 5000, 1)
        check(x, tok, forward(x, tok, dt, 1.0, 3), 1.0, 3)


# ---------------------------------------------------------------- backward


def backward(x, tok, lse, ent, dlogp, dent, dt, scale=1.0, ld=None, ldd=None, off=0, in_place=False, stream=None):
    rows, vocab = x.shape
    ld, ldd = vocab if ld is None else ld, vocab if ldd is None else ldd
    f = lambda a: None if a is None else dev(np.asarray(a, np.float32))  # noqa: E731
    dx, dtok = upload(x, dt, ld, off, 0.0), None if tok is None else dev(tok)
    bl, be, bg, bh = f(lse), f(ent), f(dlogp), f(dent)
    do = dx if in_place else out((rows, ldd), dt, off)
    before = do.numpy().reshape(rows, ld if in_place else ldd).copy()
    call("cxm_logprob_bwd_t", dx.ptr, ld, ptr(dtok), scale, bl.ptr, ptr(be), ptr(bg), ptr(bh), do.ptr, ld if in_place else ldd,
         rows, vocab, dt, stream)
    got = do.numpy().reshape(before.shape)
    assert np.array_equal(got[:, vocab:], before[:, vocab:])  # between the rows
    return from_bits(got[:, :vocab].copy(), dt)


def check_backward(x, tok, lse, ent, dlogp, dent, dt, scale, got):
    scale = float(np.float32(scale))
    l64 = lse.astype(np.float64)[:, None]
    logp = x * scale - l64
    p = np.exp(logp)
    dead = np.isinf(logp)
    logp = np.where(dead, 0.0, logp)
    rows = np.arange(len(x))
    g = np.zeros(len(x)) if dlogp is None else np.where(tok >= 0, dlogp, 0.0)
    want, size = -g[:, None] * p, np.abs(g)[:, None] * p * (6 + 4 * np.abs(logp))
    if dlogp is not None:
        want[rows, np.maximum(tok, 0)] += g
        size[rows, np.maximum(tok, 0)] += 4 * np.abs(g)
    if dent is not None:
        h, e64 = dent.astype(np.float64)[:, None], ent.astype(np.float64)[:, None]
        want -= np.where(dead, 0.0, h * p * (logp + e64))
        size += np.abs(h) * p * (np.abs(logp) + np.abs(e64)) * (10 + 4 * np.abs(logp))
        size += np.abs(g)[:, None] * p * 2
    # z - lse loses a rounding of its operands' size
    size += (np.abs(x * scale) * ~dead + np.abs(l64)) * 2 * np.abs(want) if not np.any(dead) else \
        (np.where(dead, 0.0, np.abs(np.where(dead, 0.0, x) * scale)) + np.abs(l64)) * 2 * np.abs(want)
    want *= scale
    close(got, want, HALF[dt] * np.abs(want) + U32 * scale * size + TINY[dt] + 2.0 ** -120, "dlogits")


@pytest.mark.parametrize("dt", DTYPES, ids=NAMES.get)
@pytest.mark.parametrize("rows,vocab", SHAPES)
def test_backward(hip, rows, vocab, dt):
    x, tok = logits(rows, vocab, dt, 21), given(rows, vocab, rows + 1)
    if vocab > 8:
        x[:, 5::16] = -np.inf
        tok = np.where(tok % 16 == 5, tok - 1, tok).astype(np.int32)
    rng = np.random.default_rng(vocab)
    dlogp, dent = rng.normal(size=rows).astype(np.float32), rng.normal(size=rows).astype(np.float32)
    for scale, ld, ldd, off, g, h in ((1.0, vocab, vocab, 0, dlogp, dent), (0.5, vocab + 3, vocab + 5, 1, dlogp, None),
                                      (2.0, vocab + 64, vocab, 3, None, dent)):
        r = Rows(x, scale)
        lse, ent = r.lse[:, 0].astype(np.float32), r.entropy[:, 0].astype(np.float32)
        got = backward(x, tok, lse, ent if h is not None else None, g, h, dt, scale, ld, ldd, off)
        check_backward(x, tok, lse, ent, g, h, dt, scale, got)
        if ld == vocab:
            assert np.array_equal(got, backward(x, tok, lse, ent, g, h, dt, scale, in_place=True))


@pytest.mark.parametrize("dt", DTYPES, ids=NAMES.get)
@pytest.mark.parametrize("vocab", [6, 300, 20000])
def test_backward_of_special_rows(hip, vocab, dt):
    """Rows without a gradient are zeros whatever they hold; a token outside
    the vocabulary and a row without a distribution make NaN."""
    x = logits(7, vocab, dt, 22)
    x[0] = -np.inf
    x[1, 2] = np.nan
    x[5] = -np.inf
    tok = np.array([0, 1, -1, 3, vocab + 2, 0, -1], np.int32)
    dlogp = np.array([0, 0, 5, 1, 1, 1, 1], np.float32)
    dent = np.zeros(7, np.float32)
    lse = np.array([-np.inf, np.nan, 3, Rows(x[3:4], 1.0).lse[0, 0], 3, -np.inf, np.nan], np.float32)
    ent = np.array([np.nan, np.nan, 1, Rows(x[3:4], 1.0).entropy[0, 0], 1, np.nan, np.nan], np.float32)
    for h in (None, dent):
        got = backward(x, tok, lse, ent if h is not None else None, dlogp, h, dt)
        assert np.all(got[[0, 1, 2, 6]] == 0)
        assert np.all(np.isnan(got[[4, 5]]))
        check_backward(x[3:4], tok[3:4], lse[3:4], ent[3:4], dlogp[3:4], None if h is None else h[3:4], dt, 1.0, got[3:4])


def test_gradient_is_the_slope(hip):
    """fp32 gradients of logp and entropy against central differences of float64."""
    rows, vocab, scale = 2, 30, 1.25
    x, tok = logits(rows, vocab, DT_F32, 23, 1.5), np.array([4, 17], np.int32)
    g, h = np.array([0.7, -1.3], np.float32), np.array([0.4, 1.1], np.float32)

    def loss(v):
        r = Rows(v, scale)
        return (r.logp[np.arange(rows), tok] * g + r.entropy[:, 0] * h).sum()

    fwd = forward(x, tok, DT_F32, scale)
    got = backward(x, tok, fwd["lse"], fwd["entropy"], g, h, DT_F32, scale)
    for i in ((0, 4), (0, 9), (1, 17), (1, 29)):
        e = np.zeros_like(x)
        e[i] = 1e-5
        assert abs((loss(x + e) - loss(x - e)) / 2e-5 - got[i]) <= 1e-5, i


def test_rows_past_2_31_elements(hip):
    """Offsets that 32 bits do not hold: rows 2^31 + 5 elements apart."""
    vocab, ld, dt = 5000, (1 << 31) + 5, DT_BF16
    x = logits(2, vocab, dt, 24)
    buf = DeviceArray((ld + vocab,), np.uint16)
    rows = upload(x, dt, vocab)
    for r, at in ((0, 0), (1, ld)):
        call("cxm_memcpy_d2d", buf.ptr + 2 * at, rows.ptr + 2 * r * vocab, 2 * vocab, None)
    tok = dev(np.array([7, 4999], np.int32))
    o = {k: dev(np.zeros(2, np.float32)) for k in ("logp", "entropy", "lse")}
    tl, ti = dev(np.zeros((2, 3), np.float32)), dev(np.zeros((2, 3), np.int32))
    call("cxm_logprob_fwd_t", buf.ptr, ld, tok.ptr, 1.0, o["logp"].ptr, o["entropy"].ptr, o["lse"].ptr, tl.ptr, ti.ptr, 3, 2,
         vocab, dt, None)
    got = {k: v.numpy() for k, v in o.items()}
    got.update(top_logp=tl.numpy(), top_ids=ti.numpy())
    check(x, np.array([7, 4999]), got, 1.0, 3)
    g = dev(np.array([1.0, -2.0], np.float32))
    call("cxm_logprob_bwd_t", buf.ptr, ld, tok.ptr, 1.0, o["lse"].ptr, None, g.ptr, None, buf.ptr, ld, 2, vocab, dt, None)
    both = DeviceArray((2, vocab), np.uint16)
    for r, at in ((0, 0), (1, ld)):
        call("cxm_memcpy_d2d", both.ptr + 2 * r * vocab, buf.ptr + 2 * at, 2 * vocab, None)
    check_backward(x, np.array([7, 4999]), got["lse"], None, np.array([1.0, -2.0]), None, dt, 1.0, get(both, dt))


def test_same_bits_every_time(hip):
    x, tok = logits(3, 60000, DT_BF16, 25), given(3, 60000, 3)
    want = forward(x, tok, DT_BF16, 1.0, 20)
    for _ in range(4):
        got = forward(x, tok, DT_BF16, 1.0, 20)
        assert all(np.array_equal(got[k], want[k]) for k in want)
