"""The logits' gradients of rows whose lse is so large that its rounding to fp32
is much of a probability: rows of a mask's value alone, of the type's lowest
value, and rows moved far from zero.  Against float64.

Tolerance.  log p = scale (x - m) - ln S has a rounding of x - m, of c = scale
log2(e) and of the exponent in S and here (3 gap), of ln S, its product with
log2(e) and the sum itself (4 |log p|); S's own is vocab_util's (a lane adds chunks
of up to 8 terms, at most 60 of them here, and the lanes meet in a tree: below
C).  A probability is then off by that, of itself, and by the exponential's 2; the
few products around it add a rounding each, and the output half a step."""
import numpy as np
import pytest

from cortexmind_amd._lib import DT_BF16, DT_F16, DT_F32
from layer_util import DTYPES, HALF, NAMES, TINY, U32, close, rounded
from test_distill_gpu import backward as distill_backward
from test_distill_gpu import probabilities, teacher
from test_logprob_gpu import backward, check_backward, forward
from vocab_util import C, LOWEST, Rows, logits

pytestmark = pytest.mark.gpu
VOCABS = [5, 300, 2049, 9000, 50001]
MOVED = {DT_F32: 3e5, DT_BF16: 2e4, DT_F16: 3e4}
MASK = {DT_F32: -1e12, DT_BF16: -1e30, DT_F16: -65504.0}


def rows_of(vocab, dt, seed):
    x = logits(8, vocab, dt, seed)
    x[0] = MASK[dt]
    x[1] = LOWEST[dt]
    x[2] = rounded(MOVED[dt] + 8.0 * x[2], dt)
    x[3] = rounded(-MOVED[dt] + 8.0 * x[3], dt)
    x[4] = LOWEST[dt]
    x[4, ::2] = -np.inf                 # equal ones, and none
    x[5, 1:] = MASK[dt]                 # one that is near
    x[6, :vocab // 2 + 1] = MASK[dt]    # near enough to be as any row
    return rounded(x, dt)               # (as the device has them)


def exact(x, scale):
    """p, log p (0 where p is), the entropy, and the roundings of a probability."""
    r = Rows(x, scale)
    logp = np.where(np.isinf(r.logp), 0.0, r.logp)
    off = r.log_s_err + U32 * (3 * r.gap + 4 * np.abs(logp) + 2)
    # (rows that are not far: the rounding of lse, and of what it is taken from)
    near = np.abs(r.lse) < 4096
    off = off + np.where(near, 2 * U32 * (np.abs(r.lse) + r.gap + np.abs(r.m)), 0.0)
    with np.errstate(over="ignore"):
        return r, logp, off, r.lse[:, 0].astype(np.float32), r.entropy[:, 0].astype(np.float32)


def check(got, x, tok, g, h, dt, scale):
    r, logp, off, _, ent = exact(x, scale)
    s = float(np.float32(scale))
    rows = np.arange(len(x))
    g = np.where(tok >= 0, g, 0.0)[:, None] if g is not None else np.zeros((len(x), 1))
    h = np.zeros((len(x), 1)) if h is None else h.astype(np.float64)[:, None]
    ent = ent.astype(np.float64)[:, None]
    want = -g * r.p - h * r.p * (logp + ent)
    size = np.abs(g) * r.p * (off + 6 * U32)
    size += np.abs(h) * r.p * ((np.abs(logp) + ent) * (off + 10 * U32) + off)
    given = np.zeros_like(want)
    given[rows, np.maximum(tok, 0)] = g[:, 0]
    want = s * (want + given)
    size = s * (size + 4 * U32 * np.abs(given))
    # An exponential below 2^-126 is 0: what it lacks is p (|g| + |h| |log p + H|), and p |log p| grows with p there,
    # up to 2^-126 126 ln 2 < 2^-126 88.
    none = 2.0 ** -126 * s * (np.abs(g) + np.abs(h) * (88 + ent))
    close(got, want, HALF[dt] * np.abs(want) + size + TINY[dt] + none, "dlogits")


@pytest.mark.parametrize("dt", DTYPES, ids=NAMES.get)
@pytest.mark.parametrize("vocab", VOCABS)
def test_log_probabilities(hip, vocab, dt):
    x, rng = rows_of(vocab, dt, 41), np.random.default_rng(vocab)
    tok = rng.integers(0, vocab, 8).astype(np.int32)
    tok[4] = 1  # (not one of -inf)
    g, h = rng.normal(size=8).astype(np.float32), rng.normal(size=8).astype(np.float32)
    for scale, ld, ldd, off, dg, dh in ((1.0, vocab, vocab, 0, g, h), (1.25, vocab + 3, vocab + 5, 1, g, None),
                                        (0.5, vocab + 64, vocab, 3, None, h), (1.0, vocab, vocab, 0, g, None)):
        _, _, _, lse, ent = exact(x, scale)
        assert np.isinf(lse[1]) or np.abs(lse[:4]).min() >= 4096
        got = backward(x, tok, lse, ent if dh is not None else None, dg, dh, dt, scale, ld, ldd, off)
        check(got, x, tok, dg, dh, dt, scale)
        if ld == vocab:
            assert np.array_equal(got, backward(x, tok, lse, ent if dh is not None else None, dg, dh, dt, scale, in_place=True))


@pytest.mark.parametrize("dt", DTYPES, ids=NAMES.get)
def test_rows_of_a_wave(hip, dt):
    """As many rows as give each wave one."""
    vocab = 701
    x = np.tile(rows_of(vocab, dt, 42), (140, 1))
    rng = np.random.default_rng(3)
    tok = rng.integers(0, vocab, len(x)).astype(np.int32)
    tok[4::8] |= 1
    tok[::5] = -1
    g, h = rng.normal(size=len(x)).astype(np.float32), rng.normal(size=len(x)).astype(np.float32)
    _, _, _, lse, ent = exact(x, 1.0)
    got = backward(x, tok, lse, ent, g, h, dt, ld=vocab + 1, ldd=vocab)
    check(got, x, tok, g, h, dt, 1.0)
    assert np.array_equal(got, backward(x, tok, lse, ent, g, h, dt, in_place=True))


@pytest.mark.parametrize("dt", DTYPES, ids=NAMES.get)
@pytest.mark.parametrize("vocab", [300, 50001])
def test_after_the_forward(hip, vocab, dt):
    """With the lse and entropy that the forward pass gives: a row's gradient adds up to nothing."""
    x = rows_of(vocab, dt, 43)
    tok = np.full(8, 1, np.int32)
    g, h = np.linspace(0.5, 2, 8).astype(np.float32), np.linspace(-1, 1, 8).astype(np.float32)
    for scale in (1.0, 1.25):
        f = forward(x, tok, dt, scale)
        got = backward(x, tok, f["lse"], f["entropy"], g, h, dt, scale)
        r = Rows(x, scale)
        # half a step of each, and 2 (C + 8) roundings of what adds up (an entropy's error reaches every term)
        size = np.abs(g) * 2 + np.abs(h) * (r.p * np.abs(np.where(r.p > 0, r.logp, 0.0) + r.entropy)).sum(axis=1)
        size = scale * (size + np.abs(h) * (1 + r.entropy[:, 0]) * (1 + r.E[:, 0]))
        bound = (HALF[dt] + 2 * (C + 8) * U32 * (1 + r.E[:, 0] + np.minimum(np.abs(r.lse[:, 0]), 4096) / 64)) * size
        assert np.all(np.abs(got.sum(axis=1)) <= bound + vocab * TINY[dt]), (scale, got.sum(axis=1), bound)


@pytest.mark.parametrize("dt", DTYPES, ids=NAMES.get)
@pytest.mark.parametrize("vocab", [300, 20000])
def test_special_rows(hip, vocab, dt):
    """Rows without a gradient, tokens outside the vocabulary, NaN among logits, and rows of -inf, where lse is far too."""
    x = np.tile(rows_of(vocab, dt, 44)[2], (6, 1))
    x[3, 2], x[4] = np.nan, -np.inf
    tok = np.array([-1, 3, vocab, 3, 3, 4], np.int32)
    g = np.array([5, 0, 1, 1, 1, 1], np.float32)
    lse = np.full(6, Rows(x[:1], 1.0).lse[0, 0], np.float32)
    lse[4] = -np.inf
    got = backward(x, tok, lse, None, g, None, dt)
    assert np.all(got[:2] == 0) and np.all(np.isnan(got[2])) and np.isnan(got[3, 2]) and np.all(np.isnan(got[4]))
    check(got[5:], x[5:], tok[5:], g[5:], None, dt, 1.0)


@pytest.mark.parametrize("dt", DTYPES, ids=NAMES.get)
@pytest.mark.parametrize("vocab", [300, 20000])
def test_lse_of_more_logits(hip, vocab, dt):
    """An lse that is not the row's own (of a vocabulary of which the row is a part) is taken as it is."""
    x = rounded(MOVED[dt] + 8.0 * logits(3, vocab, dt, 45), dt)
    tok, g = np.array([0, 4, -1], np.int32), np.array([1, -2, 3], np.float32)
    lse = (Rows(x, 1.0).lse[:, 0] + 3.0 + 2.0 ** -20 * MOVED[dt]).astype(np.float32)
    check_backward(x, tok, lse, None, g, None, dt, 1.0, backward(x, tok, lse, None, g, None, dt))


@pytest.mark.parametrize("dt", DTYPES, ids=NAMES.get)
@pytest.mark.parametrize("vocab,k", [(9, 5), (300, 40), (2049, 256), (9000, 17), (50001, 64)])
def test_distillation(hip, vocab, k, dt):
    x, (ids, t) = rows_of(vocab, dt, 46), teacher(8, vocab, k, vocab)
    ids[7] = -1
    dloss = np.random.default_rng(k).random(8).astype(np.float32) + 0.5
    for scale, ld, ldd, off in ((1.0, vocab, vocab, 0), (1.25, vocab + 3, vocab + 5, 1)):
        r, logp, poff, lse, _ = exact(x, scale)
        got = distill_backward(x, ids, t, lse, dloss, dt, scale, ld, ldd, off)
        q, _, tgap, _ = probabilities(ids, t, scale)
        target, tsize = np.zeros_like(r.p), np.zeros_like(r.p)
        at = (np.arange(8)[:, None], np.maximum(ids, 0))
        np.add.at(target, at, q)
        np.add.at(tsize, at, q * (C + 8 + 3 * tgap) * U32)
        g = np.where(q.sum(axis=1) > 0, dloss, 0.0)[:, None] * float(np.float32(scale))
        want = g * (r.p - target)
        close(got, want, HALF[dt] * np.abs(want) + np.abs(g) * (r.p * (poff + 4 * U32) + tsize + 4 * U32 * np.abs(r.p - target)) +
              TINY[dt] + 2.0 ** -126 * np.abs(g), "dlogits")  # (an exponential below 2^-126 is 0)
        if ld == vocab:
            assert np.array_equal(got, distill_backward(x, ids, t, lse, dloss, dt, scale, in_place=True))
