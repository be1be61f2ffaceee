"""The divergence from a teacher's distribution over its top tokens and the
logits' gradient, through the C ABI, against float64 (tolerances: vocab_util)."""
import numpy as np
import pytest

from cortexmind_amd._lib import DT_BF16, DT_F32, call
from gpu_util import dev
from layer_util import DTYPES, HALF, NAMES, TINY, U32, close, from_bits, out
from vocab_util import C, Rows, logits, upload

pytestmark = pytest.mark.gpu
SHAPES = [(1, 1, 1), (3, 5, 2), (2, 8, 8), (70, 33, 16), (5, 515, 256), (1030, 130, 40), (1100, 2049, 64), (3, 4099, 100),
          (1029, 4103, 5), (2, 16388, 256), (5, 20001, 17), (3, 65537, 64), (1, 131075, 33)]


def teacher(rows, vocab, k, seed):
    """Distinct tokens where there are enough, else some twice; a few entries missing or impossible."""
    rng = np.random.default_rng(seed)
    ids = np.stack([rng.permutation(max(vocab, k))[:k] % vocab for _ in range(rows)]).astype(np.int32)
    t = rng.normal(4.0, 2.0, (rows, k)).astype(np.float32)
    if k > 3:
        ids[::2, 1] = -1
        t[1::3, 2] = -np.inf
        ids[:, 3] = ids[:, 0]  # a token twice
    return ids, t


def probabilities(ids, t, scale):
    z = np.where(ids < 0, -np.inf, t.astype(np.float64) * float(np.float32(scale)))
    m = z.max(axis=1, keepdims=True)
    e = np.exp(z - np.where(np.isinf(m), 0.0, m))
    s = e.sum(axis=1, keepdims=True)
    with np.errstate(divide="ignore", invalid="ignore"):
        return np.where(s > 0, e / s, 0.0), np.where(e > 0, z - m - np.log(s), 0.0), np.where(e > 0, m - z, 0.0), np.log(s)


def forward(x, ids, t, dt, scale=1.0, ld=None, off=0):
    rows, vocab = x.shape
    ld = vocab if ld is None else ld
    dx, di, dtv = upload(x, dt, ld, off), dev(ids), dev(t)
    loss, lse = dev(np.full(rows, -99.0, np.float32)), dev(np.full(rows, -99.0, np.float32))
    call("cxm_distill_fwd_t", dx.ptr, ld, di.ptr, dtv.ptr, ids.shape[1], scale, loss.ptr, lse.ptr, rows, vocab, dt, None)
    return loss.numpy(), lse.numpy()


def check_forward(x, ids, t, scale, loss, lse):
    r = Rows(x, scale)
    close(lse, r.lse[:, 0], r.lse_err[:, 0], "lse")
    q, logq, tgap, logz = probabilities(ids, t, scale)
    safe = np.maximum(ids, 0)
    logp, gap = (np.take_along_axis(a, safe, 1) for a in (r.logp, r.gap))
    logp = np.where(q > 0, logp, 0.0)
    want = (q * (logq - logp)).sum(axis=1)
    # q's exponents have two roundings, its sums up to 256 entries' in a tree; each term two more
    size = (q * ((C + 3 * tgap) * (np.abs(logq) + np.abs(logp)) + 4 * gap + 4 * tgap)).sum(axis=1)
    size += (C + 4) * (1 + np.abs(logz[:, 0])) * (q.sum(axis=1) > 0) + 4 * np.abs(want)
    close(loss, want, r.log_s_err[:, 0] + U32 * size, "loss")


@pytest.mark.parametrize("dt", DTYPES, ids=NAMES.get)
@pytest.mark.parametrize("rows,vocab,k", SHAPES)
def test_forward(hip, rows, vocab, k, dt):
    x, (ids, t) = logits(rows, vocab, dt, 1), teacher(rows, vocab, k, rows)
    for scale, ld, off in ((1.0, vocab, 0), (0.5, vocab + 3, 1)):
        check_forward(x, ids, t, scale, *forward(x, ids, t, dt, scale, ld, off))


def backward(x, ids, t, lse, dloss, dt, scale=1.0, ld=None, ldd=None, off=0, in_place=False):
    rows, vocab = x.shape
    ld, ldd = vocab if ld is None else ld, vocab if ldd is None else ldd
    dx, di, dtv = upload(x, dt, ld, off, 0.0), dev(ids), dev(t)
    bl, bg = dev(np.asarray(lse, np.float32)), dev(np.asarray(dloss, np.float32))
    do = dx if in_place else out((rows, ldd), dt, off)
    before = do.numpy().reshape(rows, -1).copy()
    call("cxm_distill_bwd_t", dx.ptr, ld, di.ptr, dtv.ptr, ids.shape[1], scale, bl.ptr, bg.ptr, do.ptr, ld if in_place else ldd,
         rows, vocab, dt, None)
    got = do.numpy().reshape(before.shape)
    assert np.array_equal(got[:, vocab:], before[:, vocab:])  # between the rows
    return from_bits(got[:, :vocab].copy(), dt)


def check_backward(x, ids, t, lse, dloss, dt, scale, got):
    q, _, tgap, _ = probabilities(ids, t, scale)
    s = float(np.float32(scale))
    l64 = lse.astype(np.float64)[:, None]
    logp = x * s - l64
    p = np.exp(logp)
    target, tsize = np.zeros_like(p), np.zeros_like(p)
    rows = np.arange(len(x))[:, None]
    np.add.at(target, (rows, np.maximum(ids, 0)), q)
    np.add.at(tsize, (rows, np.maximum(ids, 0)), q * (C + 8 + 3 * tgap))
    g = np.where(q.sum(axis=1) > 0, dloss, 0.0)[:, None] * s
    want = g * (p - target)
    dead = np.isinf(logp)
    size = np.abs(g) * (p * (8 + np.where(dead, 0.0, 4 * np.abs(logp) + 2 * np.abs(x * s) + 2 * np.abs(l64))) + tsize)
    close(got, want, HALF[dt] * np.abs(want) + U32 * size + TINY[dt] + 2.0 ** -120, "dlogits")


@pytest.mark.parametrize("dt", DTYPES, ids=NAMES.get)
@pytest.mark.parametrize("rows,vocab,k", SHAPES)
def test_backward(hip, rows, vocab, k, dt):
    x, (ids, t) = logits(rows, vocab, dt, 2), teacher(rows, vocab, k, rows + 1)
    dloss = np.random.default_rng(k).random(rows).astype(np.float32) + 0.5
    if vocab > 8:
        banned = [j for j in range(5, vocab, 16) if j not in set(ids.ravel())]
        x[:, banned] = -np.inf
    for scale, ld, ldd, off in ((1.0, vocab, vocab, 0), (0.5, vocab + 3, vocab + 5, 1)):
        lse = Rows(x, scale).lse[:, 0].astype(np.float32)
        got = backward(x, ids, t, lse, dloss, dt, scale, ld, ldd, off)
        check_backward(x, ids, t, lse, dloss, dt, scale, got)
        if ld == vocab:
            assert np.array_equal(got, backward(x, ids, t, lse, dloss, dt, scale, in_place=True))


@pytest.mark.parametrize("dt", DTYPES, ids=NAMES.get)
@pytest.mark.parametrize("vocab", [9, 300, 20000])
def test_special_rows(hip, vocab, dt):
    """Rows without an entry, entries of -inf and of one token alone, ids
    outside the vocabulary, a masked token that the teacher names."""
    x = logits(8, vocab, dt, 3)
    ids = np.tile(np.arange(6, dtype=np.int32), (8, 1))
    t = np.random.default_rng(1).normal(size=(8, 6)).astype(np.float32)
    ids[0] = -1
    t[1] = -np.inf
    ids[2] = 4           # one token, six times
    ids[3, 5] = vocab
    x[4, 2] = -np.inf    # named by the teacher: infinitely far
    x[5, 2] = -np.inf
    t[5, 2] = -np.inf    # named with probability 0
    x[6] = -np.inf
    t[7, 1] = np.nan
    loss, lse = forward(x, ids, t, dt)
    assert loss[0] == 0 and loss[1] == 0 and loss[4] == np.inf
    assert np.isnan(loss[[3, 6, 7]]).all() and lse[6] == -np.inf
    keep = [2, 5]
    check_forward(x[keep], ids[keep], t[keep], 1.0, loss[keep], lse[keep])
    dloss = np.ones(8, np.float32)
    got = backward(x, ids, t, lse, dloss, dt)
    assert np.all(got[:2] == 0) and np.all(np.isnan(got[[3, 6, 7]]))
    keep = [2, 4, 5]
    check_backward(x[keep], ids[keep], t[keep], lse[keep], dloss[keep], dt, 1.0, got[keep])
    got = backward(x, ids, t, np.where(np.isfinite(lse), lse, np.nan), np.zeros(8, np.float32), dt)
    assert np.all(got[[0, 1, 2, 4, 5, 6]] == 0)


def test_teacher_from_the_top_tokens(hip):
    """The ids and log probabilities that cxm_logprob_fwd_t returns are a teacher:
    against its own logits the divergence is that of the tokens left out, and the
    largest gradient is of them."""
    rows, vocab, k, dt = 6, 20000, 64, DT_BF16
    x = logits(rows, vocab, dt, 4)
    dx, tl, ti = upload(x, dt, vocab), dev(np.zeros((rows, k), np.float32)), dev(np.zeros((rows, k), np.int32))
    call("cxm_logprob_fwd_t", dx.ptr, vocab, None, 1.0, None, None, None, tl.ptr, ti.ptr, k, rows, vocab, dt, None)
    loss, lse = dev(np.zeros(rows, np.float32)), dev(np.zeros(rows, np.float32))
    call("cxm_distill_fwd_t", dx.ptr, vocab, ti.ptr, tl.ptr, k, 1.0, loss.ptr, lse.ptr, rows, vocab, dt, None)
    kept = np.exp(tl.numpy().astype(np.float64)).sum(axis=1)
    assert np.all(np.abs(loss.numpy() + np.log(kept)) <= 1e-5)
    check_forward(x, ti.numpy(), tl.numpy(), 1.0, loss.numpy(), lse.numpy())


def test_gradient_is_the_slope(hip):
    """fp32 gradients against central differences of float64."""
    rows, vocab, k, scale = 2, 30, 7, 0.5
    x, (ids, t) = logits(rows, vocab, DT_F32, 5, 1.5), teacher(rows, vocab, k, 9)
    dloss = np.array([0.7, 1.9], np.float32)
    q, logq, _, _ = probabilities(ids, t, scale)

    def total(v):
        logp = np.take_along_axis(Rows(v, scale).logp, np.maximum(ids, 0), 1)
        return ((q * (logq - logp)).sum(axis=1) * dloss).sum()

    _, lse = forward(x, ids, t, DT_F32, scale)
    got = backward(x, ids, t, lse, dloss, DT_F32, scale)
    for i in ((0, int(ids[0, 0])), (0, 9), (1, int(ids[1, 5])), (1, 29)):
        e = np.zeros_like(x)
        e[i] = 1e-5
        assert abs((total(x + e) - total(x - e)) / 2e-5 - got[i]) <= 1e-5, i
