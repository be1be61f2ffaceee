"""The lookup of a table's rows by token and the table's gradient, through the
C ABI, against the definition in float64.

Tolerances.  The lookup is one product rounded once (to fp32, then to the
type): compared bit by bit.  A row of the gradient adds up its tokens in the
order of the tokens: at most 128 of them by one wave, then the sums of the
workgroup's 8 waves, then those of the workgroups, an eighth of them in a row and
8 more.  No sum below has more than C = 400 roundings of partial sums, each at
most sum |dy|; the scale, the addend and the output round once each."""
import numpy as np
import pytest

from cortexmind_amd._lib import DT_BF16, DT_F16, DT_F32, call
from cortexmind_amd.data import SplitMix64
from cortexmind_amd.device import DeviceArray
from gpu_util import dev
from layer_util import DTYPES, HALF, NAMES, TINY, U32, close, from_bits, get, out, rounded, to_bits, up

pytestmark = pytest.mark.gpu
C = 400


def data(rows, cols, dt, seed):
    return rounded(SplitMix64(seed + 3 * rows + cols + dt).normal((rows, cols)), dt)


def tokens(n, vocab, seed, kind="text"):
    """Ids in proportion to 1 / (id + 1), a few of them padding; or all alike,
    in order, or spread evenly."""
    u = np.random.default_rng(seed).random(n)
    t = np.minimum((np.exp(u * np.log(vocab + 1.0)) - 1).astype(np.int32), vocab - 1)
    if kind == "text":
        t[::17] = -1
    elif kind == "one":
        t[:] = vocab // 2
    elif kind == "sorted":
        t = np.sort(t)
    elif kind == "even":
        t = (u * vocab).astype(np.int32)
    elif kind == "none":
        t[:] = -5
    return t


@pytest.mark.parametrize("dt", DTYPES, ids=NAMES.get)
@pytest.mark.parametrize("n,vocab,cols", [(1, 1, 1), (1, 300, 4096), (5, 7, 3), (9, 40, 8), (70, 33, 130), (1500, 1000, 72),
                                          (2100, 500, 1003), (1030, 97, 4100)])
def test_forward(hip, n, vocab, cols, dt):
    table, t = data(vocab, cols, dt, 1), tokens(n, vocab, n)
    t[n // 2] = vocab + 3 if n > 1 else 0
    for scale, off in ((1.0, 0), (7.3, 1)):
        dy, dtab, dt_ids = out((n, cols), dt, off), up(table, dt, off), dev(t, off)
        call("cxm_embedding_fwd_t", dtab.ptr, dt_ids.ptr, scale, dy.ptr, n, vocab, cols, dt, None)
        want = to_bits(table.astype(np.float32)[np.clip(t, 0, vocab - 1)] * np.float32(scale), dt)
        got = dy.numpy().reshape(n, cols)
        ok = (t >= 0) & (t < vocab)
        assert np.array_equal(got[ok], want[ok])
        assert np.all(from_bits(got[t < 0], dt) == 0)
        assert np.all(np.isnan(from_bits(got[t >= vocab], dt)))


def backward(t, dy, dt, vocab, scale=1.0, gdt=None, off=0, before=None, stream=None):
    cols, gdt = dy.shape[1], dt if gdt is None else gdt
    dw = out((vocab, cols), gdt, off) if before is None else up(before, gdt, off)
    bdy, bt = up(dy, dt, off), dev(t, off)
    call("cxm_embedding_bwd_t", bt.ptr, bdy.ptr, scale, dw.ptr, int(before is not None), len(t), vocab, cols, dt, gdt, stream)
    return get(dw, gdt).reshape(vocab, cols)


def check_backward(got, t, dy, vocab, scale, gdt, before=None):
    ok = (t >= 0) & (t < vocab)
    want, size = np.zeros((2, vocab, dy.shape[1]))
    np.add.at(want, t[ok], dy[ok])
    np.add.at(size, t[ok], np.abs(dy[ok]))
    scale = float(np.float32(scale))
    want, size = want * scale, size * abs(scale)
    if before is not None:
        size = size + np.abs(before)
        want = want + before
    close(got, want, HALF[gdt] * np.abs(want) + C * U32 * size + TINY[gdt])
    idle = np.ones(vocab, bool)
    idle[t[ok]] = False
    assert np.all(got[idle] == (0.0 if before is None else before[idle]))


CASES = [(1, 1, 1, "even"), (1, 5, 9, "text"), (7, 3, 2, "text"), (40, 1000, 16, "text"), (300, 17, 130, "text"),
         (500, 600, 515, "even"), (64, 64, 72, "sorted"), (1000, 513, 64, "one"), (2049, 1025, 40, "text"),
         (3000, 2, 1003, "even"), (5003, 1007, 771, "text"), (9000, 30000, 24, "text"), (20000, 500, 72, "one"),
         (70000, 131, 10, "text"), (131, 140000, 8, "even"), (4096, 4096, 64, "sorted"), (200, 90, 520, "none")]


@pytest.mark.parametrize("dt,gdt", [(DT_F32, DT_F32), (DT_BF16, DT_BF16), (DT_BF16, DT_F32), (DT_F16, DT_F16), (DT_F16, DT_F32)],
                         ids=lambda d: NAMES[d])
@pytest.mark.parametrize("n,vocab,cols,kind", CASES)
def test_backward(hip, n, vocab, cols, kind, dt, gdt):
    t, dy = tokens(n, vocab, n + cols, kind), data(n, cols, dt, 5)
    check_backward(backward(t, dy, dt, vocab, 1.0, gdt), t, dy, vocab, 1.0, gdt)
    before = data(vocab, cols, gdt, 7)
    check_backward(backward(t, dy, dt, vocab, -5.7, gdt, 1, before), t, dy, vocab, -5.7, gdt, before)


@pytest.mark.parametrize("n,cols", [(131072, 64), (300000, 9)])
def test_many_tokens_of_one_id(hip, n, cols):
    """Sums over the most workgroups; small whole numbers, so that they are exact."""
    t = np.zeros(n, np.int32)
    t[::3] = 2
    dy = (np.arange(n * cols).reshape(n, cols) % 7 - 3).astype(np.float64)
    got = backward(t, dy, DT_F16, 4, 1.0, DT_F32)
    want = np.stack([dy[t == v].sum(axis=0) for v in range(4)])
    assert np.array_equal(got, want)


def test_ids_outside_the_table(hip):
    """Ids below 0 and past the table's end take no part."""
    n, vocab, cols = 600, 50, 33
    t = np.random.default_rng(3).integers(-60, 120, n).astype(np.int32)
    t[:4] = (-2 ** 31, 2 ** 31 - 1, vocab, -1)
    dy = data(n, cols, DT_F32, 9)
    check_backward(backward(t, dy, DT_F32, vocab), t, dy, vocab, 1.0, DT_F32)


def test_no_tokens(hip):
    for dt in DTYPES:
        dw = out((300, 37), dt)
        call("cxm_embedding_bwd_t", None, None, 1.0, dw.ptr, 0, 0, 300, 37, dt, dt, None)
        assert np.all(get(dw, dt) == 0)


@pytest.mark.parametrize("cols", [3, 64, 1003])
def test_neighbours_untouched(hip, cols):
    pad, n, vocab = 16, 50, 20
    t, dy, table = tokens(n, vocab, 2), data(n, cols, DT_BF16, 11), data(vocab, cols, DT_BF16, 12)
    bt, bdy, btab = dev(t), up(dy, DT_BF16), up(table, DT_BF16)
    for size in (vocab, n):
        buf = DeviceArray.from_numpy(np.full(size * cols + 2 * pad, 0x1234, np.uint16))
        if size == vocab:
            call("cxm_embedding_bwd_t", bt.ptr, bdy.ptr, 1.0, buf.ptr + 2 * pad, 0, n, vocab, cols, DT_BF16, DT_BF16, None)
        else:
            call("cxm_embedding_fwd_t", btab.ptr, bt.ptr, 1.0, buf.ptr + 2 * pad, n, vocab, cols, DT_BF16, None)
        a = buf.numpy()
        assert np.all(a[:pad] == 0x1234) and np.all(a[-pad:] == 0x1234)


def test_same_bits_every_time(hip):
    t, dy = tokens(20000, 300, 1), data(20000, 72, DT_BF16, 13)
    want = backward(t, dy, DT_BF16, 300, 1.0, DT_F32)
    for _ in range(4):
        assert np.array_equal(backward(t, dy, DT_BF16, 300, 1.0, DT_F32), want)


def test_special_values(hip):
    """A NaN or an infinity in dy reaches its token's row and no other."""
    t = np.array([3, 1, 3, 0, 2, 1], np.int32)
    dy = data(6, 20, DT_F16, 15)
    dy[0, 4], dy[4, 7] = np.nan, np.inf
    dw = backward(t, dy, DT_F16, 5)
    assert np.isnan(dw[3, 4]) and np.isinf(dw[2, 7])
    dw[3, 4] = dw[2, 7] = 0.0
    assert np.all(np.isfinite(dw))
