"""Layer norm with the residual's addition, its 8-bit output and its backward,
through the C ABI, against the definition in float64.

Tolerances.  A sum of fp32 terms s_i that a thread adds one after the other
(at most 70 here) and that then meet in a tree (at most 10 levels, and the
partials of a column's workgroups) is off by at most C U32 sum |s_i| with
C = 128 for every shape below.  The mean is then off by d = C U32 mean|h|, each
h - mean by d and a rounding; the variance by C roundings (and d^2, which is
below one for means of up to 1000 deviations); the few products around them add
a rounding each.  Outputs then have half a step of their type."""
import numpy as np
import pytest

from cortexmind_amd._lib import DT_BF16, DT_F32, call
from cortexmind_amd.data import SplitMix64
from cortexmind_amd.device import DeviceArray, Stream
from gpu_util import dev
from layer_util import DTYPES, E4M3, HALF, NAMES, TINY, U32, close, get, out, ptr, rounded, up

pytestmark = pytest.mark.gpu
EPS = 1e-5
C = 128
SHAPES = [(1, 1), (3, 7), (2, 3), (5, 8), (2, 9), (33, 100), (17, 513), (1, 4096), (4, 1003), (1030, 1000), (3, 2049),
          (1025, 2040), (2, 4100), (1025, 4100), (2, 8200), (3, 16390), (2, 32760), (2, 33000), (2, 66000), (2, 140001)]
ids = lambda s: "x".join(map(str, s))  # noqa: E731


def data(rows, cols, dt, seed, std=1.0, mean=0.0):
    g = SplitMix64(seed + 7 * rows + cols + dt)
    return rounded(g.normal((rows, cols), mean, std), dt)


def moments(h, eps=EPS):
    mean = h.mean(axis=1)
    return mean, 1.0 / np.sqrt(((h - mean[:, None]) ** 2).mean(axis=1) + eps)


def forward(x, res, w, b, dt, q8=False, off=0, eps=EPS, alias=None, stream=None):
    """(h, y or (q, scale), mean, rstd) from the entry point."""
    rows, cols = x.shape
    dx, dw = up(x, dt, off), up(w, dt, off)
    db = up(b, dt, off) if b is not None else None
    dr = up(res, dt, off) if res is not None else None
    dh = out((rows, cols), dt, off) if res is not None else None
    dy = None if q8 else out((rows, cols), dt, off)
    if alias == "y=x":
        dy = dx
    if alias == "h=x,y=res":
        dh, dy = dx, dr
    dq = dev(np.full((rows, cols), 0x55, np.uint8), off) if q8 else None
    ds = dev(np.full(rows, -1.0, np.float32)) if q8 else None
    dm, dv = dev(np.full(rows, 9.0, np.float32)), dev(np.full(rows, -1.0, np.float32))
    call("cxm_layernorm_fwd_t", dx.ptr, ptr(dr), dw.ptr, ptr(db), eps, ptr(dh), ptr(dy), ptr(dq), ptr(ds), dm.ptr, dv.ptr,
         rows, cols, dt, stream and stream.handle)
    if stream:
        stream.sync()
    y = (dq.numpy(), ds.numpy()) if q8 else get(dy, dt)
    return (get(dh, dt) if dh is not None else None), y, dm.numpy(), dv.numpy()


def check_forward(x, res, w, b, dt, got_h, y, mean, rstd, q8):
    h = x if res is None else rounded((x + res).astype(np.float32), dt)
    m64, r64 = moments(h)
    n = (h - m64[:, None]) * r64[:, None]
    y64 = n * w + (0.0 if b is None else b)
    if res is not None:
        assert np.array_equal(got_h, h)  # one fp32 sum, one rounding
    size = np.abs(h).mean(axis=1)
    close(mean, m64, C * U32 * size, "mean")
    close(rstd, r64, C * U32 * r64, "rstd")
    off = U32 * ((C + 8) * np.abs(n * w) + 2 * np.abs(y64) + np.abs(w) * (r64 * (C + 2) * size)[:, None])
    if not q8:
        close(y, y64, HALF[dt] * np.abs(y64) + off + TINY[dt], "y")
        return
    q, scale = y
    s64 = np.abs(y64).max(axis=1) / 448.0
    close(scale, s64, off.max(axis=1) / 448.0 + 4 * U32 * s64, "scale")
    # half a step of the value, or of the smallest values, around y / scale
    v = E4M3[q] * scale[:, None].astype(np.float64)
    step = np.maximum(np.abs(y64) * 2.0 ** -4, s64[:, None] * 2.0 ** -10)
    close(v, y64, step * (1 + 2.0 ** -10) + 2 * off + off.max(axis=1)[:, None], "q")


@pytest.mark.parametrize("dt", DTYPES, ids=NAMES.get)
@pytest.mark.parametrize("shape", SHAPES, ids=ids)
def test_forward(hip, shape, dt):
    rows, cols = shape
    x, w, b = data(rows, cols, dt, 1, 1.0, 3.0), data(1, cols, dt, 2, 0.2, 1.0)[0], data(1, cols, dt, 4, 0.5)[0]
    res = data(rows, cols, dt, 3, 2.0)
    for r, bias, q8 in ((None, b, False), (res, b, False), (res, None, True), (None, b, True)):
        got = forward(x, r, w, bias, dt, q8)
        check_forward(x, r, w, bias, dt, *got, q8)


@pytest.mark.parametrize("cols", [100, 1000, 4096, 40000])
def test_large_mean(hip, cols):
    """Rows whose mean is 500 deviations: the sum of squares alone would lose them."""
    x, w = data(3, cols, DT_F32, 21, 0.5, 250.0), data(1, cols, DT_F32, 22, 0.2, 1.0)[0]
    check_forward(x, None, w, None, DT_F32, *forward(x, None, w, None, DT_F32), False)


@pytest.mark.parametrize("dt", DTYPES, ids=NAMES.get)
@pytest.mark.parametrize("shape", [(5, 24), (7, 1003), (3, 4096), (2, 40000)], ids=ids)
def test_misaligned_and_in_place(hip, shape, dt):
    """Element-aligned pointers, and h and y in the places of x and res: the same bits."""
    rows, cols = shape
    x, w, res = data(rows, cols, dt, 4), data(1, cols, dt, 5, 0.2, 1.0)[0], data(rows, cols, dt, 6, 2.0)
    b = data(1, cols, dt, 7)[0]
    want = forward(x, res, w, b, dt)
    for kw in ({"off": 1}, {"off": 3}, {"alias": "h=x,y=res"}):
        got = forward(x, res, w, b, dt, **kw)
        assert all(np.array_equal(p, q) for p, q in zip(got, want)), kw
    y = forward(x, None, w, b, dt)[1]
    assert np.array_equal(y, forward(x, None, w, b, dt, alias="y=x")[1])
    (q, s), (q2, s2) = forward(x, res, w, b, dt, True)[1], forward(x, res, w, b, dt, True, off=1)[1]
    assert np.array_equal(q, q2) and np.array_equal(s, s2)


@pytest.mark.parametrize("cols", [5, 64, 1000, 40000])
def test_neighbours_untouched(hip, cols):
    """What lies before and behind the outputs stays."""
    rows, dt, pad = 3, DT_BF16, 16
    x, w = data(rows, cols, dt, 8), data(1, cols, dt, 9, 0.2, 1.0)[0]
    buf = DeviceArray.from_numpy(np.full(rows * cols + 2 * pad, 0x1234, np.uint16))
    qb = DeviceArray.from_numpy(np.full(rows * cols + 2 * pad, 0x5A, np.uint8))
    ds = dev(np.zeros(rows, np.float32))
    dx, dw = up(x, dt), up(w, dt)
    call("cxm_layernorm_fwd_t", dx.ptr, None, dw.ptr, dw.ptr, EPS, None, buf.ptr + 2 * pad, qb.ptr + pad, ds.ptr, None,
         None, rows, cols, dt, None)
    for a, v in ((buf.numpy(), 0x1234), (qb.numpy(), 0x5A)):
        assert np.all(a[:pad] == v) and np.all(a[-pad:] == v)


@pytest.mark.parametrize("dt", DTYPES, ids=NAMES.get)
@pytest.mark.parametrize("cols", [1, 6, 200, 3000, 40000])
def test_special_rows(hip, cols, dt):
    """A row of equal values gives the bias; a NaN or an infinity its whole row
    NaN; no other row changes."""
    x, w, b = data(4, cols, dt, 10), np.ones(cols), data(1, cols, dt, 11)[0]
    x[0] = 2.0  # (sums of 2 are exact)
    x[1, cols // 2] = np.nan
    x[2, cols - 1] = np.inf
    _, y, mean, rstd = forward(x, None, w, b, dt)
    assert np.array_equal(y[0], b) and mean[0] == 2.0
    assert np.all(np.isnan(y[1:3])) and np.all(np.isnan(rstd[1:3]))
    _, want, _, _ = forward(x[3:], None, w, b, dt)
    assert np.array_equal(y[3:], want)


# ---------------------------------------------------------------- backward


def backward(h, mean, rstd, w, dy, dh, dt, off=0, alias=None, stream=None, bias=True):
    rows, cols = h.shape
    bh, bw, bdy = up(h, dt, off), up(w, dt, off), up(dy, dt, off)
    bdh = up(dh, dt, off) if dh is not None else None
    bm, br = dev(np.asarray(mean, np.float32)), dev(np.asarray(rstd, np.float32))
    dx = {"h": bh, "dy": bdy, "dh": bdh}[alias] if alias else out((rows, cols), dt, off)
    dw, db = out((cols,), dt, off), (out((cols,), dt, off) if bias else None)
    call("cxm_layernorm_bwd_t", bh.ptr, bm.ptr, br.ptr, bw.ptr, bdy.ptr, ptr(bdh), dx.ptr, dw.ptr, ptr(db), rows, cols, dt,
         stream and stream.handle)
    if stream:
        stream.sync()
    return get(dx, dt), get(dw, dt), (get(db, dt) if bias else None)


def backward64(h, mean, rstd, w, dy, dh):
    n = (h - mean[:, None].astype(np.float64)) * rstd[:, None].astype(np.float64)
    g = dy * w
    mg, mgn = g.mean(axis=1, keepdims=True), (g * n).mean(axis=1, keepdims=True)
    rs = rstd[:, None].astype(np.float64)
    dx = rs * (g - mg - n * mgn) + (0.0 if dh is None else dh)
    size = rs * (8 * (np.abs(g) + np.abs(mg) + np.abs(n * mgn)) +
                 (C + 4) * (np.abs(g).mean(axis=1, keepdims=True) + np.abs(n) * np.abs(g * n).mean(axis=1, keepdims=True)))
    return dx, U32 * (size + 2 * np.abs(dx) + (0.0 if dh is None else np.abs(dh))), n


def check_backward(h, mean, rstd, w, dy, dh, dt, dx, dw, db):
    want, off, n = backward64(h, mean, rstd, w, dy, dh)
    close(dx, want, HALF[dt] * np.abs(want) + off + TINY[dt], "dx")
    for got, terms, what in ((dw, dy * n, "dw"), (db, dy, "db")):
        if got is not None:
            total = terms.sum(axis=0)
            close(got, total, HALF[dt] * np.abs(total) + (C + 4) * U32 * np.abs(terms).sum(axis=0) + TINY[dt], what)


def bwd_data(rows, cols, dt, seed=30):
    h, dy, dh = (data(rows, cols, dt, seed + i, s, m) for i, (s, m) in enumerate(((2.0, 1.0), (1.0, 0.1), (1.0, 0.0))))
    mean, rstd = (v.astype(np.float32) for v in moments(h))
    return h, mean, rstd, data(1, cols, dt, seed + 5, 0.3, 1.0)[0], dy, dh


@pytest.mark.parametrize("dt", DTYPES, ids=NAMES.get)
@pytest.mark.parametrize("shape", SHAPES + [(700, 96), (513, 2048), (600, 8448), (257, 6001), (300, 16384)],
                         ids=ids)
def test_backward(hip, shape, dt):
    h, mean, rstd, w, dy, dh = bwd_data(*shape, dt)
    for d in (None, dh):
        check_backward(h, mean, rstd, w, dy, d, dt, *backward(h, mean, rstd, w, dy, d, dt, bias=d is not None))


@pytest.mark.parametrize("dt", DTYPES, ids=NAMES.get)
@pytest.mark.parametrize("shape", [(5, 24), (70, 1003), (300, 2048), (3, 9000), (300, 8201), (2, 40000)],
                         ids=ids)
def test_backward_misaligned_and_in_place(hip, shape, dt):
    h, mean, rstd, w, dy, dh = bwd_data(*shape, dt, 50)
    want = backward(h, mean, rstd, w, dy, dh, dt)
    for kw in ({"off": 1}, {"off": 3}, {"alias": "h"}, {"alias": "dy"}, {"alias": "dh"}):
        got = backward(h, mean, rstd, w, dy, dh, dt, **kw)
        assert all(np.array_equal(a, b) for a, b in zip(got, want)), kw


def test_backward_of_no_rows(hip):
    """Empty sums: dw and db are zeros."""
    for dt in DTYPES:
        dw, db = out((37,), dt), out((37,), dt)
        call("cxm_layernorm_bwd_t", None, None, None, None, None, None, None, dw.ptr, db.ptr, 0, 37, dt, None)
        assert np.all(get(dw, dt) == 0) and np.all(get(db, dt) == 0)


def test_backward_is_the_slope_of_the_forward(hip):
    """fp32 gradients against central differences of the float64 definition."""
    rows, cols = 3, 20
    h, mean, rstd, w, dy, _ = bwd_data(rows, cols, DT_F32, 70)
    dx, dw, db = backward(h, mean, rstd, w, dy, None, DT_F32)

    def loss(hh, ww, bb):
        m, r = moments(hh)
        return ((((hh - m[:, None]) * r[:, None]) * ww + bb) * dy).sum()

    step, b = 1e-5, np.zeros(cols)
    for i in ((0, 0), (1, 7), (2, 19)):
        e = np.zeros_like(h)
        e[i] = step
        assert abs((loss(h + e, w, b) - loss(h - e, w, b)) / (2 * step) - dx[i]) <= 1e-5
    for j in (0, 11, 19):
        e = np.zeros(cols)
        e[j] = step
        assert abs((loss(h, w + e, b) - loss(h, w - e, b)) / (2 * step) - dw[j]) <= 1e-5
        assert abs((loss(h, w, b + e) - loss(h, w, b - e)) / (2 * step) - db[j]) <= 1e-5
