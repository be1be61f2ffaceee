"""The RMS norm with the residual's addition, its 8-bit output and its
backward, through the C ABI, against the definition in float64.

Tolerances.  A sum of fp32 terms s_i that a thread adds one after the other
(at most 70 here) and that then meet in a tree (at most 10 levels, and the
partials of a column's workgroups) is off by at most C U32 sum |s_i| with
C = 128 for every shape below; the few products around it add a rounding
each.  Outputs then have half a step of their type."""
import numpy as np
import pytest

from cortexmind_amd._lib import DT_BF16, DT_F32, call
from cortexmind_amd.data import SplitMix64
from cortexmind_amd.device import DeviceArray, Stream
from gpu_util import dev
from layer_util import (DTYPES, E4M3, HALF, NAMES, TINY, U32, close, e4m3_nearest, from_bits, get, out, ptr, rounded,
                        to_bits, up)

pytestmark = pytest.mark.gpu
EPS = 1e-5
C = 128
SHAPES = [(1, 1), (3, 7), (2, 3), (5, 8), (2, 9), (33, 100), (17, 513), (1, 4096), (4, 1003), (1030, 1000), (3, 2049),
          (1025, 2040), (2, 4100), (1025, 4100), (2, 8200), (3, 16390), (2, 32760), (2, 70001)]
ids = lambda s: "x".join(map(str, s))  # noqa: E731


def data(rows, cols, dt, seed, std=1.0, mean=0.0):
    g = SplitMix64(seed + 7 * rows + cols + dt)
    return rounded(g.normal((rows, cols), mean, std), dt)


def forward64(x, res, w, dt, eps=EPS):
    h = x if res is None else rounded((x + res).astype(np.float32), dt)
    rstd = 1.0 / np.sqrt((h * h).mean(axis=1) + eps)
    return h, rstd, h * rstd[:, None] * w


def forward(x, res, w, dt, q8=False, off=0, eps=EPS, alias=None, stream=None):
    """(h, y or (q, scale), rstd) from the entry point."""
    rows, cols = x.shape
    dx, dw = up(x, dt, off), up(w, dt, off)
    dr = up(res, dt, off) if res is not None else None
    dh = out((rows, cols), dt, off) if res is not None else None
    dy = None if q8 else out((rows, cols), dt, off)
    if alias == "y=x":
        dy = dx
    if alias == "h=x,y=res":
        dh, dy = dx, dr
    dq = dev(np.full((rows, cols), 0x55, np.uint8), off) if q8 else None
    ds = dev(np.full(rows, -1.0, np.float32)) if q8 else None
    dv = dev(np.full(rows, -1.0, np.float32))
    call("cxm_rmsnorm_fwd_t", dx.ptr, ptr(dr), dw.ptr, eps, ptr(dh), ptr(dy), ptr(dq), ptr(ds), dv.ptr, rows, cols, dt,
         stream)
    y = (dq.numpy(), ds.numpy()) if q8 else get(dy, dt)
    return (get(dh, dt) if dh is not None else None), y, dv.numpy()


def check_forward(x, res, w, dt, got_h, y, rstd, q8):
    h, r64, y64 = forward64(x, res, w, dt)
    if res is not None:
        assert np.array_equal(got_h, h)  # one fp32 sum, one rounding
    close(rstd, r64, C * U32 * r64, "rstd")
    if not q8:
        close(y, y64, (HALF[dt] + C * U32) * np.abs(y64) + TINY[dt], "y")
        return
    q, scale = y
    s64 = np.abs(y64).max(axis=1) / 448.0
    close(scale, s64, (C + 4) * U32 * s64, "scale")
    # half a step of the value, or of the smallest values, around y / scale
    v = E4M3[q] * scale[:, None].astype(np.float64)
    step = np.maximum(np.abs(y64) * 2.0 ** -4, s64[:, None] * 2.0 ** -10)
    close(v, y64, step * (1 + 2.0 ** -10) + 2 * C * U32 * np.abs(y64), "q")


@pytest.mark.parametrize("dt", DTYPES, ids=NAMES.get)
@pytest.mark.parametrize("shape", SHAPES, ids=ids)
def test_forward(hip, shape, dt):
    rows, cols = shape
    x, w = data(rows, cols, dt, 1), data(1, cols, dt, 2, 0.2, 1.0)[0]
    res = data(rows, cols, dt, 3, 2.0)
    for r in (None, res):
        for q8 in (False, True):
            got = forward(x, r, w, dt, q8)
            check_forward(x, r, w, dt, *got, q8)


@pytest.mark.parametrize("dt", DTYPES, ids=NAMES.get)
@pytest.mark.parametrize("shape", [(5, 24), (7, 1003), (3, 4096), (2, 40000)], ids=ids)
def test_misaligned_and_in_place(hip, shape, dt):
    """Element-aligned pointers, and h and y in the places of x and res: the same bits."""
    rows, cols = shape
    x, w, res = data(rows, cols, dt, 4), data(1, cols, dt, 5, 0.2, 1.0)[0], data(rows, cols, dt, 6, 2.0)
    h, y, rstd = forward(x, res, w, dt)
    for kw in ({"off": 1}, {"off": 3}, {"alias": "h=x,y=res"}):
        h2, y2, r2 = forward(x, res, w, dt, **kw)
        assert np.array_equal(h, h2) and np.array_equal(y, y2) and np.array_equal(rstd, r2), kw
    _, y, _ = forward(x, None, w, dt)
    _, y2, _ = forward(x, None, w, dt, alias="y=x")
    assert np.array_equal(y, y2)
    (q, s), (q2, s2) = forward(x, res, w, dt, True)[1], forward(x, res, w, dt, True, off=1)[1]
    assert np.array_equal(q, q2) and np.array_equal(s, s2)


@pytest.mark.parametrize("cols", [5, 64, 1000, 40000])
def test_neighbours_untouched(hip, cols):
    """What lies before and behind the outputs stays."""
    rows, dt = 3, DT_BF16
    x, w = data(rows, cols, dt, 8), data(1, cols, dt, 9, 0.2, 1.0)[0]
    pad = 16
    buf = DeviceArray.from_numpy(np.full(rows * cols + 2 * pad, 0x1234, np.uint16))
    qb = DeviceArray.from_numpy(np.full(rows * cols + 2 * pad, 0x5A, np.uint8))
    ds = dev(np.zeros(rows, np.float32))
    dx, dw = up(x, dt), up(w, dt)
    call("cxm_rmsnorm_fwd_t", dx.ptr, None, dw.ptr, EPS, None, buf.ptr + 2 * pad, qb.ptr + pad, ds.ptr, None, rows,
         cols, dt, None)
    for a, v in ((buf.numpy(), 0x1234), (qb.numpy(), 0x5A)):
        assert np.all(a[:pad] == v) and np.all(a[-pad:] == v)


@pytest.mark.parametrize("dt", DTYPES, ids=NAMES.get)
@pytest.mark.parametrize("cols", [6, 200, 3000, 40000])
def test_special_rows(hip, cols, dt):
    """A zero row gives zeros; a NaN its whole row; an infinity NaN at its
    place and zeros beside it; no other row changes."""
    x, w = data(4, cols, dt, 10), np.ones(cols)
    x[0] = 0.0
    x[1, cols // 2] = np.nan
    x[2, cols - 1] = np.inf
    _, y, rstd = forward(x, None, w, dt)
    assert np.all(y[0] == 0) and np.all(np.isnan(y[1])) and np.isnan(y[2, -1]) and np.all(y[2, :-1] == 0)
    assert rstd[2] == 0 and np.isnan(rstd[1])
    _, want, _ = forward(x[3:], None, w, dt)
    assert np.array_equal(y[3:], want)
    q, scale = forward(x, None, w, dt, True)[1]
    assert scale[0] == 0 and np.all(q[0] & 0x7F == 0)
    assert not np.isfinite(scale[1]) and not np.isfinite(scale[2])
    q1, s1 = forward(x[3:], None, w, dt, True)[1]
    assert np.array_equal(q[3:], q1) and scale[3] == s1[0]


def test_largest_value_is_exact_in_8_bits(hip):
    """The row's largest magnitude is stored as 448 whatever the rounding of
    its scale, and values of half the smallest step round to even."""
    for k in range(1, 40):
        x = np.array([[0.37 * k, -0.37 * k, 0.0, 1e-30, 0.01 * k]], np.float32)
        dx, q, s = dev(x), dev(np.zeros((1, 5), np.uint8)), dev(np.zeros(1, np.float32))
        call("cxm_quant_rows_t", dx.ptr, q.ptr, s.ptr, 1, 5, DT_F32, None)
        c, sc = q.numpy()[0], s.numpy()[0]
        assert E4M3[c[0]] == 448 and E4M3[c[1]] == -448 and E4M3[c[2]] == 0 and E4M3[c[3]] == 0
        assert abs(float(sc) * 448.0 - x[0, 0]) <= 2.01 * U32 * float(x[0, 0])


@pytest.mark.parametrize("dt", DTYPES, ids=NAMES.get)
@pytest.mark.parametrize("shape", [(1, 1), (3, 7), (65, 128), (5, 1003), (2, 5000), (2, 70001)], ids=ids)
def test_quant_rows(hip, shape, dt):
    rows, cols = shape
    x = data(rows, cols, dt, 12)
    dx, q, s = up(x, dt), dev(np.full(shape, 0x55, np.uint8)), dev(np.zeros(rows, np.float32))
    call("cxm_quant_rows_t", dx.ptr, q.ptr, s.ptr, rows, cols, dt, None)
    sc = s.numpy()
    want = np.abs(x).max(axis=1) / 448.0
    close(sc, want, 2 * U32 * want)  # the reciprocal of 448 and the product, a rounding each
    inv = (np.float32(1.0) / sc).astype(np.float32)
    scaled = (x.astype(np.float32) * inv[:, None]).astype(np.float64)
    assert np.array_equal(E4M3[q.numpy()], E4M3[e4m3_nearest(np.clip(scaled, -448, 448))])


# ------------------------------------------------------------- backward


def backward64(h, rstd, w, dy, dh):
    n = h * rstd[:, None]
    g = dy * w
    dx = rstd[:, None] * (g - n * (g * n).mean(axis=1, keepdims=True))
    size = rstd[:, None] * (np.abs(g) + np.abs(n) * np.abs(g * n).mean(axis=1, keepdims=True))
    if dh is not None:
        dx, size = dx + dh, size + np.abs(dh)
    return dx, size, (dy * n).sum(axis=0), np.abs(dy * n).sum(axis=0)


def backward(h, rstd, w, dy, dh, dt, off=0, alias=None, stream=None):
    rows, cols = h.shape
    b = {"h": up(h, dt, off), "dy": up(dy, dt, off), "dh": None if dh is None else up(dh, dt, off)}
    dr, dw_in = dev(rstd), up(w, dt, off)
    dx = b[alias] if alias else out((rows, cols), dt, off)
    dw = out(cols, dt, off)
    call("cxm_rmsnorm_bwd_t", b["h"].ptr, dr.ptr, dw_in.ptr, b["dy"].ptr, ptr(b["dh"]), dx.ptr, dw.ptr, rows, cols, dt,
         stream)
    return get(dx, dt), get(dw, dt)


def bwd_data(rows, cols, dt):
    h, dy = data(rows, cols, dt, 20, 2.0), data(rows, cols, dt, 21)
    dh, w = data(rows, cols, dt, 22), data(1, cols, dt, 23, 0.2, 1.0)[0]
    rstd = (1.0 / np.sqrt((h * h).mean(axis=1) + EPS)).astype(np.float32)
    return h, rstd, w, dy, dh


@pytest.mark.parametrize("dt", DTYPES, ids=NAMES.get)
@pytest.mark.parametrize("shape", SHAPES + [(5000, 33), (3, 128)], ids=ids)
def test_backward(hip, shape, dt):
    h, rstd, w, dy, dh = bwd_data(*shape, dt)
    for g in (None, dh):
        dx, dw = backward(h, rstd, w, dy, g, dt)
        want, size, want_w, size_w = backward64(h, rstd.astype(np.float64), w, dy, g)
        close(dx, want, HALF[dt] * np.abs(want) + C * U32 * size + TINY[dt], "dx")
        close(dw, want_w, HALF[dt] * np.abs(want_w) + C * U32 * size_w + TINY[dt], "dw")


@pytest.mark.parametrize("dt", DTYPES, ids=NAMES.get)
@pytest.mark.parametrize("shape", [(9, 24), (300, 1003), (2, 40000)], ids=ids)
def test_backward_in_place_and_misaligned(hip, shape, dt):
    h, rstd, w, dy, dh = bwd_data(*shape, dt)
    want = backward(h, rstd, w, dy, dh, dt)
    for kw in ({"off": 1}, {"alias": "h"}, {"alias": "dy"}, {"alias": "dh"}):
        got = backward(h, rstd, w, dy, dh, dt, **kw)
        assert all(np.array_equal(a, b) for a, b in zip(got, want)), kw


# several long rows for each workgroup, the last turn taken by some only
@pytest.mark.parametrize("dt", DTYPES, ids=NAMES.get)
@pytest.mark.parametrize("shape", [(600, 8200), (300, 12289), (513, 16384)], ids=ids)
def test_backward_of_many_long_rows(hip, shape, dt):
    h, rstd, w, dy, dh = bwd_data(*shape, dt)
    dx, dw = backward(h, rstd, w, dy, dh, dt)
    want, size, want_w, size_w = backward64(h, rstd.astype(np.float64), w, dy, dh)
    close(dx, want, HALF[dt] * np.abs(want) + C * U32 * size + TINY[dt], "dx")
    close(dw, want_w, HALF[dt] * np.abs(want_w) + C * U32 * size_w + TINY[dt], "dw")
    for kw in ({"off": 1}, {"alias": "h"}, {"alias": "dy"}, {"alias": "dh"}):
        got = backward(h, rstd, w, dy, dh, dt, **kw)
        assert np.array_equal(got[0], dx) and np.array_equal(got[1], dw), kw


def test_backward_of_no_rows(hip):
    dw = out(10, DT_F32)
    call("cxm_rmsnorm_bwd_t", None, None, None, None, None, None, dw.ptr, 0, 10, DT_F32, None)
    assert np.all(dw.numpy() == 0)
    call("cxm_rmsnorm_fwd_t", None, None, None, EPS, None, None, None, None, None, 0, 10, DT_F32, None)


def test_backward_against_differences(hip):
    """fp32 gradients of sum(dy * y) against central differences of the
    definition in float64 (step 1e-5: truncation 1e-10, rounding 1e-10)."""
    rows, cols, dt = 3, 37, DT_F32
    h, rstd, w, dy, _ = bwd_data(rows, cols, dt)
    dx, dw = backward(h, rstd, w, dy, None, dt)

    def f(a, b):
        return float((forward64(a, None, b, dt)[2] * dy).sum())

    step = 1e-5
    for r, c in ((0, 0), (1, 17), (2, 36)):
        e = np.zeros_like(h)
        e[r, c] = step
        num = (f(h + e, w) - f(h - e, w)) / (2 * step)
        assert abs(num - dx[r, c]) <= 1e-5 * (1 + np.abs(dx).max())
        e = np.zeros_like(w)
        e[c] = step
        num = (f(h, w + e) - f(h, w - e)) / (2 * step)
        assert abs(num - dw[c]) <= 1e-5 * (1 + np.abs(dw).max())


def test_runs_repeat_and_streams_agree(hip):
    """The same bits on every run and on another stream."""
    h, rstd, w, dy, dh = bwd_data(2000, 520, DT_BF16)
    want = backward(h, rstd, w, dy, dh, DT_BF16)
    s = Stream()
    for stream in (None, s.handle):
        for _ in range(2):
            got = backward(h, rstd, w, dy, dh, DT_BF16, stream=stream)
            s.sync()
            assert all(np.array_equal(a, b) for a, b in zip(got, want))
    s.close()


def test_offsets_past_32_bits(hip):
    """Rows whose elements lie past 2^32 (bf16, in place)."""
    rows, cols = 66000, 65536
    buf = DeviceArray((rows * cols,), np.uint16)
    buf.fill_bytes(0x3F)  # 0.746...
    last = data(1, cols, DT_BF16, 30)
    at = buf.ptr + 2 * (rows - 1) * cols
    bits = to_bits(last, DT_BF16)
    call("cxm_memcpy_h2d", at, bits.ctypes.data, bits.nbytes, None)
    w = up(np.ones(cols), DT_BF16)
    rstd = DeviceArray((rows,), np.float32)
    call("cxm_rmsnorm_fwd_t", buf.ptr, None, w.ptr, 0.0, None, buf.ptr, None, None, rstd.ptr, rows, cols, DT_BF16, None)
    got = np.empty(cols, np.uint16)
    call("cxm_memcpy_d2h", got.ctypes.data, at, got.nbytes, None)
    _, r64, y64 = forward64(last, None, 1.0, DT_BF16, 0.0)
    close(from_bits(got, DT_BF16), y64[0], (HALF[DT_BF16] + C * U32) * np.abs(y64[0]))
    call("cxm_memcpy_d2h", got.ctypes.data, at - 2 * cols, got.nbytes, None)
    assert np.all(from_bits(got, DT_BF16) == 1.0)
    close(rstd.numpy()[-1:], r64, C * U32 * r64)
