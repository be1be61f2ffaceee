"""The layer operators at the ends of their ranges of sizes."""
import numpy as np
import pytest

from cortexmind_amd._lib import DT_BF16, DT_F16, DT_F32, call
from cortexmind_amd.data import SplitMix64
from cortexmind_amd.device import DeviceArray
from layer_util import HALF, TINY, U32, close, from_bits, get, rounded, to_bits, up

pytestmark = pytest.mark.gpu


def test_more_rows_than_a_copy_has_workgroups(hip):
    """Rows of 18 bytes are copied to whole stages, 8 rows a workgroup, and there
    are more than one launch's 2^23 workgroups of them."""
    m, k, n, dt = 67_200_003, 9, 8, DT_F16
    period = 4099
    g = SplitMix64(91)
    x, w = rounded(g.normal((period, k)), dt), rounded(g.normal((k, n)), dt)
    dx = DeviceArray.from_numpy(np.resize(x.astype(np.float16).view(np.uint16), (m, k)))
    dw, dy = up(w, dt), DeviceArray((m, n), np.uint16)
    call("cxm_linear_fwd_t", dx.ptr, dw.ptr, None, None, None, dy.ptr, m, k, n, 0, 0, dt, None)
    y = dy.numpy()
    want, size = x @ w, np.abs(x) @ np.abs(w)
    close(y[:period].view(np.float16), want, HALF[dt] * np.abs(want) + k * U32 * size + TINY[dt])
    for r in range(period, m, period * 1024):  # the same bits in every period
        part = y[r:r + period * 1024]
        assert np.array_equal(part, np.resize(y[:period], part.shape)), r


# 2^23 - 1: rows that are copied to whole stages then take all of 2^23 values
LAST = (1 << 23) - 1
PERIOD = 1021


def across(a, dt):
    """[rows, PERIOD] repeated along the rows' LAST columns, on the device."""
    return DeviceArray.from_numpy(np.concatenate([np.resize(r, (1, LAST)) for r in to_bits(a, dt)]))


def test_longest_rows_of_k(hip):
    m, n, dt = 40, 64, DT_BF16
    g = SplitMix64(92)
    x, w = rounded(g.normal((m, PERIOD), 0.5), dt), rounded(g.normal((n, PERIOD), 0.5), dt)
    dx, dw, dy = across(x, dt), across(w, dt), DeviceArray((m, n), np.uint16)
    call("cxm_linear_fwd_t", dx.ptr, dw.ptr, None, None, None, dy.ptr, m, LAST, n, 1, 0, dt, None)
    turns, rest = divmod(LAST, PERIOD)
    want = turns * (x @ w.T) + x[:, :rest] @ w[:, :rest].T
    size = turns * (np.abs(x) @ np.abs(w).T)
    # a split's 1024 stages of 32 are added up in steps of 16, its 512 or fewer splits in turn
    close(get(dy, dt), want, HALF[dt] * np.abs(want) + (2048 + 16 + 512) * U32 * size)


def test_longest_rows_of_n(hip):
    m, k, dt = 300, 64, DT_F16
    g = SplitMix64(93)
    x, w = rounded(g.normal((m, k)), dt), rounded(g.normal((k, PERIOD)), dt)
    dx, dw, dy = up(x, dt), across(w, dt), DeviceArray((m, LAST), np.uint16)
    call("cxm_linear_fwd_t", dx.ptr, dw.ptr, None, None, None, dy.ptr, m, k, LAST, 0, 0, dt, None)
    y = dy.numpy()
    want, size = x @ w, np.abs(x) @ np.abs(w)
    close(from_bits(y[:, :PERIOD], dt), want, HALF[dt] * np.abs(want) + k * U32 * size + TINY[dt])
    for r in range(m):
        assert np.array_equal(y[r], np.resize(y[r, :PERIOD], LAST)), r


def test_longest_rows_backward(hip):
    m, n, dt = 64, 64, DT_F16
    g = SplitMix64(94)
    x, dy = rounded(g.normal((m, PERIOD)), dt), rounded(g.normal((m, n)), dt)
    w = rounded(g.normal((PERIOD, n)), dt)
    bx, bdy = across(x, dt), up(dy, dt)
    bw = DeviceArray.from_numpy(np.resize(to_bits(w, dt), (LAST, n)))
    dx, dw = DeviceArray((m, LAST), np.uint16), DeviceArray((LAST, n), np.uint16)
    call("cxm_linear_bwd_t", bx.ptr, bw.ptr, None, bdy.ptr, None, dx.ptr, dw.ptr, None, m, LAST, n, 0, 0, dt, None)
    gx, gw = dx.numpy(), dw.numpy()
    want, size = dy @ w.T, np.abs(dy) @ np.abs(w).T
    close(from_bits(gx[:, :PERIOD], dt), want, HALF[dt] * np.abs(want) + n * U32 * size + TINY[dt])
    for r in range(m):
        assert np.array_equal(gx[r], np.resize(gx[r, :PERIOD], LAST)), r
    want, size = x.T @ dy, np.abs(x).T @ np.abs(dy)
    close(from_bits(gw[:PERIOD], dt), want, HALF[dt] * np.abs(want) + m * U32 * size + TINY[dt])
    assert np.array_equal(gw, np.resize(gw[:PERIOD], (LAST, n)))


@pytest.mark.parametrize("dt", [DT_F32, DT_BF16], ids=["f32", "bf16"])
def test_longest_rows_of_the_norm_backward(hip, dt):
    """2^26 - 1 columns: the sums of dw of the last ones are past one launch's grid."""
    rows, cols, period = 2, (1 << 26) - 1, 4093
    g = SplitMix64(95)
    h, dy = rounded(g.normal((rows, period)), dt), rounded(g.normal((rows, period)), dt)
    w = rounded(g.normal((1, period), 1.0, 0.2), dt)

    def long(a):
        return DeviceArray.from_numpy(np.concatenate([np.resize(r, (1, cols)) for r in to_bits(a, dt)]))

    rstd = np.array([0.75, 1.25], np.float32)
    bh, bdy, bw, br = long(h), long(dy), long(w), DeviceArray.from_numpy(rstd)
    store = np.float32 if dt == DT_F32 else np.uint16
    dx, dw = DeviceArray((rows, cols), store), DeviceArray((cols,), store)
    call("cxm_rmsnorm_bwd_t", bh.ptr, br.ptr, bw.ptr, bdy.ptr, None, dx.ptr, dw.ptr, rows, cols, dt, None)
    n, gr = h * rstd[:, None].astype(np.float64), dy * w
    turns, rest = divmod(cols, period)
    dot = (gr * n).sum(axis=1) * turns + (gr * n)[:, :rest].sum(axis=1)
    mag = np.abs(gr * n).sum(axis=1) * (turns + 1)
    got = dw.numpy()
    want, size = (dy * n).sum(axis=0), np.abs(dy * n).sum(axis=0)
    close(from_bits(got[:period], dt), want, HALF[dt] * np.abs(want) + 4 * U32 * size + TINY[dt], "dw")
    assert np.array_equal(got, np.resize(got[:period], cols))
    # a thread's sum has 8 columns of every 8192, of four-column chunks 4 of every 4096: 2^16 terms in turn
    mean, off = dot / cols, (2 ** 16 + 32) * U32 * mag / cols
    r = rstd[:, None].astype(np.float64)
    want = r * (gr - n * mean[:, None])
    size = r * (np.abs(gr) + np.abs(n) * np.abs(mean)[:, None])
    gx = dx.numpy()
    close(from_bits(gx[:, :period], dt), want,
          HALF[dt] * np.abs(want) + 4 * U32 * size + r * np.abs(n) * off[:, None] + TINY[dt], "dx")
    for i in range(rows):
        assert np.array_equal(gx[i], np.resize(gx[i, :period], cols)), i
