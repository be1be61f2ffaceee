"""Element types, 8-bit floats and uploads of the layer operators' tests
(imported by test modules only)."""
import numpy as np

from cortexmind_amd._lib import DT_BF16, DT_F16, DT_F32
from gpu_util import dev

DTYPES = [DT_F32, DT_BF16, DT_F16]
NAMES = {DT_F32: "f32", DT_BF16: "bf16", DT_F16: "f16"}
# half a step relative to the value, and half the step of the smallest values
HALF = {DT_F32: 2.0 ** -24, DT_BF16: 2.0 ** -8, DT_F16: 2.0 ** -11}
TINY = {DT_F32: 2.0 ** -150, DT_BF16: 2.0 ** -134, DT_F16: 2.0 ** -25}
U32 = 2.0 ** -24  # one fp32 rounding
STORE = {DT_F32: np.float32, DT_BF16: np.uint16, DT_F16: np.uint16}


def to_bits(x, dt):
    """x rounded to nearest even, as the arrays the entry points take."""
    x = np.ascontiguousarray(x, np.float32)
    if dt == DT_F32:
        return x
    if dt == DT_F16:
        return x.astype(np.float16).view(np.uint16)
    u = x.view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def from_bits(b, dt):
    """The float64 values of such an array."""
    b = np.asarray(b)
    if dt == DT_F32:
        return b.astype(np.float64)
    if dt == DT_F16:
        return b.view(np.float16).astype(np.float64)
    return (b.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def rounded(x, dt):
    return from_bits(to_bits(x, dt), dt)


def _e4m3_table():
    v = np.zeros(256)
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        x = m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
        v[c] = (np.nan if (c & 127) == 127 else x) * (-1 if c & 128 else 1)
    return v


E4M3 = _e4m3_table()
_POS = E4M3[:127]


def e4m3_nearest(a):
    """Codes of |a| <= 448 rounded to nearest even, sign kept."""
    x = np.abs(np.asarray(a, np.float64))
    hi = np.clip(np.searchsorted(_POS, x, side="left"), 0, 126)
    lo = np.maximum(hi - 1, 0)
    dl, dh = x - _POS[lo], _POS[hi] - x
    pick = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    return np.where(np.signbit(a), pick | 128, pick).astype(np.uint8)


def e4m3_below(a):
    """(index of the neighbour at or below, share of the way to the one above)."""
    x = np.asarray(a, np.float64)
    lo = np.clip(np.searchsorted(_POS, x, side="right") - 1, 0, 126)
    hi = np.minimum(lo + 1, 126)
    gap = np.where(hi > lo, _POS[hi] - _POS[lo], 1.0)
    return lo, (x - _POS[lo]) / gap


def quant_rows(x):
    """(codes, scales) of rows in float64 arithmetic."""
    s = np.abs(x).max(axis=1) / 448.0
    s = np.where(s < 2.0 ** -126, 0.0, s)
    return e4m3_nearest(np.where(s[:, None] > 0, x / np.where(s > 0, s, 1.0)[:, None], 0.0)), s.astype(np.float32)


def up(x, dt, off=0):
    """Uploads x in the type; off: elements by which the pointer is misaligned."""
    return dev(to_bits(x, dt), off)


def out(shape, dt, off=0, fill=None):
    """An output buffer full of a byte pattern, so that unwritten places show."""
    a = np.full(shape, 0x7777 if dt != DT_F32 else 0, STORE[dt])
    if dt == DT_F32:
        a = np.full(shape, -7.0e30, np.float32)
    return dev(a, off)


def get(d, dt):
    return from_bits(d.numpy(), dt)


def ptr(d):
    return None if d is None else d.ptr


def close(got, want, tol, what=""):
    got, want, tol = np.broadcast_arrays(np.asarray(got, np.float64), want, tol)
    assert np.all(np.isfinite(got)), what
    err = np.abs(got - want) - tol
    worst = np.unravel_index(np.argmax(err), err.shape)
    assert np.all(err <= 0), (what, worst, got[worst], want[worst], tol[worst])
