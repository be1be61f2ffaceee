"""Arguments that the layer operators refuse on the host, before any launch:
null pointers, types, sizes and overlaps (no GPU; addresses are never read)."""
import ctypes

import pytest

from cortexmind_amd import _lib
from cortexmind_amd._lib import (ACT_EXP, ACT_GELU, ACT_NONE, ACT_RELU, ACT_SILU, DT_BF16, DT_E4M3, DT_F16, DT_F32,
                                 E_INVALID, E_TOO_LARGE, OK)

A = [0x10000000 * (i + 1) for i in range(12)]  # addresses far apart


@pytest.fixture(scope="module")
def lib():
    return _lib.lib()


def fwd(lib, x=A[0], res=A[1], w=A[2], eps=1e-5, h=A[3], y=A[4], q=None, scale=None, rstd=A[7], rows=4, cols=64,
        dt=DT_BF16):
    return lib.cxm_rmsnorm_fwd_t(x, res, w, eps, h, y, q, scale, rstd, rows, cols, dt, None)


@pytest.mark.parametrize("kw", [
    dict(x=None), dict(w=None), dict(y=None), dict(q=A[5]), dict(res=None), dict(cols=0), dict(dt=DT_E4M3), dict(dt=9),
    dict(eps=-1.0), dict(eps=float("nan")),
    dict(y=A[0] + 2), dict(h=A[1] + 128), dict(h=A[4]), dict(q=A[0], scale=A[6]), dict(q=A[5], scale=A[5] + 8),
    dict(rstd=A[4] + 64), dict(y=A[2]), dict(rstd=A[2]),
])
def test_norm_forward(lib, kw):
    assert fwd(lib, **kw) == E_INVALID


def test_norm_sizes(lib):
    assert fwd(lib, rows=0, x=None) == OK
    assert fwd(lib, cols=1 << 31) == E_TOO_LARGE
    assert fwd(lib, rows=1 << 41) == E_TOO_LARGE
    assert fwd(lib, rows=1 << 40, cols=1 << 30) == E_TOO_LARGE  # a product past 64 bits
    # grids of 2^32 threads and more
    assert fwd(lib, x=1 << 44, res=None, w=A[2], h=None, y=1 << 45, rstd=None, rows=1 << 32, cols=8) == E_TOO_LARGE
    assert bwd(lib, h=1 << 44, dy=1 << 45, dh=None, dx=1 << 46, cols=1 << 26) == E_TOO_LARGE


def bwd(lib, h=A[0], rstd=A[1], w=A[2], dy=A[3], dh=A[4], dx=A[5], dw=A[6], rows=4, cols=64, dt=DT_F16):
    return lib.cxm_rmsnorm_bwd_t(h, rstd, w, dy, dh, dx, dw, rows, cols, dt, None)


@pytest.mark.parametrize("kw", [
    dict(h=None), dict(rstd=None), dict(w=None), dict(dy=None), dict(dx=None), dict(dw=None), dict(cols=0),
    dict(dt=DT_E4M3), dict(dx=A[0] + 2), dict(dx=A[3] + 2), dict(dx=A[4] + 2), dict(dx=A[2]), dict(dw=A[2]),
    dict(dw=A[3] + 64), dict(dw=A[5] + 8), dict(dx=A[1]),
])
def test_norm_backward(lib, kw):
    assert bwd(lib, **kw) == E_INVALID


@pytest.mark.parametrize("kw", [dict(x=None), dict(q=None), dict(s=None), dict(cols=0), dict(dt=DT_E4M3), dict(q=A[0] + 4),
                                dict(s=A[0]), dict(s=A[1] + 16)])
def test_quant(lib, kw):
    a = dict(x=A[0], q=A[1], s=A[2], cols=64, dt=DT_F32)
    a.update(kw)
    assert lib.cxm_quant_rows_t(a["x"], a["q"], a["s"], 4, a["cols"], a["dt"], None) == E_INVALID


def lin(lib, x=A[0], w=A[1], bias=A[2], res=A[3], z=A[4], y=A[5], m=4, k=64, n=32, tw=0, act=ACT_GELU, dt=DT_BF16):
    return lib.cxm_linear_fwd_t(x, w, bias, res, z, y, m, k, n, tw, act, dt, None)


@pytest.mark.parametrize("kw", [
    dict(x=None), dict(w=None), dict(y=None), dict(k=0), dict(dt=DT_E4M3), dict(dt=-1), dict(act=ACT_EXP), dict(act=7),
    dict(y=A[3] + 2), dict(z=A[3]), dict(z=A[5]), dict(y=A[0]), dict(y=A[1] + 16), dict(z=A[2]), dict(z=A[0] + 100),
    dict(dt=DT_F32, y=A[3], z=None),
])
def test_linear_forward(lib, kw):
    assert lin(lib, **kw) == E_INVALID


def test_linear_sizes(lib):
    assert lin(lib, m=0, x=None) == OK and lin(lib, n=0, y=None) == OK
    for kw in (dict(k=1 << 23), dict(n=1 << 23), dict(m=1 << 31)):
        assert lin(lib, **kw) == E_TOO_LARGE
    # more tiles, and more elements of the fp32 epilogue, than a grid has
    big = dict(x=1 << 44, w=1 << 45, bias=None, res=None, z=None, y=1 << 47, m=(1 << 31) - 1, k=64, n=(1 << 23) - 1)
    for dt in (DT_BF16, DT_F32):
        assert lin(lib, dt=dt, **big) == E_TOO_LARGE


def q8(lib, x=A[0], xs=A[1], w=A[2], ws=A[3], bias=A[4], res=A[5], z=A[6], y=A[7], m=4, k=64, n=32, act=ACT_RELU,
       dt=DT_BF16):
    return lib.cxm_linear_q8_fwd(x, xs, w, ws, bias, res, z, y, m, k, n, act, dt, None)


@pytest.mark.parametrize("kw", [
    dict(x=None), dict(xs=None), dict(w=None), dict(ws=None), dict(y=None), dict(k=0), dict(dt=DT_F32), dict(dt=DT_E4M3),
    dict(act=ACT_EXP), dict(y=A[5] + 2), dict(y=A[1]), dict(z=A[3]), dict(z=A[7] + 4), dict(y=A[2] + 4),
])
def test_linear_q8(lib, kw):
    assert q8(lib, **kw) == E_INVALID


def lbwd(lib, x=A[0], w=A[1], z=A[2], dy=A[3], dz=A[4], dx=A[5], dw=A[6], db=A[7], m=4, k=64, n=32, tw=0, act=ACT_SILU,
         dt=DT_BF16):
    return lib.cxm_linear_bwd_t(x, w, z, dy, dz, dx, dw, db, m, k, n, tw, act, dt, None)


@pytest.mark.parametrize("kw", [
    dict(dy=None), dict(z=None), dict(dz=None), dict(w=None), dict(x=None), dict(m=0), dict(k=0), dict(n=0),
    dict(dt=DT_E4M3), dict(act=ACT_EXP), dict(dz=A[2] + 2), dict(dz=A[3] + 2), dict(dz=A[0]), dict(dx=A[3]),
    dict(dx=A[1]), dict(dw=A[6], db=A[6] + 64), dict(dw=A[0]), dict(db=A[4]), dict(dx=A[6]),
])
def test_linear_backward(lib, kw):
    assert lbwd(lib, **kw) == E_INVALID


def test_linear_backward_sizes(lib):
    for kw in (dict(k=1 << 23), dict(n=1 << 23), dict(m=1 << 23)):
        assert lbwd(lib, **kw) == E_TOO_LARGE
    assert lbwd(lib, act=ACT_NONE, dx=None, dw=None, db=None, dz=None, z=None) == OK  # nothing wanted


def tensors(*recs):
    t = (_lib.AdamWTensor * max(1, len(recs)))()
    for r, kw in zip(t, recs):
        d = dict(p=A[0], g=A[1], master=None, m=A[2], v=A[3], m_scale=A[4], v_scale=A[5], n=1000, decay=0.1)
        d.update(kw)
        for name, value in d.items():
            setattr(r, name, value)
    return t


@pytest.mark.parametrize("recs", [
    [dict(p=None)], [dict(g=None)], [dict(m=None)], [dict(v=None)], [dict(m_scale=None)], [dict(v_scale=None)],
    [dict(decay=-0.1)], [dict(decay=float("nan"))], [dict(decay=float("inf"))],
    [dict(), dict()],                                   # the same tensor twice
    [dict(g=A[0])], [dict(m=A[0] + 10)], [dict(v=A[2] + 999)], [dict(v_scale=A[4] + 12)],
    [dict(master=A[6]), dict(p=A[7], g=A[8], m=A[9], v=A[10], m_scale=A[11], v_scale=A[11] + 64)],  # one master of two
], ids=str)
def test_adamw_create(lib, recs):
    h = ctypes.c_void_p(None)
    assert lib.cxm_adamw_create(ctypes.byref(h), tensors(*recs), len(recs), DT_BF16, DT_BF16, DT_E4M3) == E_INVALID
    assert not h.value


def test_adamw_types(lib):
    h = ctypes.c_void_p(None)
    t = tensors(dict())
    for p, g, s in ((DT_E4M3, DT_E4M3, DT_F32), (DT_F32, DT_BF16, DT_F32), (DT_BF16, DT_F16, DT_F32),
                    (DT_BF16, DT_BF16, DT_BF16)):
        assert lib.cxm_adamw_create(ctypes.byref(h), t, 1, p, g, s) == E_INVALID
    assert lib.cxm_adamw_create(ctypes.byref(h), None, 1, DT_F32, DT_F32, DT_F32) == E_INVALID
    assert lib.cxm_adamw_create(None, t, 1, DT_F32, DT_F32, DT_F32) == E_INVALID
    assert lib.cxm_adamw_create(ctypes.byref(h), tensors(dict(master=A[6])), 1, DT_F32, DT_F32, DT_F32) == E_INVALID
    far = dict(n=1 << 40, g=1 << 44, m=1 << 45, v=1 << 46, p=1 << 47)
    assert lib.cxm_adamw_create(ctypes.byref(h), tensors(far), 1, DT_F32, DT_F32, DT_F32) == E_TOO_LARGE
    assert lib.cxm_adamw_create(ctypes.byref(h), tensors(dict(n=1 << 50)), 1, DT_F32, DT_F32, DT_F32) == E_TOO_LARGE


def test_adamw_of_nothing(lib):
    """No tensors, or empty ones: a handle whose steps do nothing."""
    for t, n in ((None, 0), (tensors(dict(n=0, p=None)), 1)):
        h = ctypes.c_void_p(None)
        assert lib.cxm_adamw_create(ctypes.byref(h), t, n, DT_F32, DT_F32, DT_F32) == OK
        step = lambda *a: lib.cxm_adamw_step(h, *a, None, 0, None)  # noqa: E731
        assert step(1e-3, 0.9, 0.999, 1e-8, 1) == OK
        assert step(1e-3, 1.0, 0.999, 1e-8, 1) == E_INVALID
        assert step(1e-3, 0.9, -0.1, 1e-8, 1) == E_INVALID
        assert step(1e-3, 0.9, 0.999, -1.0, 1) == E_INVALID
        assert step(1e-3, 0.9, 0.999, 1e-8, 0) == E_INVALID
        assert step(float("nan"), 0.9, 0.999, 1e-8, 1) == E_INVALID
        assert lib.cxm_adamw_destroy(h) == OK
    assert lib.cxm_adamw_destroy(None) == E_INVALID
    assert lib.cxm_adamw_step(None, 1e-3, 0.9, 0.999, 1e-8, 1, None, 0, None) == E_INVALID
