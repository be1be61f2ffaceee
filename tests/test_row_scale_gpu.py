"""The scales of rows and blocks in 8 bits are, bit for bit, what is declared: the
largest magnitude times the fp32 value of 1 / 448."""
import numpy as np
import pytest

from cortexmind_amd import engine
from cortexmind_amd._lib import DT_F16, DT_F32, call
from cortexmind_amd.data import SplitMix64
from gpu_util import dev
from layer_util import DTYPES, NAMES, from_bits, to_bits, up

pytestmark = pytest.mark.gpu
FLT_MIN = np.float32(2.0 ** -126)


def declared(amax):
    s = np.asarray(amax, np.float32) * (np.float32(1.0) / np.float32(448.0))
    return np.where(s < FLT_MIN, np.float32(0.0), s)


@pytest.mark.parametrize("dt", DTYPES, ids=NAMES.get)
@pytest.mark.parametrize("cols", [1, 5, 24, 1100])
def test_rows(hip, cols, dt):
    g = SplitMix64(51 + cols + dt)
    rows = 4096
    x = np.exp2(g.uniform((rows, 1), -12.0, 12.0).astype(np.float64)) * g.normal((rows, cols))
    if dt != DT_F16:  # scales around the smallest normal float, and the largest
        x[:300] *= np.exp2(np.linspace(-119.0, -115.0, 300))[:, None]
        x[300:310] = np.finfo(np.float32).max / (1.0 + np.arange(10)[:, None])
    bits = to_bits(x, dt)
    amax = np.abs(from_bits(bits, dt)).max(axis=1)
    dx, q, s = dev(bits), dev(np.zeros((rows, cols), np.uint8)), dev(np.full(rows, -1.0, np.float32))
    call("cxm_quant_rows_t", dx.ptr, q.ptr, s.ptr, rows, cols, dt, None)
    assert np.array_equal(s.numpy(), declared(amax))
    if dt != DT_F16:
        assert 0 < np.count_nonzero(s.numpy()[:300] == 0) < 300


def test_norm_rows(hip):
    """One column: y = w x / sqrt(x^2 + eps) is the row's largest magnitude."""
    g = SplitMix64(52)
    x = g.normal((5000, 1))
    dx, w = up(x, DT_F32), dev(np.array([1.37], np.float32))
    y, q, s = dev(np.zeros((5000, 1), np.float32)), dev(np.zeros((5000, 1), np.uint8)), dev(np.zeros(5000, np.float32))
    call("cxm_rmsnorm_fwd_t", dx.ptr, None, w.ptr, 1e-2, None, y.ptr, q.ptr, s.ptr, None, 5000, 1, DT_F32, None)
    assert np.array_equal(s.numpy(), declared(np.abs(y.numpy()).max(axis=1)))


def test_blocks_of_moments(hip):
    """From zero moments m is (1 - beta1) g, one product."""
    g = SplitMix64(53)
    n = 256 * 1000 + 77
    grad = (np.exp2(g.uniform((n,), -8.0, 8.0)) * g.normal((n,))).astype(np.float32)
    nb = (n + 255) // 256
    d = {"p": dev(np.zeros(n, np.float32)), "g": dev(grad), "m": dev(np.zeros(n, np.uint8)), "v": dev(np.zeros(n, np.uint8)),
         "m_scale": dev(np.zeros(nb, np.float32)), "v_scale": dev(np.zeros(nb, np.float32))}
    opt = engine.AdamW([d], state_8bit=True)
    opt.step(1e-3, 1, beta1=0.875)
    m = np.abs(np.float32(0.125) * grad)
    assert np.array_equal(d["m_scale"].numpy(), declared(np.maximum.reduceat(m, np.arange(0, n, 256))))
    opt.close()
