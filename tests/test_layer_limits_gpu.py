"""The layer operators at the ends of their ranges of sizes."""
import numpy as np
import pytest

from cortexmind_amd._lib import DT_F16, call
from cortexmind_amd.data import SplitMix64
from cortexmind_amd.device import DeviceArray
from layer_util import HALF, TINY, U32, close, get, rounded, up

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
