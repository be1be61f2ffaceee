"""Sizes below 2^31 whose launch a grid does not hold are refused on the host, before
any launch (no GPU; addresses are never read)."""
import pytest

from cortexmind_amd import _lib
from cortexmind_amd._lib import DT_BF16, DT_F32, E_TOO_LARGE


@pytest.fixture(scope="module")
def lib():
    return _lib.lib()


@pytest.mark.parametrize("dt", [DT_F32, DT_BF16])
@pytest.mark.parametrize("cols", [1, 8, 500])
def test_tokens_looked_up(lib, cols, dt):
    assert lib.cxm_embedding_fwd_t(1 << 40, 1 << 41, 1.0, 1 << 45, (1 << 28) + 1, 100, cols, dt, None) == E_TOO_LARGE


@pytest.mark.parametrize("dt", [DT_F32, DT_BF16])
def test_ids_of_a_gradient(lib, dt):
    for vocab in ((1 << 29) + 1, (1 << 31) - 1):
        assert lib.cxm_embedding_bwd_t(1 << 40, 1 << 41, 1.0, 1 << 45, 0, 8, vocab, 4, dt, dt, None) == E_TOO_LARGE


@pytest.mark.parametrize("dt", [DT_F32, DT_BF16])
def test_tokens_of_a_gradient(lib, dt):
    assert lib.cxm_embedding_bwd_t(1 << 40, 1 << 42, 1.0, 1 << 46, 0, (1 << 30) + 1, 100, 4, dt, dt, None) == E_TOO_LARGE
