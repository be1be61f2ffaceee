"""Finite logits far from zero, as masks of a large negative number are: the
largest value's product with the scale is then off by more than exponentials
hold.  Rows, halves, ends and most of a row of such values, through the three
forward entry points' sums, against float64 (tolerances: vocab_util)."""
import numpy as np
import pytest

from cortexmind_amd._lib import DT_BF16, DT_F16, DT_F32
from layer_util import DTYPES, NAMES, rounded
from test_distill_gpu import check_forward as check_loss
from test_distill_gpu import forward as distill
from test_logprob_gpu import check, forward
from vocab_util import logits

pytestmark = pytest.mark.gpu

FAR = [-1e9, -1e10, -1e12, -1e15, -1e20, -1e30, -1e32, -1e36, 1e10, 1e12, 1e30]
# fp16 holds no such values: larger scales take its own there
CASES = [(dt, m, (0.5, 0.8, 1.0, 1.25)) for dt in (DT_F32, DT_BF16) for m in FAR]
CASES += [(DT_F16, m, (1e5, 3e5, 1e12, 1e30)) for m in (-65504.0, -30000.0, -10000.0, 20000.0)]


def far_rows(vocab, dt, m, seed):
    """Whole rows, halves, ends (of less than a wave's share of a segment and of
    more), every other and all but three."""
    x = logits(8, vocab, dt, seed)
    x[0] = m
    x[1, :vocab // 2 + 1] = m
    x[2, vocab // 2:] = m
    x[3, -min(vocab, 700):] = m
    x[4, ::2] = m
    near = x[5, [0, vocab // 3, vocab - 1]].copy()
    x[5] = m
    x[5, [0, vocab // 3, vocab - 1]] = near
    x[6] = np.where(np.arange(vocab) % 3, m, 2 * m)  # two values that are both far
    return rounded(x, dt)


@pytest.mark.parametrize("dt,m,scales", CASES, ids=lambda v: NAMES.get(v, str(v)) if isinstance(v, int) else
                         f"{v:g}" if isinstance(v, float) else "")
@pytest.mark.parametrize("vocab", [7, 500, 9000, 50001])
def test_sums(hip, vocab, dt, m, scales):
    x = far_rows(vocab, dt, m, 31)
    tok = np.array([vocab - 1, 0, 0, 0, 1, vocab // 3, 1, 2], np.int32) % vocab
    for i, scale in enumerate(scales):
        top = min(vocab, (0, 6, 40, 1)[i])
        for want in (("logp", "entropy", "lse"), ("logp", "lse")):
            check(x, tok, forward(x, tok, dt, scale, top, want=want), scale, top)
    # a teacher's tokens, masked ones among them
    k = min(vocab, 5)
    rng = np.random.default_rng(vocab)
    ids = np.stack([rng.permutation(vocab)[:k] for _ in x]).astype(np.int32)
    t = rng.normal(size=ids.shape).astype(np.float32)
    for scale in (scales[1], scales[3]):
        tv = (t / max(scale, 1.0)).astype(np.float32)
        loss, lse = distill(x, ids, tv, dt, scale)
        # (twice fp16's lowest value is -inf: infinitely far from a teacher that names it)
        dead = np.isinf(np.take_along_axis(x, ids, 1)).any(axis=1)
        assert np.all(loss[dead] == np.inf)
        check_loss(x[~dead], ids[~dead], tv[~dead], scale, loss[~dead], lse[~dead])


@pytest.mark.parametrize("dt", DTYPES, ids=NAMES.get)
@pytest.mark.parametrize("m,scale", [(-1e12, 1.0), (-1e30, 1.25), (-1e15, 0.8)])
def test_sums_of_many_rows(hip, m, scale, dt):
    """Rows of a wave each."""
    if dt == DT_F16:
        m, scale = max(m, -65504.0), scale * 3e5
    x = np.tile(far_rows(1500, dt, m, 33), (140, 1))
    tok = (np.arange(len(x)) * 7 % 1500).astype(np.int32)
    for top in (0, 3):
        check(x, tok, forward(x, tok, dt, scale, top), scale, top)
