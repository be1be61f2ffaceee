"""Rows of logits, their float64 statistics and the errors that fp32 sums over
them may have (imported by test modules only).

A row's S = sum exp(z - max z) is a sum of terms that a lane adds in turn (at
most 32) and that meet in trees and in up to 64 segments: C = 128 roundings of
at most S.  A term's exponent, (x - m) scale log2(e), has three roundings, so
the term is off by 3 U32 (max z - z) and the exponential's own 2: on average
over the distribution, with E = sum p (max z - z), S is off by (C + 3 E + 4) U32
S.  E is what the entropy has beyond ln S."""
import numpy as np

from cortexmind_amd._lib import DT_BF16, DT_F16, DT_F32
from cortexmind_amd.data import SplitMix64
from gpu_util import dev
from layer_util import U32, rounded, to_bits

C = 128
LOWEST = {DT_F32: float(np.finfo(np.float32).min), DT_BF16: -(2.0 ** 128 - 2.0 ** 120), DT_F16: -65504.0}


def logits(rows, vocab, dt, seed, std=3.0, mean=0.0):
    return rounded(SplitMix64(seed + 5 * rows + vocab + dt).normal((rows, vocab), mean, std), dt)


def upload(x, dt, ld, off=0, fill=np.nan):
    """The rows ld elements apart, with `fill` between them."""
    a = np.full((x.shape[0], ld), fill)
    a[:, :x.shape[1]] = x
    return dev(to_bits(a, dt), off)


class Rows:
    """lse, log p, entropy and the bounds of their errors."""

    def __init__(self, x, scale):
        z = x * float(np.float32(scale))
        with np.errstate(invalid="ignore"):
            self.m = z.max(axis=1, keepdims=True)
            gap = np.where(z == -np.inf, np.inf, self.m - z)
        e = np.exp(-gap)
        s = e.sum(axis=1, keepdims=True)
        self.log_s = np.log(s)
        self.p = e / s
        self.gap = np.where(np.isinf(gap), 0.0, gap)
        self.E = (self.p * self.gap).sum(axis=1, keepdims=True)
        self.E2 = (self.p * self.gap ** 2).sum(axis=1, keepdims=True)
        self.lse = self.m + self.log_s
        self.logp = -gap - self.log_s  # (z - lse would lose log_s beside the type's lowest value)
        self.entropy = self.log_s + self.E
        self.rel_s = (C + 3 * self.E + 4) * U32
        self.log_s_err = self.rel_s + 2 * U32 * np.abs(self.log_s)
        self.lse_err = self.log_s_err + 2 * U32 * (np.abs(self.m) + np.abs(self.lse))
        # S's error reaches T / S and ln S; T's terms err as S's do, times the gap
        self.entropy_err = self.log_s_err + self.rel_s * self.E + U32 * ((C + 8) * self.E + 3 * self.E2) + 4 * U32 * self.entropy

    def logp_err(self, gap, logp):
        """Of log probabilities `gap` below the largest logit."""
        return self.log_s_err[:, 0] + 3 * U32 * gap + 2 * U32 * np.abs(logp)


def top_of(x, k):
    """The k largest of each row, of equal ones the first."""
    return np.stack([np.lexsort((np.arange(x.shape[1]), -r))[:k] for r in x])
