"""Arguments that the layer norm, the embedding, the log probabilities and the
distillation refuse on the host, before any launch: null pointers, types, sizes
and overlaps (no GPU; addresses are never read)."""
import pytest

from cortexmind_amd import _lib
from cortexmind_amd._lib import DT_BF16, DT_E4M3, DT_F16, DT_F32, E_INVALID, E_TOO_LARGE, OK

A = [0x10000000 * (i + 1) for i in range(12)]  # addresses far apart
INF, NAN = float("inf"), float("nan")


@pytest.fixture(scope="module")
def lib():
    return _lib.lib()


def ln(lib, x=A[0], res=A[1], w=A[2], b=A[8], eps=1e-5, h=A[3], y=A[4], q=None, scale=None, mean=A[6], rstd=A[7], rows=4,
       cols=64, dt=DT_BF16):
    return lib.cxm_layernorm_fwd_t(x, res, w, b, eps, h, y, q, scale, mean, rstd, rows, cols, dt, None)


@pytest.mark.parametrize("kw", [
    dict(x=None), dict(w=None), dict(y=None), dict(q=A[5]), dict(res=None), dict(cols=0), dict(dt=DT_E4M3), dict(dt=9),
    dict(eps=-1.0), dict(eps=NAN), dict(y=A[0] + 2), dict(h=A[1] + 128), dict(h=A[4]), dict(q=A[0], scale=A[5]),
    dict(q=A[5], scale=A[5] + 8), dict(rstd=A[4] + 64), dict(y=A[2]), dict(rstd=A[2]), dict(y=A[8]), dict(mean=A[7] + 4),
    dict(mean=A[0] + 8), dict(rstd=A[8] + 64),
])
def test_norm_forward(lib, kw):
    assert ln(lib, **kw) == E_INVALID


def lnb(lib, h=A[0], mean=A[1], rstd=A[2], w=A[3], dy=A[4], dh=A[5], dx=A[6], dw=A[7], db=A[8], rows=4, cols=64, dt=DT_F16):
    return lib.cxm_layernorm_bwd_t(h, mean, rstd, w, dy, dh, dx, dw, db, rows, cols, dt, None)


@pytest.mark.parametrize("kw", [
    dict(h=None), dict(mean=None), dict(rstd=None), dict(w=None), dict(dy=None), dict(dx=None), dict(dw=None), dict(cols=0),
    dict(dt=DT_E4M3), dict(dx=A[0] + 2), dict(dx=A[4] + 2), dict(dx=A[5] + 2), dict(dx=A[3]), dict(dw=A[3]), dict(db=A[3]),
    dict(dw=A[4] + 64), dict(dw=A[6] + 8), dict(db=A[7] + 16), dict(db=A[6]), dict(dx=A[1]), dict(dw=A[2]), dict(db=A[1]),
    dict(db=A[5]),
])
def test_norm_backward(lib, kw):
    assert lnb(lib, **kw) == E_INVALID


def test_norm_sizes(lib):
    assert ln(lib, rows=0, x=None) == OK
    assert ln(lib, cols=1 << 31) == E_TOO_LARGE
    assert ln(lib, rows=1 << 41) == E_TOO_LARGE
    assert ln(lib, rows=1 << 40, cols=1 << 30) == E_TOO_LARGE  # a product past 64 bits
    far = dict(x=1 << 44, res=None, w=A[2], h=None, y=1 << 45, mean=None, rstd=None)
    assert ln(lib, rows=1 << 32, cols=8, **far) == E_TOO_LARGE  # a grid of 2^32 threads and more
    assert lnb(lib, h=1 << 44, dy=1 << 45, dh=None, dx=1 << 46, cols=1 << 26) == E_TOO_LARGE


def emb(lib, table=A[0], ids=A[1], scale=1.0, y=A[2], tokens=8, vocab=100, cols=64, dt=DT_BF16):
    return lib.cxm_embedding_fwd_t(table, ids, scale, y, tokens, vocab, cols, dt, None)


@pytest.mark.parametrize("kw", [dict(table=None), dict(ids=None), dict(y=None), dict(scale=INF), dict(scale=NAN), dict(vocab=0),
                                dict(cols=0), dict(dt=DT_E4M3), dict(dt=-1), dict(y=A[0]), dict(y=A[0] + 12000),
                                dict(y=A[1] + 16)])
def test_embedding_forward(lib, kw):
    assert emb(lib, **kw) == E_INVALID


def embb(lib, ids=A[0], dy=A[1], scale=1.0, dw=A[2], acc=0, tokens=8, vocab=100, cols=64, dt=DT_BF16, gdt=DT_F32):
    return lib.cxm_embedding_bwd_t(ids, dy, scale, dw, acc, tokens, vocab, cols, dt, gdt, None)


@pytest.mark.parametrize("kw", [dict(ids=None), dict(dy=None), dict(dw=None), dict(scale=INF), dict(scale=NAN), dict(vocab=0),
                                dict(cols=0), dict(dt=DT_E4M3), dict(gdt=DT_F16), dict(gdt=DT_E4M3), dict(acc=2), dict(acc=-1),
                                dict(dt=DT_F32, gdt=DT_BF16), dict(dw=A[1]), dict(dw=A[1] + 1000), dict(dw=A[0])])
def test_embedding_backward(lib, kw):
    assert embb(lib, **kw) == E_INVALID


def test_embedding_sizes(lib):
    assert emb(lib, tokens=0, ids=None, table=None) == OK
    assert embb(lib, tokens=0, ids=None, dy=None, acc=1) == OK
    for f in (emb, embb):
        for kw in (dict(tokens=1 << 31), dict(vocab=1 << 31), dict(cols=1 << 31), dict(tokens=1 << 30, cols=1 << 30)):
            assert f(lib, **kw) == E_TOO_LARGE, kw
    assert emb(lib, table=1 << 40, y=1 << 45, tokens=(1 << 31) - 1, cols=16000) == E_TOO_LARGE  # a grid of 2^32 threads and more


def lp(lib, x=A[0], ld=100, tok=A[1], scale=1.0, logp=A[2], ent=A[3], lse=A[4], tl=A[5], ti=A[6], top=4, rows=8, vocab=100,
       dt=DT_BF16):
    return lib.cxm_logprob_fwd_t(x, ld, tok, scale, logp, ent, lse, tl, ti, top, rows, vocab, dt, None)


@pytest.mark.parametrize("kw", [
    dict(x=None), dict(tok=None), dict(ld=99), dict(scale=0.0), dict(scale=-1.0), dict(scale=NAN), dict(scale=INF),
    dict(vocab=0), dict(dt=DT_E4M3), dict(top=65), dict(vocab=3, ld=3), dict(tl=None), dict(ti=None),
    dict(logp=None, ent=None, lse=None, top=0), dict(logp=A[0] + 64), dict(ent=A[2] + 4), dict(lse=A[1]), dict(ti=A[5] + 8),
    dict(tl=A[0] + 1500),
])
def test_logprob_forward(lib, kw):
    assert lp(lib, **kw) == E_INVALID


def lpb(lib, x=A[0], ld=100, tok=A[1], scale=1.0, lse=A[2], ent=A[3], g=A[4], h=A[5], dx=A[6], ldd=100, rows=8, vocab=100,
        dt=DT_F16):
    return lib.cxm_logprob_bwd_t(x, ld, tok, scale, lse, ent, g, h, dx, ldd, rows, vocab, dt, None)


@pytest.mark.parametrize("kw", [
    dict(x=None), dict(tok=None), dict(lse=None), dict(ent=None), dict(g=None, h=None), dict(dx=None), dict(ld=99), dict(ldd=99),
    dict(scale=0.0), dict(scale=NAN), dict(vocab=0), dict(dt=DT_E4M3), dict(dx=A[0] + 2), dict(dx=A[0], ldd=101),
    dict(dx=A[1]), dict(dx=A[2]), dict(dx=A[3]), dict(dx=A[4]), dict(dx=A[5]),
])
def test_logprob_backward(lib, kw):
    assert lpb(lib, **kw) == E_INVALID


def di(lib, x=A[0], ld=100, ids=A[1], t=A[2], k=5, scale=1.0, loss=A[3], lse=A[4], rows=8, vocab=100, dt=DT_F32):
    return lib.cxm_distill_fwd_t(x, ld, ids, t, k, scale, loss, lse, rows, vocab, dt, None)


@pytest.mark.parametrize("kw", [dict(x=None), dict(ids=None), dict(t=None), dict(loss=None), dict(k=0), dict(k=257), dict(ld=99),
                                dict(scale=0.0), dict(scale=INF), dict(vocab=0), dict(dt=DT_E4M3), dict(loss=A[0]),
                                dict(lse=A[3] + 4), dict(loss=A[1] + 100), dict(lse=A[2] + 100)])
def test_distill_forward(lib, kw):
    assert di(lib, **kw) == E_INVALID


def dib(lib, x=A[0], ld=100, ids=A[1], t=A[2], k=5, scale=1.0, lse=A[3], g=A[4], dx=A[5], ldd=100, rows=8, vocab=100,
        dt=DT_BF16):
    return lib.cxm_distill_bwd_t(x, ld, ids, t, k, scale, lse, g, dx, ldd, rows, vocab, dt, None)


@pytest.mark.parametrize("kw", [dict(x=None), dict(ids=None), dict(t=None), dict(lse=None), dict(g=None), dict(dx=None),
                                dict(k=0), dict(k=257), dict(ld=99), dict(ldd=99), dict(scale=-2.0), dict(vocab=0),
                                dict(dt=DT_E4M3), dict(dx=A[0] + 2), dict(dx=A[0], ldd=102), dict(dx=A[1]), dict(dx=A[2]),
                                dict(dx=A[3]), dict(dx=A[4])])
def test_distill_backward(lib, kw):
    assert dib(lib, **kw) == E_INVALID


def test_vocab_sizes(lib):
    assert lp(lib, rows=0, x=None) == OK and lpb(lib, rows=0, x=None, lse=None) == OK
    assert di(lib, rows=0, x=None, ids=None) == OK and dib(lib, rows=0, x=None, dx=None) == OK
    far = dict(x=1 << 44)
    for f in (lp, lpb, di, dib):
        big = (1 << 31) - 1
        for kw in (dict(vocab=big, ld=big), dict(rows=1 << 24), dict(ld=1 << 44), dict(rows=1 << 20, ld=1 << 30)):
            assert f(lib, **far, **kw) == E_TOO_LARGE, kw
    for f in (lpb, dib):
        assert f(lib, ldd=1 << 44) == E_TOO_LARGE
    # more segments than a grid has workgroups
    many = dict(rows=1 << 23, vocab=100000, ld=100000)
    assert lp(lib, **far, tok=1 << 40, logp=1 << 41, ent=None, lse=None, top=0, **many) == E_TOO_LARGE
    assert di(lib, **far, ids=1 << 40, t=1 << 41, loss=1 << 42, lse=None, **many) == E_TOO_LARGE
    assert lpb(lib, **far, tok=1 << 40, lse=1 << 41, ent=None, g=1 << 42, h=None, dx=1 << 45, ldd=100000, **{
        k: v for k, v in many.items()}) == E_TOO_LARGE
    assert dib(lib, **far, ids=1 << 40, t=1 << 41, lse=1 << 42, g=1 << 43, dx=1 << 45, ldd=100000, **many) == E_TOO_LARGE
