"""Attention over a shared prefix and log probabilities of tokens on the host: what they refuse before any launch, and their
workspace sizes."""
import ctypes

import pytest
import torch

from qwen3_triton import _hip as H
from qwen3_triton.inference import prefix as PX
from qwen3_triton.kernels import logprobs as LP

INVALID = 100000
P = 1 << 20   # a 16-byte aligned address that no refused call touches


def prefix_call(**kw):
    a = dict(dtype=2, q=P, ql=(4096, 4096, 128), pk=P, pv=P, pl=(1024000, 128000, 128), ck=P, cv=P, cl=(102400, 12800, 128), out=P,
             ol=(4096, 4096, 128), ws=P, nbytes=1 << 40, B=4, R=1, S=1, Hq=32, Hkv=8, d=128, P=1000, C=100, start=5, dev=None, starts=0,
             scale=0.1)
    a.update(kw)
    return H.load().q3_prefix_attention(
        a['dtype'], a['q'], *a['ql'], a['pk'], a['pv'], *a['pl'], a['ck'], a['cv'], *a['cl'], a['out'], *a['ol'], a['ws'], a['nbytes'],
        a['B'], a['R'], a['S'], a['Hq'], a['Hkv'], a['d'], a['P'], a['C'], a['start'], a['dev'], a['starts'], a['scale'], None)


@pytest.mark.parametrize("bad", [
    dict(dtype=0), dict(dtype=3), dict(q=None), dict(q=P + 8), dict(ql=(4096, 4096, 130)), dict(ql=(4100, 4096, 128)), dict(pk=None),
    dict(pv=None), dict(pv=P + 4), dict(pl=(1024000, 128000, 120)), dict(pl=(1024000, 128000, 1 << 24)), dict(pl=(1024004, 128000, 128)),
    dict(ck=None), dict(cv=P + 2), dict(cl=(102400, 12800, 64)), dict(cl=(102400, 12804, 128)), dict(out=None), dict(out=P + 4),
    dict(ol=(4096, 4098, 128)), dict(ws=None), dict(ws=P + 8), dict(nbytes=16), dict(B=0), dict(R=0), dict(R=3), dict(S=0), dict(Hq=0),
    dict(Hkv=0), dict(Hkv=5), dict(d=64), dict(P=-1), dict(P=1 << 30), dict(C=0), dict(C=1 << 30), dict(start=-1), dict(start=100),
    dict(S=101, start=0), dict(dev=P, starts=0), dict(dev=P, starts=3), dict(scale=0.0), dict(scale=-1.0), dict(scale=float('nan')),
    dict(scale=1e30), dict(B=1 << 24, R=1), dict(S=1 << 29, C=1 << 29, start=0)])
def test_prefix_attention_refusals(bad):
    assert prefix_call(**bad) == INVALID


def test_prefix_workspace():
    q = lambda *a: H.query("q3_prefix_attention_workspace_bytes", *a)
    assert q(0, 1, 1, 32, 8, 1000, 90, 10) == q(4, 3, 1, 32, 8, 1000, 90, 10) == q(4, 1, 1, 32, 5, 1000, 90, 10) == q(4, 1, 1, 32, 8, -1, 90, 10) == 0
    assert q(4, 1, 1, 32, 8, 1000, 90, -1) == q(4, 1, 1, 32, 8, 1000, 90, 91) == 0
    some = q(4, 1, 1, 32, 8, 1000, 90, 10)
    assert some >= 2 * 128 * 130 * 4 and some % (128 * 130 * 4) == 0     # a slot of the prefix, a slot of its own, per query row
    assert q(64, 1, 300, 32, 8, 4000, 300, 300) == 0                     # many queries: no partials
    assert q(4, 1, 1, 32, 8, 300, 90, 10) == 0                           # few positions: none either
    # no more for a longer prefix once its splits fill the chip; never more than the splits that fill it
    assert q(32, 1, 1, 32, 8, 1 << 20, 90, 10) <= 32 * 32 * 130 * 4 * 1024
    for args in ((1, 1, 1, 8, 8, 0, 1 << 20, 1 << 20), (1, 1, 1, 1, 1, 1 << 20, 1 << 20, 1 << 20), (1 << 20, 1, 1, 1, 1, 1, 1, 1)):
        assert q(*args) >= 0


def heads(*shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device='meta')


def test_python_refuses_host_tensors():
    q, k, c = (torch.zeros(s, dtype=torch.bfloat16) for s in ((2, 1, 8, 128), (1, 2, 10, 128), (2, 2, 9, 128)))
    with pytest.raises(ValueError, match='ROCm'):
        PX.attention(q, k, k, c, c, 0)
    with pytest.raises(ValueError, match='ROCm'):
        LP.token_logprobs(torch.zeros(2, 5), torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match='ROCm'):
        LP.lm_head_logprobs(torch.zeros(2, 8), torch.zeros(5, 8), torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError):
        PX.attention(q[0], k, k, c, c, 0)
    with pytest.raises(ValueError, match='forward only'):
        PX.attention(q.requires_grad_(), k, k, c, c, 0)
    with pytest.raises(ValueError):
        LP.token_logprobs(torch.zeros(0, 5), torch.zeros(0, dtype=torch.int64))
    with pytest.raises(ValueError):
        LP.lm_head_logprobs(torch.zeros(2, 8), torch.zeros(5, 7), torch.zeros(2, dtype=torch.int64))


@pytest.mark.parametrize("kw", [dict(top=-1), dict(top=33), dict(top=6), dict(top=1.0), dict(top=True), dict(temperature=0.0),
                                dict(temperature=-1.0), dict(temperature=float('nan')), dict(temperature=float('inf')),
                                dict(ignore_index=None), dict(ignore_index=-100.0)])
def test_options(kw):
    args = dict(vocab=5, top=0, temperature=1.0, ignore_index=-100)
    LP._check_options(**args)
    with pytest.raises(ValueError):
        LP._check_options(**{**args, **kw})
    LP._check_options(**{**args, 'vocab': (1 << 30) - 1, 'top': 32})
    with pytest.raises(ValueError):
        LP._check_options(**{**args, 'vocab': 1 << 30})


def test_shifted_labels():
    x, w, y = torch.zeros(2, 3, 8), torch.zeros(5, 8), torch.zeros(2, 3, dtype=torch.int64)
    with pytest.raises(ValueError, match='ROCm'):
        LP.shifted_logprobs(x, w, y)
    for bad in (y.int(), y[:, :2], y.t().contiguous().t(), y.to('meta')):
        with pytest.raises(ValueError, match='int64'):
            LP._check_tokens(bad, x.shape[:2], x)
    LP._check_tokens(y, x.shape[:2], x)


def test_rows_of_logits():
    z = torch.zeros(4, 6, 8)
    assert LP._logit_rows(z) == (24, 8, 8)
    assert LP._logit_rows(z[:, -1]) == (4, 48, 8)
    assert LP._logit_rows(z[..., :5]) == (24, 8, 5)
    assert LP._logit_rows(z[0, 0]) == (1, 8, 8)
    for bad in (z[:, :3], z.transpose(1, 2), z[..., ::2], z[:1, :1].expand(4, 6, 8), torch.zeros(8).expand(3, 8)):
        with pytest.raises(ValueError):
            LP._logit_rows(bad)


def logprob_call(fn, **kw):
    a = dict(dtype=2, out=2, z=P, ld=1000, rows=4, vocab=1000, tok=P, ign=-100, inv=1.0, top=2, lp=P, ent=P, m=P, ls=P, tlp=P, tid=P, ws=P,
             nbytes=1 << 30, g=P, gh=P, gtop=P, dz=2 * P, ldo=1000)
    a.update(kw)
    lib = H.load()
    if fn == 'fwd':
        return lib.q3_token_logprobs(a['dtype'], a['z'], a['ld'], a['rows'], a['vocab'], a['tok'], a['ign'], a['inv'], a['top'], a['lp'],
                                     a['ent'], a['m'], a['ls'], a['tlp'], a['tid'], a['ws'], a['nbytes'], None)
    return lib.q3_token_logprobs_bwd(a['dtype'], a['out'], a['z'], a['ld'], a['rows'], a['vocab'], a['tok'], a['ign'], a['inv'], a['top'],
                                     a['tid'], a['m'], a['ls'], a['ent'], a['g'], a['gh'], a['gtop'], a['dz'], a['ldo'], None)


BOTH = [dict(dtype=3), dict(z=None), dict(z=P + 1), dict(ld=999), dict(rows=0), dict(rows=1 << 31), dict(vocab=0), dict(vocab=1 << 30, ld=1 << 30),
        dict(tok=None), dict(inv=0.0), dict(inv=-1.0), dict(inv=float('nan')), dict(inv=float('inf')), dict(top=-1), dict(top=33), dict(vocab=1),
        dict(ent=None), dict(m=None), dict(ls=None), dict(rows=(1 << 31) - 1, vocab=100000, ld=100000)]


@pytest.mark.parametrize("bad", BOTH + [dict(lp=None), dict(tlp=None), dict(tid=None),
                                        *(dict(vocab=100000, ld=100000, **x) for x in (dict(ws=None), dict(ws=P + 8), dict(nbytes=8)))])
def test_token_logprobs_refusals(bad):
    assert logprob_call('fwd', **bad) == INVALID


@pytest.mark.parametrize("bad", BOTH + [dict(dz=None), dict(dz=P), dict(dz=2 * P + 1), dict(ldo=999, ), dict(tid=None), dict(top=0), dict(out=1),
                                        dict(out=0), dict(dtype=0, out=3), dict(dtype=0, z=P + 2)])
def test_token_logprobs_gradient_refusals(bad):
    assert logprob_call('bwd', **{'ldo': 1 << 31, **bad}) == INVALID


def test_logprob_workspace():
    q = lambda *a: H.query("q3_token_logprobs_workspace_bytes", *a)
    assert q(2, 0, 10, 0) == q(3, 1, 10, 0) == q(2, 1, 10, 11) == q(2, 1, 0, 0) == 0
    assert 0 < q(2, 1, 151936, 0) <= q(2, 1, 151936, 20) <= 1 << 20
    assert q(2, 4096, 151936, 0) <= 4096 * 24 * 12
    assert q(2, 1, 1000, 5) == q(1, 3, 30000, 0) == q(0, 3, 16000, 9) == 0   # a row a workgroup: nothing to join


def head_call(**kw):
    a = dict(dtype=2, a=P, lda=128, b=P, ldb=128, M=10, N=1000, K=128, tok=P, inv=1.0, m=P, rest=P, u=P, pick=P, ldp=10, z=P, ldz=1000)
    a.update(kw)
    return H.load().q3_gemm_nt_logprobs(a['dtype'], a['a'], a['lda'], a['b'], a['ldb'], a['M'], a['N'], a['K'], a['tok'], a['inv'], a['m'],
                                        a['rest'], a['u'], a['pick'], a['ldp'], a['z'], a['ldz'], None)


@pytest.mark.parametrize("bad", [dict(dtype=0), dict(a=None), dict(a=P + 8), dict(lda=120), dict(lda=132), dict(b=None), dict(ldb=1 << 22), dict(M=0),
                                 dict(M=1 << 31, ldp=1 << 31), dict(N=0), dict(N=1001, ldz=1008), dict(N=1 << 30, ldz=1 << 30), dict(K=0),
                                 dict(K=100), dict(tok=None), dict(inv=0.0), dict(inv=float('inf')), dict(m=None), dict(rest=None), dict(u=None),
                                 dict(pick=None), dict(ldp=9), dict(z=P + 8), dict(ldz=992), dict(ldz=1004)])
def test_head_product_refusals(bad):
    assert head_call(**bad) == INVALID


@pytest.mark.parametrize("bad", [dict(m=None), dict(rest=None), dict(u=None), dict(pick=None), dict(rows=0), dict(rows=11), dict(vocab=0),
                                 dict(tok=None), dict(inv=-1.0), dict(lp=None), dict(ent=None), dict(rm=None), dict(rl=None)])
def test_head_finish_refusals(bad):
    a = dict(m=P, rest=P, u=P, ldp=10, pick=P, rows=10, vocab=1000, tok=P, ign=-100, inv=1.0, lp=P, ent=P, rm=P, rl=P)
    a.update(bad)
    assert H.load().q3_head_logprobs_finish(*a.values(), None) == INVALID


@pytest.mark.parametrize("bad", [dict(dtype=0), dict(z=None), dict(z=P + 8), dict(ldz=992), dict(ldz=1004), dict(rows=0), dict(rows=11), dict(vocab=0),
                                 dict(vocab=999), dict(vocab=1 << 30, ldz=1 << 30), dict(tok=None), dict(inv=0.0), dict(m=None), dict(rm=None),
                                 dict(rl=None), dict(lp=None), dict(ent=None)])
def test_head_gradient_refusals(bad):
    a = dict(dtype=2, z=P, ldz=1000, rows=10, vocab=1000, tok=P, ign=-100, inv=1.0, m=P, ldp=10, rm=P, rl=P, lp=P, ent=P, g=None, gh=None)
    a.update(bad)
    assert H.load().q3_head_logprobs_bwd(*a.values(), None) == INVALID


def test_forked_caches():
    """What a fork shares, counts and refuses, with tensors on the host."""
    from qwen3_triton.inference import KVCache, SharedPrefixCache
    owner = object()
    k, v = ([torch.zeros((2, 3, 50, 128), dtype=torch.bfloat16) for _ in range(2)] for _ in range(2))
    cache = KVCache(k, v, 50, 2, owner)
    with pytest.raises(ValueError):
        cache.fork(4, 10)
    cache.length = 30
    small = KVCache([t[..., :64] for t in k], [t[..., :64] for t in v], 50, 2, owner, 30)
    with pytest.raises(ValueError, match='heads of 128'):
        small.fork(4, 10)
    forked = cache.fork(4, 10)
    assert isinstance(forked, SharedPrefixCache) and forked.keys[1].shape == (8, 3, 10, 128) and forked.capacity == 40
    assert forked.length == forked.prefix_length == 30 and cache.prefix_length == 0
    assert forked.shared(1)[0].shape == (2, 3, 30, 128) and forked.shared(1)[0].data_ptr() == k[1].data_ptr()
    forked.admit(owner, 8, 10)
    cache.length = 45   # it may grow
    forked.admit(owner, 8, 10)
    for bad in ((owner, 8, 11), (owner, 2, 1), (object(), 8, 1)):
        with pytest.raises(ValueError):
            forked.admit(*bad)
    forked.length = 37
    forked.reset()
    assert forked.length == 30
    with pytest.raises(ValueError):
        forked.fork(1, 1)
    with pytest.raises(ValueError):
        forked.quantized()
    cache.valid = False
    with pytest.raises(ValueError, match='no longer'):
        forked.admit(owner, 8, 1)
    with pytest.raises(ValueError):
        cache.fork(1, 1)
    cache.reset()
    cache.length = 45   # other positions by now
    with pytest.raises(ValueError, match='no longer'):
        forked.admit(owner, 8, 1)


def long_k(m, n, k, **kw):
    d = H.GemmDesc()
    d.dtype, d.pieces, d.m, d.n, d.k, d.b_kmajor = 2, 1, m, n, k, 1
    d.a[0], d.lda[0], d.b[0], d.ldb[0], d.c[0], d.ldc[0] = P, k, P, n, P, n
    for name, value in kw.items():
        setattr(d, name, value)
    return d


def test_products_of_a_long_k():
    """The workspace holds fp32 partial products, at most 64 of them and at least 512 of k in each; a product that the other entry
    cuts into up to 8 needs no more here when its tiles fill the chip."""
    lib = H.load()
    size = lambda d: lib.q3_gemm_long_k_workspace_bytes(ctypes.addressof(d))
    few = lambda d: lib.q3_gemm_workspace_bytes(ctypes.addressof(d))
    for m, n, k in ((16, 256, 151936), (64, 1024, 151936), (1, 64, 40000), (300, 512, 50000), (1, 8, 8), (64, 1024, 512), (1, 4096, 1 << 18)):
        d = long_k(m, n, k)
        parts = size(d) / (4 * m * n)
        assert parts == int(parts) and 0 <= parts <= 64 and parts * 512 <= max(k, 512 * (parts < 2)) and few(d) / (4 * m * n) <= 8
    assert size(long_k(16, 256, 151936)) > 8 * 4 * 16 * 256
    assert size(long_k(8192, 8192, 8192)) == few(long_k(8192, 8192, 8192)) == 0
    for bad in (dict(axis=1), dict(epilogue=1, res=P, ldres=1024), dict(pieces=2), dict(m=0), dict(dtype=0), dict(k=151935)):
        d = long_k(**{**dict(m=64, n=1024, k=151936), **bad})
        assert size(d) == 0 and lib.q3_gemm_long_k(ctypes.addressof(d), P, 1 << 30, None) == INVALID
    d = long_k(64, 1024, 151936)
    assert lib.q3_gemm_long_k(None, P, 1 << 30, None) == INVALID
    assert lib.q3_gemm_long_k(ctypes.addressof(d), None, 1 << 30, None) == INVALID
    assert lib.q3_gemm_long_k(ctypes.addressof(d), P, size(d) - 1, None) == INVALID
