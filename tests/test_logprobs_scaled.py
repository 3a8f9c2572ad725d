"""What the fp16 gradient's scaled entries refuse on the host, before any launch."""
import ctypes

import pytest

from qwen3_triton import _hip as H

INVALID = 100000
P = 1 << 20   # a 16-byte aligned address that no refused call touches


@pytest.mark.parametrize("bad", [dict(rows=0), dict(rows=1 << 31), dict(vocab=0), dict(vocab=1 << 30), dict(top=-1), dict(top=33), dict(top=0), dict(tok=None),
                                 dict(inv=0.0), dict(inv=float('nan')), dict(inv=float('inf')), dict(scale=None), dict(scale=P + 2)])
def test_grad_scale_refusals(bad):
    a = dict(g=P, gh=P, gtop=P, rows=4, vocab=1000, top=2, tok=P, ign=-100, inv=1.0, scale=P)
    a.update(bad)
    assert H.load().q3_logprobs_grad_scale(*a.values(), None) == INVALID


@pytest.mark.parametrize("bad", [dict(dtype=1), dict(dtype=2, out=2), dict(out=2), dict(out=0), dict(scale=P + 1), dict(dz=P), dict(z=None)])
def test_scaled_gradient_refusals(bad):
    a = dict(dtype=0, out=1, z=P, ld=1000, rows=4, vocab=1000, tok=P, ign=-100, inv=1.0, top=2, tid=P, m=P, ls=P, ent=P, g=P, gh=P, gtop=P, dz=2 * P,
             ldo=1000, scale=P)
    a.update(bad)
    assert H.load().q3_token_logprobs_bwd_scaled(*a.values(), None) == INVALID


@pytest.mark.parametrize("bad", [dict(dtype=0), dict(dtype=2), dict(z=None), dict(z=P + 8), dict(ldz=992), dict(dz=None), dict(dz=P + 8), dict(ldo=992),
                                 dict(ldo=1004), dict(dz=P, ldo=1008), dict(rows=0), dict(rows=11), dict(vocab=999), dict(tok=None), dict(inv=0.0),
                                 dict(m=None), dict(rm=None), dict(rl=None), dict(lp=None), dict(ent=None), dict(scale=P + 2)])
def test_head_gradient_refusals(bad):
    a = dict(dtype=1, z=P, ldz=1000, dz=2 * P, ldo=1000, rows=10, vocab=1000, tok=P, ign=-100, inv=1.0, m=P, ldp=10, rm=P, rl=P, lp=P, ent=P, g=None,
             gh=None, scale=P)
    a.update(bad)
    assert H.load().q3_head_logprobs_grad(*a.values(), None) == INVALID


@pytest.mark.parametrize("bad", [(None, P, 8, P), (P, None, 8, P), (P, P, 0, P), (P, P, 8, None), (P + 2, P, 8, P), (P, P + 1, 8, P), (P, P, 8, P + 2)])
def test_unscale_refusals(bad):
    assert H.load().q3_unscale_f16(*bad, None) == INVALID


@pytest.mark.parametrize("long_k", [0, 1])
def test_scaled_product_refusals(long_k):
    lib = H.load()

    def desc(**kw):
        d = H.GemmDesc()
        d.dtype, d.pieces, d.m, d.n, d.k, d.b_kmajor = 1, 1, 64, 1024, 151936, 1
        d.a[0], d.lda[0], d.b[0], d.ldb[0], d.c[0], d.ldc[0] = P, d.k, P, d.n, P, d.n
        for name, value in kw.items():
            setattr(d, name, value)
        return d

    def call(d, scale=P, ws=P, nbytes=1 << 30):
        return lib.q3_gemm_scaled(None if d is None else ctypes.addressof(d), long_k, scale, ws, nbytes, None)
    for bad in (dict(dtype=2), dict(dtype=0), dict(b_kmajor=0), dict(axis=1), dict(epilogue=1, res=P, ldres=1024), dict(pieces=2), dict(m=0), dict(k=151935)):
        assert call(desc(**bad)) == INVALID
    d = desc()
    size = (lib.q3_gemm_long_k_workspace_bytes if long_k else lib.q3_gemm_workspace_bytes)(ctypes.addressof(d))
    assert size > 0
    assert call(None) == call(d, scale=None) == call(d, scale=P + 2) == call(d, ws=None) == call(d, nbytes=size - 1) == INVALID
