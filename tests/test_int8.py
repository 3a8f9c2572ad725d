"""The 8-bit serving entry points on the host: what they refuse before any launch, their workspace sizes, and the rule by
which a value gets its code, in the kernels' own arithmetic against exact rationals."""
import ctypes
from fractions import Fraction

import numpy as np
import pytest
import torch

from qwen3_triton import _hip as H
from qwen3_triton.inference import int8 as I8

INVALID = 100000
P = 1 << 20   # a 16-byte aligned address that no refused call touches


def test_quantise_rule_matches_exact_rationals():
    """a (127 / M) + 1.5 * 2^23 in one fma, and the exact decision within 1e-5 of a half: the same integer as the rational
    127 a / M rounded to nearest even, for 16-bit a and for products of two."""
    rng = np.random.default_rng(0)
    f32, magic = np.float32, np.float32(12582912.0)

    def fma(x, y, z):   # exact, then one rounding
        return f32(float(Fraction(float(x)) * Fraction(float(y)) + Fraction(float(z))))

    def code(a, m):
        inv = f32(127) / f32(m)
        r = fma(a, inv, magic)
        d = abs(fma(a, inv, f32(magic - r)))
        if d > f32(0.49999):
            u = 127.0 * float(a)
            k = np.floor(u / float(m))
            mid = (k + 0.5) * float(m)
            return int(k if u < mid else k + 1 if u > mid else 2 * np.rint(0.5 * k + 0.25))
        return int(r - magic)

    for _ in range(4000):
        bits = rng.choice([8, 11, 22])
        m = f32(rng.integers(1 << (bits - 1), 1 << bits)) * f32(2.0) ** int(rng.integers(-30, 30))
        n = int(rng.integers(-127, 127))
        near = float(m) * (n + 0.5) / 127   # next to a border
        a = f32(np.sign(near)) * min(f32(abs(near)), m) if rng.random() < 0.7 else f32(rng.uniform(-1, 1)) * m
        scale = 2.0 ** np.floor(np.log2(abs(float(a)) + 1e-300))
        a = f32(np.rint(float(a) / scale * 2 ** (bits - 1)) / 2 ** (bits - 1) * scale)
        if abs(a) > m:
            continue
        assert code(a, m) == round(Fraction(127) * Fraction(float(a)) / Fraction(float(m))), (a, m)


def test_rows_refusals():
    lib = H.load()
    good = dict(dtype=2, x=P, ldx=64, q=P, s=P, rows=4, h=64)

    def quant(**kw):
        a = {**good, **kw}
        return lib.q3_quant_rows(a['dtype'], a['x'], a['ldx'], a['q'], a['s'], a['rows'], a['h'], None)
    for bad in (dict(dtype=0), dict(dtype=3), dict(x=None), dict(q=None), dict(s=None), dict(rows=0), dict(rows=1 << 31), dict(h=0),
                dict(h=8), dict(h=40, ldx=40), dict(h=32784, ldx=32784), dict(h=1 << 40, ldx=1 << 40), dict(ldx=48), dict(ldx=68),
                dict(x=P + 2), dict(q=P + 4), dict(s=P + 2)):
        assert quant(**bad) == INVALID, bad

    def norm(**kw):
        a = {**good, 'w': P, 'res': P, 'ldr': 64, 'total': P, 'eps': 1e-6, **kw}
        return lib.q3_rmsnorm_quant(a['dtype'], a['x'], a['ldx'], a['res'], a['ldr'], a['w'], a['q'], a['s'], a['total'],
                                    a['rows'], a['h'], a['eps'], None)
    for bad in (dict(dtype=0), dict(w=None), dict(w=P + 2), dict(res=None), dict(total=None), dict(ldr=32), dict(ldr=68),
                dict(res=P + 2), dict(total=P + 8), dict(eps=-1.0), dict(eps=float('nan')), dict(h=24), dict(rows=0)):
        assert norm(**bad) == INVALID, bad


FIELDS = ["dtype", "pieces", "epilogue", "m", "n", "k", "end", "a", "lda", "a_scale", "b", "ldb", "b_scale", "c", "ldc", "res", "ldres"]


def gemm_desc(**kw):
    d = dict(dtype=2, pieces=1, epilogue=0, m=4, n=64, k=128, end=[64, 128, 192], a=P, lda=128, a_scale=P, b=[P] * 3, ldb=[128] * 3,
             b_scale=[P] * 3, c=[P] * 3, ldc=[64] * 3, res=0, ldres=0)
    for k, v in kw.items():
        if isinstance(v, tuple):
            d[k][v[0]] = v[1] or 0
        else:
            d[k] = v or 0
    flat = []
    for f in FIELDS:
        flat += d[f] if isinstance(d[f], list) else [d[f]]
    return H.Int8GemmDesc(*flat)


@pytest.mark.parametrize("bad", [dict(dtype=0), dict(m=0), dict(n=0), dict(k=0), dict(k=120), dict(k=1 << 17), dict(m=1 << 31), dict(n=1 << 30),
                                 dict(pieces=0), dict(pieces=4), dict(pieces=2, epilogue=1, n=128), dict(pieces=2, epilogue=3, n=128),
                                 dict(epilogue=2), dict(epilogue=4), dict(epilogue=9), dict(a=None), dict(a=P + 8), dict(a_scale=None), dict(lda=120),
                                 dict(lda=136), dict(lda=1 << 23), dict(b=(0, None)), dict(b_scale=(0, None)), dict(ldb=(0, 64)), dict(c=(0, None)),
                                 dict(ldc=(0, 63)), dict(epilogue=1), dict(epilogue=1, res=P, ldres=63), dict(epilogue=3, n=60),
                                 dict(epilogue=3, b=(1, None)), dict(epilogue=3, ldb=(1, 256)), dict(epilogue=3, c=(0, P + 2)),
                                 dict(pieces=2, n=130), dict(pieces=2, n=128, end=(0, 0)), dict(pieces=2, n=128, end=(0, 128)),
                                 dict(pieces=3, n=128), dict(pieces=2, n=128, ldc=(1, 63))])
def test_product_refusals(bad):
    d = gemm_desc(**bad)
    assert H.load().q3_gemm_int8(ctypes.addressof(d), P, 1 << 40, None) == INVALID
    assert H.load().q3_gemm_int8_workspace_bytes(ctypes.addressof(d)) == 0
    assert H.load().q3_gemm_int8(None, None, 0, None) == INVALID


def test_product_refuses_a_short_workspace():
    d = gemm_desc(m=40, n=4096, k=12288, lda=12288, ldb=(0, 12288), ldc=(0, 4096))
    need = H.load().q3_gemm_int8_workspace_bytes(ctypes.addressof(d))
    assert need > 0
    assert H.load().q3_gemm_int8(ctypes.addressof(d), P, need - 1, None) == INVALID
    assert H.load().q3_gemm_int8(ctypes.addressof(d), None, need, None) == INVALID


def test_decode_product_refusals():
    lib = H.load()

    def call(d, x=P, ldx=128, w=None, eps=1e-6):
        return lib.q3_decode_linear_int8(ctypes.addressof(d), x, ldx, w, eps, None)
    assert call(gemm_desc(m=3)) == INVALID and call(gemm_desc(m=2, k=16400)) == INVALID and call(gemm_desc(m=2, k=120)) == INVALID
    assert call(gemm_desc(m=1), x=None) == INVALID and call(gemm_desc(m=1), x=P + 2) == INVALID
    assert call(gemm_desc(m=1), ldx=64) == INVALID and call(gemm_desc(m=1), ldx=132) == INVALID
    assert call(gemm_desc(m=1), w=P + 2) == INVALID and call(gemm_desc(m=1), w=P, eps=-1.0) == INVALID
    assert call(gemm_desc(m=1, b=(0, None))) == INVALID
    assert [lib.q3_decode_linear_int8_ok(m, k) for m, k in ((0, 64), (1, 16), (2, 16384), (3, 64), (1, 24), (1, 16400), (1, 0))] == \
        [0, 1, 1, 0, 0, 0, 0]


def test_cache_refusals():
    lib = H.load()
    good = dict(dtype=2, k=P, ks=(1024, 256, 128), v=P, vs=(1024, 256, 128), ck=P, cv=P, sk=P, sv=P, tk=P, tv=P, B=1, S=4, Hh=2, d=128,
                cap=64, start=0, dev=None)

    def append(**kw):
        a = {**good, **kw}
        return lib.q3_kv8_append(a['dtype'], a['k'], *a['ks'], a['v'], *a['vs'], a['ck'], a['cv'], a['sk'], a['sv'], a['tk'], a['tv'],
                                 a['B'], a['S'], a['Hh'], a['d'], a['cap'], a['start'], a['dev'], None)
    for bad in (dict(dtype=0), dict(k=None), dict(k=P + 2), dict(v=P + 8), dict(ks=(1024, 252, 128)), dict(vs=(1020, 256, 128)),
                dict(ck=None), dict(cv=P + 1), dict(sk=None), dict(sv=None), dict(tk=None), dict(tv=P + 4), dict(B=0), dict(B=65536),
                dict(S=0), dict(Hh=0), dict(Hh=65536), dict(d=64), dict(cap=0), dict(cap=1 << 31), dict(start=-1), dict(start=61),
                dict(start=1 << 62), dict(S=1 << 62), dict(S=2, dev=P)):
        assert append(**bad) == INVALID, bad

    def fused(**kw):
        a = {**good, 'q': P, 'qs': (1024, 256, 128), 'w': (P, P, P, P), 'y': P, 'Hq': 4, 'eps': 1e-6, **kw}
        return lib.q3_kv8_norm_rope_append(a['dtype'], a['q'], *a['qs'], a['k'], *a['ks'], a['v'], *a['vs'], *a['w'], a['y'], a['ck'],
                                           a['cv'], a['sk'], a['sv'], a['tk'], a['tv'], a['B'], a['S'], a['Hq'], a['Hh'], a['d'], a['cap'],
                                           a['start'], a['dev'], a['eps'], None)
    for bad in (dict(dtype=0), dict(q=None), dict(qs=(1024, 250, 128)), dict(w=(None, P, P, P)), dict(w=(P, P + 2, P, P)), dict(w=(P, P, None, P)),
                dict(w=(P, P, P, P + 8)), dict(y=None), dict(y=P + 2), dict(Hq=0), dict(eps=-1.0), dict(k=None), dict(vs=(1024, 256, 100)),
                dict(start=61), dict(S=2, dev=P), dict(d=64), dict(tk=None)):
        assert fused(**bad) == INVALID, bad

    def read(**kw):
        a = {**good, 'out': 2, 'length': 10, **kw}
        return lib.q3_kv8_read(a['dtype'], a['out'], a['ck'], a['cv'], a['sk'], a['sv'], a['tk'], a['tv'], a['k'], a['v'], a['B'],
                               a['Hh'], a['d'], a['cap'], a['length'], None)
    for bad in (dict(dtype=0), dict(out=3), dict(out=-1), dict(ck=None), dict(k=None), dict(v=P + 2), dict(length=0), dict(length=65),
                dict(d=32), dict(B=0)):
        assert read(**bad) == INVALID, bad


def test_attention_refusals():
    lib = H.load()
    good = dict(dtype=2, q=P, qs=(1024, 1024, 128), ck=P, cv=P, sk=P, sv=P, tk=P, tv=P, o=P, os=(1024, 1024, 128), ws=P, wsb=1 << 40, B=1, S=1,
                Hq=8, Hkv=2, d=128, cap=64, start=0, dev=None)

    def attn(**kw):
        a = {**good, **kw}
        return lib.q3_kv8_attention(a['dtype'], a['q'], *a['qs'], a['ck'], a['cv'], a['sk'], a['sv'], a['tk'], a['tv'], a['o'], *a['os'],
                                    a['ws'], a['wsb'], a['B'], a['S'], a['Hq'], a['Hkv'], a['d'], a['cap'], a['start'], a['dev'], a.get('scale', 0.1), None)
    for bad in (dict(dtype=0), dict(q=None), dict(q=P + 2), dict(qs=(1024, 1024, 124)), dict(ck=None), dict(cv=P + 8), dict(sk=None),
                dict(sv=None), dict(tk=P + 2), dict(tv=None), dict(o=None), dict(o=P + 4), dict(os=(1024, 1022, 128)), dict(B=0), dict(B=65536),
                dict(S=0), dict(Hq=1), dict(Hq=7), dict(Hkv=0), dict(B=8192, Hkv=8), dict(d=64), dict(cap=0), dict(cap=1 << 31), dict(start=-1),
                dict(start=64), dict(S=65), dict(start=1 << 62), dict(S=2, dev=P), dict(cap=4096, start=4095, wsb=16), dict(cap=4096, start=4095, ws=None),
                dict(scale=0.0), dict(scale=-1.0), dict(scale=float('nan')), dict(scale=float('inf'))):
        assert attn(**bad) == INVALID, bad
    assert lib.q3_kv8_attention_workspace_bytes(1, 1, 7, 2, 64) == 0 and lib.q3_kv8_attention_workspace_bytes(0, 1, 8, 2, 64) == 0
    # a captured step's workspace, sized for the capacity, holds every shorter span's
    sizes = [lib.q3_kv8_attention_workspace_bytes(1, 1, 32, 8, n) for n in range(64, 65536, 64)]
    assert sizes == sorted(sizes) and sizes[-1] > 0


def test_python_refusals_without_a_device():
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match='ROCm device'):
        I8.quantize_rows(x)
    with pytest.raises(ValueError, match='forward only'):
        I8.quantize_rows(x.requires_grad_())
    with torch.no_grad(), pytest.raises(ValueError, match='ROCm device'):
        I8.quantize_rows(x)
    c = I8.LayerCache.empty(1, 2, 70, device='cpu')
    assert c.capacity == 128 and c.v.shape == (1, 2, 2, 128, 64) and c.k_scale.shape == (1, 2, 2)
    assert c.nbytes == 2 * 2 * 128 * 128 + 2 * 2 * 2 * 4 + 2 * 2 * 64 * 128 * 2
    with pytest.raises(ValueError):
        I8.LayerCache.empty(1, 2, 0, device='cpu')
    with pytest.raises(ValueError):
        I8.LayerCache.empty(1, 2, 64, device='cpu', head_dim=64)
    with pytest.raises(TypeError):
        I8.LayerCache.empty(1, 2, 64, device='cpu', dtype=torch.float32)
    with pytest.raises(ValueError, match='one to three'):
        I8.projections(x, x, [])


def test_gradients_are_refused():
    x = torch.zeros(1, 32)
    q, w, one = torch.zeros(1, 32, dtype=torch.int8), torch.zeros(8, 32, dtype=torch.int8), torch.ones(1)
    learned = torch.ones(8, requires_grad=True)
    for call in (lambda: I8.linear(q, one, w, learned), lambda: I8.linear(q, one.clone().requires_grad_(), w, torch.ones(8)),
                 lambda: I8.gate_up_swiglu(q, one, w, torch.ones(8), w, learned),
                 lambda: I8.projections(q, one, [(w, torch.ones(8)), (w, learned)]),
                 lambda: I8.decode_linear(x.bfloat16(), [(w, learned)])):
        with pytest.raises(ValueError, match='forward only'):
            call()
    cos = torch.zeros(1, 1, 128, dtype=torch.bfloat16, requires_grad=True)
    t = torch.zeros(1, 1, 1, 128, dtype=torch.bfloat16)
    cache = I8.LayerCache.empty(1, 1, 64, device='cpu')
    with pytest.raises(ValueError, match='forward only'):
        I8.norm_rope_append(t, t, t, t[0, 0, 0], t[0, 0, 0], cos, cos, cache, 0)
    with pytest.raises(ValueError, match='no gradient'):
        I8.LayerCache(cache.k, cache.v, cache.k_scale.requires_grad_(), cache.v_scale, cache.k_tail, cache.v_tail)


def test_decode_linear_ok_of_nothing():
    for shape in ((), (0,), (3, 0), (0, 32)):
        assert not I8.decode_linear_ok(torch.zeros(shape, dtype=torch.bfloat16))
    assert I8.decode_linear_ok(torch.zeros(2, 16384)) and not I8.decode_linear_ok(torch.zeros(3, 16384))


def tiny_model():
    """A small inference model on the CPU (no kernel runs)."""
    import oracle as O
    from transformers import Qwen3Config
    from qwen3_triton.inference import TritonQwen3Inference
    sizes = dict(vocab_size=64, hidden_size=128, intermediate_size=256, num_hidden_layers=2, num_attention_heads=2,
                 num_key_value_heads=1, head_dim=128)
    state = {k: v.bfloat16() for k, v in O.init_params(O.OracleConfig(**sizes), seed=2, std=0.05).items()}
    config = Qwen3Config(**sizes, tie_word_embeddings=False, max_position_embeddings=256)
    return TritonQwen3Inference(config).load_hf_state_dict(state), state


def test_replaced_weights_end_captured_steps():
    from types import SimpleNamespace
    from qwen3_triton.inference.model import _check_captured
    model, state = tiny_model()
    step = SimpleNamespace(model=model, _weights=model._weights)
    model.load_state_dict(state)   # copied in place
    _check_captured(step)
    for load in (lambda: model.load_hf_state_dict(state), lambda: model.load_state_dict(state, assign=True),
                 lambda: model.load_state_dict({k: v for k, v in state.items() if 'norm' in k}, strict=False, assign=True)):
        step._weights = model._weights
        load()
        with pytest.raises(RuntimeError, match='capture again'):
            _check_captured(step)


def tiny_int8_model(monkeypatch):
    from qwen3_triton.inference import TritonQwen3Inference
    model, state = tiny_model()
    with monkeypatch.context() as m:   # the codes' values do not matter here
        m.setattr(TritonQwen3Inference, 'device', property(lambda self: torch.device('cuda')))
        m.setattr(I8, 'quantize_rows', lambda w: (w.to(torch.int8), w.float().abs().amax(1) / 127))
        m.setattr(I8, 'check_rows', lambda w: None)
        model.quantize_weights()
    return model, state


def test_weights_loaded_beside_int8_are_refused(monkeypatch):
    """The codes stand for the projections until load_hf_state_dict takes them away: no other load is left without effect."""
    from types import SimpleNamespace
    from qwen3_triton.inference import KVCache
    from qwen3_triton.inference.model import _check_captured
    model, state = tiny_int8_model(monkeypatch)
    step = SimpleNamespace(model=model, _weights=model._weights)
    before = dict(model.named_parameters())
    for kw in (dict(assign=True), dict(), dict(strict=False, assign=True)):
        with pytest.raises(ValueError, match='load_hf_state_dict'):
            model.load_state_dict(state, **kw)
    assert all(p is before[n] for n, p in model.named_parameters()) and len(model._int8) == 2
    _check_captured(step)
    # what is not in int8 can be loaded
    rest = {k: v + 1 for k, v in state.items() if '_proj' not in k}
    model.load_state_dict(rest, strict=False)
    assert torch.equal(model.lm_head.weight, rest['lm_head.weight'])
    # a part of the model, or one weight, behind its back
    ids, up = torch.zeros(1, 3, dtype=torch.int64), 'layers.1.mlp.up_proj.weight'

    def set_one(m):
        m.model.layers[0].self_attn.k_proj.weight = torch.nn.Parameter(state['model.layers.0.self_attn.k_proj.weight'])
    for change in (lambda m: m.model.load_state_dict({up: state['model.' + up]}, strict=False, assign=True), set_one):
        model, _ = tiny_int8_model(monkeypatch)
        step = SimpleNamespace(model=model, _weights=model._weights)
        _check_captured(step)
        change(model)
        with pytest.raises(RuntimeError, match='beside its int8'):
            model(ids, past_key_values=KVCache([], [], 16, 1, model._cache_owner))
        with pytest.raises(RuntimeError, match='beside its int8'):
            _check_captured(step)
        model.load_hf_state_dict(state)
        assert model._int8 is None and all(torch.equal(p, state[n]) for n, p in model.named_parameters())


def test_a_failed_load_over_int8(monkeypatch):
    """Names that fit nothing leave the model in int8; a load that reached the projections does not leave the old codes."""
    model, state = tiny_int8_model(monkeypatch)
    with pytest.raises(RuntimeError):
        model.load_hf_state_dict({'x.' + k: v for k, v in state.items()})
    assert len(model._int8) == 2
    model._int8.check()
    with pytest.raises(RuntimeError):
        model.load_hf_state_dict({k: v for k, v in state.items() if 'layers.1' not in k})
    assert model._int8 is None
    model.load_hf_state_dict(state)
    assert all(torch.equal(p, state[n]) for n, p in model.named_parameters())


@pytest.mark.parametrize("grad", [True, False])
def test_tangents_are_refused(grad):
    """Inputs of forward-mode differentiation, whose tangents the outputs would not carry."""
    import torch.autograd.forward_ad as fw
    x, q, w, one = torch.ones(1, 32).bfloat16(), torch.zeros(1, 32, dtype=torch.int8), torch.zeros(8, 32, dtype=torch.int8), torch.ones(1)
    t = torch.zeros(1, 1, 1, 128, dtype=torch.bfloat16)
    cache = I8.LayerCache.empty(1, 1, 64, device='cpu')
    with fw.dual_level(), torch.set_grad_enabled(grad):
        dual = lambda a: fw.make_dual(a, torch.ones_like(a))  # noqa: E731
        for call in (lambda: I8.quantize_rows(dual(x)), lambda: I8.rms_norm(x, dual(x[0]), 1e-6), lambda: I8.rms_norm(x, x[0], 1e-6, residual=dual(x)),
                     lambda: I8.linear(q, one, w, dual(torch.ones(8))), lambda: I8.linear(q, dual(one), w, torch.ones(8)),
                     lambda: I8.linear(q, one, w, torch.ones(8), residual=dual(torch.ones(1, 8).bfloat16())),
                     lambda: I8.decode_linear(dual(x), [(w, torch.ones(8))]), lambda: I8.append(dual(t), t, cache, 0),
                     lambda: I8.norm_rope_append(t, t, t, t[0, 0, 0], t[0, 0, 0], dual(t[0]), t[0], cache, 0),
                     lambda: I8.attention(dual(t), cache, 0)):
            with pytest.raises(ValueError, match='forward only'):
                call()
        with pytest.raises(ValueError, match='no gradient'):
            I8.LayerCache(cache.k, cache.v, dual(cache.k_scale), cache.v_scale, cache.k_tail, cache.v_tail)
        with pytest.raises(ValueError, match='ROCm device'):   # no tangent among them: the next check's turn
            I8.quantize_rows(x)


def test_cache_knows_its_quantised_blocks(monkeypatch):
    from qwen3_triton.inference import Int8KVCache
    monkeypatch.setattr(torch.cuda, 'is_current_stream_capturing', lambda: False)
    c = I8.LayerCache.empty(1, 1, 256, device='cpu')

    def check(ok):
        for n in range(257):
            if ok(n):
                c.require_whole(n)
            else:
                with pytest.raises(ValueError, match='quantised block'):
                    c.require_whole(n)
    check(lambda n: True)   # nothing known yet
    I8._note(c, 0, 200, None)
    check(lambda n: n % 64 == 0 or n > 192)
    owner = object()
    cache = Int8KVCache([], [], 256, 1, owner, 100, layers=[c])
    with pytest.raises(ValueError, match='quantised block'):
        cache.admit(owner, 1, 1)
    cache.reset()
    cache.admit(owner, 1, 1)
    I8._note(c, 200, 20, None)
    I8._note(c, 220, 36, None)   # the block's end: the tail still holds 192 .. 219
    check(lambda n: n % 64 == 0 or 192 < n <= 220)
    I8._note(c, 210, 46, None)   # other positions from 210 on
    check(lambda n: n % 64 == 0 or 192 < n <= 210)
    I8._note(c, 64, 64, None)   # started again at 64: what lies behind 128 is no longer held
    check(lambda n: n % 64 == 0 or n > 128)
    I8._note(c, 128, 127, None)
    check(lambda n: n % 64 == 0 or n > 192)
    I8._note(c, 255, 1, torch.zeros(1, dtype=torch.int64))
    check(lambda n: True)
