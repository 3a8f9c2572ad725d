"""The inference model in 8 bits: int8 weights, an int8 cache, and both, against the same steps in 64 bits; the captured
paths against the eager one; chunked prefill; conversions between the caches."""
import pytest
import torch

import oracle as O
from _util import max_rel, seeded

from qwen3_triton.inference import CapturedGreedyRequest, DecodeSession, Int8KVCache, TritonQwen3Inference, int8

pytestmark = pytest.mark.gpu

CFG = O.OracleConfig(vocab_size=1000, hidden_size=512, intermediate_size=1040, num_hidden_layers=3, num_attention_heads=8,
                     num_key_value_heads=2, head_dim=128)
BF = torch.bfloat16

# Two computations that both quantise an activation row, from values that differ in their last bf16 bits, need not agree on
# the codes: at worst their rounding errors are independent, each uniform over a step M / 127, so the rows differ by
# M / 127 / sqrt(6) in the root mean square.  M / rms is about 4 for the normed rows and attention outputs (512 nearly
# normal values) and about 8 for the SwiGLU outputs: 1.3 % and 2.6 % of a row.  Three layers of three such rows and one of
# these, none of which outweighs the residual stream: sqrt(3 (3 * 1.3^2 + 2.6^2)) = 5.9 % of the logits, on top of nothing
# else that counts; the largest of them against the largest logit alike.  Bf16 weights have no such rows: the forward gate.
GATE = {False: 2e-2, True: 6e-2}


def hf_config(oc):
    from transformers import Qwen3Config
    return Qwen3Config(vocab_size=oc.vocab_size, hidden_size=oc.hidden_size, intermediate_size=oc.intermediate_size,
                       num_hidden_layers=oc.num_hidden_layers, num_attention_heads=oc.num_attention_heads,
                       num_key_value_heads=oc.num_key_value_heads, head_dim=oc.head_dim, rope_theta=oc.rope_theta,
                       rms_norm_eps=oc.rms_norm_eps, tie_word_embeddings=False, max_position_embeddings=4096)


def build(weights8):
    params = {k: v.to(BF) for k, v in O.init_params(CFG, seed=2, std=0.05).items()}
    model = TritonQwen3Inference(hf_config(CFG)).load_hf_state_dict({k: v.cuda() for k, v in params.items()})
    return model.quantize_weights() if weights8 else model, params


@pytest.fixture(scope="module", params=[False, True], ids=["w16", "w8"])
def model(request):
    return (*build(request.param), request.param)


def rounded(x):
    return x.to(BF).double()


def codes64(a):
    m = a.abs().amax(-1, keepdim=True)
    return (127.0 * a / m).round() * (m / 127.0)


def forward64(p, ids, weights8, cache8):
    """All positions' logits in 64 bits, with the values stored in bf16 and in 8 bits where the model stores them so."""
    c = CFG
    b, s = ids.shape
    d, hq, hkv = c.head_dim, c.num_attention_heads, c.num_key_value_heads

    def proj(x, name):
        w = p[name].double()
        return rounded((codes64(x) @ codes64(w).t()) if weights8 else x @ w.t())

    def norm(x, name):
        w = p[name].double()
        y = x * w / (x.square().mean(-1, keepdim=True) + c.rms_norm_eps).sqrt()
        return y if weights8 else rounded(y)   # quantised as it is, or stored in bf16

    inv = 1.0 / (c.rope_theta ** (torch.arange(0, d, 2).double() / d))
    ang = torch.arange(s).double()[:, None] * inv
    cos, sin = (rounded(torch.cat([f(ang)] * 2, -1))[None, :, None] for f in (torch.cos, torch.sin))

    def head_norm_rope(x, name):
        w = p[name].double()
        y = x * w / (x.square().mean(-1, keepdim=True) + c.rms_norm_eps).sqrt()
        rot = torch.cat([-y[..., d // 2:], y[..., :d // 2]], -1)
        return rounded(y * cos + rot * sin)

    def held(x):   # [B, S, H, D] as the cache gives it back: whole blocks in 8 bits
        n = s // 64 * 64
        if not cache8 or n == 0:
            return x
        blocks = x[:, :n].view(b, n // 64, 64, hkv, d).permute(0, 1, 3, 2, 4).reshape(b, n // 64, hkv, 64 * d)
        back = codes64(blocks).view(b, n // 64, hkv, 64, d).permute(0, 1, 3, 2, 4).reshape(b, n, hkv, d)
        return torch.cat([back, x[:, n:]], 1)

    x = p["model.embed_tokens.weight"].double()[ids]
    mask = torch.ones(s, s, dtype=torch.bool).triu(1)
    for i in range(c.num_hidden_layers):
        pre = f"model.layers.{i}."
        h = norm(x, pre + "input_layernorm.weight")
        q, k, v = (proj(h, pre + f"self_attn.{n}_proj.weight").view(b, s, -1, d) for n in "qkv")
        q = head_norm_rope(q, pre + "self_attn.q_norm.weight")
        k = held(head_norm_rope(k, pre + "self_attn.k_norm.weight")).repeat_interleave(hq // hkv, 2)
        v = held(v).repeat_interleave(hq // hkv, 2)
        z = torch.einsum("bshd,bthd->bhst", q, k) * d ** -0.5
        y = rounded(torch.einsum("bhst,bthd->bshd", torch.softmax(z.masked_fill(mask, -1e300), -1), v).reshape(b, s, -1))
        x = rounded(x + proj(y, pre + "self_attn.o_proj.weight"))
        h = norm(x, pre + "post_attention_layernorm.weight")
        if weights8:
            g, u = ((codes64(h) @ codes64(p[pre + f"mlp.{n}_proj.weight"].double()).t()) for n in ("gate", "up"))
        else:
            g, u = (proj(h, pre + f"mlp.{n}_proj.weight") for n in ("gate", "up"))
        x = rounded(x + proj(rounded(g * torch.sigmoid(g) * u), pre + "mlp.down_proj.weight"))
    w = p["model.norm.weight"].double()
    h = rounded(x * w / (x.square().mean(-1, keepdim=True) + c.rms_norm_eps).sqrt())
    return h @ p["lm_head.weight"].double().t()


@pytest.mark.parametrize("cache_dtype", [BF, torch.int8], ids=["c16", "c8"])
@pytest.mark.parametrize("b,s", [(1, 5), (2, 64), (1, 150), (3, 200)])
def test_prefill_logits(model, cache_dtype, b, s):
    """Every position's logits against the same steps in 64 bits."""
    m, params, weights8 = model
    ids = torch.randint(0, CFG.vocab_size, (b, s), generator=seeded(s))
    cache = m.new_cache(b, s, dtype=cache_dtype)
    got = m(ids.cuda(), past_key_values=cache, logits_to_keep=s).logits
    want = forward64(params, ids, weights8, cache_dtype == torch.int8)
    assert isinstance(cache, Int8KVCache) == (cache_dtype == torch.int8) and cache.length == s
    assert max_rel(got, want) <= GATE[weights8]


@pytest.mark.parametrize("b", [1, 3, 17])
def test_decode_steps_follow_the_whole_sequence(model, b):
    """Teacher-forced decode steps over a block's end: each step's logits against a whole prefill of what the cache then
    holds (a block that is finished later is still exact in the step's cache, so only steps whose last block is whole, or
    sequences below one block, see the same cache)."""
    m, params, weights8 = model
    ids = torch.randint(0, CFG.vocab_size, (b, 140), generator=seeded(b))
    for first in (50, 120):
        cache = m.new_cache(b, 140, dtype=torch.int8)
        m(ids[:, :first].cuda(), past_key_values=cache)
        for t in range(first, 140):
            got = m(ids[:, t:t + 1].cuda(), past_key_values=cache).logits
            if t + 1 in (55, 64, 128, 140):
                want = forward64(params, ids[:, :t + 1], weights8, True)[:, -1:]
                # earlier positions' layers saw their own block unquantised while the whole prefill sees it quantised: an
                # 8-bit rounding (1 / 254 of a block's largest value, below 2 % of its rms) of some keys and values beside it
                assert max_rel(got, want) <= GATE[weights8] + 2e-2, t
        assert cache.length == 140


@pytest.mark.parametrize("b,s", [(1, 60), (2, 130), (17, 40)])
def test_captured_paths_reproduce_generate(model, b, s):
    """DecodeSession (its graph replayed at every position, over a block's end) and CapturedGreedyRequest, token for token."""
    m, _, _ = model
    ids = torch.randint(0, CFG.vocab_size, (b, s), generator=seeded(s + b)).cuda()
    new = 12
    eager = m.generate(ids, max_new_tokens=new, eos_token_id=[], pad_token_id=0, cache_dtype=torch.int8)
    sess = DecodeSession(m, b, s + 300, cache_dtype=torch.int8)   # a longer capacity: other spans, the same sums
    for _ in range(2):
        sess.prefill(ids)
        if sess.graph is None:
            sess.capture()
        for _ in range(new - 1):
            sess.step()
        torch.cuda.synchronize()
        assert torch.equal(sess.tokens(), eager)
        sess.reset()
    req = CapturedGreedyRequest(m, ids, max_new_tokens=new, cache_dtype=torch.int8)
    for _ in range(2):
        assert torch.equal(req(ids).clone(), eager)


def test_two_captured_sessions_side_by_side(model):
    """Two sessions of one model, their graphs replayed in turn: each keeps its own tokens."""
    m, _, _ = model
    prompts = [torch.randint(0, CFG.vocab_size, (1, n), generator=seeded(n)).cuda() for n in (30, 61)]
    want = [m.generate(p, max_new_tokens=8, eos_token_id=[], pad_token_id=0, cache_dtype=torch.int8) for p in prompts]
    sessions = [DecodeSession(m, 1, 200, cache_dtype=torch.int8) for _ in prompts]
    for sess, p in zip(sessions, prompts):
        sess.prefill(p)
        sess.capture()
    for _ in range(7):
        for sess in sessions:
            sess.step()
    torch.cuda.synchronize()
    for sess, w in zip(sessions, want):
        assert torch.equal(sess.tokens(), w)


def test_chunked_prefill_holds_the_same_blocks(model):
    """The first layer's cache after one prefill and after chunks: the same codes and scales, bit for bit (its keys and values
    depend on the tokens alone), whatever the chunks."""
    m, _, weights8 = model
    ids = torch.randint(0, CFG.vocab_size, (2, 200), generator=seeded(1)).cuda()
    caches = []
    for cuts in ((200,), (1, 63, 64, 65, 190, 200), (100, 200)):
        cache, at = m.new_cache(2, 200, dtype=torch.int8), 0
        for end in cuts:
            m(ids[:, at:end].contiguous(), past_key_values=cache)
            at = end
        caches.append(cache.layers[0])
    if weights8:   # integer sums: a projection is the same whatever the number of rows
        for c in caches[1:]:
            for x, y in zip((c.k[:, :, :192], c.v[:, :, :3], c.k_scale[:, :, :3], c.k_tail[:, :, :8]),
                            (caches[0].k[:, :, :192], caches[0].v[:, :, :3], caches[0].k_scale[:, :, :3], caches[0].k_tail[:, :, :8])):
                assert torch.equal(x, y)


def test_cache_conversions(model):
    """16 bits -> 8 -> 16: the positions of whole blocks as quantised, the rest as they were; decoding goes on in both."""
    m, _, weights8 = model
    ids = torch.randint(0, CFG.vocab_size, (2, 150), generator=seeded(5)).cuda()
    cache = m.new_cache(2, 160)
    m(ids, past_key_values=cache)
    c8 = cache.quantized()
    assert isinstance(c8, Int8KVCache) and c8.length == 150 and c8.capacity == 160
    # per head and layer: 64 positions' tail in 16 bits beside 8 bits and 4 bytes a block
    assert m.new_cache(1, 4096, dtype=torch.int8).nbytes == 3 * 2 * 2 * (4096 * 128 + 64 * 4 + 64 * 128 * 2)
    back = c8.dequantized()
    assert type(back) is type(cache) and back.length == 150
    for k, k0 in zip(back.keys + back.values, cache.keys + cache.values):
        assert torch.equal(k[:, :, 128:150], k0[:, :, 128:150])
        big = k0[:, :, :128].double().reshape(2, 2, 2, -1).abs().amax(-1)[..., None]
        err = (k[:, :, :128].double() - k0[:, :, :128].double()).reshape(2, 2, 2, -1).abs()
        # half a step of M / 127, and the value's rounding to bf16
        assert bool((err <= big / 254 * (1 + 2.0 ** -20) + big * 2.0 ** -8).all())
    tok = ids[:, :1].contiguous()
    a = m(tok, past_key_values=c8).logits
    b = m(tok, past_key_values=back).logits
    assert c8.length == back.length == 151 and max_rel(a, b.float()) <= GATE[weights8] + 2e-2
    assert m.new_cache(1, 10, dtype=torch.int8).dequantized().length == 0
    assert m.new_cache(1, 10).quantized().length == 0


def test_weights_in_8_bits_and_back():
    model, params = build(False)
    before = {k for k, _ in model.named_parameters()}
    ids = torch.randint(0, CFG.vocab_size, (1, 20), generator=seeded(3)).cuda()
    want = model(ids, logits_to_keep=20).logits
    model.quantize_weights()
    with pytest.raises(ValueError, match='already'):
        model.quantize_weights()
    got = model(ids, logits_to_keep=20).logits
    assert not torch.equal(got, want) and max_rel(got, want.float()) <= 0.1   # three layers of 8-bit roundings
    bf16 = sum(p.numel() * 2 for n, p in params.items() if '_proj' in n)
    assert sum(w.nbytes for w in model._int8) < 0.52 * bf16
    model.load_hf_state_dict({k: v.cuda() for k, v in params.items()})
    assert torch.equal(model(ids, logits_to_keep=20).logits, want) and {k for k, _ in model.named_parameters()} == before
    with pytest.raises(TypeError):
        model.new_cache(1, 10, dtype=torch.float32)


def test_integer_sums_do_not_depend_on_the_batch():
    gen = seeded(2)
    x = torch.randn(600, 512, generator=gen).to(BF).cuda()
    w = int8.quantize_rows(torch.randn(520, 512, generator=gen).to(BF).cuda())
    q, s = int8.quantize_rows(x)
    whole = int8.linear(q, s, *w)
    for m in (1, 5, 16, 17, 40, 130, 300):
        assert torch.equal(int8.linear(q[:m], s[:m], *w), whole[:m])


def test_replaced_weights_end_captured_steps_and_state():
    """A captured step reads the weights that it was captured with: once they are freed it refuses to replay."""
    model, params = build(False)
    ids = torch.arange(12, device='cuda').view(1, 12)
    session = DecodeSession(model, 1, 32)
    session.prefill(ids)
    session.capture()
    session.step()
    request = CapturedGreedyRequest(model, ids, max_new_tokens=3)
    request(ids)
    assert model.state_dict()
    model.quantize_weights()
    with pytest.raises(RuntimeError, match='capture again'):
        session.step()
    with pytest.raises(RuntimeError, match='capture again'):
        request(ids)
    with pytest.raises(ValueError, match='no state'):
        model.state_dict()
    session.capture()
    session.step()
    request = CapturedGreedyRequest(model, ids, max_new_tokens=3)
    assert torch.equal(request(ids), model.generate(ids, max_new_tokens=3, eos_token_id=()))
    model.load_hf_state_dict({k: v.cuda() for k, v in params.items()})
    with pytest.raises(RuntimeError, match='capture again'):
        request(ids)
    assert model.state_dict()
    with pytest.raises(ValueError, match='already'):
        model.new_cache(1, 16, dtype=torch.int8).quantized()


@pytest.mark.parametrize("heads,kv,cache_dtype", [(144, 18, BF), (144, 18, torch.int8), (144, 9, torch.int8), (130, 2, torch.int8)])
def test_more_heads_than_a_fused_product_takes(heads, kv, cache_dtype):
    """The output projection's rows (18432 and 16640 values) are longer than decode_linear's.  More than 8 heads of a group
    decode over the int8 cache only: attention over the 16-bit one refuses them, whatever the weights."""
    oc = O.OracleConfig(vocab_size=200, hidden_size=128, intermediate_size=256, num_hidden_layers=1, num_attention_heads=heads,
                        num_key_value_heads=kv, head_dim=128)
    model = TritonQwen3Inference.random_init(hf_config(oc), seed=3, std=0.05).quantize_weights()
    ids = torch.arange(9, device='cuda').view(1, 9)
    out = model.generate(ids, max_new_tokens=4, eos_token_id=(), cache_dtype=cache_dtype)
    assert torch.equal(out, CapturedGreedyRequest(model, ids, max_new_tokens=4, cache_dtype=cache_dtype)(ids))


@pytest.mark.parametrize("load", ["load_hf_state_dict", "load_state_dict", "half a load"])
def test_a_reload_ends_captured_steps(load):
    """Without int8 too: the old tensors are gone, and a step captured on them refuses to replay."""
    model, params = build(False)
    ids = torch.arange(12, device='cuda').view(1, 12)
    session = DecodeSession(model, 1, 32)
    session.prefill(ids)
    session.capture()
    session.step()
    request = CapturedGreedyRequest(model, ids, max_new_tokens=3)
    want = request(ids).clone()
    state = {k: v.cuda() for k, v in params.items()}
    if load == "load_hf_state_dict":
        model.load_hf_state_dict(state)
    elif load == "load_state_dict":
        model.load_state_dict(state, assign=True)
    else:
        del state["lm_head.weight"]
        with pytest.raises((KeyError, RuntimeError)):
            model.load_hf_state_dict(state)
    with pytest.raises(RuntimeError, match='capture again'):
        session.step()
    with pytest.raises(RuntimeError, match='capture again'):
        request(ids)
    assert torch.equal(CapturedGreedyRequest(model, ids, max_new_tokens=3)(ids), want)
    # weights copied into the tensors that are there: what a captured step reads is the new ones
    request = CapturedGreedyRequest(model, ids, max_new_tokens=3)
    model.load_state_dict({k: v.cuda() for k, v in params.items()})
    assert torch.equal(request(ids), want)


def test_weights_beside_int8_are_refused():
    model, params = build(True)
    state = {k: v.cuda() for k, v in params.items()}
    ids = torch.arange(12, device='cuda').view(1, 12)
    want = model(ids).logits
    request = CapturedGreedyRequest(model, ids, max_new_tokens=3)
    with pytest.raises(ValueError, match='load_hf_state_dict'):
        model.load_state_dict(state, assign=True)
    assert torch.equal(model(ids).logits, want)
    model.model.layers[1].mlp.up_proj.load_state_dict({'weight': state['model.layers.1.mlp.up_proj.weight']}, assign=True)
    for call in (lambda: model(ids), lambda: request(ids), lambda: model.generate(ids, max_new_tokens=2)):
        with pytest.raises(RuntimeError, match='beside its int8'):
            call()
    model.load_hf_state_dict(state)
    assert torch.equal(model(ids).logits, build(False)[0](ids).logits)
    assert torch.equal(model.quantize_weights()(ids).logits, want)


def test_weights_that_cannot_be_quantised_leave_the_model_as_it_was():
    """One weight of the last layer does not start on 16 bytes: quantize_weights refuses before any bf16 weight is gone."""
    model, params = build(False)
    ids = torch.arange(12, device='cuda').view(1, 12)
    want = model(ids).logits
    proj = model.model.layers[-1].mlp.down_proj
    good = proj.weight
    flat = torch.empty(good.numel() + 1, dtype=BF, device='cuda')
    flat[1:].copy_(good.detach().flatten())
    proj.weight = torch.nn.Parameter(flat[1:].view_as(good), requires_grad=False)
    with pytest.raises(ValueError, match='16 bytes'):
        model.quantize_weights()
    proj.weight = good
    assert model._int8 is None and torch.equal(model(ids).logits, want)
    model.quantize_weights()
    assert max_rel(model(ids).logits, want.float()) <= 0.1


def test_an_int8_cache_is_not_wound_back_into_a_block(model):
    """Its length can go back to a multiple of 64 or within the unfinished block; elsewhere the next step refuses."""
    m, _, _ = model
    ids = torch.randint(0, CFG.vocab_size, (1, 150), generator=seeded(8)).cuda()
    cache = m.new_cache(1, 200, dtype=torch.int8)
    m(ids, past_key_values=cache)
    want = m(ids[:, 140:145].contiguous(), past_key_values=cache).logits
    for back in (100, 127):
        cache.length = back
        with pytest.raises(ValueError, match='quantised block'):
            m(ids[:, :1].contiguous(), past_key_values=cache)
        with pytest.raises(ValueError, match='quantised block'):
            cache.dequantized()
        assert cache.valid
    cache.length = 150   # a tail position: the same tokens again
    assert torch.equal(m(ids[:, 140:145].contiguous(), past_key_values=cache).logits, want)
    cache.length = 128
    m(ids[:, 128:].contiguous(), past_key_values=cache)
    cache.reset()
    m(ids[:, :70].contiguous(), past_key_values=cache)
    assert cache.length == 70


def test_chunked_prefill_holds_alike_blocks(model):
    """With bf16 weights too: a projection's sums depend on the number of its rows (the kernel that forms them), so its bf16
    result may lie one rounding aside (2^-7 of it).  Values follow it; keys by twice that of either dim after the norm, 2^-6 of
    |n c| + |r s| <= sqrt(2) of the block's largest, and round once more (2^-7).  Each side's code is half a step from its value."""
    m, _, _ = model
    ids = torch.randint(0, CFG.vocab_size, (2, 200), generator=seeded(1)).cuda()
    held = []
    for cuts in ((200,), (1, 63, 64, 65, 190, 200), (100, 200)):
        cache, at = m.new_cache(2, 200, dtype=torch.int8), 0
        for end in cuts:
            m(ids[:, at:end].contiguous(), past_key_values=cache)
            at = end
        held.append([t[:, :, :192].double() for t in int8.read(cache.layers[0], 200, dtype=torch.float32)])
    for other in held[1:]:
        for a, b in zip(held[0], other):
            block = a.view(2, -1, 3, 64 * 128)
            most = block.abs().amax(-1, keepdim=True) * (1 + 2.0 ** -5)   # either side's M
            step = most * (2.0 ** -6 * 2 ** 0.5 + 2.0 ** -7 + 1 / 127)
            assert bool(((block - b.view_as(block)).abs() <= step).all())


@pytest.mark.parametrize("b", [1, 2, 3, 17])
def test_decode_steps_over_a_16_bit_cache(model, b):
    """Teacher-forced decode steps, every projection at its few-row forms, against the whole sequence in 64 bits."""
    m, params, weights8 = model
    ids = torch.randint(0, CFG.vocab_size, (b, 75), generator=seeded(b + 40))
    cache = m.new_cache(b, 75)
    m(ids[:, :60].cuda(), past_key_values=cache)
    got = torch.cat([m(ids[:, t:t + 1].cuda(), past_key_values=cache).logits for t in range(60, 75)], 1)
    assert max_rel(got, forward64(params, ids, weights8, False)[:, 60:]) <= GATE[weights8]


def test_head_norms_with_an_eps_each(model):
    """Norms whose eps were set apart: the int8 cache's tail holds the keys that the 16-bit cache holds."""
    m, _, _ = model
    ids = torch.randint(0, CFG.vocab_size, (1, 40), generator=seeded(4)).cuda()
    norms = [layer.self_attn.k_norm for layer in m.model.layers]
    keys = []
    eps = norms[0].eps
    try:
        for e in (eps, 1.0):
            for norm in norms:
                norm.eps = e
            c8, c16 = m.new_cache(1, 64, dtype=torch.int8), m.new_cache(1, 64)
            a, b = (m(ids, past_key_values=c).logits for c in (c8, c16))
            assert torch.equal(c8.layers[0].k_tail[:, :, :40], c16.keys[0][:, :, :40]) and max_rel(a, b.float()) <= GATE[True]
            step = [m(ids[:, :1].contiguous(), past_key_values=c).logits for c in (c8, c16)]
            assert max_rel(step[0], step[1].float()) <= GATE[True]
            keys.append(c16.keys[0][:, :, :40].clone())
    finally:
        for norm in norms:
            norm.eps = eps
    assert not torch.equal(*keys)
