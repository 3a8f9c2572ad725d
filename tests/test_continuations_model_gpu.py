"""Many continuations of one prompt through the models: a forked cache against the whole sequences in 64 bits, decoding after it
(eager and captured), scores of continuations, and log probabilities in training.

Gates: logits within 2 % of their largest (the bf16 forward gate).  A log probability moves by at most twice what a logit does; an
entropy by at most sum p |log p + H| <= 2 H times that, and its second order is below it (2 H + 1)."""
import pytest
import torch

import oracle as O
from _util import cosine, max_rel, seeded

from qwen3_triton.configuration import OptimizationOptions
from qwen3_triton.inference import DecodeSession, SharedPrefixCache, TritonQwen3Inference
from qwen3_triton.model import PrecisionQwen3ForCausalLM

pytestmark = pytest.mark.gpu

CFG = O.OracleConfig(vocab_size=1000, hidden_size=512, intermediate_size=1040, num_hidden_layers=3, num_attention_heads=8,
                     num_key_value_heads=2, head_dim=128)
BF = torch.bfloat16


def hf_config(oc):
    from transformers import Qwen3Config
    return Qwen3Config(vocab_size=oc.vocab_size, hidden_size=oc.hidden_size, intermediate_size=oc.intermediate_size,
                       num_hidden_layers=oc.num_hidden_layers, num_attention_heads=oc.num_attention_heads,
                       num_key_value_heads=oc.num_key_value_heads, head_dim=oc.head_dim, rope_theta=oc.rope_theta,
                       rms_norm_eps=oc.rms_norm_eps, tie_word_embeddings=oc.tie_word_embeddings, max_position_embeddings=4096)


def build(weights8=False):
    params = {k: v.to(BF) for k, v in O.init_params(CFG, seed=2, std=0.05).items()}
    model = TritonQwen3Inference(hf_config(CFG)).load_hf_state_dict({k: v.cuda() for k, v in params.items()})
    return (model.quantize_weights() if weights8 else model), params


@pytest.fixture(scope="module")
def model():
    return build()


def logits64(params, ids):
    return O.model_forward_reference(ids, {k: v.double() for k, v in params.items()}, CFG, dtype=torch.float64)[0]


def ids_of(b, s, seed):
    return torch.randint(0, CFG.vocab_size, (b, s), generator=seeded(seed))


@pytest.mark.parametrize("prompt,rows,chunks", [(100, 3, (17, 1, 1, 5)), (64, 1, (1, 1)), (1, 4, (70, 2)), (333, 9, (1, 40))])
def test_forked_cache_against_whole_sequences(model, prompt, rows, chunks):
    model, params = model
    head, tail = ids_of(2, prompt, prompt), ids_of(2 * rows, sum(chunks), rows)
    whole = logits64(params, torch.cat([head.repeat_interleave(rows, 0), tail], 1))[:, prompt:]
    cache = model.new_cache(2, prompt + 30)
    model(head.cuda(), past_key_values=cache)
    forked = cache.fork(rows, sum(chunks))
    assert isinstance(forked, SharedPrefixCache) and forked.batch_size == 2 * rows and forked.length == prompt
    for again in range(2):   # and once more after a reset; what the prompt's cache appends meanwhile does not matter
        at = 0
        for n in chunks:
            out = model(tail[:, at:at + n].cuda(), past_key_values=forked, logits_to_keep=n).logits
            assert max_rel(out, whole[:, at:at + n]) <= 2e-2
            at += n
        with pytest.raises(ValueError, match='free positions'):
            model(tail[:, :1].cuda(), past_key_values=forked)
        forked.reset()
        model(tail[:2, :7].cuda(), past_key_values=cache)
    cache.reset()
    with pytest.raises(ValueError, match='no longer'):
        model(tail[:, :1].cuda(), past_key_values=forked)


def test_forked_cache_with_int8_weights():
    """The same step after shared and after copied positions differs by the attention's rounding only; codes next to it may turn by
    a step: the gate of two computations that quantise such rows, 6 %."""
    model, _ = build(weights8=True)
    head, tail = ids_of(1, 90, 1).cuda(), ids_of(4, 3, 2).cuda()
    cache = model.new_cache(1, 90)
    model(head, past_key_values=cache)
    forked, copied = cache.fork(4, 5), model.new_cache(4, 95)
    model(head.expand(4, -1).contiguous(), past_key_values=copied)
    for ids in (tail, tail[:, :1].contiguous()):
        a, b = (model(ids, past_key_values=c).logits for c in (forked, copied))
        assert max_rel(a, b) <= 6e-2


def test_decoding_after_a_fork(model):
    """``generate`` on a forked cache and a captured session give the same tokens, and each is the 64-bit model's choice (or within
    the measured error of it)."""
    model, params = model
    head, tail = ids_of(2, 150, 5), ids_of(6, 12, 6)
    cache = model.new_cache(2, 150)
    model(head.cuda(), past_key_values=cache)
    forked = cache.fork(3, 12 + 19)
    tokens = model.generate(tail.cuda(), max_new_tokens=20, eos_token_id=[], pad_token_id=0, past_key_values=forked)
    assert tokens.shape == (6, 32) and torch.equal(tokens[:, :12], tail.cuda()) and forked.length == 150 + 31
    z = logits64(params, torch.cat([head.repeat_interleave(3, 0), tokens.cpu()], 1))[:, 150 + 11:-1]
    err = 2e-2 * float(z.abs().max())
    picked = z.gather(-1, tokens[:, 12:].cpu()[..., None])[..., 0]
    assert bool((z.max(-1).values - picked <= 2 * err).all())
    session = DecodeSession(model, 6, 40, prefix=cache)
    for _ in range(2):
        session.prefill(tail.cuda())
        session.step()                # eager
        if session.graph is None:
            session.capture()
        for _ in range(18):
            session.step()
        assert torch.equal(session.tokens()[:, :32], tokens)
        session.reset()
    cache.reset()
    with pytest.raises(ValueError, match='no longer'):
        session.prefill(tail.cuda())


def test_scores_of_continuations(model):
    """Answers to one prompt scored after its shared positions, whole sequences scored at once, and the 64-bit model; the
    alternatives are the 64-bit model's up to the logits' error."""
    model, params = model
    prompt, answers = ids_of(1, 200, 7), ids_of(5, 31, 8)
    z = logits64(params, torch.cat([prompt.expand(5, -1), answers], 1))
    d = 2e-2 * float(z.abs().max())
    lp64 = (z[:, 199:-1] / 0.8).log_softmax(-1)
    want = lp64.gather(-1, answers[..., None])[..., 0]
    ent = -(lp64.exp() * lp64).sum(-1)
    # the prompt's last token goes with the answers, so that their first tokens are scored too
    cache = model.new_cache(1, 199)
    model(prompt[:, :199].cuda(), past_key_values=cache)
    ids = torch.cat([prompt[:, 199:].expand(5, -1), answers], 1).cuda()
    out = model.score(ids, past_key_values=cache.fork(5, 32), temperature=0.8)
    assert out.logprobs.shape == (5, 31)
    assert float((out.logprobs.cpu() - want).abs().max()) <= 2 * d / 0.8
    assert bool(((out.entropy.cpu() - ent).abs() <= 2 * d / 0.8 * (2 * ent + 1)).all())
    whole = model.score(torch.cat([prompt.expand(5, -1), answers], 1).cuda(), temperature=0.8)
    assert whole.logprobs.shape == (5, 230)
    assert float((whole.logprobs[:, 199:].cpu() - want).abs().max()) <= 2 * d / 0.8
    top = model.score(ids, past_key_values=cache.fork(5, 32), top=4, temperature=0.8)
    assert top.top_tokens.shape == (5, 31, 4)
    kth = z[:, 199:-1].sort(dim=-1, descending=True).values[..., 3]
    assert bool((z[:, 199:-1].gather(-1, top.top_tokens.cpu()).min(-1).values >= kth - 2 * d).all())
    # only some positions
    labels = ids.clone()
    labels[:, :10] = -100
    some = model.score(ids, past_key_values=cache.fork(5, 32), labels=labels, temperature=0.8)
    assert bool((some.logprobs[:, :9] == 0).all()) and torch.equal(some.logprobs[:, 9:], out.logprobs[:, 9:])


@pytest.mark.parametrize("s", [1, 3])
def test_positions_appended_where_the_device_says(s):
    """Norm, rotation and append with a start that is read on the device: the bits of the host's start, and nothing outside the caches."""
    from qwen3_triton.kernels import _ops
    b, hq, hk, d, c = 3, 8, 2, 128, 20
    gen = seeded(s)
    q, k, v = (torch.randn((b, s, h, d), generator=gen).to(BF).cuda() for h in (hq, hk, hk))
    wq, wk = (torch.rand(d, generator=gen).to(BF).cuda() for _ in range(2))
    cos, sin = (torch.randn((b, s, d), generator=gen).to(BF).cuda() for _ in range(2))
    fresh = torch.randn((2, b, hk, c, d), generator=gen).to(BF).cuda()
    for start in (0, 7, c - s, c - 1, c, c + 5, -1, -s, 1 << 40, -(1 << 40)):
        got, want = fresh.clone(), fresh.clone()
        y = _ops.norm_rope_qk_cache_fwd(q, k, v, wq, wk, cos, sin, got[0], got[1], 0, 1e-6, torch.tensor([start]).cuda())
        big = torch.zeros((2, b, hk, c + 2 * s, d), dtype=BF, device='cuda')   # room on both sides
        inside = max(-s, min(start, c))
        x = _ops.norm_rope_qk_cache_fwd(q, k, v, wq, wk, cos, sin, big[0], big[1], inside + s, 1e-6)
        lo, hi = max(inside, 0), min(inside + s, c)
        want[:, :, :, lo:hi] = big[:, :, :, lo + s:hi + s]
        assert torch.equal(y, x) and torch.equal(got, want), start


def test_refusals(model):
    model, _ = model
    cache = model.new_cache(2, 20)
    with pytest.raises(ValueError, match='no positions'):
        cache.fork(2, 5)
    model(ids_of(2, 10, 0).cuda(), past_key_values=cache)
    for bad in ((0, 5), (2, 0), (1.0, 5), (2, True)):
        with pytest.raises(ValueError, match='positive'):
            cache.fork(*bad)
    forked = cache.fork(2, 5)
    with pytest.raises(ValueError, match='holds batch'):
        model(ids_of(2, 1, 0).cuda(), past_key_values=forked)
    for what in (lambda: forked.fork(2, 5), forked.quantized, lambda: cache.quantized().fork(2, 5)):
        with pytest.raises(ValueError):
            what()
    with pytest.raises(ValueError, match='free positions'):
        model.generate(ids_of(4, 3, 0).cuda(), max_new_tokens=4, eos_token_id=[], past_key_values=forked)
    with pytest.raises(ValueError, match='int8'):
        model.generate(ids_of(4, 1, 0).cuda(), max_new_tokens=2, past_key_values=forked, cache_dtype=torch.int8)
    other, _ = build()
    with pytest.raises(ValueError, match='another model'):
        other(ids_of(4, 1, 0).cuda(), past_key_values=forked)
    with pytest.raises(ValueError, match='prefix'):
        DecodeSession(other, 4, 10, prefix=cache)
    with pytest.raises(ValueError, match='prefix'):
        DecodeSession(model, 3, 10, prefix=cache)
    with pytest.raises(ValueError, match='at least 2'):
        model.score(ids_of(2, 1, 0).cuda())
    with pytest.raises(ValueError, match='labels'):
        model.score(ids_of(2, 5, 0).cuda(), labels=ids_of(2, 4, 0).cuda())
    for bad in (dict(top=33), dict(temperature=0.0), dict(ignore_index=None)):   # refused before the cache takes the chunk
        with pytest.raises(ValueError):
            model.score(ids_of(4, 3, 0).cuda(), past_key_values=forked, **bad)
    assert forked.valid and forked.length == forked.prefix_length
    long = cache.fork(1, model.config.max_position_embeddings)
    with pytest.raises(ValueError, match='positions'):
        model(ids_of(2, model.config.max_position_embeddings - 9, 0).cuda(), past_key_values=long)
    assert long.valid and long.length == long.prefix_length


@pytest.mark.parametrize("dtype", [torch.float32, BF])
def test_policy_gradient_step(dtype):
    """Log probabilities and entropies of a batch with masked prompts, an advantage-weighted loss of both, and its gradients in every
    parameter, against the 64-bit model (the gates of the training step: logits within 2 %, in fp32 1e-4; gradients' cosine)."""
    tiny = O.OracleConfig()
    params = O.init_params(tiny, seed=0, std=0.02)
    ids = torch.randint(0, tiny.vocab_size, (3, 90), generator=seeded(0))
    labels = ids.clone()
    labels[:, :20] = -100
    labels[1, 70:] = -100
    adv, bonus = torch.randn((3, 1), generator=seeded(1)), 0.01
    model = PrecisionQwen3ForCausalLM(hf_config(tiny), OptimizationOptions(), require_8b_shape=False)
    model.load_hf_state_dict({k: v.to(dtype) for k, v in params.items()})
    model = model.to("cuda")
    out = model.logprobs(ids.cuda(), labels.cuda(), temperature=0.9)
    loss = -(out.logprobs * adv.cuda()).sum() - bonus * out.entropy.sum()
    loss.backward()
    leaf = {k: v.to(dtype).double().requires_grad_() for k, v in params.items()}
    z = O.model_forward_reference(ids, leaf, tiny, dtype=torch.float64)[0][:, :-1] / 0.9
    lp = z.log_softmax(-1)
    keep = labels[:, 1:] != -100
    got = torch.where(keep, lp.gather(-1, labels[:, 1:].clamp_min(0)[..., None])[..., 0], 0.0)
    ent = torch.where(keep, -(lp.exp() * lp).sum(-1), 0.0)
    eloss = -(got * adv).sum() - bonus * ent.sum()
    eloss.backward()
    gate = 2e-2 if dtype == BF else 1e-4
    d = gate * float(z.detach().abs().max())
    assert float((out.logprobs.detach().cpu() - got.detach()).abs().max()) <= 2 * d
    assert bool((out.logprobs.detach().cpu()[~keep] == 0).all()) and bool((out.entropy.detach().cpu()[~keep] == 0).all())
    for name, p in model.named_parameters():
        assert cosine(p.grad, leaf[name].grad) >= (0.999 if dtype == BF else 0.99999), name
