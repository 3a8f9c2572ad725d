"""Performance cases of the operators for many continuations of one prompt: attention over a prefix that rows share
(``qwen3_triton.inference.prefix``) and log probabilities of given tokens (``qwen3_triton.kernels.logprobs``), from one token to
4096.

The shapes are Qwen3-8B's (hidden 4096, 32 query and 8 key/value heads of 128, 151936 tokens).  With ``own`` false, ``run``
computes each operator from elementary torch operations; with ``own`` true it calls the package.

The operators' definitions:

* shared prefix: B rows in R groups of B / R; the rows of group r continue prefix r (keys and values [R, Hkv, P, D], held once)
  with positions of their own ([B, Hkv, C, D]).  Query s of row b, at its own position start_b + s, sees the whole prefix and its
  row's positions 0 .. start_b + s: o = softmax(q k^T / sqrt(D)) v over both.
* token log probabilities: with x = logits / temperature (32 bits) and p = softmax(x), of each row: log p[token], the entropy
  -sum p log p, and the ``top`` largest log p with their tokens (ties: the lowest token first).  A token of -100 leaves its row out:
  zeros.  Backward: dlogits = (g_i [i = token] - p_i (g + g_h (log p_i + entropy))) / temperature for upstream gradients g of the
  log probability and g_h of the entropy.
* the same straight from hidden states and the LM head's weight, logits = h W^T, whose gradients are dh = dlogits W and
  dW = dlogits^T h.
"""
import math
import os
import sys

import torch

own = False

H, HQ, HKV, D, V = 4096, 32, 8, 128, 151936   # Qwen3-8B
IGNORE = -100
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # Four answers to a short question, their eighth token: the smallest attention, all latency.
        {"name": "prefix_b4_p200", "kind": "prefix", "groups": 1, "rows": 4, "seq": 1, "prefix": 200, "start": 7, "ragged": False, "dtype": "bf16"},
        # 32 requests behind a common system prompt of 8192 tokens, at their 512th token.
        {"name": "prefix_b32_p8192", "kind": "prefix", "groups": 1, "rows": 32, "seq": 1, "prefix": 8192, "start": 511, "ragged": False, "dtype": "bf16"},
        # Rollouts: four prompts with eight samples each, which have come to different lengths.
        {"name": "prefix_g4x8_p2047_f16", "kind": "prefix", "groups": 4, "rows": 32, "seq": 1, "prefix": 2047, "start": 700, "ragged": True, "dtype": "f16"},
        # 64 users of one long document, at different lengths.
        {"name": "prefix_b64_p32768", "kind": "prefix", "groups": 1, "rows": 64, "seq": 1, "prefix": 32768, "start": 1000, "ragged": True, "dtype": "bf16"},
        # Eight questions of 200 tokens about a document of 4001, prefilled together.
        {"name": "prefix_b8_s200_p4001", "kind": "prefix", "groups": 1, "rows": 8, "seq": 200, "prefix": 4001, "start": 0, "ragged": False, "dtype": "bf16"},
        # A decode step that reports its token with twenty alternatives: one row, all latency.
        {"name": "logprobs_t1_top20", "kind": "logprobs", "rows": 1, "vocab": V, "top": 20, "temperature": 1.0, "masked": 0.0, "grad": False, "dtype": "bf16"},
        # Scoring prompts of 4096 tokens from their logits.
        {"name": "logprobs_t4096", "kind": "logprobs", "rows": 4096, "vocab": V, "top": 0, "temperature": 1.0, "masked": 0.0, "grad": False, "dtype": "bf16"},
        # The same with five alternatives, sampled at a temperature under a grammar that forbids a third of the tokens, in fp32.
        {"name": "logprobs_t777_top5_f32", "kind": "logprobs", "rows": 777, "vocab": V, "top": 5, "temperature": 0.7, "masked": 0.3, "grad": False, "dtype": "f32"},
        # A policy-gradient step on logits: log probabilities and entropies of 2048 sampled tokens, and their gradient.
        {"name": "logprobs_t2048_grad", "kind": "logprobs", "rows": 2048, "vocab": V, "top": 0, "temperature": 1.0, "masked": 0.0, "grad": True, "dtype": "bf16"},
        # Eight rows scored straight from their hidden states: the LM head's weight, streamed once.
        {"name": "lm_head_t8", "kind": "lm_head", "rows": 8, "h": H, "vocab": V, "temperature": 1.0, "grad": False, "dtype": "bf16"},
        # The old policy's log probabilities of a ragged batch of 999 tokens.
        {"name": "lm_head_t999_f16", "kind": "lm_head", "rows": 999, "h": H, "vocab": V, "temperature": 1.0, "grad": False, "dtype": "f16"},
        # The policy-gradient step of 4096 tokens straight from the hidden states: three products with the LM head.
        {"name": "lm_head_t4096_grad", "kind": "lm_head", "rows": 4096, "h": H, "vocab": V, "temperature": 1.0, "grad": True, "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["prefix", "prefix", "prefix", "logprobs", "logprobs", "lm_head"])
    dtype = rng.choice(["bf16", "f16"])
    if kind == "prefix":
        groups = rng.choice([1, 1, 1, 2, 4])
        seq = rng.choice([1, 1, 1, rng.randint(2, 16), _log_int(rng, 17, 300)])
        rows = groups * _log_int(rng, 1, max(1, 64 // groups if seq <= 16 else 8 // groups))
        return {"kind": kind, "groups": groups, "rows": rows, "seq": seq, "prefix": _log_int(rng, 1, 32768 if seq <= 16 else 8192),
                "start": _log_int(rng, 1, 2000) - 1, "ragged": rng.random() < 0.5, "dtype": dtype}
    if kind == "logprobs":
        grad = rng.random() < 0.4
        return {"kind": kind, "rows": _log_int(rng, 1, 2048 if grad else 4096), "vocab": _log_int(rng, 1000, V),
                "top": 0 if grad else rng.choice([0, 1, rng.randint(2, 20)]), "temperature": rng.choice([1.0, 1.0, 0.7, 1.3]),
                "masked": rng.choice([0.0, 0.0, 0.3]), "grad": grad, "dtype": rng.choice([dtype, dtype, "f32"])}
    grad = rng.random() < 0.4
    return {"kind": kind, "rows": _log_int(rng, 1, 4096), "h": 64 * _log_int(rng, 4, H // 64), "vocab": 8 * _log_int(rng, 125, V // 8),
            "temperature": rng.choice([1.0, 1.0, 0.7]), "grad": grad, "dtype": "bf16" if grad else dtype}


# ------------------------------------------------------------------------------------------ inputs
def _heads(shape, gen, wide, dtype):
    x = torch.randn(shape, generator=gen, device="cuda")
    if wide:   # keys after the norm and the rotation: some channels are larger
        x[..., ::16] *= 4.0
    return x.to(dtype)


def _tokens(rows, vocab, gen, banned=None):
    """One token a row, some rows left out (padding)."""
    t = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
    if banned is not None:   # a token that may not follow is not what followed
        t = torch.where(banned.gather(1, t[:, None])[:, 0], 0, t)
    if rows > 16:
        t[torch.randint(0, rows, (rows // 16,), generator=gen, device="cuda")] = IGNORE
    return t


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    s = {"case": dict(case), "dtype": dtype}
    if case["kind"] == "prefix":
        r, b, seq, start = case["groups"], case["rows"], case["seq"], case["start"]
        cap = -(-(start + seq) // 64) * 64 + 64
        for name, wide in (("k", True), ("v", False)):
            s["prefix_" + name] = _heads((r, HKV, case["prefix"], D), gen, wide, dtype)
            s["cache_" + name] = _heads((b, HKV, cap, D), gen, wide, dtype)
        s["q"] = _heads((b, seq, HQ, D), gen, False, dtype)
        s["starts"] = torch.randint(0, start + 1, (b,), generator=gen, device="cuda") if case["ragged"] else None
        return s
    rows, vocab = case["rows"], case["vocab"]
    # how sure the model is: from rows that are almost certain of their token to flat ones
    sure = torch.rand((rows, 1), generator=gen, device="cuda") ** 2 * 14.0
    if case["kind"] == "logprobs":
        x = torch.randn((rows, vocab), generator=gen, device="cuda") * 2.0
        banned = None
        if case["masked"]:
            banned = torch.rand((rows, vocab), generator=gen, device="cuda") < case["masked"]
            banned[:, 0] = False
        t = _tokens(rows, vocab, gen, banned)
        at = t.clamp_min(0)[:, None]
        x.scatter_(1, at, x.gather(1, at) + sure)
        if banned is not None:
            x.masked_fill_(banned, -math.inf)
        s["logits"] = x.to(dtype)
        del x, banned
    else:
        h = case["h"]
        s["weight"] = (torch.randn((vocab, h), generator=gen, device="cuda") * (1.5 / math.sqrt(h))).to(dtype)
        t = _tokens(rows, vocab, gen)
        x = torch.randn((rows, h), generator=gen, device="cuda")
        x += s["weight"][t.clamp_min(0)].float() * (sure / 2.25)   # |w|^2 is 2.25
        s["hidden"] = x.to(dtype)
    s["tokens"] = t
    if case["grad"]:   # advantages, and the entropy bonus
        s["g"] = torch.randn((rows,), generator=gen, device="cuda")
        s["gh"] = 0.1 * torch.rand((rows,), generator=gen, device="cuda")
        for name in ("logits", "hidden", "weight"):
            if name in s:
                s[name].requires_grad_(True)
    return s


# ------------------------------------------------------------------------------------------ one pass
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _package():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "qwen3-triton_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from qwen3_triton.inference import prefix
    from qwen3_triton.kernels import logprobs
    return prefix, logprobs


def _run_own(s):
    prefix, logprobs = _package()
    case = s["case"]
    if case["kind"] == "prefix":
        return {"o": prefix.attention(s["q"], s["prefix_k"], s["prefix_v"], s["cache_k"], s["cache_v"], case["start"], s["starts"])}
    if case["kind"] == "logprobs":
        leaves = [s["logits"]]
        out = logprobs.token_logprobs(s["logits"], s["tokens"], top=case["top"], temperature=case["temperature"])
    else:
        leaves = [s["hidden"], s["weight"]]
        out = logprobs.lm_head_logprobs(s["hidden"], s["weight"], s["tokens"], temperature=case["temperature"])
    got = {"logprobs": out.logprobs, "entropy": out.entropy}
    if case["grad"]:
        grads = torch.autograd.grad([out.logprobs, out.entropy], leaves, [s["g"], s["gh"]])
        got = {name: x.detach() for name, x in got.items()}
        got.update(zip(("dlogits",) if len(leaves) == 1 else ("dhidden", "dweight"), grads))
    if case.get("top"):
        got.update(top_logprobs=out.top_logprobs, top_tokens=out.top_tokens)
    return got


def _plain_prefix(s):
    case = s["case"]
    r, b, seq, p = case["groups"], case["rows"], case["seq"], case["prefix"]
    n, g, cap = b // r, HQ // HKV, s["cache_k"].shape[2]
    q = s["q"].float().view(b, seq, HKV, g, D).permute(0, 2, 3, 1, 4)   # [B, Hkv, G, S, D]
    shared = q.reshape(r, n, HKV, g * seq, D).transpose(1, 2).reshape(r, HKV, n * g * seq, D)
    zp = torch.matmul(shared, s["prefix_k"].float().transpose(2, 3).contiguous()).view(r, HKV, n, g, seq, p)
    zp = zp.transpose(1, 2).reshape(b, HKV, g, seq, p)
    zc = torch.matmul(q.reshape(b, HKV, g * seq, D), s["cache_k"].float().transpose(2, 3).contiguous()).view(b, HKV, g, seq, cap)
    starts = torch.full((b,), case["start"], device="cuda") if s["starts"] is None else s["starts"]
    last = starts[:, None] + torch.arange(seq, device="cuda")[None, :]
    seen = torch.arange(cap, device="cuda")[None, None, :] <= last[:, :, None]   # [B, S, C]
    zc = torch.where(seen[:, None, None], zc, -math.inf)
    scale = D ** -0.5
    top = torch.maximum(zp.amax(-1, keepdim=True), zc.amax(-1, keepdim=True))
    pp, pc = torch.exp((zp - top) * scale), torch.exp((zc - top) * scale)
    total = pp.sum(-1, keepdim=True) + pc.sum(-1, keepdim=True)
    pp = pp.view(r, n, HKV, g * seq, p).transpose(1, 2).reshape(r, HKV, n * g * seq, p)
    op = torch.matmul(pp, s["prefix_v"].float()).view(r, HKV, n, g, seq, D).transpose(1, 2).reshape(b, HKV, g, seq, D)
    oc = torch.matmul(pc.view(b, HKV, g * seq, cap), s["cache_v"].float()).view(b, HKV, g, seq, D)
    return {"o": ((op + oc) / total).permute(0, 3, 1, 2, 4).reshape(b, seq, HQ, D).to(s["dtype"])}


def _plain_rows(logits, temperature, tokens, top):
    """Of rows of logits in 32 bits: the outputs, and what the gradient needs."""
    x = logits / temperature
    keep = tokens != IGNORE
    at = torch.where(keep, tokens, 0)[:, None]
    d, first = x.max(dim=1, keepdim=True)
    d = x - d
    e = torch.exp(d)
    e.scatter_(1, first, 0.0)                      # the largest term is 1: the others' sum keeps its small parts
    rest = e.sum(1)
    e.scatter_(1, first, 1.0)
    log_total, total = torch.log1p(rest), 1.0 + rest
    weighted = torch.where(e > 0, e * d, 0.0).sum(1)
    entropy = log_total - weighted / total
    logp = d.gather(1, at)[:, 0] - log_total
    got = {"logprobs": torch.where(keep, logp, 0.0), "entropy": torch.where(keep, entropy, 0.0)}
    if top:
        ids = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :top]
        got["top_logprobs"] = torch.where(keep[:, None], d.gather(1, ids) - log_total[:, None], 0.0)
        got["top_tokens"] = torch.where(keep[:, None], ids, 0)
    return got, (keep, at, d, e, total, log_total)


def _plain_grad(s, got, kept):
    keep, at, d, e, total, log_total = kept
    p = e / total[:, None]
    logp = torch.where(e > 0, d - log_total[:, None], 0.0)
    dx = -p * (s["g"][:, None] + s["gh"][:, None] * (logp + got["entropy"][:, None]))
    one = torch.zeros_like(dx).scatter_(1, at, 1.0)
    dx += s["g"][:, None] * one
    return torch.where(keep[:, None], dx, 0.0) / s["case"]["temperature"]


def _run_plain(s):
    with torch.no_grad():
        case = s["case"]
        if case["kind"] == "prefix":
            return _plain_prefix(s)
        if case["kind"] == "logprobs":
            x = s["logits"].float()
        else:
            x = torch.matmul(s["hidden"].float(), s["weight"].float().t())
        got, kept = _plain_rows(x, case["temperature"], s["tokens"], case.get("top", 0))
        if case["grad"]:
            dx = _plain_grad(s, got, kept)
            if case["kind"] == "logprobs":
                got["dlogits"] = dx.to(s["dtype"])
            else:
                got["dhidden"] = torch.matmul(dx, s["weight"].float()).to(s["dtype"])
                got["dweight"] = torch.matmul(dx.t(), s["hidden"].float()).to(s["dtype"])
        return got


# ------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "prefix":
        r, b, seq, p = case["groups"], case["rows"], case["seq"], case["prefix"]
        start = case["start"] / 2 if case["ragged"] else case["start"]   # on average
        held = 2 * HKV * D * (r * p + b * (start + seq)) * size
        pairs = b * (seq * (p + start) + seq * (seq + 1) / 2)
        return {"bytes": int(held) + 2 * b * seq * HQ * D * size, "flops": int(4 * HQ * D * pairs)}
    rows, vocab, top = case["rows"], case["vocab"], case.get("top", 0)
    small = rows * (16 + 12 * top + (8 if case["grad"] else 0))
    if case["kind"] == "logprobs":
        return {"bytes": rows * vocab * size * (2 if case["grad"] else 1) + small, "flops": rows * vocab * (14 if case["grad"] else 6)}
    h = case["h"]
    ways = 2 if case["grad"] else 1
    return {"bytes": ways * size * h * (rows + vocab) + small, "flops": 2 * rows * vocab * h * (3 if case["grad"] else 1)}


# ------------------------------------------------------------------------------------------ the same in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    f64 = torch.float64
    with torch.no_grad():
        if case["kind"] == "prefix":
            b, seq, n, group = case["rows"], case["seq"], case["rows"] // case["groups"], HQ // HKV
            starts = [case["start"]] * b if s["starts"] is None else s["starts"].tolist()
            o = torch.empty((b, seq, HQ, D), dtype=f64, device="cuda")
            for i in range(b):
                for h in range(HKV):
                    end, p = starts[i] + seq, case["prefix"]
                    k = torch.cat((s["prefix_k"][i // n, h], s["cache_k"][i, h, :end])).to(f64)
                    v = torch.cat((s["prefix_v"][i // n, h], s["cache_v"][i, h, :end])).to(f64)
                    q = s["q"][i, :, h * group:(h + 1) * group].to(f64).transpose(0, 1)
                    hidden = torch.ones((seq, p + end), dtype=torch.bool, device="cuda").triu(p + starts[i] + 1)
                    z = (q.reshape(group * seq, D) @ k.t() / math.sqrt(D)).view(group, seq, p + end)
                    w = z.masked_fill(hidden, -math.inf).softmax(-1).view(group * seq, p + end) @ v
                    o[i, :, h * group:(h + 1) * group] = w.view(group, seq, D).transpose(0, 1)
            return {"o": o}
        tokens = s["tokens"]
        left_out = tokens == IGNORE
        x = s["logits"].to(f64) if case["kind"] == "logprobs" else s["hidden"].to(f64) @ s["weight"].to(f64).t()
        x /= case["temperature"]
        logp = x.log_softmax(1)
        p = logp.exp()
        entropy = -(p * logp.clamp_min(-1e300)).sum(1)
        picked = logp.gather(1, tokens.clamp_min(0).unsqueeze(1)).squeeze(1)
        out = {"logprobs": picked.masked_fill(left_out, 0.0), "entropy": entropy.masked_fill(left_out, 0.0)}
        if case.get("top"):
            best = x.sort(dim=1, descending=True, stable=True).indices[:, :case["top"]]
            out["top_logprobs"] = logp.gather(1, best).masked_fill(left_out.unsqueeze(1), 0.0)
            out["top_tokens"] = best.masked_fill(left_out.unsqueeze(1), 0)
        if case["grad"]:
            g, gh = s["g"].to(f64).unsqueeze(1), s["gh"].to(f64).unsqueeze(1)
            grad = logp.clamp_(min=-1e300).add_(entropy.unsqueeze(1)).mul_(gh).add_(g).mul_(p).neg_()
            grad.scatter_add_(1, tokens.clamp_min(0).unsqueeze(1), g)
            grad.masked_fill_(left_out.unsqueeze(1), 0.0).div_(case["temperature"])
            if case["kind"] == "logprobs":
                out["dlogits"] = grad
            else:
                out["dhidden"] = grad @ s["weight"].to(f64)
                out["dweight"] = grad.t() @ s["hidden"].to(f64)
        return out
