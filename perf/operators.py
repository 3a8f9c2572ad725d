"""Performance cases of the 8-bit serving operators (``qwen3_triton.inference.int8``), from one token to 8192.

The shapes are Qwen3-8B's (hidden 4096, intermediate 12288, 32 query and 8 key/value heads of 128).  With ``own``
false, ``run`` computes each operator from elementary torch operations; with ``own`` true it calls the package.

The operators' definitions:

* rows in 8 bits: a row ``a`` of M = max |a| is held as q = the integer nearest to 127 a / M (ties to even) and the
  scale M / 127.  RMSNorm in 8 bits takes t = round(x + residual) to the activation type, a = t * weight, and the
  scale M / 127 / sqrt(mean t^2 + eps): the row's 1 / rms is common to the row and leaves q as it is.
* product in 8 bits: y = round((sum_k q[m, k] w[n, k]) * s[m] * ws[n] (+ residual)); gate/up: silu(g) * u of two such.
* cache in 8 bits: blocks of 64 positions, quantised as a whole like a row, per key/value head, once their last token
  is there; positions of the last, unfinished block stay in the activation type (the tail).  Buffers per layer:
  k [B, Hkv, cap, D], v [B, Hkv, cap / 64, D, 64], scales [B, Hkv, cap / 64], k_tail [B, Hkv, 64, D],
  v_tail [B, Hkv, D, 64].
* attention over it: causal, grouped queries at positions start .. start + S - 1 against positions 0 .. start + S - 1.
"""
import math
import os
import sys

import torch

own = False

H, I, HQ, HKV, D = 4096, 12288, 32, 8, 128   # Qwen3-8B
EPS = 1e-6
BLOCK = 64
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


# ------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # Decoding, one request: the norm before the gate/up projection, with the attention's residual.
        {"name": "norm_b1", "kind": "norm", "rows": 1, "h": H, "residual": True, "dtype": "bf16"},
        # Prefill of four prompts of 2048 tokens: the same norm at 8192 tokens.
        {"name": "norm_t8192", "kind": "norm", "rows": 8192, "h": H, "residual": True, "dtype": "bf16"},
        # A ragged prompt's SwiGLU output, quantised for the down projection.
        {"name": "rows_t1500_f16", "kind": "rows", "rows": 1500, "h": I, "dtype": "f16"},
        # Decoding, one request: the stacked Q/K/V projection.
        {"name": "linear_b1_qkv", "kind": "linear", "m": 1, "n": 6144, "k": H, "residual": False, "dtype": "bf16"},
        # Decoding for 32 users: the down projection with its residual.
        {"name": "linear_b32_down", "kind": "linear", "m": 32, "n": H, "k": I, "residual": True, "dtype": "bf16"},
        # A ragged prompt: the output projection with its residual, in fp16.
        {"name": "linear_t333_f16", "kind": "linear", "m": 333, "n": H, "k": H, "residual": True, "dtype": "f16"},
        # Prefill of four prompts of 2048 tokens: gate/up + SwiGLU, the largest product of a layer.
        {"name": "gate_up_t8192", "kind": "gate_up", "m": 8192, "n": I, "k": H, "dtype": "bf16"},
        # Decoding for 8 users: the token that completes a block, and the cache of 1024 positions read back.
        {"name": "cache_b8_t1024", "kind": "cache", "batch": 8, "start": 1023, "seq": 1, "dtype": "bf16"},
        # A prompt of 8192 tokens written into an empty cache, and read back.
        {"name": "cache_b1_s8192", "kind": "cache", "batch": 1, "start": 0, "seq": 8192, "dtype": "bf16"},
        # Decoding, one request after a 2048-token prompt: the smallest attention, all latency.
        {"name": "attn_b1_t2048", "kind": "attn", "batch": 1, "start": 2047, "seq": 1, "dtype": "bf16"},
        # Decoding for 8 users at a long ragged context.
        {"name": "attn_b8_t20001", "kind": "attn", "batch": 8, "start": 20000, "seq": 1, "dtype": "f16"},
        # A chunk of a long prompt: 1024 queries behind 3000 cached positions.
        {"name": "attn_b1_s1024", "kind": "attn", "batch": 1, "start": 3000, "seq": 1024, "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["norm", "rows", "linear", "linear", "gate_up", "cache", "attn", "attn"])
    dtype = rng.choice(["bf16", "f16"])
    if kind in ("norm", "rows"):
        c = {"kind": kind, "rows": _log_int(rng, 1, 8192), "h": 16 * _log_int(rng, 8, 768 if kind == "rows" else 256), "dtype": dtype}
        if kind == "norm":
            c["residual"] = rng.random() < 0.7
        return c
    if kind in ("linear", "gate_up"):
        c = {"kind": kind, "m": _log_int(rng, 1, 8192), "n": _log_int(rng, 100, I), "k": 16 * _log_int(rng, 16, 768), "dtype": dtype}
        if kind == "linear":
            c["residual"] = rng.random() < 0.5
        else:
            c["n"], c["k"] = 8 * (c["n"] // 8), min(c["k"], H)
        return c
    if kind == "cache":
        batch, seq = _log_int(rng, 1, 8), _log_int(rng, 1, 4096)
        start = rng.choice([0, BLOCK * _log_int(rng, 1, 64), _log_int(rng, 1, 4000)])
        # The chunk starts a block, or ends one, or stays within one: then a second call finds the tail it needs.
        if start % BLOCK and (start % BLOCK + seq) > BLOCK:
            seq = -(-(start + seq) // BLOCK) * BLOCK - start
        return {"kind": kind, "batch": min(batch, max(1, 8192 // (start + seq))), "start": start, "seq": seq, "dtype": dtype}
    seq = rng.choice([1, 1, 1, rng.randint(2, 16), _log_int(rng, 17, 1024)])
    start = _log_int(rng, 1, 3000 if seq > 16 else 20000) - 1
    batch = _log_int(rng, 1, 8) if seq == 1 else 1
    return {"kind": kind, "batch": batch, "start": start, "seq": seq, "dtype": dtype}


# ------------------------------------------------------------------------------------------ inputs
def _activations(rows, h, dtype, gen):
    """Hidden states: a few channels are many times larger than the others, as in trained models."""
    x = torch.randn((rows, h), generator=gen, device="cuda")
    wide = torch.randint(0, h, (max(1, h // 512),), generator=gen, device="cuda")
    x[:, wide] *= 8.0
    return x.to(dtype)


def _codes(rows, k, gen, wide):
    """Rows in 8 bits as a program holds them, with their scales: activations (``wide``) or weight channels."""
    x = torch.randn((rows, k), generator=gen, device="cuda") * (1.0 if wide else 0.02)
    m = x.abs().amax(1)
    return torch.round(x * (127.0 / m)[:, None]).to(torch.int8), m / 127.0


def _heads(shape, gen, wide, dtype):
    x = torch.randn(shape, generator=gen, device="cuda")
    if wide:   # keys after the norm and the rotation: some channels are larger
        x[..., ::16] *= 4.0
    return x.to(dtype)


def _cache_state(batch, length, capacity, dtype, gen):
    """A cache that holds ``length`` positions: whole blocks in 8 bits, the rest in the tail."""
    blocks, full = -(-capacity // BLOCK), length // BLOCK
    c = {
        "k": torch.zeros((batch, HKV, blocks * BLOCK, D), dtype=torch.int8, device="cuda"),
        "v": torch.zeros((batch, HKV, blocks, D, BLOCK), dtype=torch.int8, device="cuda"),
        "k_scale": torch.zeros((batch, HKV, blocks), device="cuda"),
        "v_scale": torch.zeros((batch, HKV, blocks), device="cuda"),
        "k_tail": torch.zeros((batch, HKV, BLOCK, D), dtype=dtype, device="cuda"),
        "v_tail": torch.zeros((batch, HKV, D, BLOCK), dtype=dtype, device="cuda"),
    }
    if full:
        k = _heads((batch, HKV, full, BLOCK * D), gen, True, dtype).float()
        v = _heads((batch, HKV, full, BLOCK * D), gen, False, dtype).float()
        for name, x in (("k", k), ("v", v)):
            m = x.abs().amax(-1)
            q = torch.round(x * (127.0 / m)[..., None]).to(torch.int8).view(batch, HKV, full, BLOCK, D)
            c[name + "_scale"][:, :, :full] = m / 127.0
            if name == "k":
                c["k"][:, :, :full * BLOCK] = q.reshape(batch, HKV, full * BLOCK, D)
            else:
                c["v"][:, :, :full] = q.transpose(3, 4)
    rest = length - full * BLOCK
    if rest:
        c["k_tail"][:, :, :rest] = _heads((batch, HKV, rest, D), gen, True, dtype)
        c["v_tail"][:, :, :, :rest] = _heads((batch, HKV, D, rest), gen, False, dtype)
    return c


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    kind = case["kind"]
    s = {"case": dict(case), "dtype": dtype}
    if kind in ("norm", "rows"):
        s["x"] = _activations(case["rows"], case["h"], dtype, gen)
        if kind == "norm":
            s["w"] = (1.0 + 0.1 * torch.randn((case["h"],), generator=gen, device="cuda")).to(dtype)
            s["res"] = _activations(case["rows"], case["h"], dtype, gen) if case["residual"] else None
    elif kind in ("linear", "gate_up"):
        s["q"], s["s"] = _codes(case["m"], case["k"], gen, True)
        s["w"] = [_codes(case["n"], case["k"], gen, False) for _ in range(2 if kind == "gate_up" else 1)]
        s["res"] = torch.randn((case["m"], case["n"]), generator=gen, device="cuda").to(dtype) if case.get("residual") else None
    elif kind == "cache":
        b, start, seq = case["batch"], case["start"], case["seq"]
        s["cache"] = _cache_state(b, start, start + seq, dtype, gen)
        s["k"] = _heads((b, seq, HKV, D), gen, True, dtype)
        s["v"] = _heads((b, seq, HKV, D), gen, False, dtype)
    else:
        b, start, seq = case["batch"], case["start"], case["seq"]
        s["cache"] = _cache_state(b, start + seq, start + seq, dtype, gen)
        s["q"] = _heads((b, seq, HQ, D), gen, False, dtype)
    return s


# ------------------------------------------------------------------------------------------ one pass
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _package():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "qwen3-triton_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from qwen3_triton.inference import int8
    return int8


def _run_own(s):
    ops = _package()
    case, kind = s["case"], s["case"]["kind"]
    if kind == "rows":
        q, scale = ops.quantize_rows(s["x"])
        return {"values": q * scale[:, None]}
    if kind == "norm":
        if s["res"] is None:
            q, scale = ops.rms_norm(s["x"], s["w"], EPS)
            return {"values": q * scale[:, None]}
        q, scale, total = ops.rms_norm(s["x"], s["w"], EPS, residual=s["res"])
        return {"values": q * scale[:, None], "total": total}
    if kind == "linear":
        (w, ws), = s["w"]
        return {"y": ops.linear(s["q"], s["s"], w, ws, dtype=s["dtype"], residual=s["res"])}
    if kind == "gate_up":
        (wg, sg), (wu, su) = s["w"]
        return {"y": ops.gate_up_swiglu(s["q"], s["s"], wg, sg, wu, su, dtype=s["dtype"])}
    cache = ops.LayerCache(**s["cache"])
    if kind == "cache":
        ops.append(s["k"], s["v"], cache, case["start"])
        k, v = ops.read(cache, case["start"] + case["seq"])
        return {"k": k, "v": v}
    return {"o": ops.attention(s["q"], cache, case["start"])}


def _nearest(a, m):
    """The integers nearest to 127 a / m, by whole rows of the last axis (64 bits: values next to a border)."""
    a, m = a.double(), m.double()
    return torch.round(torch.where(m > 0, 127.0 * a / m, 0.0))


def _plain_block(x):
    """[..., 64, D] in the activation type -> (codes, scale)."""
    m = x.float().abs().amax((-2, -1))
    return _nearest(x, m[..., None, None]).to(torch.int8), m / 127.0


def _plain_append(k, v, c, start):
    b, seq, heads, d = k.shape
    end, first = start + seq, start // BLOCK
    full, off = end // BLOCK, start - first * BLOCK
    # the positions from the first touched block on: what the tail holds of it, then the new ones
    ks = torch.cat([c["k_tail"][:, :, :off], k.transpose(1, 2)], 2)
    vs = torch.cat([c["v_tail"][:, :, :, :off].transpose(2, 3), v.transpose(1, 2)], 2)
    n = full - first
    if n > 0:
        q, scale = _plain_block(ks[:, :, :n * BLOCK].reshape(b, heads, n, BLOCK, d))
        c["k"][:, :, first * BLOCK:full * BLOCK] = q.reshape(b, heads, n * BLOCK, d)
        c["k_scale"][:, :, first:full] = scale
        q, scale = _plain_block(vs[:, :, :n * BLOCK].reshape(b, heads, n, BLOCK, d))
        c["v"][:, :, first:full] = q.transpose(3, 4)
        c["v_scale"][:, :, first:full] = scale
    rest = ks.shape[2] - max(n, 0) * BLOCK
    if rest:
        c["k_tail"][:, :, :rest] = ks[:, :, -rest:]
        c["v_tail"][:, :, :, :rest] = vs[:, :, -rest:].transpose(2, 3)


def _plain_read(c, length):
    """Keys and values [B, Hkv, length, D] in 32 bits."""
    b, heads, _, d = c["k"].shape
    full = length // BLOCK
    rest = length - full * BLOCK
    k = c["k"][:, :, :full * BLOCK].float().view(b, heads, full, BLOCK, d) * c["k_scale"][:, :, :full, None, None]
    v = c["v"][:, :, :full].float().transpose(3, 4) * c["v_scale"][:, :, :full, None, None]
    k, v = k.reshape(b, heads, full * BLOCK, d), v.reshape(b, heads, full * BLOCK, d)
    if rest:
        k = torch.cat([k, c["k_tail"][:, :, :rest].float()], 2)
        v = torch.cat([v, c["v_tail"][:, :, :, :rest].transpose(2, 3).float()], 2)
    return k, v


def _run_plain(s):
    case, kind, dtype = s["case"], s["case"]["kind"], s["dtype"]
    if kind in ("norm", "rows"):
        t = s["x"]
        if s.get("res") is not None:
            t = (t.float() + s["res"].float()).to(dtype)
        a = t.float() * s["w"].float() if kind == "norm" else t.float()
        m = a.abs().amax(1)
        scale = m / 127.0
        if kind == "norm":
            scale = scale * torch.rsqrt(t.float().square().mean(1) + EPS)
        values = _nearest(a, m[:, None]).to(torch.int8) * scale[:, None]
        return {"values": values, "total": t} if s.get("res") is not None else {"values": values}
    if kind in ("linear", "gate_up"):
        x = s["q"].float()
        ys = [torch.matmul(x, w.float().t()) * s["s"][:, None] * ws for w, ws in s["w"]]
        if kind == "gate_up":
            return {"y": (ys[0] / (1.0 + torch.exp(-ys[0])) * ys[1]).to(dtype)}
        y = ys[0]
        if s["res"] is not None:
            y = y + s["res"].float()
        return {"y": y.to(dtype)}
    start, seq = case["start"], case["seq"]
    if kind == "cache":
        _plain_append(s["k"], s["v"], s["cache"], start)
        k, v = _plain_read(s["cache"], start + seq)
        return {"k": k.to(dtype), "v": v.to(dtype)}
    k, v = _plain_read(s["cache"], start + seq)
    b, g, total = case["batch"], HQ // HKV, start + seq
    q = s["q"].float().view(b, seq, HKV, g, D).permute(0, 2, 3, 1, 4).reshape(b, HKV, g * seq, D)
    z = torch.matmul(q, k.transpose(2, 3).contiguous()).view(b, HKV, g, seq, total) * D ** -0.5
    if seq > 1:
        pos = torch.arange(total, device="cuda")
        z = torch.where(pos[None, :] <= start + torch.arange(seq, device="cuda")[:, None], z, -math.inf)
    p = torch.exp(z - z.amax(-1, keepdim=True))
    o = torch.matmul(p.view(b, HKV, g * seq, total), v).view(b, HKV, g, seq, D) / p.sum(-1, keepdim=True)
    return {"o": o.permute(0, 3, 1, 2, 4).reshape(b, seq, HQ, D).to(dtype)}


# ------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    kind = case["kind"]
    if kind in ("norm", "rows"):
        r, h = case["rows"], case["h"]
        per = 3 + (4 if case.get("residual") else 0)
        return {"bytes": r * h * per + 4 * r + (2 * h if kind == "norm" else 0), "flops": 6 * r * h}
    if kind in ("linear", "gate_up"):
        m, n, k = case["m"], case["n"], case["k"]
        ws = 2 if kind == "gate_up" else 1
        out = m * n * (4 if case.get("residual") else 2)
        return {"bytes": m * k + ws * n * k + 4 * (m + ws * n) + out, "flops": 2 * m * n * k * ws}
    b, start, seq = case["batch"], case["start"], case["seq"]
    total = start + seq
    held = 2 * b * HKV * D * total
    if kind == "cache":
        # the new tokens in, their codes out; the whole cache in, its values in 16 bits out
        return {"bytes": 2 * b * HKV * D * seq * 3 + held * 3, "flops": 2 * held}
    pairs = seq * start + seq * (seq + 1) // 2
    return {"bytes": held + 4 * b * seq * HQ * D, "flops": 4 * b * HQ * D * pairs}


# ------------------------------------------------------------------------------------------ the same in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    kind, f64 = case["kind"], torch.float64
    if kind in ("norm", "rows"):
        total = None
        t = s["x"].to(f64)
        if s.get("res") is not None:
            total = t + s["res"].to(f64)
            t = total.to(s["dtype"]).to(f64)   # the sum of two 16-bit numbers rounds once, from 64 bits as from 32
        a = t * s["w"].to(f64) if kind == "norm" else t
        top = a.abs().max(dim=1, keepdim=True).values
        values = (127.0 * a / top).round() * (top / 127.0)
        if kind == "norm":
            values = values / (t.pow(2).mean(dim=1, keepdim=True) + EPS).sqrt()
        return {"values": values} if total is None else {"values": values, "total": total}
    if kind in ("linear", "gate_up"):
        y = [(s["q"].to(f64) @ w.to(f64).t()) * s["s"].to(f64).unsqueeze(1) * ws.to(f64).unsqueeze(0) for w, ws in s["w"]]
        if kind == "gate_up":
            return {"y": y[0] * torch.sigmoid(y[0]) * y[1]}
        return {"y": y[0] if s["res"] is None else y[0] + s["res"].to(f64)}
    start, seq, c = case["start"], case["seq"], s["cache"]
    total = start + seq
    if kind == "cache":
        out = {}
        for name in ("k", "v"):
            new, held = s[name].to(f64), start // BLOCK
            scale = c[name + "_scale"][:, :, :held].to(f64)
            if name == "k":
                old = c["k"][:, :, :held * BLOCK].to(f64) * scale.repeat_interleave(BLOCK, 2).unsqueeze(3)
                tail = c["k_tail"][:, :, :start % BLOCK].to(f64)
            else:
                old = (c["v"][:, :, :held].to(f64) * scale[..., None, None]).permute(0, 1, 2, 4, 3).flatten(2, 3)
                tail = c["v_tail"][..., :start % BLOCK].to(f64).permute(0, 1, 3, 2)
            fresh = torch.cat((tail, new.permute(0, 2, 1, 3)), 2)
            pieces = [old]
            for piece in fresh.split(BLOCK, 2):
                if piece.shape[2] == BLOCK:
                    top = piece.abs().flatten(2).max(2).values[..., None, None]
                    held_scale = (top.float() / 127.0).to(f64)   # a scale is a 32-bit number
                    piece = (127.0 * piece / top).round() * held_scale
                pieces.append(piece)
            out[name] = torch.cat(pieces, 2)
        return out
    full, group = total // BLOCK, HQ // HKV
    o = torch.empty((case["batch"], seq, HQ, D), dtype=f64, device="cuda")
    visible = torch.ones((seq, total), dtype=torch.bool, device="cuda").tril(start)
    for b in range(case["batch"]):
        for h in range(HKV):
            ks = c["k_scale"][b, h, :full].to(f64).repeat_interleave(BLOCK)
            vs = c["v_scale"][b, h, :full].to(f64).repeat_interleave(BLOCK)
            k = torch.cat((c["k"][b, h, :full * BLOCK].to(f64) * ks[:, None], c["k_tail"][b, h, :total - full * BLOCK].to(f64)))
            v = c["v"][b, h, :full].to(f64).permute(0, 2, 1).flatten(0, 1) * vs[:, None]
            v = torch.cat((v, c["v_tail"][b, h, :, :total - full * BLOCK].to(f64).t()))
            for j in range(h * group, (h + 1) * group):
                z = s["q"][b, :, j].to(f64) @ k.t() / math.sqrt(D)
                o[b, :, j] = z.masked_fill(~visible, -math.inf).softmax(dim=1) @ v
    return {"o": o}
