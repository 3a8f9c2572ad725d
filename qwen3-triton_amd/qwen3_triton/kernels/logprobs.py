"""Log probabilities of given tokens, with the entropy of their distributions and the most likely alternatives, from logits or
straight from hidden states and the LM head's weight; differentiable.

Of each row, with p = softmax(logits / temperature): log p[token], -sum p log p, and the ``top`` largest log p with their tokens
(equal logits: the lower token first).  Everything is formed and returned in fp32.  The reference has a mean cross-entropy and
an argmax only; nothing here has a counterpart in it.
"""
from typing import NamedTuple, Optional

import torch
import torch.autograd.forward_ad as _forward_ad
from torch.autograd.function import once_differentiable

from .. import _hip as H
from ._ops import cast, ce_shift_labels
from .linear import MAX_LD, gemm, gemm_nt_into, gemm_ok, matmul_into

MAX_TOP = 32
MAX_GRAD_VOCAB = MAX_LD - 64   # of lm_head_logprobs: what the products with the logits' gradient take, whichever of them run
IGNORE_INDEX = -100
_FLOATS = (torch.float32, torch.bfloat16, torch.float16)


class TokenLogprobs(NamedTuple):
    """Of tokens [...]: ``logprobs`` and ``entropy`` fp32 [...], and with ``top`` = K > 0 the K most likely tokens in order,
    ``top_logprobs`` fp32 and ``top_tokens`` int64 [..., K] (else None)."""
    logprobs: torch.Tensor
    entropy: torch.Tensor
    top_logprobs: Optional[torch.Tensor] = None
    top_tokens: Optional[torch.Tensor] = None


def _check_options(vocab, top, temperature, ignore_index):
    if type(top) is not int or not 0 <= top <= min(MAX_TOP, vocab):
        raise ValueError(f'top must be an int in [0, {min(MAX_TOP, vocab)}]')
    if vocab >= 1 << 30:
        raise ValueError('fewer than 2^30 tokens required')
    if not 1e-6 <= temperature <= 1e6:
        raise ValueError('a temperature in [1e-6, 1e6] required')
    if type(ignore_index) is not int:
        raise ValueError('ignore_index must be an int')


def _check_tokens(tokens, shape, ref):
    if tokens.dtype != torch.int64 or tokens.shape != shape or tokens.device != ref.device or not tokens.is_contiguous():
        raise ValueError(f'contiguous int64 tokens {tuple(shape)} on the same device required')


def _logit_rows(logits):
    """logits [..., V] as (rows, row stride, V): rows at one stride, each contiguous."""
    v = logits.shape[-1]
    rows = logits.numel() // v
    if logits.is_contiguous():
        return rows, v, v
    try:
        m = logits.view(rows, v)
    except RuntimeError:
        raise ValueError('logits whose rows lie at one stride required; no hidden layout copy') from None
    if v > 1 and m.stride(1) != 1 or rows > 1 and m.stride(0) < v:
        raise ValueError('contiguous rows of logits that do not overlap required; no hidden layout copy')
    return rows, m.stride(0) if rows > 1 else v, v


def _forward(z, rows, ld, v, tokens, ignore_index, temperature, top, keep, outs=None, at=0):
    """q3_token_logprobs of rows of z -> (log probability, entropy, alternatives' log probabilities, their tokens, [row maximum, row
    log] where ``keep`` says that a gradient needs them); into rows ``at`` .. of ``outs`` where those are given."""
    if outs is None:
        outs = _outputs(z, rows, top, keep)
    lp, ent, tlp, tid, kept = outs
    nbytes = H.query("q3_token_logprobs_workspace_bytes", H.code(z.dtype), rows, v, top)
    ws = H.workspace(nbytes, z.device) if nbytes else None
    m, ls = (None, None) if kept is None else (kept.data_ptr() + 4 * at, kept.data_ptr() + 4 * (kept.shape[1] + at))
    H.launch(z, "q3_token_logprobs", H.code(z.dtype), z.data_ptr(), ld, rows, v, tokens.data_ptr() + 8 * at, ignore_index,
             1.0 / temperature, top, lp.data_ptr() + 4 * at, ent.data_ptr() + 4 * at, m, ls,
             None if tlp is None else tlp.data_ptr() + 4 * top * at, None if tid is None else tid.data_ptr() + 8 * top * at,
             None if ws is None else ws.data_ptr(), nbytes)
    return outs


def _outputs(ref, rows, top, keep):
    f = torch.float32
    return (ref.new_empty(rows, dtype=f), ref.new_empty(rows, dtype=f), ref.new_empty((rows, top), dtype=f) if top else None,
            ref.new_empty((rows, top), dtype=torch.int64) if top else None, ref.new_empty((2, rows), dtype=f) if keep else None)


def _shaped(shape, top, lp, ent, tlp, tid, _=None):
    """The results for tokens of ``shape``."""
    if len(shape) != 1:
        lp, ent = lp.view(shape), ent.view(shape)
        if top:
            tlp, tid = tlp.view(*shape, top), tid.view(*shape, top)
    return lp, ent, tlp, tid


def _backward(z, rows, ld, v, tokens, ignore_index, temperature, top, top_tokens, kept, ent, g, gh, gtop, dz, ldo, at=0, scale=None):
    """q3_token_logprobs_bwd of rows ``at`` .. ``at`` + rows - 1 (z and dz start there), times ``scale``."""
    def p(t, width=4):
        return None if t is None else t.data_ptr() + at * width
    args = (H.code(z.dtype), H.code(dz.dtype), z.data_ptr(), ld, rows, v, p(tokens, 8), ignore_index, 1.0 / temperature, top,
            p(top_tokens, 8 * top), p(kept), p(kept[1]), p(ent), p(g), p(gh), p(gtop, 4 * top), dz.data_ptr(), ldo)
    if scale is None:
        H.launch(z, "q3_token_logprobs_bwd", *args)
    else:
        H.launch(z, "q3_token_logprobs_bwd_scaled", *args, scale.data_ptr())


def _upstream(g):
    return None if g is None else g.float().contiguous()


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, ignore_index, temperature, top):
        rows, ld, v = _logit_rows(logits)
        outs = _forward(logits, rows, ld, v, tokens, ignore_index, temperature, top, True)
        ctx.save_for_backward(logits, tokens, outs[4], outs[1], outs[3])
        ctx.rest = ignore_index, temperature, top
        ctx.set_materialize_grads(False)
        lp, ent, tlp, tid = _shaped(logits.shape[:-1], top, *outs)
        if not top:
            return lp, ent
        ctx.mark_non_differentiable(tid)
        return lp, ent, tlp, tid

    @staticmethod
    @once_differentiable
    def backward(ctx, g, gh, gtop=None, _=None):
        logits, tokens, kept, ent, tid = ctx.saved_tensors
        ignore_index, temperature, top = ctx.rest
        rows, ld, v = _logit_rows(logits)
        dz = torch.empty(logits.shape, device=logits.device, dtype=logits.dtype)
        _backward(logits, rows, ld, v, tokens, ignore_index, temperature, top, tid, kept, ent, _upstream(g), _upstream(gh),
                  _upstream(gtop), dz, v)
        return dz, None, None, None, None


def _recorded(*tensors):
    """Whether autograd has to see a call on these (a forward-mode tangent has to, to be refused)."""
    return torch.is_grad_enabled() and any(t.requires_grad for t in tensors) or _forward_ad._current_level >= 0


def token_logprobs(logits, tokens, *, top=0, temperature=1.0, ignore_index=IGNORE_INDEX):
    """``TokenLogprobs`` of tokens [...] (int64) under logits [..., V] in fp32, bf16 or fp16 (rows at one stride, such as
    ``logits[:, -1]``); nothing is shifted: row i's token is what row i's logits predict.

    A position whose token is ``ignore_index`` is left out: zeros, and no gradient.  Any other token outside [0, V) has the log
    probability NaN (it is not looked for on the host: nothing here synchronises), and so has every token of a row that holds
    a NaN or +inf or only -inf.  Logits of -inf (tokens ruled out) have probability 0.  The gradient reaches the logits from all
    of ``logprobs``, ``entropy`` and ``top_logprobs``."""
    if logits.ndim < 1 or logits.numel() < 1:
        raise ValueError('nonempty [..., V] logits required')
    H.require_device(logits)
    if logits.dtype not in _FLOATS:
        raise TypeError(f'float32, bfloat16 or float16 logits required, not {logits.dtype}')
    shape, temperature = logits.shape[:-1], float(temperature)
    _check_options(logits.shape[-1], top, temperature, ignore_index)
    _check_tokens(tokens, shape, logits)
    rows, ld, v = _logit_rows(logits)
    if _recorded(logits):
        return TokenLogprobs(*_TokenLogprobs.apply(logits, tokens, ignore_index, temperature, top))
    return TokenLogprobs(*_shaped(shape, top, *_forward(logits, rows, ld, v, tokens, ignore_index, temperature, top, False)))


# ---------------------------------------------------------------- from hidden states
_CHUNK_BYTES = 1 << 30   # of fp32 logits at a time


def _chunks(rows, v):
    step = max(1, min(rows, _CHUNK_BYTES // (4 * v)))
    step = step if step == rows or step < 256 else step // 256 * 256
    return [(r, min(r + step, rows)) for r in range(0, rows, step)]


def _logits(x, w, z):
    """z = x w^T in fp32."""
    if x.dtype != torch.float32 and x.shape[1] % 8 == 0 and x.data_ptr() % 16 == 0 and w.data_ptr() % 16 == 0:
        gemm_nt_into(x, x.shape[1], w, w.shape[1], z, x.shape[0], w.shape[0], x.shape[1])
    else:
        matmul_into(x, w.t(), z)


def _fused_ok(x, w, top):
    """The logits' product with their statistics in its epilogue (matrix cores; alternatives need whole rows of logits)."""
    return not top and x.shape[1] % 64 == 0 and gemm_ok(x, w) and w.shape[0] % 8 == 0 and w.shape[0] < MAX_LD and x.shape[0] < (1 << 31) - 256


def _fused_product(x, w, tokens, temperature, store):
    """(maxima [groups of 128 columns, T], the groups' other two statistics, logits of the tokens, 16 bits of each logit [T, V]
    for the gradient or None)"""
    t, h = x.shape
    v = w.shape[0]
    f = torch.float32
    groups = x.new_empty((-(-v // 128), t), dtype=f)
    rest = x.new_empty((2 * groups.numel() + t,), dtype=f)
    z = x.new_empty((t, v)) if store else None   # 16 bits; the gradient takes its place
    p, step = rest.data_ptr(), 4 * groups.numel()
    H.call("q3_gemm_nt_logprobs", H.code(x.dtype), x.data_ptr(), h, w.data_ptr(), h, t, v, h, tokens.data_ptr(), 1.0 / temperature,
           groups.data_ptr(), p, p + step, p + 2 * step, t, None if z is None else z.data_ptr(), v, H.stream())
    return groups, rest, z


def _head_forward(x, weight, tokens, ignore_index, temperature, top, keep):
    """(``_forward``'s results, the fused form's (groups' maxima, stored logits))"""
    t, v = x.shape[0], weight.shape[0]
    with H.on(x):
        if _fused_ok(x, weight, top):
            outs = _outputs(x, t, 0, True)
            groups, rest, z = _fused_product(x, weight, tokens, temperature, keep)
            p, step, kept = rest.data_ptr(), 4 * groups.numel(), outs[4].data_ptr()
            H.call("q3_head_logprobs_finish", groups.data_ptr(), p, p + step, t, p + 2 * step, t, v, tokens.data_ptr(), ignore_index,
                   1.0 / temperature, outs[0].data_ptr(), outs[1].data_ptr(), kept, kept + 4 * t, H.stream())
            return outs, (groups, z)
        outs = _outputs(x, t, top, keep)
        chunks = _chunks(t, v)
        z = torch.empty((chunks[0][1], v), device=x.device, dtype=torch.float32)
        for r, end in chunks:
            _logits(x[r:end], weight, z[:end - r])
            _forward(z, end - r, v, v, tokens, ignore_index, temperature, top, keep, outs, r)
    return outs, (None, None)


class _LMHeadLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, tokens, ignore_index, temperature, top):
        outs, (groups, z) = _head_forward(hidden.view(-1, weight.shape[1]), weight, tokens, ignore_index, temperature, top, True)
        ctx.save_for_backward(hidden, weight, tokens, outs[4], outs[1], outs[3], groups, outs[0] if groups is not None else None, z)
        ctx.rest, ctx.consumed, ctx.captured = (ignore_index, temperature, top), False, False
        ctx.set_materialize_grads(False)
        lp, ent, tlp, tid = _shaped(hidden.shape[:-1], top, *outs)
        if not top:
            return lp, ent
        ctx.mark_non_differentiable(tid)
        return lp, ent, tlp, tid

    @staticmethod
    @once_differentiable
    def backward(ctx, g, gh, gtop=None, _=None):
        hidden, weight, tokens, kept, ent, tid, groups, lp, z = ctx.saved_tensors
        ignore_index, temperature, top = ctx.rest
        v, h = weight.shape
        x = hidden.view(-1, h)
        t = x.shape[0]
        g, gh, gtop = _upstream(g), _upstream(gh), _upstream(gtop)
        again = ctx.consumed
        ctx.captured = ctx.captured or torch.cuda.is_current_stream_capturing()
        ctx.consumed = again or not ctx.captured
        with H.on(x):
            dx = torch.empty_like(x) if ctx.needs_input_grad[0] else None
            scale = _grad_scale(x, g, gh, gtop, v, top, tokens, ignore_index, temperature)
            if groups is not None:
                if again:   # a second backward: the same logits once more
                    z = _fused_product(x, weight, tokens, temperature, True)[2]
                # The gradient takes the stored logits' place, except where replays of a captured pass read them again.
                dz = z if ctx.consumed else torch.empty_like(z)
                H.call("q3_head_logprobs_grad", H.code(x.dtype), z.data_ptr(), v, dz.data_ptr(), v, t, v, tokens.data_ptr(), ignore_index,
                       1.0 / temperature, groups.data_ptr(), t, kept.data_ptr(), kept.data_ptr() + 4 * t, lp.data_ptr(), ent.data_ptr(),
                       None if g is None else g.data_ptr(), None if gh is None else gh.data_ptr(), _address(scale), H.stream())
                dw = _products(dz, x, weight, dx, ctx.needs_input_grad[1], scale)
            else:
                whole = gemm_ok(x, weight) and v % 8 == 0   # dW = dz^T x and dX = dz W from one dz [T, V]
                chunks = _chunks(t, v)
                z = torch.empty((chunks[0][1], v), device=x.device, dtype=torch.float32)
                dz = torch.empty((t if whole else chunks[0][1], v), device=x.device, dtype=x.dtype)
                dw = part = None
                if not whole and ctx.needs_input_grad[1]:
                    dw = torch.empty((v, h), device=x.device, dtype=torch.float32)
                if not whole and dx is not None and scale is not None:
                    part = torch.empty((chunks[0][1], h), device=x.device, dtype=torch.float32)
                for r, end in chunks:
                    n, at = end - r, r if whole else 0
                    _logits(x[r:end], weight, z[:n])
                    _backward(z, n, v, v, tokens, ignore_index, temperature, top, tid, kept, ent, g, gh, gtop, dz[at:], v, r, scale)
                    if not whole and dx is not None:
                        matmul_into(dz[:n], weight, dx[r:end] if part is None else part[:n])
                        if part is not None:
                            _unscale(part[:n], dx[r:end], scale)
                    if dw is not None:
                        matmul_into(dz[:n].t(), x[r:end], dw, accumulate=r > 0)
                if whole:
                    dw = _products(dz, x, weight, dx, ctx.needs_input_grad[1], scale)
                elif dw is not None and scale is not None:
                    dw = _unscale(dw, torch.empty_like(weight), scale)
                elif dw is not None and dw.dtype != weight.dtype:
                    dw = cast(dw, weight.dtype)
        return None if dx is None else dx.view(hidden.shape), dw, None, None, None, None


def _address(t):
    return None if t is None else t.data_ptr()


def _grad_scale(x, g, gh, gtop, v, top, tokens, ignore_index, temperature):
    """[factor, its inverse] of the logits' gradient in fp16, chosen on the device from the upstream gradients; None for types with
    fp32's exponents.  Single values of it, p g, would be lost where dX and dW, which sum over them, are not."""
    if x.dtype != torch.float16:
        return None
    scale = x.new_empty(2, dtype=torch.float32)
    H.call("q3_logprobs_grad_scale", _address(g), _address(gh), _address(gtop), x.shape[0], v, top, tokens.data_ptr(), ignore_index,
           1.0 / temperature, scale.data_ptr(), H.stream())
    return scale


def _unscale(x, out, scale):
    H.call("q3_unscale_f16", x.data_ptr(), out.data_ptr(), x.numel(), scale.data_ptr(), H.stream())
    return out


def _products(dz, x, weight, dx, need_dw, scale):
    """dX = dz W into ``dx`` (None: not wanted); returns dW = dz^T x or None.  ``scale``: that of dz."""
    (t, v), h = dz.shape, x.shape[1]
    inverse = None if scale is None else scale.data_ptr() + 4
    if dx is not None:
        gemm([dz], [weight], [dx], t, h, v, kmajor=(False, True), long_k=True, scale=inverse)
    if not need_dw:
        return None
    dw = torch.empty_like(weight)
    gemm([dz], [x], [dw], v, h, t, kmajor=(True, True), scale=inverse)
    return dw


def lm_head_logprobs(hidden, weight, tokens, *, top=0, temperature=1.0, ignore_index=IGNORE_INDEX):
    """``token_logprobs`` of the logits ``hidden @ weight.T`` (hidden [..., H], weight [V, H], both fp32, bf16 or fp16), which
    are formed in fp32; the gradient reaches hidden and weight (V up to 2^22 - 64).

    16-bit operands with H a multiple of 64 and V of 8, without alternatives: the results are formed beside the product, and no
    logits are written unless a gradient is wanted; then 16 bits of each are kept for it (their distance to the largest of 128),
    which its own rounding takes the place of.  Otherwise the logits are written in fp32, 1 GiB of rows at a time.  The products
    that give the gradient take the logits' in the operands' type, in fp16 at a scale of its own: no loss scale is needed for it."""
    if hidden.ndim < 1 or weight.ndim != 2 or hidden.numel() < 1 or weight.numel() < 1 or hidden.shape[-1] != weight.shape[1]:
        raise ValueError('nonempty hidden [..., H] and weight [V, H] required')
    H.require_device(hidden, weight)
    if hidden.dtype not in _FLOATS or weight.dtype != hidden.dtype:
        raise TypeError(f'hidden and weight of one dtype, float32, bfloat16 or float16, required, not {hidden.dtype} and {weight.dtype}')
    if not hidden.is_contiguous() or not weight.is_contiguous():
        raise ValueError('contiguous hidden and weight required; no hidden layout copy')
    temperature = float(temperature)
    _check_options(weight.shape[0], top, temperature, ignore_index)
    _check_tokens(tokens, hidden.shape[:-1], hidden)
    if _recorded(hidden, weight):
        if weight.shape[0] > MAX_GRAD_VOCAB:
            raise ValueError(f'a gradient takes at most {MAX_GRAD_VOCAB} tokens')
        return TokenLogprobs(*_LMHeadLogprobs.apply(hidden, weight, tokens, ignore_index, temperature, top))
    return TokenLogprobs(*_shaped(hidden.shape[:-1], top, *_head_forward(hidden.view(-1, weight.shape[1]), weight, tokens, ignore_index,
                                                                         temperature, top, False)[0]))


def shifted_logprobs(hidden, weight, labels, *, ignore_index=IGNORE_INDEX, **options):
    """``lm_head_logprobs`` of a causal model: of labels[:, 1:] (labels int64 [B, S]) after hidden[:, :-1], [B, S - 1].  ``options``: its
    others.  The hidden states are taken as they lie; the last ones of each row are left out."""
    H.require_device(hidden, weight)
    if hidden.ndim != 3:
        raise ValueError('hidden states [B, S, H] required')
    _check_tokens(labels, hidden.shape[:2], hidden)
    with H.on(labels):
        tokens = ce_shift_labels(labels, ignore_index).view(labels.shape)
    out = lm_head_logprobs(hidden, weight, tokens, ignore_index=ignore_index, **options)
    return TokenLogprobs(*(None if t is None else t[:, :-1] for t in out))
