"""Serving in 8 bits: rows, RMSNorm, matrix products and a key/value cache in int8 with fp32 scales, and attention over
that cache.  Forward only (inputs that require a gradient or carry a tangent are refused); bf16 or fp16 around the codes.

One rule for every group of values with one scale (a token's row, a weight's output channel, 64 cached positions of a
head): with M the largest magnitude, a value is held as the integer nearest to 127 a / M (ties to even) and the scale is
M / 127.  A group that holds an infinity or a NaN gets the scale NaN, and what is formed from it is NaN.

``TritonQwen3Inference.quantize_weights`` and ``new_cache(..., dtype=torch.int8)`` run the model on these.  The reference
serves in 16 bits only; nothing here has a counterpart in it.
"""
from dataclasses import dataclass

import torch
import torch.autograd.forward_ad as _forward_ad

from .. import _hip as H

KV_BLOCK = 64     # cached positions that share a scale
MAX_ROW = 32768   # values that quantize_rows / rms_norm take per row
MAX_K = 1 << 17   # int32 sums of products of 8-bit codes stay exact below

_FLOATS = (torch.bfloat16, torch.float16)


def _dual(t):
    """Whether t carries a tangent of forward-mode differentiation (which torch.no_grad does not end)."""
    return _forward_ad._current_level >= 0 and _forward_ad.unpack_dual(t).tangent is not None


def _forward_only(*tensors):
    if torch.is_grad_enabled() or _forward_ad._current_level >= 0:
        for t in tensors:
            if t is not None and (t.requires_grad and torch.is_grad_enabled() or _dual(t)):
                raise ValueError('operators of inference are forward only: run them under torch.no_grad or detach the inputs')


def _launch(t, name, *args):
    """Launch on t's device and its current stream (appended to ``args``), whatever device is current."""
    if t.get_device() == torch._C._cuda_getDevice():
        return H.call(name, *args, H.stream())
    with torch.cuda.device(t.device):
        return H.call(name, *args, H.stream())


def _on_device(x, *others):
    """x on a ROCm device and the others beside it (the quick form of ``_hip.require_device``, which names what is wrong)."""
    dev = x.get_device()
    if dev < 0:
        H.require_device(x)
    for t in others:
        if t.get_device() != dev:
            H.require_device(x, t)


def _require_float(t, what):
    if t.dtype not in _FLOATS:
        raise TypeError(f'{what}: bfloat16 or float16 required, not {t.dtype}')


def _rows(x, what):
    """x [..., K] as (rows, row stride, K): whole rows of 16-byte chunks at one stride."""
    k, n = x.shape[-1] if x.ndim else 0, x.numel()
    if n == 0:
        raise ValueError(f'{what}: nonempty [..., K] required')
    rows, ld = n // k, k
    if not x.is_contiguous():
        if x.ndim != 2 or x.stride(1) != 1 and k > 1:
            raise ValueError(f'{what}: contiguous, or a matrix of contiguous rows; no hidden layout copy')
        if rows > 1:
            ld = x.stride(0)
    if ld < k or (ld * x.element_size()) % 16 or x.data_ptr() % 16:
        raise ValueError(f'{what}: rows must start on 16 bytes and not overlap')
    return rows, ld, k


# ---------------------------------------------------------------- rows
def check_rows(x):
    """Rows that ``quantize_rows`` takes, as (rows, row stride, row length); what it refuses is raised."""
    _on_device(x)
    _require_float(x, 'rows')
    rows, ld, k = _rows(x, 'rows')
    if k % 16 or k > MAX_ROW:
        raise ValueError(f'rows: a row length that is a multiple of 16 and at most {MAX_ROW} required, not {k}')
    return rows, ld, k


def _check_norm(x, weight, eps, k):
    if weight.shape != (k,) or weight.dtype != x.dtype or not weight.is_contiguous() or weight.data_ptr() % 16 or \
            not float(eps) >= 0.0:
        raise ValueError(f'a contiguous 16-byte aligned norm weight of {k} {x.dtype} values and a nonnegative eps required')


def _codes_like(x):
    return torch.empty_like(x, dtype=torch.int8, memory_format=torch.contiguous_format), \
        x.new_empty(x.shape[:-1], dtype=torch.float32)


def quantize_rows(x):
    """x [..., K] -> (codes int8 [..., K], scales fp32 [...]): each row on its own."""
    _forward_only(x)
    rows, ld, k = check_rows(x)
    q, scale = _codes_like(x)
    _launch(x, "q3_quant_rows", H.code(x.dtype), x.data_ptr(), ld, q.data_ptr(), scale.data_ptr(), rows, k)
    return q, scale


def rms_norm(x, weight, eps, *, residual=None):
    """RMSNorm of x [..., K] in 8 bits: (codes, scales), and with ``residual`` (codes, scales, total) where
    total = x + residual, rounded once, is what the norm is taken of."""
    _forward_only(x, weight, residual)
    rows, ld, k = check_rows(x)
    _on_device(x, weight)
    _check_norm(x, weight, eps, k)
    if residual is None:
        q, scale = _codes_like(x)
        _launch(x, "q3_rmsnorm_quant", H.code(x.dtype), x.data_ptr(), ld, None, 0, weight.data_ptr(), q.data_ptr(),
                scale.data_ptr(), None, rows, k, float(eps))
        return q, scale
    _on_device(x, residual)
    if residual.shape != x.shape or residual.dtype != x.dtype:
        raise ValueError('a residual of the shape and dtype of x required')
    ldr = _rows(residual, 'residual')[1]
    q, scale = _codes_like(x)
    total = torch.empty_like(x, memory_format=torch.contiguous_format)
    _launch(x, "q3_rmsnorm_quant", H.code(x.dtype), x.data_ptr(), ld, residual.data_ptr(), ldr, weight.data_ptr(),
            q.data_ptr(), scale.data_ptr(), total.data_ptr(), rows, k, float(eps))
    return q, scale, total


# ---------------------------------------------------------------- products
def _check_codes(q, scale):
    _on_device(q, scale)
    if q.dtype != torch.int8:
        raise TypeError(f'int8 codes required, not {q.dtype}')
    rows, ld, k = _rows(q, 'codes')
    if scale.dtype != torch.float32 or scale.numel() != rows or not scale.is_contiguous():
        raise ValueError('contiguous float32 scales, one per row of codes, required')
    if k % 16 or k >= MAX_K or ld >= 1 << 23:
        raise ValueError(f'a row length that is a multiple of 16 and below {MAX_K} required, not {k} ({ld} apart)')
    return rows, ld, k


def _check_weight(x, k, w, ws):
    _on_device(x, w, ws)
    if w.dtype != torch.int8 or w.ndim != 2 or w.shape[1] != k:
        raise ValueError('an int8 weight [N, K] of the input\'s K required')
    if ws.dtype != torch.float32 or ws.ndim != 1 or ws.shape[0] != w.shape[0] or not ws.is_contiguous():
        raise ValueError('contiguous float32 scales, one per weight row, required')
    ld = _rows(w, 'weight')[1]
    if ld >= 1 << 23:
        raise ValueError('weight rows are too far apart')
    return w.data_ptr(), ld, ws.data_ptr()


def _desc(x, operand, rows, k, weights, outs, epilogue, dtype, residual):
    """``q3_int8_gemm_desc``; ``operand``: the left one's (codes, row stride, scales), x: a tensor of its device."""
    res = ldres = 0
    if residual is not None:
        _on_device(x, residual)
        if residual.shape != outs[0].shape or residual.dtype != dtype or not residual.is_contiguous():
            raise ValueError('a contiguous residual of the result\'s shape and dtype required')
        res, ldres = residual.data_ptr(), residual.shape[-1]
    if len(weights) == 1:
        (w, ws), = weights
        p, ld, s = _check_weight(x, k, w, ws)
        n = w.shape[0]
        return H.Int8GemmDesc(H.code(dtype), 1, epilogue, rows, n, k, n, 0, 0, *operand, p, 0, 0, ld, 0, 0, s, 0, 0,
                              outs[0].data_ptr(), 0, 0, n, 0, 0, res, ldres)
    p, ld, s, ends, end = [0, 0, 0], [0, 0, 0], [0, 0, 0], [0, 0, 0], 0
    for i, (w, ws) in enumerate(weights):
        p[i], ld[i], s[i] = _check_weight(x, k, w, ws)
        end += w.shape[0]
        ends[i] = end
    n = end if epilogue != H.GEMM_GATE_UP else weights[0][0].shape[0]
    c, ldc = [0, 0, 0], [0, 0, 0]
    for i, y in enumerate(outs):
        c[i], ldc[i] = y.data_ptr(), y.shape[-1]
    return H.Int8GemmDesc(H.code(dtype), len(outs), epilogue, rows, n, k, *ends, *operand, *p, *ld, *s, *c, *ldc, res, ldres)


def _product(q, scale, weights, outs, epilogue, dtype, residual=None):
    _forward_only(scale, residual, *(ws for _, ws in weights))
    rows, ld, k = _check_codes(q, scale)
    d = _desc(q, (q.data_ptr(), ld, scale.data_ptr()), rows, k, weights, outs, epilogue, dtype, residual)
    nbytes = H.query("q3_gemm_int8_workspace_bytes", d) if rows > 16 else 0   # up to 16 rows never take any
    ws = H.workspace(nbytes, q.device) if nbytes else None
    _launch(q, "q3_gemm_int8", d, None if ws is None else ws.data_ptr(), nbytes)


def _out(q, n, dtype):
    if dtype not in _FLOATS:
        raise TypeError(f'a bfloat16 or float16 result required, not {dtype}')
    if q.ndim == 2:
        return q.new_empty((q.shape[0], n), dtype=dtype)
    return q.new_empty((*q.shape[:-1], n), dtype=dtype)


def linear(q, scale, weight, weight_scale, *, dtype=torch.bfloat16, residual=None):
    """(codes [..., K], scales [...]) x (weight codes [N, K], scales [N]) -> [..., N] in ``dtype``: exact integer sums,
    scaled in fp32, plus ``residual`` [..., N], rounded once."""
    y = _out(q, weight.shape[0], dtype)
    _product(q, scale, ((weight, weight_scale),), (y,), H.GEMM_PLAIN if residual is None else H.GEMM_RESIDUAL, dtype, residual)
    return y


def projections(q, scale, weights, *, dtype=torch.bfloat16):
    """``linear`` by up to three weights [(codes, scales), ...] of one input in one launch (Q, K and V)."""
    if not 1 <= len(weights) <= 3:
        raise ValueError('one to three weights required')
    outs = [_out(q, w.shape[0], dtype) for w, _ in weights]
    _product(q, scale, weights, outs, H.GEMM_PLAIN, dtype)
    return outs


def _check_gate_up(gate, up):
    if gate.shape != up.shape or gate.stride() != up.stride():
        raise ValueError('gate and up weights of one shape and layout required')
    if gate.shape[0] % 8:
        raise ValueError('a number of gate/up channels that is a multiple of 8 required')


def gate_up_swiglu(q, scale, gate, gate_scale, up, up_scale, *, dtype=torch.bfloat16):
    """silu(x Wg^T) * (x Wu^T) of codes x and weights [N, K] (N a multiple of 8), formed in fp32 and rounded once."""
    _check_gate_up(gate, up)
    y = _out(q, gate.shape[0], dtype)
    _product(q, scale, ((gate, gate_scale), (up, up_scale)), (y,), H.GEMM_GATE_UP, dtype)
    return y


def decode_linear_ok(x):
    """Whether ``decode_linear`` takes rows like x [..., K]: at most 2, of at most 16384 values."""
    k = x.shape[-1] if x.ndim else 0
    return k > 0 and bool(H.query("q3_decode_linear_int8_ok", x.numel() // k, k))


def decode_linear(x, weights, *, norm_weight=None, eps=1e-6, gate_up=False, residual=None):
    """A decode step's product straight from 16-bit rows x [..., K]: ``quantize_rows`` (with ``norm_weight`` ``rms_norm``) and
    ``projections`` of up to three weights [(codes, scales), ...] in one launch -> a list; with ``gate_up`` the SwiGLU of
    two -> one tensor; with ``residual`` [..., N] one weight's product plus it -> one tensor."""
    _forward_only(x, norm_weight, residual, *(ws for _, ws in weights))
    rows, ld, k = check_rows(x)
    if not decode_linear_ok(x):
        raise ValueError('decode_linear takes at most 2 rows of at most 16384 values')
    if norm_weight is not None:
        _on_device(x, norm_weight)
        _check_norm(x, norm_weight, eps, k)
    if gate_up:
        if len(weights) != 2 or residual is not None:
            raise ValueError('gate and up weights and no residual required')
        _check_gate_up(weights[0][0], weights[1][0])
        outs, epilogue = [_out(x, weights[0][0].shape[0], x.dtype)], H.GEMM_GATE_UP
    else:
        if not 1 <= len(weights) <= (3 if residual is None else 1):
            raise ValueError('one to three weights required, one with a residual')
        outs = [_out(x, w.shape[0], x.dtype) for w, _ in weights]
        epilogue = H.GEMM_PLAIN if residual is None else H.GEMM_RESIDUAL
    d = _desc(x, (0, 0, 0), rows, k, weights, outs, epilogue, x.dtype, residual)
    _launch(x, "q3_decode_linear_int8", d, x.data_ptr(), ld, None if norm_weight is None else norm_weight.data_ptr(),
            float(eps))
    return outs[0] if gate_up or residual is not None else outs


# ---------------------------------------------------------------- cache
@dataclass(frozen=True)
class LayerCache:
    """One layer's keys and values in 8 bits, head dim 128, capacity C in blocks of 64 positions (Cb = ceil(C / 64)):

    ``k`` int8 [B, Hkv, 64 Cb, 128]; ``v`` int8 [B, Hkv, Cb, 128, 64], transposed within a block; ``k_scale`` and
    ``v_scale`` fp32 [B, Hkv, Cb]; ``k_tail`` [B, Hkv, 64, 128] and ``v_tail`` [B, Hkv, 128, 64]: the positions of the last,
    unfinished block in 16 bits, at slot position % 64.

    A block is quantised once, from its 16-bit values, when its last position is appended; so what the cache holds does
    not depend on how the tokens were cut into chunks.  Positions are appended in order: the cache cannot be wound back
    into a block that is already quantised (start again from 0 or another multiple of 64), nor read there, since the tail
    holds another block's positions by then.  The object knows how far its own ``append`` calls went and refuses both; it does
    not know what a captured or device-positioned call appends (after one it checks nothing more), nor what its buffers
    held before or are given through another object."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor
    k_tail: torch.Tensor
    v_tail: torch.Tensor

    @classmethod
    def empty(cls, batch, heads, capacity, *, device, dtype=torch.bfloat16, head_dim=128):
        """Buffers for ``capacity`` positions (their contents are whatever the memory held: nothing reads a position that
        was not appended)."""
        if head_dim != 128:
            raise ValueError('head_dim 128 required')
        if min(batch, heads, capacity) < 1:
            raise ValueError('a batch, heads and capacity of at least 1 required')
        if dtype not in _FLOATS:
            raise TypeError(f'bfloat16 or float16 required, not {dtype}')
        cb = -(-capacity // KV_BLOCK)
        i8, f32 = dict(device=device, dtype=torch.int8), dict(device=device, dtype=torch.float32)
        return cls(torch.empty((batch, heads, cb * KV_BLOCK, 128), **i8), torch.empty((batch, heads, cb, 128, KV_BLOCK), **i8),
                   torch.empty((batch, heads, cb), **f32), torch.empty((batch, heads, cb), **f32),
                   torch.empty((batch, heads, KV_BLOCK, 128), device=device, dtype=dtype),
                   torch.empty((batch, heads, 128, KV_BLOCK), device=device, dtype=dtype))

    @property
    def capacity(self):
        return self.k.shape[2]

    @property
    def nbytes(self):
        return sum(t.numel() * t.element_size()
                   for t in (self.k, self.v, self.k_scale, self.v_scale, self.k_tail, self.v_tail))

    def __post_init__(self):
        """The buffers are what the kernels take, once and for all (the fields cannot be set again)."""
        k, v, ks, vs, kt, vt = tensors = (self.k, self.v, self.k_scale, self.v_scale, self.k_tail, self.v_tail)
        b, h, c, d = k.shape if k.ndim == 4 else (0, 0, 0, 0)
        cb = c // KV_BLOCK
        if d != 128 or c % KV_BLOCK or min(b, h, c) < 1 or v.shape != (b, h, cb, d, KV_BLOCK) or ks.shape != (b, h, cb) or \
                vs.shape != (b, h, cb) or kt.shape != (b, h, KV_BLOCK, d) or vt.shape != (b, h, d, KV_BLOCK):
            raise ValueError('cache buffers of matching shapes (head dim 128, blocks of 64) required')
        if k.dtype != torch.int8 or v.dtype != torch.int8 or ks.dtype != torch.float32 or vs.dtype != torch.float32 or \
                kt.dtype not in _FLOATS or vt.dtype != kt.dtype:
            raise TypeError('int8 codes, float32 scales and 16-bit tails of one dtype required')
        dev = k.device
        for t in tensors:
            if t.device != dev or not t.is_contiguous() or t.data_ptr() % 16 and t.dtype != torch.float32:
                raise ValueError('contiguous, 16-byte aligned cache buffers on one device required')
            if t.requires_grad or _dual(t):
                raise ValueError('cache buffers take no gradient')
        self._know(None, 0)

    def _know(self, end, tail):
        """Note that the cache holds the positions before ``end`` (None: not known; -1: not known from now on), and the tail
        those of its block before ``tail`` (a block's last append leaves there what was before it)."""
        object.__setattr__(self, '_end', end)
        object.__setattr__(self, '_tail', tail)

    def require_whole(self, n):
        """Raise if n, where an append is to start or a read to end, lies inside a block that is quantised already (and no
        longer in the tail)."""
        end = self._end
        if n % KV_BLOCK and end is not None and n < end // KV_BLOCK * KV_BLOCK and \
                not self._tail // KV_BLOCK * KV_BLOCK < n <= self._tail:
            raise ValueError(f'position {n} lies inside a quantised block of a cache of {end} positions: only a multiple of '
                             f'{KV_BLOCK}, or a position of the unfinished block, can be gone back to')

    def pointers(self):
        return (self.k.data_ptr(), self.v.data_ptr(), self.k_scale.data_ptr(), self.v_scale.data_ptr(),
                self.k_tail.data_ptr(), self.v_tail.data_ptr())


def _check_heads(t, cache, what):
    """t [B, S, heads, 128] of the cache's batch and dtype, every head's row 16 bytes of its own; returns its strides."""
    _on_device(cache.k, t)
    if t.ndim != 4 or t.numel() == 0:
        raise ValueError(f'{what}: [B, S, heads, 128] required')
    b, s, h, d = t.shape
    if b != cache.k.shape[0] or d != 128:
        raise ValueError(f'{what}: [B, S, heads, 128] of the cache\'s batch required')
    if t.dtype != cache.k_tail.dtype:
        raise TypeError(f'{what}: {cache.k_tail.dtype} required, not {t.dtype}')
    sb, ss, sh, sd = t.stride()
    sb, ss, sh = sb if b > 1 else 0, ss if s > 1 else 0, sh if h > 1 else 0   # a lone index's stride is never used
    if sd != 1 or (sb | ss | sh) % 8 or t.data_ptr() % 16:
        raise ValueError(f'{what}: contiguous, 16-byte aligned heads required')
    return sb, ss, sh


def _check_span(start, s, cache, start_dev, new):
    """``new``: whether the s positions are to be appended or are there."""
    if start_dev is not None:
        if s != 1:
            raise ValueError('device-resident positions are for single-token decode steps')
        _on_device(cache.k, start_dev)
        if start_dev.dtype != torch.int64 or start_dev.numel() != 1:
            raise ValueError('a device position is one int64')
        return 0
    if type(start) is not int or start < 0 or start + s > cache.capacity:
        raise ValueError(f'positions {start} .. {start} + {s} - 1 do not fit a cache of {cache.capacity}')
    cache.require_whole(start if new else start + s)
    return start


def _note(cache, start, s, start_dev):
    """After an append.  What a captured one appends, and when, is not known here."""
    if start_dev is not None or cache._end == -1 or torch.cuda.is_current_stream_capturing():
        cache._know(-1, 0)
        return
    end, tail = start + s, cache._tail
    if end % KV_BLOCK:
        tail = end
    elif start % KV_BLOCK:
        tail = start
    elif tail > start:   # the positions that it held are others now
        tail = 0
    cache._know(end, tail)


def append(k, v, cache, start, start_dev=None):
    """Append k, v [B, S, Hkv, 128] to a ``LayerCache`` that holds the positions before ``start`` (with ``start_dev``, one
    token at that device int64, read when the kernel runs; positions outside the capacity are skipped)."""
    _forward_only(k, v)
    ks, vs = _check_heads(k, cache, 'keys'), _check_heads(v, cache, 'values')
    b, s, h, d = k.shape
    if v.shape != k.shape or h != cache.k.shape[1]:
        raise ValueError('keys and values of one shape, with the cache\'s heads, required')
    start = _check_span(start, s, cache, start_dev, True)
    _launch(k, "q3_kv8_append", H.code(k.dtype), k.data_ptr(), *ks, v.data_ptr(), *vs, *cache.pointers(), b, s, h, d,
            cache.capacity, start, None if start_dev is None else start_dev.data_ptr())
    _note(cache, start, s, start_dev)


def _check_norm_rope(q, q_norm_weight, k_norm_weight, cos, sin, eps):
    b, s, _, d = q.shape
    for t, shape in ((q_norm_weight, (d,)), (k_norm_weight, (d,)), (cos, (b, s, d)), (sin, (b, s, d))):
        _on_device(q, t)
        if t.shape != shape or t.dtype != q.dtype or not t.is_contiguous() or t.data_ptr() % 16:
            raise ValueError(f'contiguous, 16-byte aligned {q.dtype} norm weights [128] and tables [B, S, 128] required')
    if not float(eps) >= 0.0:
        raise ValueError('a nonnegative eps required')


def norm_rope_append(q, k, v, q_norm_weight, k_norm_weight, cos, sin, cache, start, start_dev=None, *, eps=1e-6):
    """Per-head RMSNorm and rotation of q [B, S, Hq, 128] and k [B, S, Hkv, 128] as projected (tables cos, sin [B, S, 128])
    and ``append`` of those keys and v, in one launch; returns the normed and rotated q, contiguous."""
    _forward_only(q, k, v, q_norm_weight, k_norm_weight, cos, sin)
    qs, ks, vs = (_check_heads(t, cache, what) for t, what in ((q, 'queries'), (k, 'keys'), (v, 'values')))
    b, s, hq, d = q.shape
    h = k.shape[2]
    if v.shape != k.shape or k.shape[1] != s or h != cache.k.shape[1]:
        raise ValueError('queries, keys and values of one batch and length, with the cache\'s heads, required')
    _check_norm_rope(q, q_norm_weight, k_norm_weight, cos, sin, eps)
    start = _check_span(start, s, cache, start_dev, True)
    out = q.new_empty((b, s, hq, d))
    _launch(q, "q3_kv8_norm_rope_append", H.code(q.dtype), q.data_ptr(), *qs, k.data_ptr(), *ks, v.data_ptr(), *vs,
            q_norm_weight.data_ptr(), k_norm_weight.data_ptr(), cos.data_ptr(), sin.data_ptr(), out.data_ptr(),
            *cache.pointers(), b, s, hq, h, d, cache.capacity, start, None if start_dev is None else start_dev.data_ptr(),
            float(eps))
    _note(cache, start, s, start_dev)
    return out


def read(cache, length, *, dtype=None):
    """The ``length`` positions that the cache holds back as k, v [B, Hkv, length, 128] in ``dtype`` (the tail's by default).
    Fewer than it holds can be read up to a multiple of 64, or to a position of its unfinished block."""
    _on_device(cache.k)
    b, h, capacity, _ = cache.k.shape
    if type(length) is not int or not 1 <= length <= capacity:
        raise ValueError(f'length must be an int in [1, {capacity}]')
    cache.require_whole(length)
    dtype = cache.k_tail.dtype if dtype is None else dtype
    k, v = (cache.k.new_empty((b, h, length, 128), dtype=dtype) for _ in range(2))
    _launch(k, "q3_kv8_read", H.code(cache.k_tail.dtype), H.code(dtype), *cache.pointers(), k.data_ptr(), v.data_ptr(), b, h,
            128, capacity, length)
    return k, v


def attention(q, cache, start, start_dev=None, *, scale=None):
    """q [B, S, Hq, 128] at positions start .. start + S - 1, causal, against the cache's positions up to each query's own
    (appended before; where the cache holds more, ``start + S`` as ``read``'s length); returns [B, S, Hq, 128].  With
    ``start_dev`` (S = 1) the position is read on the device and the launch spans the whole capacity, so a captured step
    replays at any position."""
    _forward_only(q)
    qs = _check_heads(q, cache, 'queries')
    b, s, hq, d = q.shape
    hkv = cache.k.shape[1]
    if hq % hkv:
        raise ValueError('query heads must be a multiple of key/value heads')
    start = _check_span(start, s, cache, start_dev, False)
    scale = d ** -0.5 if scale is None else float(scale)
    if not 0.0 < scale < 1e30:
        raise ValueError('a positive softmax scale required')
    out = q.new_empty((b, s, hq, d))
    nbytes = H.query("q3_kv8_attention_workspace_bytes", b, s, hq, hkv, start + s if start_dev is None else cache.capacity)
    ws = H.workspace(nbytes, q.device) if nbytes else None
    _launch(q, "q3_kv8_attention", H.code(q.dtype), q.data_ptr(), *qs, *cache.pointers(), out.data_ptr(), s * hq * d, hq * d, d,
            None if ws is None else ws.data_ptr(), nbytes, b, s, hq, hkv, d, cache.capacity, start,
            None if start_dev is None else start_dev.data_ptr(), scale)
    return out
