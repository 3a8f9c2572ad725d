"""Attention for rows that continue shared prefixes (several answers to one prompt, many requests behind one system prompt):
the prefix's keys and values are held once, and read once for all of its rows.  Forward only, bf16 or fp16, head dim 128.

``KVCache.fork`` makes the cache that ``TritonQwen3Inference`` runs on it.  The reference gives every row a copy of its prompt;
nothing here has a counterpart in it.
"""
import torch

from .. import _hip as H
from .int8 import _FLOATS, _forward_only, _on_device

HEAD_DIM = 128
MAX_STRIDE = 1 << 24   # elements between positions, below


def _cache_strides(k, v, what):
    """Strides (batch, head, position) of keys and values [.., heads, positions, 128] that lie alike."""
    shape = k.shape
    if len(shape) != 4 or v.shape != shape or shape[3] != HEAD_DIM:
        raise ValueError(f'{what}: keys and values [batch, heads, positions, {HEAD_DIM}] of one shape required')
    sk, sv = k.stride(), v.stride()
    if sk != sv or not _strides_ok(*sk):   # maybe that of an index that is alone (never used), or nothing is there
        sk, sv = ([s if n > 1 else d for n, s, d in zip(shape, t, (0, 0, HEAD_DIM, 1))] for t in (sk, sv))
        if 0 in shape:
            return 0, 0, HEAD_DIM
        if sk != sv:
            raise ValueError(f'{what}: keys and values of one layout required')
    if not _strides_ok(*sk) or (k.data_ptr() | v.data_ptr()) % 16:
        raise ValueError(f'{what}: contiguous, 16-byte aligned positions required; no hidden layout copy')
    return sk[0], sk[1], sk[2]


def _strides_ok(sb, sh, ss, sd):
    return sd == 1 and not (sb | sh | ss) % 8 and HEAD_DIM <= ss < MAX_STRIDE


def attention(q, prefix_k, prefix_v, cache_k, cache_v, start, start_dev=None, *, scale=None):
    """q [B, S, Hq, 128] of B rows, which continue R prefixes (keys and values [R, Hkv, P, 128], row b prefix b // (B // R);
    P may be 0) with positions of their own (cache_k, cache_v [B, Hkv, C, 128]), at their own positions start .. start + S - 1,
    appended before: each query sees its whole prefix and its row's positions up to its own.  Returns [B, S, Hq, 128].

    With ``start_dev`` (device int64, one value or one a row) the positions are read on the device when the kernel runs, also
    in a captured graph's replays, and ``start`` counts for nothing; own positions outside [0, C) are not there (a query that then
    sees nothing at all gets zeros).  Keys and values behind a row's last position may hold anything."""
    _forward_only(q, prefix_k, prefix_v, cache_k, cache_v)
    if q.ndim != 4 or q.numel() == 0 or q.shape[3] != HEAD_DIM:
        raise ValueError(f'queries: [B, S, heads, {HEAD_DIM}] required')
    _on_device(q, prefix_k, prefix_v, cache_k, cache_v)
    ps, cs = _cache_strides(prefix_k, prefix_v, 'prefix'), _cache_strides(cache_k, cache_v, 'own positions')
    b, s, hq, d = q.shape
    r, hkv, p, _ = prefix_k.shape
    c = cache_k.shape[2]
    dt = q.dtype
    if dt not in _FLOATS or prefix_k.dtype != dt or prefix_v.dtype != dt or cache_k.dtype != dt or cache_v.dtype != dt:
        raise TypeError(f'bfloat16 or float16 queries, keys and values of one dtype required, not {dt}')
    if r < 1 or b % r or cache_k.shape[:2] != (b, hkv) or hkv < 1 or hq % hkv:
        raise ValueError('a whole number of rows per prefix, own positions of every row, and query heads that are a multiple of '
                         'the key/value heads required')
    qb, qs, qh, qd = q.stride()
    qb, qs, qh = qb if b > 1 else 0, qs if s > 1 else 0, qh if hq > 1 else 0
    if qd != 1 or (qb | qs | qh) % 8 or q.data_ptr() % 16:
        raise ValueError('queries: contiguous, 16-byte aligned heads required')
    if c < s:
        raise ValueError(f'{s} positions do not fit {c}')
    starts = 0
    if start_dev is None:
        if type(start) is not int or start < 0 or start + s > c:
            raise ValueError(f'positions {start} .. {start} + {s} - 1 do not fit {c}')
    else:
        _on_device(q, start_dev)
        starts, start = start_dev.numel(), 0
        if start_dev.dtype != torch.int64 or starts not in (1, b) or not start_dev.is_contiguous():
            raise ValueError(f'device positions are one int64, or one for each of the {b} rows')
    scale = d ** -0.5 if scale is None else float(scale)
    if not 0.0 < scale < 1e30:
        raise ValueError('a positive softmax scale required')
    if b * s * hq >= 1 << 31 or max(p, c) >= 1 << 30 or b >= 1 << 24:
        raise ValueError('fewer than 2^31 query rows, 2^30 positions and 2^24 rows required')
    out = q.new_empty((b, s, hq, d))
    nbytes = H.query("q3_prefix_attention_workspace_bytes", b, r, s, hq, hkv, p, c, start + s if start_dev is None else c)
    ws = H.workspace(nbytes, q.device) if nbytes else None
    H.launch(q, "q3_prefix_attention", H.code(dt), q.data_ptr(), qb, qs, qh, prefix_k.data_ptr(), prefix_v.data_ptr(), *ps,
             cache_k.data_ptr(), cache_v.data_ptr(), *cs, out.data_ptr(), s * hq * d, hq * d, d,
             None if ws is None else ws.data_ptr(), nbytes, b, r, s, hq, hkv, d, p, c, start,
             None if start_dev is None else start_dev.data_ptr(), starts, scale)
    return out
