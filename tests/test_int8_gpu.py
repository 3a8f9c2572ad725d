"""The 8-bit serving operators (``inference/int8.py``) against their definitions in 64 bits.

Codes are compared for equality: the rule (the integer nearest to 127 a / M, ties to even) leaves nothing to rounding.
Tolerances elsewhere count roundings: u = eps / 2 of the output type once, 2^-24 per fp32 operation, and for attention the
rounding of the probabilities (2^-11 in fp16 over 8-bit blocks; the tail's, in the activation type) on sum p |v|.
"""
import math

import pytest
import torch

from _util import seeded

from qwen3_triton.inference import int8 as I8

pytestmark = pytest.mark.gpu

DT = [torch.bfloat16, torch.float16]
F64 = torch.float64


def randn(*shape, gen, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=gen) * scale).to(dtype)


def codes64(a):
    """a [..., n] in 64 bits -> (codes, M): one scale per row of the last axis."""
    m = a.abs().amax(-1)
    return torch.where(m[..., None] > 0, (127.0 * a / m[..., None]).round(), torch.zeros_like(a)), m


def close(y, ref, tol):
    bad = (y.double().cpu() - ref).abs() > tol
    assert torch.isfinite(y).all() and not bool(bad.any()), \
        (int(bad.sum()), float(((y.double().cpu() - ref).abs() - tol).max()))


# ---------------------------------------------------------------- rows
def row_cases(h, dtype, gen):
    """Rows where the rule can go wrong: ordinary, outliers, zeros, ties, tiny and huge magnitudes."""
    x = randn(9, h, gen=gen)
    x[1, ::7] *= 40
    x[2] = 0
    x[3] = torch.arange(h) % 128 - 0.5      # M 126.5 or 127 with ties
    x[3, 0] = 127
    x[4] = (torch.arange(h) % 255 - 127) / 2  # ties at M = 63.5: 127 x / M = 2 x
    x[4, 1] = 63.5
    x[5] *= 2.0 ** (-110 if dtype == torch.bfloat16 else -20)
    x[6] *= 2.0 ** (120 if dtype == torch.bfloat16 else 12)
    x[7] = 0
    x[7, h // 2] = -3.0
    x[8] = -1.5
    return x.to(dtype)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("h", [16, 48, 128, 512, 528, 1024, 1040, 2048, 4096, 4112, 8192, 12288, 16400, 32768])
def test_quantize_rows(h, dtype):
    x = row_cases(h, dtype, seeded(h))
    q, s = I8.quantize_rows(x.cuda())
    want, m = codes64(x.double())
    assert torch.equal(q.cpu().double(), want)
    assert torch.equal(s.cpu(), m.float() / 127.0)
    q1, s1 = I8.quantize_rows(x[1:2].cuda().view(1, 1, h))
    assert torch.equal(q1.view(1, h), q[1:2]) and torch.equal(s1.view(1), s[1:2]) and q1.shape == (1, 1, h)


def test_quantize_rows_strided_and_nonfinite():
    x = randn(7, 256, gen=seeded(1), dtype=torch.bfloat16).cuda()
    q, s = I8.quantize_rows(x[:, :128])
    want, wants = I8.quantize_rows(x[:, :128].contiguous())
    assert torch.equal(q, want) and torch.equal(s, wants)
    y = x.clone()
    y[1, 3], y[2, 200], y[3, 0] = math.nan, math.inf, -math.inf
    q, s = I8.quantize_rows(y)
    assert torch.isnan(s[1:4]).all() and torch.isfinite(s[[0, 4, 5, 6]]).all()
    assert torch.equal(q[[0, 4, 5, 6]], I8.quantize_rows(x)[0][[0, 4, 5, 6]])


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("rows,h", [(1, 4096), (3, 16), (130, 256), (5, 1040), (2, 2048), (33, 4096), (2, 12288), (1, 32768)])
def test_rms_norm(rows, h, dtype, residual):
    gen = seeded(rows + h)
    x, r = randn(rows, h, gen=gen, dtype=dtype), randn(rows, h, gen=gen, dtype=dtype)
    x[0, ::5] *= 16
    w = (1 + 0.1 * torch.randn(h, generator=gen)).to(dtype)
    out = I8.rms_norm(x.cuda(), w.cuda(), 1e-6, residual=r.cuda() if residual else None)
    t = (x.float() + r.float()).to(dtype) if residual else x
    if residual:
        assert torch.equal(out[2].cpu(), t)
    want, m = codes64(t.double() * w.double())
    assert torch.equal(out[0].cpu().double(), want)
    ref = m / 127.0 / (t.double().square().mean(-1) + 1e-6).sqrt()
    # the sum of squares over h / 8 ... terms a thread, then butterflies; 1 / h, + eps, the root (2 ulp), two products
    tol = (math.ceil(math.log2(h)) + 40) * 2.0 ** -24
    assert float(((out[1].double().cpu() - ref) / ref).abs().max()) <= tol


def test_rms_norm_zero_row_eps_and_strided_residual():
    gen = seeded(5)
    x, r = randn(3, 512, gen=gen, dtype=torch.bfloat16).cuda(), randn(3, 1024, gen=gen, dtype=torch.bfloat16).cuda()
    w = torch.ones(512, dtype=torch.bfloat16, device="cuda")
    x[1] = 0
    q, s = I8.rms_norm(x, w, 0.0)
    assert not q[1].any() and torch.isnan(s[1])   # 0 * rsqrt(0), as the 16-bit norm's
    q, s = I8.rms_norm(x, w, 1e-6)
    assert not q[1].any() and float(s[1]) == 0.0
    a = I8.rms_norm(x, w, 1e-6, residual=r[:, :512])
    b = I8.rms_norm(x, w, 1e-6, residual=r[:, :512].contiguous())
    assert all(torch.equal(p, o) for p, o in zip(a, b))


# ---------------------------------------------------------------- products
def product_inputs(m, n, k, gen):
    q = torch.randint(-127, 128, (m, k), generator=gen, dtype=torch.int8)
    w = torch.randint(-127, 128, (n, k), generator=gen, dtype=torch.int8)
    s, ws = torch.rand(m, generator=gen) * 1e-2 + 1e-3, torch.rand(n, generator=gen) * 1e-3 + 1e-4
    return q, s, w, ws


def product64(q, s, w, ws):
    return (q.double() @ w.double().t()) * s.double()[:, None] * ws.double()


SIZES = [(1, 1, 16), (1, 64, 128), (2, 100, 48), (3, 7, 1040), (8, 256, 4096), (16, 300, 512), (17, 256, 256), (33, 64, 144),
         (65, 130, 2048), (100, 1000, 80), (128, 128, 128), (200, 512, 12288), (256, 256, 64), (300, 264, 528), (513, 520, 1024)]


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_linear(m, n, k, residual, dtype):
    gen = seeded(m * 7 + n * 3 + k)
    q, s, w, ws = product_inputs(m, n, k, gen)
    res = randn(m, n, gen=gen, dtype=dtype) if residual else None
    y = I8.linear(q.cuda(), s.cuda(), w.cuda(), ws.cuda(), dtype=dtype, residual=None if res is None else res.cuda())
    p = product64(q, s, w, ws)
    ref = p + (res.double() if residual else 0)
    # int -> fp32, two scales, the residual's sum: four fp32 roundings; one to the output type
    close(y, ref, ref.abs() * torch.finfo(dtype).eps / 2 * (1 + 2.0 ** -10) + (p.abs() + ref.abs()) * 4 * 2.0 ** -24 + 1e-7)


@pytest.mark.parametrize("m", [1, 5, 16, 40, 300])
def test_linear_largest_sums(m):
    """Codes of +-127 (and the -128 that a caller's own weights may hold) at the largest K: sums up to 2^31 - 2^18."""
    k = (1 << 17) - 16
    q = torch.full((m, k), -128, dtype=torch.int8)
    w = torch.full((24, k), -128, dtype=torch.int8)
    w[1] = 127
    w[2, ::2] = 127
    s, ws = torch.full((m,), 2.0 ** -20), torch.full((24,), 2.0 ** -10)
    y = I8.linear(q.cuda(), s.cuda(), w.cuda(), ws.cuda())
    ref = product64(q, s, w, ws)
    close(y, ref, ref.abs() * 2.0 ** -8 * (1 + 2.0 ** -10))


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("m", [1, 7, 16, 31, 130, 515])
def test_projections_in_one_launch(m, dtype):
    gen = seeded(m)
    q, s, _, _ = product_inputs(m, 8, 512, gen)
    ws = [product_inputs(1, n, 512, gen)[2:] for n in (256, 64, 72)]
    outs = I8.projections(q.cuda(), s.cuda(), [(w.cuda(), x.cuda()) for w, x in ws], dtype=dtype)
    for y, (w, x) in zip(outs, ws):
        assert torch.equal(y, I8.linear(q.cuda(), s.cuda(), w.cuda(), x.cuda(), dtype=dtype))
        ref = product64(q, s, w, x)
        close(y, ref, ref.abs() * (torch.finfo(dtype).eps / 2 * (1 + 2.0 ** -10) + 2.0 ** -21) + 1e-7)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("m,n,k", [(1, 8, 16), (1, 688, 256), (5, 104, 1040), (16, 256, 4096), (17, 72, 128), (128, 512, 512),
                                   (300, 264, 64), (520, 776, 256)])
def test_gate_up_swiglu(m, n, k, dtype):
    gen = seeded(m + n + k)
    q, s, wg, sg = product_inputs(m, n, k, gen)
    _, _, wu, su = product_inputs(1, n, k, gen)
    y = I8.gate_up_swiglu(q.cuda(), s.cuda(), wg.cuda(), sg.cuda(), wu.cuda(), su.cuda(), dtype=dtype)
    g, u = product64(q, s, wg, sg), product64(q, s, wu, su)
    ref = g * torch.sigmoid(g) * u
    # g and u carry 3 fp32 roundings each; silu's relative sensitivity to g is at most 1 + |g|; exp2, rcp and its argument
    # (1.44 g rounded) a few ulp each, again times |g| in the exponent
    rel = torch.finfo(dtype).eps / 2 * (1 + 2.0 ** -10) + (12 + 6 * g.abs()) * 2.0 ** -23
    close(y, ref, ref.abs() * rel + 1e-7)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("m,k", [(1, 16), (1, 4096), (2, 4096), (2, 528), (1, 4112), (1, 12288), (2, 12288), (2, 16384), (1, 8208)])
def test_decode_linear(m, k, norm, dtype):
    """One launch against quantize_rows / rms_norm and the product: the same codes, so the same bits but for the norm's scale,
    whose sum of squares is taken in another order."""
    gen = seeded(m + k)
    x, nw = randn(m, k, gen=gen, dtype=dtype).cuda(), (1 + 0.1 * torch.randn(k, generator=gen)).to(dtype).cuda()
    x[0, ::9] *= 20
    ws = [I8.quantize_rows(randn(n, k, gen=gen, dtype=dtype, scale=0.05).cuda()) for n in (100, 40, 24, 100)]
    res = randn(m, 100, gen=gen, dtype=dtype).cuda()
    kw = dict(norm_weight=nw, eps=1e-6) if norm else {}
    q, s = I8.rms_norm(x, nw, 1e-6) if norm else I8.quantize_rows(x)
    pairs = list(zip(I8.decode_linear(x, ws[:3], **kw), I8.projections(q, s, ws[:3], dtype=dtype)))
    pairs.append((I8.decode_linear(x, ws[:1], residual=res, **kw), I8.linear(q, s, *ws[0], dtype=dtype, residual=res)))
    even = [(w[:96], t[:96].contiguous()) for w, t in (ws[0], ws[3])]
    pairs.append((I8.decode_linear(x, even, gate_up=True, **kw), I8.gate_up_swiglu(q, s, *even[0], *even[1], dtype=dtype)))
    for got, want in pairs:
        if norm:   # one output rounding apart where the scales differ in their last bits (sums below 2^-17 apart)
            ref = want.double().cpu()
            close(got, ref, ref.abs() * torch.finfo(dtype).eps * (1 + 2.0 ** -8) + 2.0 ** -16)
        else:
            assert torch.equal(got, want)


@pytest.mark.parametrize("m", [1, 2, 9, 16])
@pytest.mark.parametrize("k", [272, 2048, 4352])
def test_few_rows_many_channels(m, k):
    """More channels than the workgroups of a launch take in one go: each goes on to others, over the pieces' borders."""
    gen = seeded(m + k)
    dtype = torch.bfloat16
    x = randn(m, k, gen=gen, dtype=dtype).cuda()
    q, s = I8.quantize_rows(x)
    _, _, w, ws = product_inputs(1, 17016, k, gen)
    wd, wsd = w.cuda(), ws.cuda()
    ref = product64(q.cpu(), s.cpu(), w, ws)
    tol = torch.finfo(dtype).eps / 2 * (1 + 2.0 ** -10) + 2.0 ** -21
    y = I8.linear(q, s, wd, wsd)
    close(y, ref, ref.abs() * tol + 1e-7)
    ends = (0, 8216, 8240, 17016)
    pieces = [(wd[a:b], wsd[a:b]) for a, b in zip(ends, ends[1:])]
    for got, a, b in zip(I8.projections(q, s, pieces), ends, ends[1:]):
        assert torch.equal(got, y[:, a:b])
    even = [(wd[:8504], wsd[:8504]), (wd[8512:], wsd[8512:])]
    g, u = ref[:, :8504], ref[:, 8512:]
    z = I8.gate_up_swiglu(q, s, *even[0], *even[1])
    want = g * torch.sigmoid(g) * u
    close(z, want, want.abs() * (torch.finfo(dtype).eps / 2 * (1 + 2.0 ** -10) + (12 + 6 * g.abs()) * 2.0 ** -23) + 1e-7)
    if m <= 2:
        for got, a, b in zip(I8.decode_linear(x, pieces), ends, ends[1:]):
            assert torch.equal(got, y[:, a:b])
        assert torch.equal(I8.decode_linear(x, even, gate_up=True), z)


def test_decode_linear_refusals_and_nonfinite_rows():
    x = randn(3, 64, gen=seeded(1), dtype=torch.bfloat16).cuda()
    w = I8.quantize_rows(randn(32, 64, gen=seeded(2), dtype=torch.bfloat16).cuda())
    for bad in (lambda: I8.decode_linear(x, [w]), lambda: I8.decode_linear(x[:1], [w] * 4), lambda: I8.decode_linear(x[:1], []),
                lambda: I8.decode_linear(x[:1], [w, w, w], gate_up=True), lambda: I8.decode_linear(x[:1], [w, w], residual=x[:1, :32]),
                lambda: I8.decode_linear(x[:1, :48], [w]), lambda: I8.decode_linear(x[:1], [w], norm_weight=x[0, :32])):
        with pytest.raises(ValueError):
            bad()
    x[1, 5] = math.nan
    y, = I8.decode_linear(x[:2], [w])
    assert torch.isnan(y[1]).all() and torch.equal(y[:1], I8.decode_linear(x[:1], [w])[0])


def test_linear_strided_and_last_columns_untouched():
    gen = seeded(9)
    q, s, w, ws = product_inputs(20, 40, 256, gen)
    wide = torch.cat([q, torch.full_like(q, 99)], 1).cuda()
    y = I8.linear(wide[:, :256], s.cuda(), w.cuda(), ws.cuda())
    assert torch.equal(y, I8.linear(q.cuda(), s.cuda(), w.cuda(), ws.cuda()))
    wwide = torch.cat([w, torch.full_like(w, 77)], 1).cuda()
    assert torch.equal(y, I8.linear(q.cuda(), s.cuda(), wwide[:, :256], ws.cuda()))
    s2 = s.clone()
    s2[3] = math.nan
    z = I8.linear(q.cuda(), s2.cuda(), w.cuda(), ws.cuda())
    keep = [i for i in range(20) if i != 3]
    assert torch.isnan(z[3]).all() and torch.equal(z[keep], y[keep])


# ---------------------------------------------------------------- cache
def filled(b, h, total, dtype, gen, *, cuts=(), capacity=None, wide=True):
    """(cache, k, v): ``total`` positions appended in the chunks that ``cuts`` make, into poisoned buffers."""
    k, v = randn(b, total, h, 128, gen=gen, dtype=dtype), randn(b, total, h, 128, gen=gen, dtype=dtype)
    if wide:
        k[..., ::16] *= 6
        v[:, ::3] *= 0.1
    c = poisoned(b, h, capacity or total, dtype)
    at = 0
    for end in (*cuts, total):
        I8.append(k[:, at:end].cuda(), v[:, at:end].cuda(), c, at)
        at = end
    return c, k, v


def poisoned(b, h, capacity, dtype):
    c = I8.LayerCache.empty(b, h, capacity, device="cuda", dtype=dtype)
    c.k.fill_(111), c.v.fill_(-111)
    for t in (c.k_scale, c.v_scale, c.k_tail, c.v_tail):
        t.fill_(math.nan)
    return c


def held64(k, v):
    """What a cache holds of k, v [B, T, H, 128], as values [B, H, T, 128] in 64 bits, and the codes and scales."""
    full = k.shape[1] // 64
    out, parts = [], []
    for x in (k, v):
        x = x.double().transpose(1, 2)
        b, h, t, d = x.shape
        blocks = x[:, :, :full * 64].reshape(b, h, full, 64 * d)
        q, m = codes64(blocks)
        scale = (m.float() / 127.0)
        val = (q * scale.double()[..., None]).view(b, h, full * 64, d)
        out.append(torch.cat([val, x[:, :, full * 64:]], 2))
        parts.append((q.view(b, h, full, 64, d), scale))
    return out, parts


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("total,cuts", [(1, ()), (63, ()), (64, ()), (65, ()), (64, (63,)), (128, (1, 2, 64, 127)), (200, (130,)),
                                        (257, (63, 64, 65, 191, 192)), (300, (100, 200)), (130, tuple(range(1, 130)))])
def test_append_and_read(total, cuts, dtype):
    b, h = 2, 3
    c, k, v = filled(b, h, total, dtype, seeded(total + len(cuts)), cuts=cuts, capacity=total + 70)
    values, parts = held64(k, v)
    full, rest = total // 64, total % 64
    blocks = c.k_scale.shape[2]
    (qk, sk), (qv, sv) = parts
    got_k = c.k.cpu().view(b, h, blocks, 64, 128)
    assert torch.equal(got_k[:, :, :full].double(), qk) and torch.equal(c.v.cpu()[:, :, :full].transpose(3, 4).double(), qv)
    assert torch.equal(c.k_scale.cpu()[:, :, :full], sk) and torch.equal(c.v_scale.cpu()[:, :, :full], sv)
    # behind the last position everything is as it was
    assert (got_k[:, :, full:] == 111).all() and (c.v.cpu()[:, :, full:] == -111).all()
    assert torch.isnan(c.k_scale[:, :, full:]).all() and torch.isnan(c.v_scale[:, :, full:]).all()
    if rest:
        assert torch.equal(c.k_tail.cpu()[:, :, :rest], k.transpose(1, 2)[:, :, full * 64:])
        assert torch.equal(c.v_tail.cpu()[..., :rest].transpose(2, 3), v.transpose(1, 2)[:, :, full * 64:])
    for out in (dtype, torch.float32, torch.bfloat16):
        rk, rv = I8.read(c, total, dtype=out)
        for got, want in ((rk, values[0]), (rv, values[1])):
            u = torch.finfo(out).eps / 2
            tol = want.abs() * (u * (1 + 2.0 ** -10) + 2.0 ** -23) + (2.0 ** -25 if out == torch.float16 else 0)
            close(got, want, tol)


def test_append_strided_sources_and_nonfinite_block():
    gen = seeded(3)
    b, s, h = 2, 130, 2
    qkv = randn(b, s, 4 * h, 128, gen=gen, dtype=torch.bfloat16).cuda()
    k, v = qkv[:, :, h:2 * h], qkv[:, :, 2 * h:3 * h]
    c, d = poisoned(b, h, s, torch.bfloat16), poisoned(b, h, s, torch.bfloat16)
    I8.append(k, v, c, 0)
    I8.append(k.contiguous(), v.contiguous(), d, 0)
    for x, y in zip(I8.read(c, s), I8.read(d, s)):
        assert torch.equal(x, y)
    k2 = k.clone()
    k2[0, 70, 1, 5] = math.inf
    I8.append(k2, v, c, 0)
    rk, rv = I8.read(c, s)
    assert torch.isnan(rk[0, 1, 64:128]).all() and torch.equal(rv, I8.read(d, s)[1])
    rk[0, 1, 64:128] = I8.read(d, s)[0][0, 1, 64:128]
    assert torch.equal(rk, I8.read(d, s)[0])


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("b,hq,h,cuts", [(1, 4, 1, (1, 2)), (2, 8, 2, (70, 71, 130)), (3, 5, 5, (64, 65, 128)), (1, 32, 8, (200, 201))])
def test_norm_rope_append(b, hq, h, cuts, dtype):
    """Norm + rotation + append in chunks: the keys within their roundings of 64 bits, and the cache bit for bit that of the
    same keys appended; whatever the chunks."""
    gen = seeded(sum(cuts))
    t = cuts[-1]
    qkv = randn(b, t, hq + 2 * h, 128, gen=gen, dtype=dtype)
    wq, wk = ((1 + 0.1 * torch.randn(128, generator=gen)).to(dtype) for _ in range(2))
    ang = torch.rand(b, t, 64, generator=gen) * 6.28
    cos, sin = (torch.cat([f(ang)] * 2, -1).to(dtype) for f in (torch.cos, torch.sin))
    dev = qkv.cuda()

    def ref(x, w):
        x = x.double()
        n = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
        rot = torch.cat([-n[..., 64:], n[..., :64]], -1)
        c, s = cos.double()[:, :, None], sin.double()[:, :, None]
        return n * c + rot * s, n.abs() * c.abs() + rot.abs() * s.abs()

    def run(cuts):
        c, qs, at = poisoned(b, h, t + 64, dtype), [], 0
        for end in cuts:
            part = dev[:, at:end]
            qs.append(I8.norm_rope_append(part[:, :, :hq], part[:, :, hq:hq + h], part[:, :, hq + h:], wq.cuda(), wk.cuda(),
                                          cos[:, at:end].contiguous().cuda(), sin[:, at:end].contiguous().cuda(), c, at))
            at = end
        return c, torch.cat(qs, 1)
    c, q = run(cuts)
    want, mag = ref(qkv[:, :, :hq], wq)
    # the norm: a sum of 128 squares, rsqrt, two products; the rotation: two products and a sum
    close(q, want, want.abs() * torch.finfo(dtype).eps / 2 * (1 + 2.0 ** -8) + mag * 2.0 ** -19 + 2.0 ** -24)
    whole, qw = run((t,))
    assert torch.equal(q, qw)
    # the keys as 16-bit numbers: those of a cache that never fills a block
    keys = []
    for at in range(0, t, 63):
        d, end = poisoned(b, h, 64, dtype), min(t, at + 63)
        part = dev[:, at:end]
        I8.norm_rope_append(part[:, :, :hq], part[:, :, hq:hq + h], part[:, :, hq + h:], wq.cuda(), wk.cuda(),
                            cos[:, at:end].contiguous().cuda(), sin[:, at:end].contiguous().cuda(), d, 0)
        keys.append(d.k_tail[:, :, :end - at].transpose(1, 2))
    k = torch.cat(keys, 1)
    want, mag = ref(qkv[:, :, hq:hq + h], wk)
    close(k, want, want.abs() * torch.finfo(dtype).eps / 2 * (1 + 2.0 ** -8) + mag * 2.0 ** -19 + 2.0 ** -24)
    plain = poisoned(b, h, t + 64, dtype)
    I8.append(k, dev[:, :, hq + h:], plain, 0)
    n, rest = t // 64, t % 64
    for x in (c, whole):
        assert torch.equal(x.k, plain.k) and torch.equal(x.v, plain.v)
        assert torch.equal(x.k_scale[:, :, :n], plain.k_scale[:, :, :n]) and torch.equal(x.v_scale[:, :, :n], plain.v_scale[:, :, :n])
        assert torch.equal(x.k_tail[:, :, :rest], plain.k_tail[:, :, :rest]) and torch.equal(x.v_tail[..., :rest], plain.v_tail[..., :rest])


# ---------------------------------------------------------------- attention
def attention64(q, k, v, start, scale, full):
    """In 64 bits, k, v [B, Hkv, T, 128]: o, sum p |v| over the 8-bit blocks and over the tail, the largest score's sum of
    magnitudes, and (largest p) * sum |v| over the 8-bit blocks that a query sees."""
    b, s, hq, d = q.shape
    hkv, t = k.shape[1], k.shape[2]
    qf = q.double().transpose(1, 2).reshape(b, hkv, hq // hkv, s, d)
    z = torch.matmul(qf, k[:, :, None].transpose(3, 4)) * scale
    zerr = torch.matmul(qf.abs(), k[:, :, None].abs().transpose(3, 4)).amax((-1), keepdim=True) * scale
    mask = torch.arange(t)[None] > start + torch.arange(s)[:, None]
    p = torch.softmax(z.masked_fill(mask, -math.inf), -1)
    shape = lambda x: x.reshape(b, hq, s, d).transpose(1, 2)  # noqa: E731
    o = torch.matmul(p, v[:, :, None])
    n = full * 64
    a8 = torch.matmul(p[..., :n], v[:, :, None, :n].abs())
    at = torch.matmul(p[..., n:], v[:, :, None, n:].abs())
    seen = torch.matmul((~mask[:, :n]).double().expand(b, hkv, 1, s, n), v[:, :, None, :n].abs()) * p.amax(-1, keepdim=True)
    return shape(o), shape(a8), shape(at), zerr.reshape(b, hq, s, 1).transpose(1, 2), shape(seen)


def check_attention(o, q, values, start, scale, dtype):
    full = (start + q.shape[1]) // 64
    ref, a8, at, zerr, seen = attention64(q, *values, start, scale, full)
    u = torch.finfo(dtype).eps / 2
    # a score: 128 products summed in fp32 (any order: 128 * 2^-24 of the sum of magnitudes), two scales, log2(e): in the
    # exponent, twice (numerator and sum).  p (relative to the largest) in fp16: 2^-11 where normal; below, 2^-25 absolute,
    # of a value scale that is at least 1 / 16 of O's unit.  The tail's p in the activation type, fp16's again 2^-25 absolute.
    # Sums over t and the joins: 2^-16.
    dz = zerr * 136 * 2.0 ** -24 * 2
    tol = ref.abs() * u * (1 + 2.0 ** -8) + (a8 + at) * (dz + 2.0 ** -16) + a8 * 2.0 ** -11 + at * u + seen * 2.0 ** -21 + 2.0 ** -24
    close(o, ref, tol)


ATT = [(1, 4, 4, 1, 0), (1, 4, 1, 1, 62), (2, 8, 2, 1, 63), (1, 8, 2, 1, 64), (3, 8, 2, 1, 200), (1, 5, 1, 1, 127), (1, 16, 1, 1, 300),
       (1, 32, 1, 1, 500), (2, 12, 4, 1, 1000), (1, 32, 8, 1, 4095), (1, 4, 2, 2, 63), (1, 8, 2, 4, 60), (1, 8, 2, 5, 1000),
       (2, 4, 1, 16, 0), (1, 8, 2, 64, 0), (1, 8, 2, 65, 0), (1, 8, 2, 100, 30), (1, 4, 4, 300, 0), (2, 8, 2, 129, 500),
       (1, 7, 1, 70, 100), (1, 64, 2, 9, 77), (1, 8, 2, 700, 100)]


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("b,hq,hkv,s,start", ATT)
def test_attention(b, hq, hkv, s, start, dtype):
    gen = seeded(b + hq + s + start)
    c, k, v = filled(b, hkv, start + s, dtype, gen, cuts=(start,) if start else (), capacity=start + s + 100)
    q = randn(b, s, hq, 128, gen=gen, dtype=dtype)
    o = I8.attention(q.cuda(), c, start)
    check_attention(o, q, held64(k, v)[0], start, 128 ** -0.5, dtype)


@pytest.mark.parametrize("dtype", DT)
def test_attention_value_scales_far_apart(dtype):
    """Blocks whose value scales differ by up to 2^40: O changes its units, and a block that dominates is exact whatever the
    others' scales; strided queries and an own softmax scale."""
    gen = seeded(8)
    b, h, t = 1, 2, 64 * 9 + 10
    k, v = randn(b, t, h, 128, gen=gen, dtype=dtype), randn(b, t, h, 128, gen=gen)
    exps = [0, -3, 5, -6, 3, -7, 8, 0, 4, 0] if dtype == torch.float16 else [0, -20, 5, -40, 17, -13, 18, -22, 20, 0]
    for i, e in enumerate(exps):
        v[:, 64 * i:64 * (i + 1)] *= 2.0 ** e
    v[:, 64:128, 1] = 0   # a block of zeros: scale 0
    k[:, 192:256, 1] = 0
    k[:, t - 74:t - 10, 0] = 0   # the last whole block, which some of the queries below see in part
    v = v.to(dtype)
    c = poisoned(b, h, t, dtype)
    I8.append(k.cuda(), v.cuda(), c, 0)
    for s in (1, 3, 40, 100):
        wide = randn(b, s, 6, 256, gen=gen, dtype=dtype, scale=2.0).cuda()
        q = wide[:, :, 1:5, 64:192]
        o = I8.attention(q, c, t - s, scale=0.3)
        check_attention(o, q.cpu(), held64(k, v)[0], t - s, 0.3, dtype)


def test_cache_started_again_at_a_block():
    """Positions appended again from a multiple of 64 on: as if the earlier ones had never been."""
    gen = seeded(7)
    c, k, v = filled(2, 2, 200, torch.bfloat16, gen)
    k2, v2 = (randn(2, 90, 2, 128, gen=gen, dtype=torch.bfloat16).cuda() for _ in range(2))
    fresh = poisoned(2, 2, 200, torch.bfloat16)
    for start in (128, 64, 0):
        I8.append(k2, v2, c, start)
        if start:
            I8.append(k[:, :start].cuda(), v[:, :start].cuda(), fresh, 0)
        I8.append(k2, v2, fresh, start)
        for got, want in zip(I8.read(c, start + 90), I8.read(fresh, start + 90)):
            assert torch.equal(got, want), start


def test_attention_masked_nonfinite_positions():
    """A NaN key or value reaches the queries that see its position (or, once quantised, its block), no others."""
    gen = seeded(4)
    b, hq, h, s, start = 1, 4, 2, 40, 70   # positions 70 .. 109: the tail holds 64 .. 109
    c, k, v = filled(b, h, start + s, torch.bfloat16, gen, cuts=(start,))
    q = randn(b, s, hq, 128, gen=gen, dtype=torch.bfloat16).cuda()
    want = I8.attention(q, c, start)
    c.k_tail[0, 0, 100 - 64, 3] = math.nan
    got = I8.attention(q, c, start)
    assert torch.equal(got[:, :100 - start], want[:, :100 - start]) and torch.equal(got[:, :, 2:], want[:, :, 2:])
    assert torch.isnan(got[:, 100 - start:, :2]).all()
    # whole blocks: two of them, queries in both; a NaN scale of the second leaves the queries of the first alone
    c, k, v = filled(b, h, 128, torch.bfloat16, gen)
    q = randn(b, 128, hq, 128, gen=gen, dtype=torch.bfloat16).cuda()
    want = I8.attention(q, c, 0)
    for scales in (c.k_scale, c.v_scale):
        keep = scales.clone()
        scales[0, 1, 1] = math.nan
        got = I8.attention(q, c, 0)
        assert torch.equal(got[:, :64], want[:, :64]) and torch.equal(got[:, :, :2], want[:, :, :2])
        assert torch.isnan(got[:, 64:, 2:]).all()
        scales.copy_(keep)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("s", [4, 40], ids=["few", "many"])
def test_attention_masked_nonfinite_tail_values(s, dtype):
    """An infinite or NaN value in the tail: NaN for the queries that see its position, nothing for the others."""
    gen = seeded(5)
    b, hq, h, total = 2, 4, 2, 110
    c, k, v = filled(b, h, total, dtype, gen)
    q = randn(b, s, hq, 128, gen=gen, dtype=dtype).cuda()
    start = total - s
    want = I8.attention(q, c, start)
    for pos, dim, x in ((total - 1, 0, math.nan), (total - 3, 77, math.inf), (total - 2, 127, -math.inf), (64, 5, math.nan)):
        keep = c.v_tail[1, 1, dim, pos - 64].clone()
        c.v_tail[1, 1, dim, pos - 64] = x
        got = I8.attention(q, c, start)
        sees = max(pos - start, 0)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1, :, :2], want[1, :, :2]), (pos, dim)
        assert torch.equal(got[1, :sees, 2:], want[1, :sees, 2:]) and torch.isnan(got[1, sees:, 2:]).all(), (pos, dim)
        c.v_tail[1, 1, dim, pos - 64] = keep


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("s", [1, 20])
def test_attention_many_tiny_weights(s, dtype):
    """One strong key beside 40000 weak ones, whose weights of about e^-11 are subnormal in fp16 where the strong one's is 1."""
    total = 40000
    gen = seeded(11)
    k, v = torch.zeros(1, total, 1, 128), 1 + 0.01 * torch.randn(1, total, 1, 128, generator=gen)
    k[..., 0] = -11 * 128 ** 0.5 / 8
    k[0, 70], v[0, 70] = 0, -1
    q = torch.zeros(1, s, 4, 128)
    q[..., 0] = 8
    c = I8.LayerCache.empty(1, 1, total, device="cuda", dtype=dtype)
    I8.append(k.to(dtype).cuda(), v.to(dtype).cuda(), c, 0)
    y = I8.attention(q.to(dtype).cuda(), c, total - s)[0, -1].double().cpu()
    kk, vv = (x[0, 0].double().cpu() for x in I8.read(c, total, dtype=torch.float32))
    w = torch.softmax(8.0 * kk[:, 0] * 128 ** -0.5, 0) @ vv
    # P and its sum each rounded by at most 2^-11 (fp16; here the weak ones all alike), subnormal ones by 2^-25 of a weight of
    # 2^-16: 2^-9; |v| is 1; the output's own rounding
    assert ((y - w).abs() <= 2 * (2.0 ** -11 + 2.0 ** -9) + w.abs() * torch.finfo(dtype).eps / 2).all()


@pytest.mark.parametrize("s", [1, 70])
def test_attention_nonfinite_values_of_no_weight(s):
    """A block of values that were not finite makes a query that sees it NaN, however small the block's weight."""
    gen = seeded(6)
    k, v = (randn(1, 192 + s, 1, 128, gen=gen, dtype=torch.float32) for _ in range(2))
    q = randn(1, s, 2, 128, gen=gen, dtype=torch.float32)
    k[:, :64] = -40.0   # its scores lie thousands below the others': weights of 0
    q += 40.0
    c = poisoned(1, 1, 192 + s, torch.bfloat16)
    I8.append(k.bfloat16().cuda(), v.bfloat16().cuda(), c, 0)
    assert torch.isfinite(I8.attention(q.bfloat16().cuda(), c, 192)).all()
    c.v_scale[0, 0, 0] = math.nan
    assert torch.isnan(I8.attention(q.bfloat16().cuda(), c, 192)).all()


def test_cache_past_32_bits():
    """2.2 million positions of 8 heads: codes, 16-bit sources and read-back values past 2^31 elements.  The last head against
    the same calls on a cache of that head alone."""
    total, h, dtype = 2_200_037, 8, torch.bfloat16
    gen = torch.Generator(device="cuda").manual_seed(8)
    k, v = (torch.randn((1, total, h, 128), generator=gen, device="cuda", dtype=dtype) for _ in range(2))
    c = I8.LayerCache.empty(1, h, total, device="cuda", dtype=dtype)
    one = I8.LayerCache.empty(1, 1, total, device="cuda", dtype=dtype)
    at = 0
    for end in (1_500_000, total):
        I8.append(k[:, at:end], v[:, at:end], c, at)
        I8.append(k[:, at:end, 7:], v[:, at:end, 7:], one, at)
        at = end
    full, rest = total // 64, total % 64
    assert torch.equal(c.k[:, 7:, :full * 64], one.k[:, :, :full * 64]) and torch.equal(c.v[:, 7:, :full], one.v[:, :, :full])
    assert torch.equal(c.k_tail[:, 7:, :rest], one.k_tail[:, :, :rest])
    for got, want in zip(I8.read(c, total), I8.read(one, total)):
        assert torch.equal(got[:, 7:], want)
    del k, got, want
    top = float(v[:, :, 7].abs().max())
    for s in (1, 40):
        q = torch.randn((1, s, 16, 128), generator=gen, device="cuda", dtype=dtype) * 4
        a = I8.attention(q, c, total - s)[:, :, 14:].double()
        b = I8.attention(q[:, :, 14:], one, total - s).double()
        # two splits of one sum: P rounded to fp16 in either (2^-11 of sum p |v| <= top), fp32 sums and joins, an output rounding
        tol = 2 * top * (2.0 ** -11 + 2.0 ** -15)
        assert ((a - b).abs() <= tol + b.abs() * torch.finfo(dtype).eps * (1 + 2.0 ** -8)).all()
        # the outputs stand clear of it, so that another head's would show: scores of deviation 4 leave the largest of 2.2
        # million (about 5 deviations up) more than a hundredth of the sum, 2.2e6 e^8 against e^20 and more: 0.07 of a value
        assert float(b.abs().max()) > 10 * tol


def test_rows_past_32_bits():
    """70000 rows of 32768: values and codes past 2^31 elements; rows here and there against calls on those rows alone."""
    gen = torch.Generator(device="cuda").manual_seed(9)
    x = torch.randn((70000, 32768), generator=gen, device="cuda", dtype=torch.bfloat16)
    w = torch.rand(32768, generator=gen, device="cuda").bfloat16()
    wq, ws = I8.quantize_rows(x[:48])
    parts = (slice(0, 3), slice(65530, 65545), slice(69990, 70000))
    q, s = I8.quantize_rows(x)
    y = I8.linear(q, s, wq, ws)
    for p in parts:
        a, b = I8.quantize_rows(x[p])
        assert torch.equal(q[p], a) and torch.equal(s[p], b) and torch.equal(y[p], I8.linear(a, b, wq, ws))
    del q, s, y
    q, s, total = I8.rms_norm(x, w, 1e-6, residual=x)
    for p in parts:
        for got, want in zip((q[p], s[p], total[p]), I8.rms_norm(x[p], w, 1e-6, residual=x[p])):
            assert torch.equal(got, want)


def test_device_positions_and_graph_replay():
    """One captured step (append + attention at a device position) replayed over a block's end against eager calls."""
    gen = seeded(6)
    b, hq, h, cap, start = 2, 8, 2, 200, 120
    c, k, v = filled(b, h, start, torch.bfloat16, gen, capacity=cap)
    d = I8.LayerCache(*(t.clone() for t in (c.k, c.v, c.k_scale, c.v_scale, c.k_tail, c.v_tail)))
    pos = torch.tensor([start], device="cuda")
    new = [[randn(b, 1, n, 128, gen=gen, dtype=torch.bfloat16).cuda() for n in (hq, h, h)] for _ in range(20)]
    q, kk, vv = (t.clone() for t in new[0])
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=stream):
        I8.append(kk, vv, c, 0, pos)
        o = I8.attention(q, c, 0, pos)
        pos += 1
    torch.cuda.current_stream().wait_stream(stream)
    for i, (a, bk, bv) in enumerate(new):
        q.copy_(a), kk.copy_(bk), vv.copy_(bv)
        graph.replay()
        I8.append(bk, bv, d, start + i)
        eager = I8.attention(a, d, start + i)
        k, v = torch.cat([k, bk.cpu()], 1), torch.cat([v, bv.cpu()], 1)
        values = held64(k, v)[0]
        for got in (o, eager):   # the two split the positions differently
            check_attention(got, a.cpu(), values, start + i, 128 ** -0.5, torch.bfloat16)
    n = (start + 20) // 64
    assert torch.equal(c.k[:, :, :n * 64], d.k[:, :, :n * 64]) and torch.equal(c.v[:, :, :n], d.v[:, :, :n])
    # positions outside the capacity are skipped
    bits = lambda: [t.clone() for t in (c.k, c.v, c.k_tail.view(torch.int16), c.v_tail.view(torch.int16))]  # noqa: E731
    keep = bits()
    for bad in (c.capacity, c.capacity + 5, -1):
        I8.append(kk, vv, c, 0, torch.tensor([bad], device="cuda"))
    assert all(torch.equal(x, y) for x, y in zip(keep, bits()))


def test_refusals_on_the_device():
    q = torch.zeros(1, 1, 34, 128, dtype=torch.bfloat16, device="cuda")
    w, t = torch.ones(128, dtype=torch.bfloat16, device="cuda"), torch.ones(1, 1, 128, dtype=torch.bfloat16, device="cuda")
    c = poisoned(1, 2, 64, torch.bfloat16)
    kv = q[:, :, :2]
    for bad in (lambda: I8.norm_rope_append(q, kv, kv, w, w, t, t, c, 64), lambda: I8.norm_rope_append(q, kv, kv, w, w, t, t, c, 0, eps=-1.0),
                lambda: I8.norm_rope_append(q, kv, kv, w[:64], w, t, t, c, 0), lambda: I8.norm_rope_append(q, kv, kv, w, w, t[0], t, c, 0),
                lambda: I8.norm_rope_append(q, q[:, :, :1], q[:, :, :1], w, w, t, t, c, 0),
                lambda: I8.attention(q[:, :, :32], c, 0, scale=0.0), lambda: I8.attention(q[:, :, :33], c, 0),
                lambda: I8.attention(q[:, :, :32], c, 64), lambda: I8.attention(q[:, :, :32], c, -1),
                lambda: I8.append(kv, q[:, :, :1], c, 0), lambda: I8.append(kv.expand(1, 2, 2, 128), kv.expand(1, 2, 2, 128), c, 63),
                lambda: I8.read(c, 65), lambda: I8.read(c, 0), lambda: I8.append(kv, kv, c, True)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        I8.attention(q.half()[:, :, :32], c, 0)


def test_determinism_and_side_stream():
    gen = seeded(12)
    c, k, v = filled(1, 2, 700, torch.bfloat16, gen)
    q = randn(1, 1, 8, 128, gen=gen, dtype=torch.bfloat16).cuda()
    want = I8.attention(q, c, 699)
    x = randn(5, 1024, gen=gen, dtype=torch.bfloat16).cuda()
    w = I8.quantize_rows(randn(300, 1024, gen=gen, dtype=torch.bfloat16).cuda())
    y = I8.linear(*I8.quantize_rows(x), *w)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for _ in range(3):
            assert torch.equal(I8.attention(q, c, 699), want)
            assert torch.equal(I8.linear(*I8.quantize_rows(x), *w), y)
    torch.cuda.current_stream().wait_stream(stream)


# ---------------------------------------------------------------- a layer of them together
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("s", [1, 3, 70])
def test_chain(s, dtype):
    """norm -> Q/K/V -> cache -> attention -> output projection with its residual -> norm with its residual -> gate/up, each
    step against its own definition on the step's own inputs."""
    gen = seeded(s)
    hid, hq, h, start = 512, 4, 2, 100
    x = randn(1, s, hid, gen=gen, dtype=dtype).cuda()
    nw = (1 + 0.1 * torch.randn(hid, generator=gen)).to(dtype).cuda()
    ws = [I8.quantize_rows(randn(n, k, gen=gen, dtype=dtype, scale=0.05).cuda())
          for n, k in ((hq * 128, hid), (h * 128, hid), (h * 128, hid), (hid, hq * 128), (1024, hid), (1024, hid))]
    c, k0, v0 = filled(1, h, start, dtype, gen, capacity=start + s)
    a, sa = I8.rms_norm(x, nw, 1e-6)
    q, k, v = I8.projections(a, sa, ws[:3], dtype=dtype)
    q, k, v = q.view(1, s, hq, 128), k.view(1, s, h, 128), v.view(1, s, h, 128)
    I8.append(k, v, c, start)
    o = I8.attention(q, c, start)
    values = held64(torch.cat([k0, k.cpu()], 1), torch.cat([v0, v.cpu()], 1))[0]
    check_attention(o, q.cpu(), values, start, 128 ** -0.5, dtype)
    b, sb = I8.quantize_rows(o.view(1, s, -1))
    y = I8.linear(b, sb, *ws[3], dtype=dtype, residual=x)
    p = product64(b.cpu().view(s, -1), sb.cpu().view(s), *(t.cpu() for t in ws[3]))
    ref = p + x.double().cpu().view(s, hid)
    close(y.view(s, hid), ref, ref.abs() * torch.finfo(dtype).eps / 2 * (1 + 2.0 ** -10) + (p.abs() + ref.abs()) * 2.0 ** -22)
    d, sd, total = I8.rms_norm(y, nw, 1e-6, residual=x)
    assert torch.equal(total, (y.float() + x.float()).to(dtype))
    z = I8.gate_up_swiglu(d, sd, *ws[4], *ws[5], dtype=dtype)
    g, u = (product64(d.cpu().view(s, -1), sd.cpu().view(s), *(t.cpu() for t in w)) for w in ws[4:])
    ref = g * torch.sigmoid(g) * u
    close(z.view(s, -1), ref, ref.abs() * (torch.finfo(dtype).eps / 2 * (1 + 2.0 ** -10) + (12 + 6 * g.abs()) * 2.0 ** -23) + 1e-7)


@pytest.mark.parametrize("t,s", [(2, 1), (5, 5), (40, 1), (63, 1), (17, 17), (63, 40), (63, 63)])
def test_attention_short_contexts(t, s):
    """Below 64 positions every one of them is in the tail: outputs as near to 64 bits as their own rounding to bf16 lets them."""
    gen = seeded(t + s)
    c, k, v = filled(2, 2, t, torch.bfloat16, gen, wide=False)
    q = randn(2, s, 8, 128, gen=gen, dtype=torch.bfloat16, scale=0.3)
    o = I8.attention(q.cuda(), c, t - s)
    ref, _, at, zerr, _ = attention64(q, *held64(k, v)[0], t - s, 128 ** -0.5, 0)
    # scores and sums as in check_attention; P in two bf16 terms: what the first leaves (2^-8 of it) is rounded by 2^-8
    dz = zerr * 136 * 2.0 ** -24 * 2
    close(o, ref, ref.abs() * 2.0 ** -8 * (1 + 2.0 ** -8) + at * (dz + 2.0 ** -16 + 2.0 ** -16) + 2.0 ** -24)


@pytest.mark.parametrize("exps", [(0, -55, -110), (0, -40, -80, -120), (0, -30, -60, -90, -120), (0, -55, -110, 4, -70, -100), (-60, 0, -110)])
@pytest.mark.parametrize("s", [1, 40])
def test_attention_value_scales_that_keep_falling(s, exps):
    """Blocks whose values fall by more in all than a 32-bit sum in one unit could follow: the large ones' values stay finite."""
    gen = seeded(len(exps))
    for tail in (0, 10):
        t = 64 * len(exps) + tail
        k, v = randn(1, t, 2, 128, gen=gen, dtype=torch.bfloat16), randn(1, t, 2, 128, gen=gen)
        for i, e in enumerate(exps):
            v[:, 64 * i:64 * (i + 1)] *= 2.0 ** e
        v[:, 64 * len(exps):] *= 2.0 ** exps[-1]
        v = v.bfloat16()
        c = poisoned(1, 2, t, torch.bfloat16)
        I8.append(k.cuda(), v.cuda(), c, 0)
        q = randn(1, s, 4, 128, gen=gen, dtype=torch.bfloat16)
        check_attention(I8.attention(q.cuda(), c, t - s), q, held64(k, v)[0], t - s, 128 ** -0.5, torch.bfloat16)


def test_attention_value_scales_that_keep_falling_over_a_full_launch():
    """The same where the rows fill the CUs, so that each wave goes over several of the blocks."""
    gen = seeded(3)
    exps, b = (20, -36, -92, -118), 512
    t = 64 * 4 * len(exps)
    k, v = randn(1, t, 1, 128, gen=gen, dtype=torch.bfloat16), randn(1, t, 1, 128, gen=gen)
    for i, e in enumerate(exps):   # four waves take every fourth block each
        v[:, 256 * i:256 * (i + 1)] *= 2.0 ** e
    v = v.bfloat16()
    c = poisoned(b, 1, t, torch.bfloat16)
    I8.append(k.cuda().expand(b, t, 1, 128), v.cuda().expand(b, t, 1, 128), c, 0)
    q = randn(1, 1, 2, 128, gen=gen, dtype=torch.bfloat16)
    o = I8.attention(q.cuda().expand(b, 1, 2, 128), c, t - 1)
    check_attention(o[:1], q, held64(k, v)[0], t - 1, 128 ** -0.5, torch.bfloat16)
    assert torch.equal(o, o[:1].expand_as(o))


@pytest.mark.parametrize("s", [1, 40])
def test_attention_key_scales_that_vanish(s):
    """Keys so small that their scale times the softmax scale is below the least 32-bit number: every score is 0."""
    gen = seeded(2)
    t = 64 * 3
    k, v = randn(1, t, 2, 128, gen=gen, scale=2.0 ** -100).bfloat16(), randn(1, t, 2, 128, gen=gen, dtype=torch.bfloat16)
    c = poisoned(1, 2, t, torch.bfloat16)
    I8.append(k.cuda(), v.cuda(), c, 0)
    q = randn(1, s, 4, 128, gen=gen, dtype=torch.bfloat16, scale=4.0)
    check_attention(I8.attention(q.cuda(), c, t - s, scale=1e-20), q, held64(k, v)[0], t - s, 1e-20, torch.bfloat16)


def test_going_back_into_a_quantised_block_is_refused():
    """The tail holds the unfinished block alone: shorter reads and earlier appends go to a whole block or to a tail position."""
    gen = seeded(9)
    c, k, v = filled(1, 2, 200, torch.bfloat16, gen, cuts=(100,))   # tail: positions 192 .. 199
    q = randn(1, 3, 4, 128, gen=gen, dtype=torch.bfloat16).cuda()
    new = randn(1, 3, 2, 128, gen=gen, dtype=torch.bfloat16).cuda()
    w, t = torch.ones(128, dtype=torch.bfloat16, device="cuda"), torch.ones(1, 3, 128, dtype=torch.bfloat16, device="cuda")
    bits = lambda: [x.clone() for x in (c.k, c.v, c.k_tail.view(torch.int16), c.v_tail.view(torch.int16))]  # noqa: E731
    keep = bits()
    for bad in (lambda: I8.read(c, 50), lambda: I8.read(c, 191), lambda: I8.attention(q, c, 100), lambda: I8.attention(q, c, 188),
                lambda: I8.append(new, new, c, 70), lambda: I8.append(new, new, c, 191),
                lambda: I8.norm_rope_append(q, new, new, w, w, t, t, c, 1)):
        with pytest.raises(ValueError, match='quantised block'):
            bad()
    assert all(torch.equal(a, b) for a, b in zip(keep, bits()))
    values = held64(k, v)[0]
    for n in (64, 128, 192, 195, 200):   # what it holds still
        for got, want in zip(I8.read(c, n, dtype=torch.float32), values):
            close(got, want[:, :, :n], want[:, :, :n].abs() * 2.0 ** -22)
        check_attention(I8.attention(q, c, n - 3), q.cpu(), [x[:, :, :n] for x in values], n - 3, 128 ** -0.5, torch.bfloat16)
    I8.append(new, new, c, 194)   # over the tail's own positions
    k[:, 194:197], v[:, 194:197] = new.cpu(), new.cpu()
    for got, want in zip(I8.read(c, 197, dtype=torch.float32), held64(k[:, :197], v[:, :197])[0]):
        close(got, want, want.abs() * 2.0 ** -22)
    I8.append(new, new, c, 128)   # back to a block: the positions from there on are others
    with pytest.raises(ValueError, match='quantised block'):
        I8.read(c, 120)
    assert torch.equal(I8.read(c, 131)[0][:, :, 128:], new.transpose(1, 2))
    # device positions, and captured calls, are not known on the host
    I8.append(new[:, :1], new[:, :1], c, 0, torch.tensor([131], device="cuda"))
    assert torch.equal(I8.read(c, 132)[0][:, :, 131:], new[:, :1].transpose(1, 2))
    d, stream, graph = poisoned(1, 2, 200, torch.bfloat16), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    kd, vd = k.cuda(), v.cuda()
    with torch.cuda.graph(graph, stream=stream):
        I8.append(kd, vd, d, 0)
    torch.cuda.current_stream().wait_stream(stream)
    I8.append(kd[:, :10], vd[:, :10], d, 0)
    assert torch.equal(I8.read(d, 10)[0], kd[:, :10].transpose(1, 2))
    for _ in range(2):
        graph.replay()
        for got, want in zip(I8.read(d, 200, dtype=torch.float32), held64(k, v)[0]):
            close(got, want, want.abs() * 2.0 ** -22)
        I8.append(kd[:, :10], vd[:, :10], d, 0)


@pytest.mark.parametrize("b,hq,h", [(1, 8, 2), (3, 32, 8)])
@pytest.mark.parametrize("dtype", DT)
def test_captured_step_over_several_splits(b, hq, h, dtype):
    """A captured step in a long capacity, at lengths of several splits (which follow from the position alone): the bits of the
    eager call, and both against 64 bits."""
    gen = seeded(b)
    lengths, cap = (255, 300, 769, 1500, 3000), 6000
    k, v = randn(b, lengths[-1] + 1, h, 128, gen=gen, dtype=dtype), randn(b, lengths[-1] + 1, h, 128, gen=gen, dtype=dtype)
    kd, vd = k.cuda(), v.cuda()
    c, pos = poisoned(b, h, cap, dtype), torch.zeros(1, dtype=torch.int64, device="cuda")
    q, kk, vv = (torch.zeros(b, 1, n, 128, dtype=dtype, device="cuda") for n in (hq, h, h))
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=stream):
        I8.append(kk, vv, c, 0, pos)
        o = I8.attention(q, c, 0, pos)
    torch.cuda.current_stream().wait_stream(stream)
    for n in lengths:
        I8.append(kd[:, :n], vd[:, :n], c, 0)
        d = I8.LayerCache(*(t.clone() for t in (c.k, c.v, c.k_scale, c.v_scale, c.k_tail, c.v_tail)))
        new = randn(b, 1, hq, 128, gen=gen, dtype=dtype)
        q.copy_(new), kk.copy_(kd[:, n:n + 1]), vv.copy_(vd[:, n:n + 1]), pos.fill_(n)
        graph.replay()
        I8.append(kd[:, n:n + 1], vd[:, n:n + 1], d, n)
        assert torch.equal(o, I8.attention(q, d, n)), n
        check_attention(o, new, held64(k[:, :n + 1], v[:, :n + 1])[0], n, 128 ** -0.5, dtype)


def test_going_back_over_a_block_s_last_token():
    """A block's last append leaves the tail as it was: that token can be taken back, and another one appended."""
    gen = seeded(10)
    for cut in (127, 100):
        c, k, v = filled(1, 2, 128, torch.bfloat16, gen, cuts=(cut,))
        close(I8.read(c, cut, dtype=torch.float32)[0], held64(k[:, :cut], v[:, :cut])[0][0], 2.0 ** -22 * k.double().transpose(1, 2)[:, :, :cut].abs() + 2.0 ** -22)
        k2, v2 = (randn(1, 128 - cut, 2, 128, gen=gen, dtype=torch.bfloat16, scale=0.5) for _ in range(2))
        I8.append(k2.cuda(), v2.cuda(), c, cut)
        fresh = poisoned(1, 2, 128, torch.bfloat16)
        I8.append(torch.cat([k[:, :cut], k2], 1).cuda(), torch.cat([v[:, :cut], v2], 1).cuda(), fresh, 0)
        for got, want in zip(I8.read(c, 128), I8.read(fresh, 128)):
            assert torch.equal(got, want)
        with pytest.raises(ValueError, match='quantised block'):
            I8.append(k2.cuda()[:, :1], v2.cuda()[:, :1], c, {127: 62, 100: 101}[cut])
