"""Log probabilities of tokens, entropies, alternatives and gradients against the formulas in 64 bits.

Tolerances (e = 2^-24, c = 1 / temperature, d = z - max z): an exponential has three roundings in its argument, which matter
for |c d| up to 20 (below, it is less than 2^-28 of the sum), and two of its own; a sum is a chain of at most 64 additions in a
thread, 8 over the workgroup and 8 over the slices.  Together the sum is off by less than 160 e of itself, and so is its logarithm in
absolute terms.  A log probability adds two roundings of c d: 4 e c |d|.  The entropy's second part is off by 160 + 4 c |d| (20 of
them at most) e of itself, and it is at most the entropy."""
import math

import pytest
import torch

from _util import seeded

from qwen3_triton.kernels import logprobs
from qwen3_triton.kernels.logprobs import MAX_TOP, lm_head_logprobs, token_logprobs

pytestmark = pytest.mark.gpu
E = 2.0 ** -24
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def rows_of(t, v, dtype, seed=0, masked=0.0, sure=10.0):
    gen = seeded(seed + t + v)
    z = torch.randn((t, v), generator=gen) * 2
    ids = torch.randint(0, v, (t,), generator=gen)
    z[torch.arange(t), ids] += torch.rand(t, generator=gen) * sure
    if masked:
        ban = torch.rand((t, v), generator=gen) < masked
        ban[torch.arange(t), ids] = False
        z[ban] = float('-inf')
    return z.to(dtype).cuda(), ids.cuda()


def reference(z, ids, temperature=1.0, ignore=-100):
    """(log softmax, log probabilities, entropies, tolerances of both), float64."""
    x = z.double() / temperature
    lp = x.log_softmax(-1)
    p = lp.exp()
    h = -(p * torch.where(p > 0, lp, 0.0)).sum(-1)
    left = ids == ignore
    got = lp.gather(-1, ids.clamp(0, z.shape[-1] - 1)[..., None])[..., 0]
    d = got + (x.max(-1).values - x.logsumexp(-1)).abs()
    t_lp = E * (160 + 4 * d.abs())
    t_h = E * (160 + 240 * h)
    return lp, torch.where(left, 0.0, got), torch.where(left, 0.0, h), t_lp, t_h


def near(got, want, tol):
    worst = float(((got.double() - want).abs() / tol).nan_to_num(nan=1e9).max())
    assert worst <= 1.0, f'{worst:.2f} times the tolerance'


SHAPES = [(1, 1), (1, 2), (3, 7), (2, 1000), (5, 2047), (4, 2048), (3, 2049), (1, 16385), (2, 151936), (300, 4099), (1100, 2600), (130, 65537), (3, 32761), (3, 32762),
          (3, 16381), (3, 16382)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,v", SHAPES)
def test_against_64_bits(t, v, dtype):
    print(f"logprobs {t} {v} {dtype}", flush=True)
    z, ids = rows_of(t, v, dtype)
    if t > 2:
        ids[1] = -100
    for temperature in (1.0, 0.7, 1.3):
        out = token_logprobs(z, ids, temperature=temperature)
        assert out.top_logprobs is None and out.top_tokens is None and out.logprobs.dtype == out.entropy.dtype == torch.float32
        _, lp, h, t_lp, t_h = reference(z, ids, temperature)
        near(out.logprobs, lp, t_lp)
        near(out.entropy, h, t_h)
        if t > 2:
            assert float(out.logprobs[1]) == float(out.entropy[1]) == 0.0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,v,top", [(1, 1, 1), (2, 5, 5), (3, 33, 32), (1, 151936, 20), (2, 2049, 1), (700, 5001, 5), (5, 300001, 32), (1030, 2100, 3),
                                     (3, 32761, 20), (3, 32762, 20), (3, 16381, 7), (3, 16382, 7), (300, 33000, 4)])
def test_alternatives(t, v, top, dtype):
    print(f"top {t} {v} {top} {dtype}", flush=True)
    z, ids = rows_of(t, v, dtype, masked=0.3 if v > 100 else 0.0)
    plain = token_logprobs(z, ids, temperature=0.7)
    out = token_logprobs(z, ids, top=top, temperature=0.7)
    assert torch.equal(out.logprobs, plain.logprobs) and torch.equal(out.entropy, plain.entropy)
    want = z.float().sort(dim=-1, descending=True, stable=True).indices[:, :top]
    assert torch.equal(out.top_tokens, want)
    lp, _, _, _, _ = reference(z, ids, 0.7)
    best = lp.gather(-1, want)
    near(out.top_logprobs, best, E * (160 + 4 * (best - lp.max(-1, keepdim=True).values).abs() + 4 * lp.max(-1, keepdim=True).values.abs()))


@pytest.mark.parametrize("v", [40000, 30000, 9000])   # a row in several workgroups, in one
@pytest.mark.parametrize("dtype", DTYPES)
def test_alternatives_of_awkward_rows(dtype, v):
    """Rows of equals, sorted rows either way, the largest all in one thread's values, few values that are not ruled out."""
    top = 32
    ramp = torch.linspace(-8, 8, v)
    rows = [torch.zeros(v), ramp, ramp.flip(0), torch.full((v,), -3.0), torch.zeros(v)]
    n = min(16, v // 2048)
    rows[3][8 * 256 * torch.arange(n)[:, None] + torch.arange(8)] = 4.0 + torch.rand((n, 8), generator=seeded(1))
    rows[4] = torch.full((v,), float('-inf'))
    rows[4][torch.tensor([5, v - 1, v // 2])] = torch.tensor([-0.0, 0.0, 1.0])
    for reps in (1, 60):   # small slices and large ones
        z = torch.stack(rows).repeat(reps, 1).to(dtype).cuda()
        out = token_logprobs(z, torch.zeros(z.shape[0], dtype=torch.int64, device='cuda'), top=top)
        assert torch.equal(out.top_tokens, z.float().sort(dim=-1, descending=True, stable=True).indices[:, :top])
        assert out.top_tokens[4, :4].tolist() == [v // 2, 5, v - 1, 0] and float(out.top_logprobs[4, 3]) == -float('inf')


@pytest.mark.parametrize("v,top", [(5000, 0), (5000, 6), (40000, 0), (40000, 6)])
def test_rows_left_out(v, top):
    """Zeros, whatever the row holds, and the other rows as they are alone."""
    z, ids = rows_of(6, v, torch.bfloat16)
    ids[2], ids[5] = -100, -100
    z[2], z[5] = float('nan'), float('inf')
    out = token_logprobs(z, ids, top=top)
    keep = torch.tensor([0, 1, 3, 4]).cuda()
    alone = token_logprobs(z[keep], ids[keep], top=top)
    for a, b in zip(out, alone):
        if a is not None:
            assert torch.equal(a[keep], b) and not bool(a[[2, 5]].any())


def test_rows_without_a_distribution():
    """NaN, +inf and rows of -inf only give NaN for that row and nothing else; tokens outside the vocabulary give NaN."""
    for v in (50, 30000):
        z, ids = rows_of(8, v, torch.float32)
        clean = token_logprobs(z, ids, top=3)
        z[1, v // 2], z[2, 3], z[3] = float('nan'), float('inf'), float('-inf')
        ids[4], ids[5] = v, -1
        out = token_logprobs(z, ids, top=3)
        assert bool(out.logprobs[1:6].isnan().all()) and bool(out.entropy[1:4].isnan().all()) and bool(out.top_logprobs[1:4].isnan().all())
        assert int(out.top_tokens[1, 0]) == v // 2 and out.top_tokens[3].tolist() == [0, 1, 2] and int(out.top_tokens[2, 0]) == 3
        for a, b in zip(out, clean):
            assert torch.equal(a[[0, 6, 7]], b[[0, 6, 7]])
        assert torch.equal(out.entropy[4:6], clean.entropy[4:6]) and torch.equal(out.top_tokens[4:6], clean.top_tokens[4:6])


def test_a_sure_row_keeps_its_digits():
    """One token has all but 1e-9 of the probability: 1 - p, -log p and the entropy come out to their own digits."""
    z = torch.full((1, 1000), -27.0, device='cuda')
    z[0, 7] = 0.0
    zr = z.requires_grad_()
    out = token_logprobs(zr, torch.tensor([7], device='cuda'))
    lp, want, h, _, _ = reference(z.detach(), torch.tensor([7], device='cuda'))
    (g,) = torch.autograd.grad(out.logprobs.sum(), zr)
    p = lp.exp()
    for got, exact in ((out.logprobs, want), (out.entropy, h), (g[0, 7:8], -torch.expm1(want)), (g[0, :7], -p[0, :7])):
        assert float(((got.double() - exact) / exact).abs().max()) <= 300 * E


def grads(z, ids, g, gh, gtop, top_ids, temperature, ignore=-100):
    """(dlogits, its tolerance before rounding), float64."""
    x = z.double() / temperature
    lp = x.log_softmax(-1)
    p = lp.exp()
    lp = torch.where(p > 0, lp, -1e30)
    h = -(p * torch.where(p > 0, lp, 0.0)).sum(-1, keepdim=True)
    up = g[:, None].double() + gtop.double().sum(-1, keepdim=True)
    spread = torch.where(p > 0, lp, 0.0)
    dz = -p * (up + gh[:, None].double() * (spread + h))
    mag = p * (g.abs()[:, None] + gtop.abs().sum(-1, keepdim=True) + gh.abs()[:, None] * (spread.abs() + h + 1)).double()
    one = torch.zeros_like(x).scatter_add_(-1, ids.clamp(0)[:, None], g[:, None].double())
    one.scatter_add_(-1, top_ids, gtop.double())
    left = (ids == ignore)[:, None]
    tol = E * (320 + 8 * spread.abs()) * (mag + one.abs()) / temperature
    return torch.where(left, 0.0, (dz + one) / temperature), tol


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,v,top", [(1, 1, 0), (3, 9, 3), (2, 2049, 0), (700, 3001, 0), (4, 151936, 0), (40, 20003, 5)])
def test_gradient(t, v, top, dtype):
    z, ids = rows_of(t, v, dtype, masked=0.2 if v > 100 else 0.0)
    if t > 2:
        ids[1] = -100
    gen = seeded(t)
    g, gh = torch.randn(t, generator=gen).cuda(), torch.randn(t, generator=gen).cuda()
    gtop = torch.randn((t, top), generator=gen).cuda()
    zr = z.clone().requires_grad_()
    out = token_logprobs(zr, ids, top=top, temperature=0.8)
    outs, ups = [out.logprobs, out.entropy], [g, gh]
    if top:
        outs, ups = outs + [out.top_logprobs], ups + [gtop]
        assert not out.top_tokens.requires_grad
    (dz,) = torch.autograd.grad(outs, zr, ups, retain_graph=True)
    assert dz.dtype == dtype
    tid = out.top_tokens if top else torch.zeros((t, 0), dtype=torch.int64, device='cuda')
    u, tiny = torch.finfo(dtype).eps / 2, torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    want, tol = grads(z, ids, g, gh, gtop, tid, 0.8)
    near(dz, want, u * want.abs() + tol + tiny)
    # each output by itself
    for i, (o, up) in enumerate(zip(outs, ups)):
        (one,) = torch.autograd.grad(o, zr, up, retain_graph=True)
        parts = [torch.zeros_like(x) for x in (g, gh, gtop)]
        parts[i] = up
        want, tol = grads(z, ids, *parts, tid, 0.8)
        near(one, want, u * want.abs() + tol + tiny)


def test_gradient_against_differences():
    """Central differences of the outputs themselves along random directions, |direction| <= 1: the third derivative of a log
    probability along one is at most 8 (a third central moment of values within 2), of an entropy at most 8 (3 + |log p| <= 12)."""
    z, ids = rows_of(6, 40, torch.float32)
    gen = seeded(5)
    g, gh, gt = (torch.randn(s, generator=gen).cuda() for s in ((6,), (6,), (6, 3)))

    def loss(x):
        out = token_logprobs(x, ids, top=3, temperature=1.0)
        return ((out.logprobs * g).sum().double() + (out.entropy * gh).sum().double() + (out.top_logprobs * gt).sum().double())
    zr = z.clone().requires_grad_()
    (dz,) = torch.autograd.grad(loss(zr), zr)
    step = 2.0 ** -7
    size = float(g.abs().sum() + 15 * gh.abs().sum() + gt.abs().sum())
    for i in range(4):
        v = (torch.rand(z.shape, generator=seeded(i)) * 2 - 1).cuda()
        fd = (loss(z + step * v) - loss(z - step * v)) / (2 * step)
        tol = size * 8 * step ** 2 / 6 + size * 400 * E * 10 / step
        assert abs(float(fd) - float((dz.double() * v).sum())) <= tol


def test_layouts_and_streams():
    b, s, v = 3, 5, 2051
    z = torch.randn((b, s, v), generator=seeded(0)).bfloat16().cuda()
    ids = torch.randint(0, v, (b, s), generator=seeded(1)).cuda()
    whole = token_logprobs(z, ids, top=4)
    assert whole.logprobs.shape == (b, s) and whole.top_tokens.shape == (b, s, 4)
    last = token_logprobs(z[:, -1], ids[:, -1].contiguous(), top=4)           # rows s v apart
    for a, w in zip(last, whole):
        assert torch.equal(a, w[:, -1])
    cut = token_logprobs(z[..., :2000], ids.clamp_max(1999), top=4)           # a vocabulary that ends before the row
    _, lp, h, t_lp, t_h = reference(z[..., :2000], ids.clamp_max(1999))      # a thread's values go by 16-byte boundaries: other
    near(cut.logprobs, lp, t_lp)                                             # rows' starts, other orders of the same sums
    near(cut.entropy, h, t_h)
    assert torch.equal(cut.top_tokens, token_logprobs(z[..., :2000].contiguous(), ids.clamp_max(1999), top=4).top_tokens)
    one = token_logprobs(z[0, 0], ids[0, 0], top=4)
    assert one.logprobs.shape == () and torch.equal(one.top_tokens, whole.top_tokens[0, 0])
    zr = z.clone().requires_grad_()
    (d1,) = torch.autograd.grad(token_logprobs(zr[:, 2], ids[:, 2].contiguous()).entropy.sum(), zr)
    (d2,) = torch.autograd.grad(token_logprobs(zr, ids).entropy[:, 2].sum(), zr)
    assert torch.equal(d1, d2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = token_logprobs(z, ids, top=4)
    side.synchronize()
    for a, w in zip(got, whole):
        assert torch.equal(a, w)


def test_captured_calls():
    """Forward and backward in one captured graph, replayed on other inputs beside eager calls; a second graph of other sizes."""
    def make(t, v, top):
        z = torch.zeros((t, v), dtype=torch.bfloat16, device='cuda', requires_grad=True)
        ids = torch.zeros(t, dtype=torch.int64, device='cuda')
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        up = torch.ones(t, device='cuda')
        with torch.cuda.graph(g, stream=stream):
            out = token_logprobs(z, ids, top=top)
            (dz,) = torch.autograd.grad([out.logprobs, out.entropy], z, [up, up])
        torch.cuda.current_stream().wait_stream(stream)
        return g, z, ids, [x.detach() for x in out if x is not None] + [dz], up
    graphs = [make(3, 5000, 4), make(70, 901, 0)]
    for i in range(3):
        for g, z, ids, outs, up in graphs:
            zi, ii = rows_of(*z.shape, torch.bfloat16, seed=i)
            with torch.no_grad():
                z.copy_(zi)
            ids.copy_(ii)
            g.replay()
            torch.cuda.synchronize()
            top = outs[2].shape[-1] if len(outs) == 5 else 0
            zr = zi.clone().requires_grad_()
            out = token_logprobs(zr, ii, top=top)
            (dz,) = torch.autograd.grad([out.logprobs, out.entropy], zr, [up, up])
            for a, w in zip(outs, [x.detach() for x in out if x is not None] + [dz]):
                assert torch.equal(a, w)
            del out, dz, zr


# ------------------------------------------------------------------------------------------ from hidden states
def head(t, h, v, dtype, seed=0):
    gen = seeded(seed + t + h + v)
    w = (torch.randn((v, h), generator=gen) * (1.5 / h ** 0.5)).to(dtype)
    ids = torch.randint(0, v, (t,), generator=gen)
    x = (torch.randn((t, h), generator=gen) + w[ids].float() * torch.rand((t, 1), generator=gen) * 4).to(dtype)
    if t > 2:
        ids[1] = -100
    return x.cuda(), w.cuda(), ids.cuda()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,h,v", [(1, 64, 8), (3, 64, 1000), (8, 256, 4096), (17, 128, 4104), (300, 192, 1032), (129, 64, 300), (5, 72, 1000),
                                   (6, 50, 77), (40, 64, 1001), (257, 320, 2600)])
def test_lm_head(t, h, v, dtype):
    """Against 64 bits.  A logit is a sum of h products: off by at most (h + 8) 2^-24 sum |x w|, which moves a log probability or
    an entropy (times its largest |log p| + entropy) by at most twice that.  The gradient of a logit is rounded to the type
    before the products with it; every product rounds its sum once.  For 16-bit types it is formed from the logit's distance to a
    maximum in steps of 64 / 65535 in base 2: half of one moves a probability by 0.5 ln 2 64 / 65535 (3.4e-4) of itself, and
    probabilities below 2^-64 of another may be 2^-64 of it."""
    print(f"lm head {t} {h} {v} {dtype}", flush=True)
    x, w, ids = head(t, h, v, dtype)
    g, gh = torch.randn(t, generator=seeded(1)).cuda(), 0.2 * torch.randn(t, generator=seeded(2)).cuda()
    check_head(x, w, ids, g, gh, 0.9, t)


def check_head(x, w, ids, g, gh, temperature, n, top=0):
    """The last n rows; the others have no upstream gradient.  With ``top`` the alternatives have one too."""
    (t, h), v, dtype = x.shape, w.shape[0], x.dtype
    xr, wr = x.clone().requires_grad_(), w.clone().requires_grad_()
    out = lm_head_logprobs(xr, wr, ids, temperature=temperature, top=top)
    gtop = torch.randn((t, top), generator=seeded(3)).cuda()
    dx, dw = torch.autograd.grad([x for x in out[:3] if x is not None], [xr, wr], [g, gh, gtop][:3 if top else 2])
    assert dx.shape == x.shape and not bool(dx[:t - n].any())
    x, ids, g, gh, dx = x[-n:], ids[-n:], g[-n:], gh[-n:], dx[-n:]
    z = x.double() @ w.double().t()
    dot = (h + 8) * E * (x.double().abs() @ w.double().abs().t())
    lp, want, ent, t_lp, t_h = reference(z, ids, temperature)
    e = 2 * dot.amax(-1) / temperature
    near(out.logprobs[-n:], want, t_lp + e)
    span = (-lp.min(-1).values) + ent + 1
    near(out.entropy[-n:], ent, t_h + e * span)
    tid = out.top_tokens if top else torch.zeros((n, 0), dtype=torch.int64, device='cuda')
    if top:
        near(out.top_logprobs, torch.where((ids == -100)[:, None], 0.0, lp.gather(-1, tid)), (t_lp + e)[:, None] + 4 * E * lp.abs().amax())
    dz, tol = grads(z, ids, g, gh, gtop[-n:], tid, temperature)
    p = lp.exp()
    one = torch.zeros_like(z).scatter_(-1, ids.clamp(0)[:, None], 1.0).scatter_(-1, tid, 1.0)
    wide = (g.abs()[:, None] + gtop[-n:].abs().sum(-1, keepdim=True) + gh.abs()[:, None] * (3 + lp.abs() + ent[:, None])) / temperature
    u = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    step = 0.0 if dtype == torch.float32 else 0.5 * 0.6931472 * 64 / 65535 * 1.01
    tol = tol + u * dz.abs() + tiny + (p + one * (1 - p)) * wide * e[:, None] + p * wide * step + 2.0 ** -64 * wide * (step > 0)
    tol = torch.where((ids == -100)[:, None], 0.0, tol)
    for got, exact, bound in ((dx, dz @ w.double(), tol @ w.double().abs() + (v + 8) * E * (dz.abs() @ w.double().abs())),
                              (dw, dz.t() @ x.double(), tol.t() @ x.double().abs() + (t + 8) * E * (dz.abs().t() @ x.double().abs()))):
        assert got.dtype == dtype
        near(got, exact, bound + u * exact.abs() + tiny)


@pytest.mark.parametrize("dtype", DTYPES)
def test_lm_head_alternatives_and_needs(dtype):
    """The alternatives' order is that of the logits where they differ by more than the sums' error; a gradient of one operand
    only; shapes of any number of dimensions."""
    x, w, ids = head(24, 128, 2000, dtype)
    z = x.double() @ w.double().t()
    out = lm_head_logprobs(x.view(2, 12, 128), w, ids.view(2, 12), top=7)
    assert out.top_tokens.shape == (2, 12, 7) and out.logprobs.shape == (2, 12)
    keep = ids != -100
    got = z.gather(-1, out.top_tokens.view(24, 7))[keep]
    dot = 136 * E * (x.double().abs() @ w.double().abs().t()).amax(-1)[keep]
    assert bool(((got[:, :-1] - got[:, 1:]) >= -2 * dot[:, None]).all())
    kth = z.sort(dim=-1, descending=True).values[keep][:, 6]
    assert bool((got[:, -1] >= kth - 2 * dot).all())
    plain = lm_head_logprobs(x, w, ids)
    for need in ((True, False), (False, True)):
        xr, wr = x.clone().requires_grad_(need[0]), w.clone().requires_grad_(need[1])
        o = lm_head_logprobs(xr, wr, ids)
        assert torch.equal(o.logprobs, plain.logprobs)
        (got,) = torch.autograd.grad(o.entropy.sum(), xr if need[0] else wr)
        assert bool(got.isfinite().all())


# a tile of each kind above 64 rows, two of them beside each other, weights beyond the caches, and dX with its sum over the vocabulary in more than eight parts
@pytest.mark.parametrize("t,h,v", [(200, 64, 32008), (1000, 64, 16376), (100, 192, 9000), (500, 1024, 40000), (8, 1024, 140000), (100, 1024, 140000), (16, 256, 70000), (40, 128, 36000)])
def test_lm_head_of_other_sizes(t, h, v):
    test_lm_head(t, h, v, torch.bfloat16)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", [1000, 1001])   # dX and dW from one dz, and chunk by chunk
@pytest.mark.parametrize("top", [0, 4])
def test_lm_head_in_chunks(v, top, dtype, monkeypatch):
    """Logits a few rows at a time."""
    monkeypatch.setattr(logprobs, '_CHUNK_BYTES', 4 * v * 30)
    t = 70
    assert logprobs._chunks(t, v) == [(0, 30), (30, 60), (60, 70)]
    x, w, ids = head(t, 72, v, dtype)
    check_head(x, w, ids, torch.randn(t, generator=seeded(1)).cuda(), torch.randn(t, generator=seeded(2)).cuda(), 0.9, t, top)


@pytest.mark.parametrize("h", [128, 72])   # with the statistics beside the product, and without
def test_lm_head_backward_again_and_of_one_result(h):
    """A second backward of one forward gives the first one's bits (the first takes the stored logits' place), and the gradients of the
    log probabilities alone and of the entropies alone are those with zeros for the other."""
    x, w, ids = head(70, h, 1000, torch.bfloat16)
    g = torch.randn(70, generator=seeded(1)).cuda()
    xr, wr = x.clone().requires_grad_(), w.clone().requires_grad_()
    out = lm_head_logprobs(xr, wr, ids)
    runs = [torch.autograd.grad([out.logprobs, out.entropy], (xr, wr), [g, g], retain_graph=True) for _ in range(3)]
    for run in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(run, runs[0]))
    zero = torch.zeros_like(g)
    for i in range(2):
        one = torch.autograd.grad(out[i], (xr, wr), g, retain_graph=True)
        both = torch.autograd.grad([out.logprobs, out.entropy], (xr, wr), [zero if j != i else g for j in range(2)], retain_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(one, both))
    with torch.no_grad():
        xr.mul_(2)
    with pytest.raises(RuntimeError, match='modified'):
        torch.autograd.grad(out.entropy.sum(), wr)


def test_lm_head_gradient_against_differences():
    """As test_gradient_against_differences, along directions of hidden states and of the weight that move no logit by more than 1 a
    unit; a logit's own sum (and the rounding of the moved operand) is off by at most (h + 8) 2^-24 sum |x w|, which moves a log
    probability by twice that and an entropy by its largest |log p| + entropy + 1 <= 15 times as much."""
    t, h, v = 6, 48, 40
    x, w, ids = head(t, h, v, torch.float32)
    gen = seeded(5)
    g, gh, gt = (torch.randn(s, generator=gen).cuda() for s in ((t,), (t,), (t, 3)))

    def loss(x, w):
        out = lm_head_logprobs(x, w, ids, top=3)
        return ((out.logprobs * g).sum().double() + (out.entropy * gh).sum().double() + (out.top_logprobs * gt).sum().double())
    xr, wr = x.clone().requires_grad_(), w.clone().requires_grad_()
    dx, dw = torch.autograd.grad(loss(xr, wr), (xr, wr))
    step = 2.0 ** -7
    size = float(g.abs().sum() + 15 * gh.abs().sum() + gt.abs().sum())
    e = 2 * (h + 8) * E * float((x.double().abs() @ w.double().abs().t()).amax())
    tol = size * 8 * step ** 2 / 6 + size * (400 * E * 10 + e) / step
    for i in range(4):
        vx, vw = ((torch.rand(s.shape, generator=seeded(10 * i + j)) * 2 - 1).cuda() for j, s in enumerate((x, w)))
        vx /= (vx @ w.t()).abs().amax()
        vw /= (x @ vw.t()).abs().amax()
        fd = (loss(x + step * vx, w) - loss(x - step * vx, w)) / (2 * step)
        assert abs(float(fd) - float((dx.double() * vx).sum())) <= tol
        fd = (loss(x, w + step * vw) - loss(x, w - step * vw)) / (2 * step)
        assert abs(float(fd) - float((dw.double() * vw).sum())) <= tol


def test_lm_head_captured():
    """Forward and backward in captured graphs, replayed on other inputs beside eager calls."""
    def make(t, h, v):
        x, w = (torch.zeros(s, dtype=torch.bfloat16, device='cuda', requires_grad=True) for s in ((t, h), (v, h)))
        ids = torch.zeros(t, dtype=torch.int64, device='cuda')
        up = torch.ones(t, device='cuda')
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            out = lm_head_logprobs(x, w, ids)
            grads = torch.autograd.grad([out.logprobs, out.entropy], (x, w), [up, up])
        torch.cuda.current_stream().wait_stream(stream)
        return g, x, w, ids, [out.logprobs.detach(), out.entropy.detach(), *grads], up
    graphs = [make(9, 64, 40000), make(130, 72, 904), make(300, 128, 1032)]
    for i in range(3):
        for g, x, w, ids, outs, up in graphs:
            xi, wi, ii = head(*x.shape, w.shape[0], torch.bfloat16, seed=i)
            with torch.no_grad():
                x.copy_(xi)
                w.copy_(wi)
            ids.copy_(ii)
            g.replay()
            torch.cuda.synchronize()
            xr, wr = xi.clone().requires_grad_(), wi.clone().requires_grad_()
            out = lm_head_logprobs(xr, wr, ii)
            grads = torch.autograd.grad([out.logprobs, out.entropy], (xr, wr), [up, up])
            for a, b in zip(outs, [out.logprobs.detach(), out.entropy.detach(), *grads]):
                assert torch.equal(a, b)
            del out, grads, xr, wr


def test_offsets_beyond_32_bits():
    """More than 2^31 logits: the last rows against 64 bits, none of the gradient before them."""
    t, v, n = 16640, 131080, 300
    ids = torch.randint(0, v, (t,), generator=seeded(0)).cuda()
    up = torch.zeros(t, device='cuda')
    up[-n:] = torch.randn(n, generator=seeded(1)).cuda()
    z = torch.zeros((t, v), dtype=torch.float16, device='cuda')
    assert z.numel() > 1 << 31
    z[-n:] = torch.randn((n, v), generator=seeded(2)).half().cuda()
    z.requires_grad_()
    out = token_logprobs(z, ids, top=3)
    (dz,) = torch.autograd.grad([out.logprobs, out.entropy], z, [up, up])
    near(out.logprobs[:-n], torch.full((t - n,), -math.log(v), dtype=torch.float64, device='cuda'), E * (160 + 4 * math.log(v)))
    assert not bool(dz[:-n].any()) and torch.equal(out.top_tokens[0], torch.arange(3, device='cuda'))
    lp, want, h, t_lp, t_h = reference(z.detach()[-n:], ids[-n:])
    near(out.logprobs[-n:], want, t_lp)
    near(out.entropy[-n:], h, t_h)
    assert torch.equal(out.top_tokens[-n:], lp.sort(dim=-1, descending=True, stable=True).indices[:, :3])
    none = torch.zeros((n, 0), device='cuda')
    want, tol = grads(z.detach()[-n:], ids[-n:], up[-n:], up[-n:], none, none.long(), 1.0)
    u, tiny = torch.finfo(z.dtype).eps / 2, 2.0 ** -25
    near(dz[-n:], want, u * want.abs() + tol + tiny)
    del out, z, dz, lp, want, tol
    x, w, _ = head(t, 64, v, torch.bfloat16)
    check_head(x, w, ids, up, up, 1.0, n)


def test_lm_head_calls_alike_give_the_same_bits():
    x, w, ids = head(500, 256, 8192, torch.bfloat16)
    runs = []
    for _ in range(2):
        xr, wr = x.clone().requires_grad_(), w.clone().requires_grad_()
        out = lm_head_logprobs(xr, wr, ids)
        runs.append([out.logprobs, out.entropy, *torch.autograd.grad((out.logprobs * 0.3 + out.entropy).sum(), (xr, wr))])
    for a, b in zip(*runs):
        assert torch.equal(a, b)


def test_largest_top():
    z, ids = rows_of(3, 70000, torch.bfloat16)
    assert token_logprobs(z, ids, top=MAX_TOP).top_tokens.shape == (3, MAX_TOP)
