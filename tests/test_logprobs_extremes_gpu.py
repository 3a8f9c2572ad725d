"""Log probabilities where numbers are extreme: finite masks, temperatures near their bounds, infinite logits, gradients beyond fp16's
range; and backward passes that are captured, offloaded or formed again.

Tolerances are those of the plain cases (test_logprobs_gpu.py), and a probability below 2^-126 may come out of the exponential as 0."""
import pytest
import torch

from _util import seeded
from test_logprobs_gpu import E, check_head, grads, head, near, reference

from qwen3_triton.kernels.linear import MAX_LD
from qwen3_triton.kernels.logprobs import MAX_GRAD_VOCAB, lm_head_logprobs, token_logprobs

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def close(got, want, tol):
    """``near``, where equal infinities are near too and what fp32 rounds to an infinity (2^128 - 2^103 and more) is one."""
    want = torch.where(want < -3.40282357e38, float('-inf'), want)
    same = got.double() == want
    near(torch.where(same, 0.0, got), torch.where(same, 0.0, want), torch.where(same, 1.0, tol))


def check_rows(z, ids, temperature, top=5):
    """Results, alternatives and gradients of rows against 64 bits."""
    t, v = z.shape
    gen = seeded(t)
    g, gh = torch.randn(t, generator=gen).cuda(), torch.randn(t, generator=gen).cuda()
    gtop = torch.randn((t, top), generator=gen).cuda()
    zr = z.clone().requires_grad_()
    out = token_logprobs(zr, ids, top=top, temperature=temperature)
    lp, want, h, t_lp, t_h = reference(z, ids, temperature)
    close(out.logprobs, want, t_lp)
    near(out.entropy, h, t_h)
    order = z.float().sort(dim=-1, descending=True, stable=True).indices[:, :top]
    assert torch.equal(out.top_tokens, order)
    best = lp.gather(-1, order)
    close(out.top_logprobs, best, E * (160 + 4 * (best - lp.amax(-1, keepdim=True)).abs() + 4 * lp.amax(-1, keepdim=True).abs()))
    plain = token_logprobs(z, ids, temperature=temperature)
    assert torch.equal(plain.logprobs, out.logprobs) and torch.equal(plain.entropy, out.entropy)
    (dz,) = torch.autograd.grad([out.logprobs, out.entropy, out.top_logprobs], zr, [g, gh, gtop])
    want, tol = grads(z, ids, g, gh, gtop, out.top_tokens, temperature)
    p_lp = torch.where(lp.exp() > 0, lp, 0.0).abs()
    none = 2.0 ** -126 * (g.abs()[:, None] + gtop.abs().sum(-1, keepdim=True) + gh.abs()[:, None] * (p_lp + h[:, None] + 1)) / temperature
    fin = torch.finfo(z.dtype)
    near(dz, want, fin.eps / 2 * want.abs() + tol + none + fin.smallest_normal * fin.eps / 2)


@pytest.mark.parametrize("dtype,mask", [*((d, m) for d in (F32, BF16) for m in (-1e4, -1e9, -1e10, -1e20, -1e29, -2e30, None)), (F16, -6e4), (F16, None)])
@pytest.mark.parametrize("v", [700, 9000, 70001])   # one vector or less a thread, a row in one workgroup, in several
def test_finite_masks(v, dtype, mask):
    """Values ruled out by a finite number (None: the type's lowest): here and there, in blocks, all but a few, all."""
    mask = torch.finfo(dtype).min if mask is None else mask
    print(f"masks {v} {dtype} {mask}", flush=True)
    gen = seeded(v)
    z = torch.randn((8, v), generator=gen) * 2
    ids = torch.randint(0, v, (8,), generator=gen)
    z[1, torch.rand(v, generator=gen) < 0.3] = mask
    z[2] = mask
    z[2, ids[2]] = 1.5
    z[3] = mask                                # a row of equals
    z[4, :v // 2] = mask
    z[5, 16:32] = mask
    z[6, :-3] = mask
    z[7], z[7, v // 3], ids[7] = mask, 2.0, v // 2   # the token is one of those ruled out
    for reps in (1, 150):   # 1200 rows: large slices of a thread
        zr, ir = z.repeat(reps, 1).to(dtype).cuda(), ids.repeat(reps).cuda()
        for temperature in (1.0, 0.5, 0.1):
            if reps == 1 or temperature == 0.5 and v < 10000:
                check_rows(zr, ir, temperature)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("v", [700, 9000, 70001])
def test_smallest_temperature(v, dtype):
    """Large logits at a temperature of 1e-6: what counts is their difference to the largest."""
    z = torch.full((3, v), 3000.3)
    z[1, ::2] = 2999.0
    z[2, v // 2] = 3100.0
    check_rows(z.to(dtype).cuda(), torch.tensor([0, 1, v // 2]).cuda(), 1e-6)
    check_rows(-z.to(dtype).cuda(), torch.tensor([0, 1, v // 2]).cuda(), 1e-6)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("v", [50, 5000, 30000, 70001, 151936])
def test_alternatives_of_rows_with_infinite_logits(v, dtype):
    """As many +inf as there are alternatives or more, alone and with NaN, all in different threads or in one: NaN first of all, then
    +inf, equals by their tokens."""
    gen = seeded(v)
    z = torch.randn((6, v), generator=gen)
    inf, nan = float('inf'), float('nan')
    far = (torch.arange(12) * (v // 12) + 3) % v
    z[0, v // 2] = inf
    z[1, far] = inf
    z[2, far], z[2, far[5]] = inf, nan
    z[3, 8:16], z[3, 13] = inf, nan            # in one thread's values
    z[4], z[4, 7] = -inf, inf
    z[5] = inf
    for reps in (1, 200):
        if reps * v > 10 ** 7:
            continue
        zr = z.repeat(reps, 1).to(dtype).cuda()
        ids = torch.zeros(zr.shape[0], dtype=torch.int64, device='cuda')
        key = zr.double().nan_to_num(nan=3e300, posinf=2e300)
        want = key.sort(dim=-1, descending=True, stable=True).indices
        for top in (1, 2, 5, 12):
            out = token_logprobs(zr, ids, top=top)
            assert torch.equal(out.top_tokens, want[:, :top]), top
            assert bool(out.logprobs.isnan().all()) and bool(out.entropy.isnan().all()) and bool(out.top_logprobs.isnan().all())


@pytest.mark.parametrize("size", [1.0, 1e12, 1e25])
def test_large_gradients_of_entropies(size):
    """Tokens of no probability add nothing to an entropy's gradient, however large it is."""
    t, v = 6, 9000
    gen = seeded(3)
    z = torch.randn((t, v), generator=gen) * 2
    z[:, ::3], z[2, 1::3], z[3, 5:] = float('-inf'), -1e20, -1e4
    ids = torch.tensor([1, 2, 2, 0, 3, 8])   # some of them ruled out
    z, ids = z.cuda(), ids.cuda()
    g, gh = torch.zeros(t, device='cuda'), size * torch.randn(t, generator=gen).cuda()
    zr = z.clone().requires_grad_()
    (dz,) = torch.autograd.grad(token_logprobs(zr, ids).entropy, zr, gh)
    none = torch.zeros((t, 0), device='cuda')
    want, tol = grads(z, ids, g, gh, none, none.long(), 1.0)
    near(dz, want, E * want.abs() + tol + 2.0 ** -126 * 1e3 * size)
    # and from hidden states, some of whose logits are -inf, one group of 128 of them all
    x, w, ids = head(t, 64, 1024, BF16)
    x[:, 0], w[:, 0] = 1.0, 0.0
    w[128:256, 0], w[300, 0] = float('-inf'), float('-inf')
    wr = w.clone().requires_grad_()
    (dw,) = torch.autograd.grad(lm_head_logprobs(x, wr, ids).entropy, wr, gh)
    keep = w[:, 0] == 0
    want, tol = grads(x.double() @ w.double().t(), ids, g, gh, none, none.long(), 1.0)
    bound = (2.0 ** -7 * want.abs() + tol).t() @ x.double().abs()   # dz and dW round to bf16 once each
    lp = (x.double() @ w.double().t()).log_softmax(-1)
    p, span = lp.exp(), torch.where(lp.exp() > 0, lp.abs(), 0.0).amax(-1, keepdim=True)
    off = 2 * 72 * E * (x.double().abs() @ w[keep].double().abs().t()).amax(-1, keepdim=True) + 3.5e-4   # a probability, of itself
    bound += (p * gh.abs()[:, None] * (2 * span + 3) * off).t() @ x.double().abs()
    exact = want.t() @ x.double()
    assert bool((dw[~keep] == 0).all())
    near(dw[keep], exact[keep], bound[keep] + 2.0 ** -8 * exact[keep].abs() + 2.0 ** -64 * size * 1e2)


def test_lm_head_gradient_at_small_temperatures():
    """Whole-number logits, exact in fp32, with several equal largest: each of k such tokens has the probability 1 / k.  A step of the
    stored distance moves it by 3.4e-4; the gradient and the product round once each."""
    gen = seeded(0)
    h, v = 64, 1024
    w = torch.randint(-2, 3, (v, h), generator=gen).float()
    for seed in range(24):
        x = torch.randint(-2, 3, (1, h), generator=seeded(seed)).float()
        x[0, 0] = 1.0
        best = int((x @ w.t()).argmax())
        wr = w.clone()
        wr[(torch.arange(4) * 250 + best + 1) % v] = w[best]
        z = (x @ wr.t())[0].double()
        for temperature in (0.01, 1e-3, 1e-4):
            weight = wr.half().cuda().requires_grad_()
            out = lm_head_logprobs(x.half().cuda(), weight, torch.tensor([best]).cuda(), temperature=temperature)
            (dw,) = torch.autograd.grad(out.logprobs.sum(), weight)
            p = (z / temperature).softmax(-1)
            want = -p / temperature
            want[best] += 1 / temperature
            u = 2.0 ** -11
            tol = want.abs() * (2 * u + 1.01 * 3.4e-4 + 400 * E) + 2.0 ** -24 + 2.0 ** -64 / temperature
            near(dw[:, 0].cpu(), want, tol)


def test_lm_head_gradient_beside_ruled_out_tokens():
    """Weights of -inf against a hidden feature of 1: whole groups of tokens whose logits are -inf.  Their probability is 0, and the
    gradient of the weight is that of the others alone."""
    t, h, v = 20, 64, 1024
    x, w, ids = head(t, h, v, BF16)
    x[:, 0], w[:, 0] = 1.0, 0.0
    ids %= 256
    keep = torch.ones(v, dtype=torch.bool)
    keep[256:512], keep[700:] = False, False
    w[~keep.cuda(), 0] = float('-inf')
    g, gh = torch.randn(t, generator=seeded(1)).cuda(), torch.randn(t, generator=seeded(2)).cuda()
    got = []
    for weight in (w, w[keep.cuda()].contiguous()):
        ids2 = torch.where(ids < 0, ids, ids)   # the first 256 tokens stand in both
        wr = weight.clone().requires_grad_()
        out = lm_head_logprobs(x, wr, ids2)
        (dw,) = torch.autograd.grad([out.logprobs, out.entropy], wr, [g, gh])
        got.append((out.logprobs, out.entropy, dw))
    assert bool((got[0][2][~keep.cuda()] == 0).all())
    for a, b in zip(got[0], got[1]):
        a = a[keep.cuda()] if a.ndim == 2 else a
        # the groups are others: sums in another order, and distances to other maxima (0.034 % of each probability, twice)
        scale = float(b.double().abs().max())
        assert bool(a.isfinite().all()) and float((a.double() - b.double()).abs().max()) <= (2.0 ** -7 + 7e-4) * scale


@pytest.mark.parametrize("top", [0, 3])
@pytest.mark.parametrize("t,h,v", [(512, 64, 32000), (300, 72, 20000), (200, 64, 20001), (16, 256, 70000)])
@pytest.mark.parametrize("size", [2.0 ** -14, 2.0 ** -24, 2.0 ** 18])
def test_fp16_gradients_of_any_size(size, t, h, v, top):
    """Upstream gradients that leave the gradient of single logits far below fp16's smallest number, or above its largest; dX and dW
    are right wherever they fit the type themselves.  A logit's gradient may lose half a step of its own and 2^-38 of the largest that any could be, B."""
    print(f"fp16 {size} {t} {h} {v} {top}", flush=True)
    gen = seeded(t)
    w = torch.randn((v, h), generator=gen) * 0.02
    x = torch.randn((t, h), generator=gen)
    up = 1.0 if size > 1 else 2.0 ** 6   # hidden states and weights that carry small gradients into fp16's range
    w[:, 0], x[:, 1] = up, 8 * up
    w[:, 1], x[:, 0] = 0.0, 0.0
    x, w = x.half().cuda(), w.half().cuda()
    ids = torch.randint(0, v, (t,), generator=gen).cuda()
    ids[1] = -100
    g, gh = size * torch.randn(t, generator=gen).cuda(), 0.1 * size * torch.randn(t, generator=gen).cuda()
    g[1] = float('inf')   # a row that is left out
    gtop = size * torch.randn((t, top), generator=gen).cuda()
    xr, wr = x.clone().requires_grad_(), w.clone().requires_grad_()
    out = lm_head_logprobs(xr, wr, ids, top=top)
    dx, dw = torch.autograd.grad([o for o in out[:3] if o is not None], [xr, wr], [g, gh, gtop][:3 if top else 2])
    g[1] = 0.0
    gh[1] = 0.0
    tid = out.top_tokens if top else torch.zeros((t, 0), dtype=torch.int64, device='cuda')
    if top:
        gtop[1] = 0.0
    z = x.double() @ w.double().t()
    e = 2 * ((h + 8) * E * (x.double().abs() @ w.double().abs().t())).amax(-1)
    lp, _, ent, _, _ = reference(z, ids)
    dz, tol = grads(z, ids, g, gh, gtop, tid, 1.0)
    one = torch.zeros_like(z).scatter_(-1, ids.clamp(0)[:, None], 1.0).scatter_(-1, tid, 1.0)
    wide = g.abs()[:, None] + gtop.abs().sum(-1, keepdim=True) + gh.abs()[:, None] * (3 + lp.abs() + ent[:, None])
    largest = float((g.abs() + gtop.abs().sum(-1) + gh.abs() * (1 + torch.log(torch.tensor(float(v))))).max())
    p = lp.exp()
    tol = tol + 2.0 ** -11 * dz.abs() + (p + one * (1 - p)) * wide * e[:, None] + p * wide * 3.5e-4 + 2.0 ** -64 * wide + 2.0 ** -38 * largest
    tol = torch.where((ids == -100)[:, None], 0.0, tol)
    for got, exact, bound in ((dx, dz @ w.double(), tol @ w.double().abs() + (v + 8) * E * (dz.abs() @ w.double().abs())),
                              (dw, dz.t() @ x.double(), tol.t() @ x.double().abs() + (t + 8) * E * (dz.abs().t() @ x.double().abs()))):
        bound = bound + 2.0 ** -11 * exact.abs() + 2.0 ** -25
        fits, over = exact.abs() + bound < 65504, exact.abs() - bound >= 65520   # fp16's largest, and from where on it rounds to infinity
        near(torch.where(fits, got, 0.0), torch.where(fits, exact, 0.0), bound)
        assert bool(fits.any()) and bool((got[over] == exact[over].sign() * float('inf')).all())


def test_lm_head_of_a_very_long_vocabulary():
    """The most tokens that a gradient takes, and more: log probabilities still, but no gradient, which is refused before any work."""
    t, h = 3, 64
    for v in (MAX_GRAD_VOCAB, MAX_GRAD_VOCAB - 1, MAX_LD + 8):
        w = (torch.randn((v, h), generator=seeded(0)) * 0.1).bfloat16().cuda()
        x = torch.randn((t, h), generator=seeded(1)).bfloat16().cuda()
        ids = torch.randint(0, v, (t,), generator=seeded(2)).cuda()
        for top in (0, 2):
            if v <= MAX_GRAD_VOCAB:
                check_head(x, w, ids, torch.ones(t, device='cuda'), torch.ones(t, device='cuda'), 1.0, t, top)
                continue
            out = lm_head_logprobs(x, w, ids, top=top)
            dot = 72 * E * (x.double().abs() @ w.double().abs().t()).amax(-1)
            _, lp, _, t_lp, _ = reference(x.double() @ w.double().t(), ids)
            near(out.logprobs, lp, t_lp + 2 * dot)
            for need in (0, 1):
                with pytest.raises(ValueError, match='gradient'):
                    lm_head_logprobs(x.clone().requires_grad_(need == 0), w.detach().requires_grad_(need == 1), ids, top=top)


# ------------------------------------------------------------------------------------------ backward passes
def step(x, w, ids, g):
    xr, wr = x.clone().requires_grad_(), w.clone().requires_grad_()
    out = lm_head_logprobs(xr, wr, ids)
    return torch.autograd.grad([out.logprobs, out.entropy], (xr, wr), [g, g])


def test_saved_tensor_hooks_see_the_stored_logits():
    """Offloading and recomputation work on all that the forward keeps: the 16 bits of each logit too."""
    t, h, v = 70, 128, 1000
    x, w, ids = head(t, h, v, BF16)
    g = torch.randn(t, generator=seeded(1)).cuda()
    want = step(x, w, ids, g)
    seen = []
    with torch.autograd.graph.saved_tensors_hooks(lambda s: (seen.append(s.numel() * s.element_size()), s.cpu())[1], lambda s: s.cuda()):
        got = step(x, w, ids, g)
    assert 2 * t * v in seen and all(torch.equal(a, b) for a, b in zip(got, want))
    xr, wr = x.clone().requires_grad_(), w.clone().requires_grad_()
    out = torch.utils.checkpoint.checkpoint(lambda a, b: lm_head_logprobs(a, b, ids)[:2], xr, wr, use_reentrant=False)
    got = torch.autograd.grad(out, (xr, wr), [g, g])
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("before", [0, 1])   # eager backward passes before the captured one
def test_captured_backward_of_an_eager_forward(before):
    """Replays of a backward pass alone, with other upstream gradients, beside eager work that takes and frees memory."""
    t, h, v = 70, 128, 1000
    x, w, ids = head(t, h, v, BF16)
    up = torch.zeros(t, device='cuda')
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        xr, wr = x.clone().requires_grad_(), w.clone().requires_grad_()
        out = lm_head_logprobs(xr, wr, ids)
        for _ in range(before):
            torch.autograd.grad([out.logprobs, out.entropy], (xr, wr), [up, up], retain_graph=True)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        got = torch.autograd.grad([out.logprobs, out.entropy], (xr, wr), [up, up], retain_graph=True)
    torch.cuda.current_stream().wait_stream(stream)
    for i in range(4):
        g = torch.randn(t, generator=seeded(i)).cuda()
        want = step(x, w, ids, g)
        junk = [torch.full((t, v), float('nan'), dtype=BF16, device='cuda') for _ in range(4)]
        up.copy_(g)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i
        if i:   # an eager one between the replays
            eager = torch.autograd.grad([out.logprobs, out.entropy], (xr, wr), [g, g], retain_graph=True)
            assert all(torch.equal(a, b) for a, b in zip(eager, want)), i
        del junk, want
