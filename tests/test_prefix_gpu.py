"""Attention over a shared prefix against the formula in 64 bits.

Tolerance, element by element, with u the rounding of the type (half its eps): the output rounds once, u |o|; each weight P
rounds once in the numerator, u sum p |v|, and in the sum it is divided by, u |o|.  fp32: a score is a sum of 128 products, off by
at most 128 2^-24 sum |q k|, and one fma and one exp2 of it by 4 2^-24 |score|; a score's error e moves the output by at
most 2 e sum p |v|.  In fp16 a weight below 2^-14 of a row's largest keeps an absolute 2^-25 (the largest is at least 1)."""
import pytest
import torch

from _util import seeded

from qwen3_triton.inference import prefix as PX

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16]


def expected(q, pk, pv, ck, cv, starts, scale=None):
    """(o, tolerance) in float64 on the GPU; ``starts``: one per row."""
    b, s, hq, d = q.shape
    r, hkv, p, _ = pk.shape
    g, n = hq // hkv, b // r
    scale = d ** -0.5 if scale is None else scale
    u = torch.finfo(q.dtype).eps / 2
    o = torch.zeros((b, s, hq, d), dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(o)
    for i in range(b):
        end = min(max(starts[i] + s, 0), ck.shape[2])
        for h in range(hkv):
            k = torch.cat((pk[i // n, h], ck[i, h, :end])).double()
            v = torch.cat((pv[i // n, h], cv[i, h, :end])).double()
            x = q[i, :, h * g:(h + 1) * g].double().transpose(0, 1)   # [G, S, D]
            z = (x @ k.t()) * scale
            own = torch.arange(k.shape[0], device=q.device) - p
            seen = (own[None, :] < 0) | (own[None, :] <= starts[i] + torch.arange(s, device=q.device)[:, None])
            z = z.masked_fill(~seen, float('-inf'))
            some = seen.any(1)
            w = torch.where(some[None, :, None], z.softmax(-1), 0.0)
            clean = torch.where(v.isfinite(), v, 0.0)
            out, a = w @ clean, w @ clean.abs()
            err = 0.0
            if k.shape[0]:
                mag = 128 * 2.0 ** -24 * (x.abs() @ torch.where(k.isfinite(), k, 0.0).abs().t()) * scale + 4 * 2.0 ** -24 * z.abs()
                err = torch.where(seen & z.isfinite(), mag, 0.0).amax(-1, keepdim=True)
            small = k.shape[0] * 2.0 ** -25 * clean.abs().amax(0) if q.dtype == torch.float16 and k.shape[0] else 0.0
            t = u * (2 * out.abs() + a) + 2 * err * a + small + 2.0 ** -25
            o[i, :, h * g:(h + 1) * g] = out.transpose(0, 1)
            tol[i, :, h * g:(h + 1) * g] = t.transpose(0, 1)
    return o, tol


def inputs(r, n, s, hq, hkv, p, c, dtype, seed=0):
    gen = seeded(seed + 7 * s + p + c)

    def rn(*shape, wide=False):
        x = torch.randn(shape, generator=gen)
        if wide:
            x[..., ::16] *= 4.0
        return x.to(dtype).cuda()
    return (rn(r * n, s, hq, 128), rn(r, hkv, p, 128, wide=True), rn(r, hkv, p, 128), rn(r * n, hkv, c, 128, wide=True),
            rn(r * n, hkv, c, 128))


def check(got, q, pk, pv, ck, cv, starts, scale=None):
    o, tol = expected(q, pk, pv, ck, cv, starts, scale)
    worst = float(((got.double() - o).abs() / tol).nan_to_num(nan=1e9).max())
    assert worst <= 1.0, f'{worst:.2f} times the tolerance'


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("r,n,s,hq,hkv,p,start", [
    (1, 1, 1, 4, 1, 1, 0), (1, 4, 1, 32, 8, 200, 7), (1, 3, 1, 8, 8, 64, 63), (2, 5, 1, 6, 2, 65, 64), (1, 2, 1, 16, 1, 129, 200),
    (1, 9, 1, 8, 1, 63, 1000), (4, 2, 1, 16, 4, 700, 128), (1, 40, 1, 8, 2, 1000, 33), (1, 1, 1, 32, 8, 5000, 3000),
    (1, 33, 1, 4, 1, 257, 0), (3, 1, 1, 3, 1, 100, 100), (1, 4, 1, 14, 2, 70, 5),
    (1, 2, 2, 8, 2, 100, 0), (1, 3, 17, 8, 2, 64, 50), (2, 2, 33, 4, 4, 130, 64), (1, 1, 300, 8, 2, 77, 100), (1, 2, 65, 16, 2, 1, 1),
    (1, 8, 100, 32, 8, 333, 10), (1, 24, 40, 32, 8, 90, 3), (1, 1, 64, 4, 1, 64, 0), (2, 16, 130, 16, 8, 65, 77),
    (1, 24, 56, 32, 8, 90, 3), (2, 16, 250, 16, 8, 65, 77), (1, 4, 2, 32, 8, 300, 9), (1, 1, 8, 32, 8, 700, 100),
    (1, 4, 1, 32, 8, 1500, 7), (1, 8, 1, 32, 8, 2000, 300), (2, 5, 1, 6, 2, 1100, 64), (1, 4, 4, 8, 2, 1500, 60), (3, 11, 1, 8, 8, 600, 70),
    (1, 65, 1, 32, 8, 200, 9), (1, 1, 1, 71, 1, 1000, 20), (1, 2, 4, 16, 4, 900, 600)])
def test_against_64_bits(r, n, s, hq, hkv, p, start, dtype):
    print(f"prefix {r}x{n} S{s} {hq}/{hkv} P{p} start {start} {dtype}", flush=True)
    t = inputs(r, n, s, hq, hkv, p, start + s + 9, dtype)
    check(PX.attention(*t, start), *t, [start] * (r * n))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,s,start", [(1, 1, 0), (3, 1, 500), (2, 70, 0), (2, 5, 64)])
def test_without_a_prefix(n, s, start, dtype):
    t = inputs(1, n, s, 8, 2, 0, start + s, dtype)
    check(PX.attention(*t, start), *t, [start] * n)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("r,n,s,p", [(1, 6, 1, 200), (2, 3, 1, 64), (1, 6, 3, 31), (1, 6, 1, 0), (1, 6, 140, 10), (1, 24, 140, 70), (1, 24, 190, 70), (1, 4, 4, 100)])
def test_a_position_for_each_row_read_on_the_device(r, n, s, p, dtype):
    b, c = r * n, 700
    t = inputs(r, n, s, 16, 8, p, c, dtype)
    starts = torch.randint(0, c - s + 1, (b,), generator=seeded(n + s)).tolist()
    # the first position, the last, one before the capacity's end, rows without own positions, one far outside either way
    starts[:5] = [0, c - s, -s, -s - 3, -1][:b]
    check(PX.attention(*t, 0, torch.tensor(starts).cuda()), *t, starts)
    far = list(starts)
    far[0], far[1] = c + 5, -(1 << 40)
    got = PX.attention(*t, 0, torch.tensor(far).cuda())
    check(got, *t, far)
    if p == 0:
        assert bool((got[2] == 0).all()) and bool((got[3] == 0).all())
    one = torch.tensor([70]).cuda()
    assert torch.equal(PX.attention(*t, 0, one), PX.attention(*t, 70))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("s,n", [(1, 4), (3, 4), (150, 4), (70, 20)])
def test_what_lies_behind_the_last_position_counts_for_nothing(s, n, dtype):
    """Infinities, NaN and the type's lowest value behind the prefix and behind each row's own positions."""
    p, c = 77, 400
    q, pk, pv, ck, cv = inputs(1, n, s, *((8, 2) if n == 4 else (32, 8)), 200, c, dtype)
    starts = [0, 100, 63, c - s - 1] * (n // 4)
    want = PX.attention(q, pk[:, :, :p], pv[:, :, :p], ck, cv, 0, torch.tensor(starts).cuda())
    check(want, q, pk[:, :, :p], pv[:, :, :p], ck, cv, starts)
    for bad in (float('nan'), float('inf'), -float('inf'), torch.finfo(dtype).min):
        k2, v2, ck2, cv2 = (t.clone() for t in (pk, pv, ck, cv))
        k2[:, :, p:], v2[:, :, p:] = bad, bad
        for i, start in enumerate(starts):
            ck2[i, :, start + s:], cv2[i, :, start + s:] = bad, bad
        assert torch.equal(PX.attention(q, k2[:, :, :p], v2[:, :, :p], ck2, cv2, 0, torch.tensor(starts).cuda()), want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,s,start,p", [(2, 40, 20, 70), (24, 40, 20, 70), (2, 18, 20, 70), (24, 56, 20, 70), (2, 4, 28, 70), (2, 4, 28, 3000), (2, 4, 35, 70)])
def test_a_value_that_is_not_finite_stays_with_the_queries_that_see_it(n, s, start, p, dtype):
    t = inputs(1, n, s, 32, 8, p, 120, dtype)
    cv = t[4]
    cv[:, :, 30, 5], cv[:, :, 37, 8], cv[0, :, 33, :] = float('inf'), float('nan'), -float('inf')
    got = PX.attention(*t, start)
    o, tol = expected(*t, [start] * n)
    pos = start + torch.arange(s, device='cuda')
    bad = torch.zeros((n, s, 128), dtype=torch.bool, device='cuda')
    bad[:, pos >= 30, 5] = True
    bad[:, pos >= 37, 8] = True
    bad[0, pos >= 33, :] = True
    bad = bad[:, :, None, :].expand_as(got)
    assert bool((~got.isfinite() == bad).all())
    assert float(torch.where(bad, 0.0, (got.double() - o).abs() / tol).max()) <= 1.0
    assert bool(got[1, pos >= 37, :, 8].isnan().all()) and bool((got[1, pos >= 30, :, 5] == float('inf')).all())


def test_a_key_that_is_not_a_number_stays_with_its_row():
    t = inputs(1, 4, 1, 8, 2, 100, 80, torch.bfloat16)
    t[3][1, :, 20] = float('nan')
    got = PX.attention(*t, 40)
    assert bool(got[1].isnan().all()) and bool(got[[0, 2, 3]].isfinite().all())
    t[1][:, :, 3] = float('nan')
    assert bool(PX.attention(*t, 40).isnan().all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_layouts(dtype):
    """Queries with heads before positions, keys and values of heads side by side, and slices of larger buffers."""
    r, n, s, hq, hkv, p, c = 2, 2, 5, 8, 2, 90, 70
    t = inputs(r, n, s, hq, hkv, p, c, dtype)
    want = PX.attention(*t, 60)
    q2 = t[0].transpose(1, 2).contiguous().transpose(1, 2)
    rest = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in t[1:]]   # [.., positions, heads, 128]
    assert torch.equal(PX.attention(q2, *rest, 60), want)
    big = [torch.cat((x, x), 2)[:, :, :x.shape[2]] for x in t[1:]]
    assert torch.equal(PX.attention(t[0], *big, 60), want)
    both = torch.stack(t[1:3], 0)
    assert torch.equal(PX.attention(t[0], both[0], both[1], *t[3:], 60), want)
    check(PX.attention(*t, 60, scale=0.01), *t, [60] * 4, 0.01)
    check(PX.attention(*t, 60, scale=3.0), *t, [60] * 4, 3.0)


def test_rows_that_share_a_prefix_are_rows_with_copies_of_it():
    t = inputs(1, 6, 1, 16, 4, 333, 50, torch.bfloat16)
    q, pk, pv, ck, cv = t
    copies = PX.attention(q, pk.expand(6, -1, -1, -1).contiguous(), pv.expand(6, -1, -1, -1).contiguous(), ck, cv, 30)
    check(copies, *t, [30] * 6)


def test_captured_steps_and_other_streams():
    """One captured call replayed as the position moves on, against the eager call of that position, bit for bit; two graphs at
    once; and a call on a stream of its own."""
    n, c, p = 5, 900, 300
    t = inputs(1, n, 1, 16, 8, p, c, torch.bfloat16)
    q, pk, pv, ck, cv = t
    at = torch.zeros(1, dtype=torch.int64, device='cuda')
    rows = torch.zeros(n, dtype=torch.int64, device='cuda')
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graphs = []
    for dev in (at, rows):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            o = PX.attention(*t, 0, dev)
        graphs.append((g, o))
    torch.cuda.current_stream().wait_stream(stream)
    for i, pos in enumerate([0, 1, 63, 64, 500, c - 1, 12]):
        q.copy_(torch.randn(q.shape, generator=seeded(i)).to(q.dtype))
        at.fill_(pos)
        ragged = [(pos + 37 * j) % c for j in range(n)]
        rows.copy_(torch.tensor(ragged))
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert torch.equal(graphs[0][1], PX.attention(*t, pos))
        check(graphs[1][1], *t, ragged)
        for j in (0, n - 1):   # a row's sums do not depend on where the others stand
            assert torch.equal(graphs[1][1][j], PX.attention(*t, ragged[j])[j])
    want = PX.attention(*t, 100)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = PX.attention(*t, 100)
    side.synchronize()
    assert torch.equal(got, want)


def test_offsets_beyond_32_bits():
    """Own positions of the last rows and a prefix's last head start behind 2^31 elements."""
    b, hkv, c, p = 36, 8, 65536, 1 << 21
    free, _ = torch.cuda.mem_get_info()
    if free < 60 << 30:
        pytest.skip("needs 60 GiB")
    gen = torch.Generator(device='cuda').manual_seed(1)
    bf = dict(dtype=torch.bfloat16, device='cuda')
    ck, cv = torch.empty((b, hkv, c, 128), **bf), torch.empty((b, hkv, c, 128), **bf)
    starts = [c - 1 - 700 * (i % 3) for i in range(b)]
    ck[-2:].normal_(generator=gen)
    cv[-2:].normal_(generator=gen)
    q = torch.randn((b, 1, 16, 128), generator=gen, device='cuda').bfloat16()
    pk, pv = (torch.randn((1, hkv, 50, 128), generator=gen, device='cuda').bfloat16() for _ in range(2))
    got = PX.attention(q, pk, pv, ck, cv, 0, torch.tensor(starts).cuda())
    check(got[-2:], q[-2:], pk, pv, ck[-2:], cv[-2:], starts[-2:])
    del ck, cv
    pk, pv = torch.zeros((1, hkv, p, 128), **bf), torch.zeros((1, hkv, p, 128), **bf)
    assert pk.numel() >= 1 << 31
    for t in (pk, pv):
        t[:, -1, -3000:].normal_(generator=gen)
    ck, cv = (torch.randn((2, hkv, 9, 128), generator=gen, device='cuda').bfloat16() for _ in range(2))
    got = PX.attention(q[:2], pk, pv, ck, cv, 4)[:, :, -2:]
    check(got, q[:2, :, -2:], pk[:, -1:], pv[:, -1:], ck[:, -1:], cv[:, -1:], [4, 4])
