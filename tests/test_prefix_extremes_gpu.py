"""Attention over a shared prefix where values or keys are not finite: what is seen counts, in every form of the kernel."""
import pytest
import torch

from _util import seeded
from test_prefix_gpu import DTYPES, expected, inputs

from qwen3_triton.inference import prefix as PX

pytestmark = pytest.mark.gpu

# single queries and short chunks in one pass over few positions, in jobs behind many, and tiles of longer chunks in either
FORMS = [(1, 6, 1, 8, 2, 100, 9), (1, 6, 2, 8, 2, 100, 9), (1, 6, 4, 8, 2, 128, 0), (2, 3, 3, 8, 2, 70, 5), (1, 1, 4, 8, 2, 3000, 9), (1, 2, 2, 8, 2, 3000, 0),
         (1, 1, 16, 4, 4, 2048, 70), (1, 9, 1, 8, 2, 3000, 5), (2, 2, 3, 8, 2, 1500, 0), (1, 4, 4, 8, 2, 3000, 3), (1, 3, 40, 8, 2, 100, 9),
         (1, 3, 40, 8, 2, 3000, 9), (1, 24, 56, 32, 8, 200, 3)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("r,n,s,hq,hkv,p,start", FORMS)
def test_values_of_the_prefix_that_are_not_finite(r, n, s, hq, hkv, p, start, dtype):
    """Every query sees the whole prefix: infinite where a value is infinite, not a number where one is none, in every row."""
    print(f"values {r}x{n} S{s} P{p} start {start} {dtype}", flush=True)
    t = inputs(r, n, s, hq, hkv, p, start + s + 9, dtype)
    pv = t[2]
    pv[:, :, 60, 5], pv[:, :, p - 1, 8], pv[0, :, p // 2, 11] = float('inf'), float('nan'), -float('inf')
    got = PX.attention(*t, start)
    o, tol = expected(*t, [start] * (r * n))
    bad = torch.zeros_like(got, dtype=torch.bool)
    bad[..., 5], bad[..., 8], bad[:n, ..., 11] = True, True, True
    assert bool((~got.isfinite() == bad).all())
    assert bool(got[..., 8].isnan().all())
    assert float(torch.where(bad, 0.0, (got.double() - o).abs() / tol).max()) <= 1.0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("start", [0, 5, 61])
@pytest.mark.parametrize("r,n,s,hq,hkv,p", sorted({f[:6] for f in FORMS}))
def test_own_keys_that_are_not_numbers(r, n, s, hq, hkv, p, start, dtype):
    """All of a row's own keys, beside positions that are not there yet: its queries are not numbers, the others' stay as they were."""
    t = inputs(r, n, s, hq, hkv, p, 160, dtype)
    want = PX.attention(*t, start)
    row = r * n - 1
    t[3][row, :, :start + s] = float('nan')
    got = PX.attention(*t, start)
    assert bool(got[row].isnan().all())
    assert torch.equal(got[:row], want[:row])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("r,n,s,hq,hkv,p,start", FORMS)
def test_keys_of_the_prefix_that_are_not_numbers(r, n, s, hq, hkv, p, start, dtype):
    """The last part of a prefix, whose last block has positions that are not there: nobody behind it has a number."""
    t = inputs(r, n, s, hq, hkv, p, start + s + 9, dtype)
    want = PX.attention(*t, start)
    t[1][0, :, p - p // 3:] = float('nan')
    got = PX.attention(*t, start)
    assert bool(got[:n].isnan().all())
    assert torch.equal(got[n:], want[n:])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("r,n,s,hq,hkv,p,start", FORMS)
def test_very_large_scores(r, n, s, hq, hkv, p, start, dtype):
    """Scores of 2^34 and more, exact in fp32 and at least 2^30 apart where they differ: each query's output is the mean of the values at
    its largest one."""
    t = inputs(r, n, s, hq, hkv, p, start + s + 9, dtype)
    gen = seeded(p + s)
    t[0].copy_((2 ** 15 * (1 - 2 * torch.randint(0, 2, t[0].shape[:3], generator=gen)))[..., None])
    for k in (t[1], t[3]):
        k.copy_((2 ** 12 * torch.randint(-8, 9, k.shape[:3], generator=gen))[..., None])
    got = PX.attention(*t, start)
    o, _ = expected(*t, [start] * (r * n))
    a, _ = expected(t[0], t[1], t[2].abs(), t[3], t[4].abs(), [start] * (r * n))
    u = torch.finfo(dtype).eps / 2   # the output's rounding; weights of 2^x, equal ones alike, and their sum in fp32
    tol = u * o.abs() + (u + 2.0 ** -14) * a + 2.0 ** -24
    assert float(((got.double() - o).abs() / tol).nan_to_num(nan=1e9).max()) <= 1.0
