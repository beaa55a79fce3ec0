"""Low-rank adapters over more rows than one round of small tiles covers, against
FP64, with the bound of fewer rows: x and t = x A^T keep 21 bits or more, sums are
FP32, so with T = sum_k |x_k A_rk|

  off <= 2^-18 |scale| sum_r T_r |B_nr| + 2^-22 (|base| + |out|)."""
import pytest
import torch

import htpg

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def run(gpu, m, k, n, adapters, max_rank, src, order):
    g = torch.Generator(device=gpu).manual_seed(m + k + adapters)
    r = lambda *s: torch.randn(*s, generator=g, device=gpu)  # noqa: E731
    x, base = r(m, k), r(m, n)
    a, b = (r(adapters, max_rank, k) / k**0.5).to(src), r(adapters, n, max_rank).to(src)
    ranks = torch.randint(0, max_rank + 1, (adapters,), generator=g, device=gpu, dtype=torch.int32)
    ranks[0] = max_rank
    scales = 0.5 + torch.rand(adapters, generator=g, device=gpu)
    if order == "mixed":
        ids = torch.randint(-1, adapters + 1, (m,), generator=g, device=gpu, dtype=torch.int32)
    else:  # requests one after another, their borders anywhere in a tile
        ids = (torch.arange(m, device=gpu) * adapters // m).int()
    for j in range(adapters):  # what lies past a rank is never seen
        a[j, int(ranks[j]):], b[j, :, int(ranks[j]):] = float("nan"), float("inf")
    out = torch.full((m, n), float("nan"), device=gpu)
    prm = htpg.lora_params(out, base, x, a, b)
    assert htpg.lora_run(prm, out, base, x, ids, a, b, ranks, scales) == 0
    assert htpg.check_device() == 0
    want, size = base.double(), torch.zeros(m, n, dtype=torch.float64, device=gpu)
    for j in range(adapters):
        rows, rank = torch.nonzero(ids == j)[:, 0], int(ranks[j])
        aa, bb, xx, s = a[j, :rank].double(), b[j, :, :rank].double(), x[rows].double(), float(scales[j])
        want[rows] += s * (xx @ aa.T) @ bb.T
        size[rows] = s * (xx.abs() @ aa.abs().T) @ bb.abs().T
    off = (out.double() - want).abs()
    bound = 2.0**-18 * size + 2.0**-22 * (base.abs().double() + want.abs())
    assert bool((off <= bound).all()), f"off by {(off / bound).max().item():.2f} of the bound"


@pytest.mark.parametrize("order", ["mixed", "in order"])
@pytest.mark.parametrize("m,k,n,adapters,max_rank,src", [
    (5000, 136, 64, 3, 16, F16),
    (16385, 264, 72, 7, 64, F16),   # one row past whole tiles
    (9999, 520, 40, 40, 32, BF16),  # more kinds of rows in a tile than its warps
    (20000, 1032, 64, 1, 24, F16),  # one adapter: no row out of order
    (6001, 72, 136, 300, 8, BF16),  # a kind for nearly every row of a tile
    (8191, 328, 64, 5, 128, F16),
])
def test_many_rows(gpu, m, k, n, adapters, max_rank, src, order):
    run(gpu, m, k, n, adapters, max_rank, src, order)
