"""Low-rank adapters beside a shared projection (htpg_lora_run) against a
plain implementation in FP64.

Bound: adapter weights are exact operands; x and t = x A^T are carried in parts
that keep 21 bits or more, and sums are FP32 over at most 2^5 roundings in a row
between exact regroupings of up to 2^14 terms, so with T = sum_k |x_k A_rk|

  off <= 2^-18 |scale| sum_r T_r |B_nr| + 2^-22 (|base| + |out|)."""
import pytest
import torch

import htpg

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def reference(base, x, ids, a, b, ranks, scales):
    out, size = base.double(), torch.zeros_like(base, dtype=torch.float64)
    for j in range(a.shape[0]):
        rows, r = torch.nonzero(ids == j)[:, 0], min(max(int(ranks[j]), 0), a.shape[1])
        aa, bb, s = a[j, :r].double(), b[j, :, :r].double(), float(scales[j])
        xx = x[rows].double()
        out[rows] += s * (xx @ aa.T) @ bb.T
        size[rows] = abs(s) * (xx.abs() @ aa.abs().T) @ bb.abs().T
    return out, size


def close(got, base, *rest):
    want, size = reference(base, *rest)
    bound = 2.0**-18 * size + 2.0**-22 * (base.abs().double() + want.abs()) + 1e-37
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), f"off by {(off / bound).max().item():.2f} of the bound"


def inputs(gpu, m, k, n, adapters, rank, src, seed=0):
    g = torch.Generator(device=gpu).manual_seed(seed + m * 31 + n)
    r = lambda *s: torch.randn(*s, generator=g, device=gpu)
    x = r(m, k)
    x = torch.where(torch.rand(m, k, generator=g, device=gpu) < 0.01, x * 20, x)
    return (x, r(m, n), torch.randint(-1, adapters + 1, (m,), generator=g, device=gpu, dtype=torch.int32),
            (r(adapters, rank, k) / k**0.5).to(src), r(adapters, n, rank).to(src),
            torch.full((adapters,), rank, dtype=torch.int32, device=gpu), 0.5 + torch.rand(adapters, generator=g, device=gpu))


def call(x, base, ids, a, b, ranks, scales, out=None):
    out = torch.full((x.shape[0], b.shape[1]), float("nan"), device=x.device) if out is None else out
    prm = htpg.lora_params(out, base, x, a, b)
    assert htpg.lora_run(prm, out, base, x, ids, a, b, ranks, scales) == 0
    assert htpg.check_device() == 0
    return out


@pytest.mark.parametrize("src", [F16, BF16])
@pytest.mark.parametrize("m,k,n,adapters,rank", [
    (1, 8, 8, 1, 8), (1, 4096, 1000, 1, 16), (4, 512, 14336, 4, 16), (16, 14336, 512, 16, 8), (17, 1152, 4608, 3, 64),
    (33, 1544, 200, 40, 128), (64, 776, 1536, 5, 32), (77, 768, 776, 2, 24), (129, 6144, 1536, 7, 40),
    (1000, 1536, 1544, 6, 32), (2500, 264, 392, 300, 8), (4096, 512, 512, 3, 128), (300, 40, 24, 2, 72),
])
def test_matches_fp64(gpu, m, k, n, adapters, rank, src):
    x, base, ids, a, b, ranks, scales = inputs(gpu, m, k, n, adapters, rank, src)
    close(call(x, base, ids, a, b, ranks, scales), base, x, ids, a, b, ranks, scales)
    # whole requests one after another, as prompts come
    ids = (torch.arange(m, device=gpu) * adapters // m).int()
    close(call(x, base, ids, a, b, ranks, scales), base, x, ids, a, b, ranks, scales)


@pytest.mark.parametrize("m", [3, 40, 500])
@pytest.mark.parametrize("src", [F16, BF16])
def test_ragged_ranks_and_what_lies_past_them(gpu, m, src):
    x, base, ids, a, b, _, scales = inputs(gpu, m, 328, 456, 8, 32, src)
    ranks = torch.tensor([0, 1, 7, 8, 17, 32, 99, -4], dtype=torch.int32, device=gpu)
    for j in range(8):
        r = min(max(int(ranks[j]), 0), 32)
        a[j, r:], b[j, :, r:] = float("nan"), float("inf")
    close(call(x, base, ids, a, b, ranks, scales), base, x, ids, a, b, ranks, scales)


@pytest.mark.parametrize("m", [2, 30, 300])
def test_base_forms_and_strides(gpu, m):
    k, n = 264, 520
    x, base, ids, a, b, ranks, scales = inputs(gpu, m, k, n, 3, 16, F16)
    want = (base, x, ids, a, b, ranks, scales)
    out = base.clone()
    call(x, out, ids, a, b, ranks, scales, out=out)  # in place
    close(out, *want)
    out = call(x, None, ids, a, b, ranks, scales)
    close(out, torch.zeros_like(base), *want[1:])
    xs = torch.full((m, k + 12), float("nan"), device=gpu)
    xs[:, :k] = x
    bs = torch.full((m, n + 4), float("nan"), device=gpu)
    bs[:, :n] = base
    os_ = torch.full((m, n + 8), 3.0, device=gpu)
    call(xs[:, :k], bs[:, :n], ids, a, b, ranks, scales, out=os_[:, :n])
    close(os_[:, :n], *want)
    assert bool((os_[:, n:] == 3).all())


@pytest.mark.parametrize("m", [5, 100])
def test_rows_keep_their_own_values(gpu, m):
    """A row without an adapter is its base bit for bit, and NaN or infinity in one row's x changes no other row."""
    x, base, ids, a, b, ranks, scales = inputs(gpu, m, 256, 264, 4, 16, F16)
    ids[:] = torch.arange(m, device=gpu) % 4
    ids[1], ids[3] = -1, 2**31 - 1
    plain = call(x, base, ids, a, b, ranks, scales)
    assert torch.equal(plain[1], base[1]) and torch.equal(plain[3], base[3])
    x[0, 7], x[2, 9] = float("nan"), float("inf")
    x[1, 0] = float("nan")  # not read into anything
    out = call(x, base, ids, a, b, ranks, scales)
    assert bool(out[0].isnan().all()) and not bool(out[2].isfinite().any())
    rest = [i for i in range(m) if i not in (0, 2)]
    assert torch.equal(out[rest], plain[rest])


@pytest.mark.parametrize("m", [4, 50, 200])
def test_large_and_small_magnitudes(gpu, m):
    x, base, ids, a, b, ranks, scales = inputs(gpu, m, 512, 264, 3, 16, F16)
    for f in (1e6, 1e-6, 1e-12):
        close(call(x * f, base * f, ids, a, b, ranks, scales), base * f, x * f, ids, a, b, ranks, scales)


def test_same_bits_every_time_on_any_stream(gpu):
    for m in (4, 600):
        args = inputs(gpu, m, 1536, 1536, 5, 32, F16)
        x, base, ids, a, b, ranks, scales = args
        first = call(*args)
        prm = htpg.lora_params(first, base, x, a, b)
        streams = [torch.cuda.Stream() for _ in range(3)]
        outs = [torch.empty_like(first) for _ in streams]
        torch.cuda.synchronize()
        for _ in range(3):
            for st, o in zip(streams, outs):
                assert htpg.lora_run(prm, o, base, x, ids, a, b, ranks, scales, stream=st) == 0
        torch.cuda.synchronize()
        for o in outs:
            assert torch.equal(o, first)
