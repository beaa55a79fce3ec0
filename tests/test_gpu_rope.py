"""Per-head norm, rotary positions and conversion (htpg_qkv_rope) and the
position table (htpg_rope_table) against a plain implementation in FP64.

Bounds.  u = 2^-24 (FP32), h = the output type's half ulp (2^-24, 2^-11,
2^-8).  A normed element: the sum of up to 512 squares by lanes has at most 16
terms in a row and 5 tree steps, so its relative error is below 21 u, halved by
the root; root, reciprocal, two products and the mean add less than 8 u: 20 u in
all.  A rotated pair adds three roundings on |a| + |b|: 24 u (|a| + |b|).  The
store adds h |y| (and 2^-25 for FP16 results below the normal range)."""
import math

import pytest
import torch

import htpg

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
HALF_ULP = {F32: 2.0**-24, F16: 2.0**-11, BF16: 2.0**-8}
EPS = 1e-6


def rotated(x, table, pos, rot, half, weight):
    """FP64: x [b][s][h][d] -> (y, |a| + |b| of each element's pair)."""
    x = x.double()
    if weight is not None:
        x = x / (x.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * weight.double()
    size = x.abs()
    y = x.clone()
    if rot:
        i = torch.arange(rot // 2, device=x.device)
        a, b = (i, i + rot // 2) if half else (2 * i, 2 * i + 1)
        cs = table.double()[pos.long()][:, :, None]
        y[..., a] = x[..., a] * cs[..., 0] - x[..., b] * cs[..., 1]
        y[..., b] = x[..., a] * cs[..., 1] + x[..., b] * cs[..., 0]
        size = size.clone()
        size[..., a] = x[..., a].abs() + x[..., b].abs()
        size[..., b] = size[..., a]
    return y, size


def close(got, want, size):
    h = HALF_ULP[got.dtype]
    bound = 24 * 2.0**-24 * size * 1.5 + h * want.abs() * 1.01 + 2.0**-25
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), f"off by {(off / bound).max().item():.2f} of the bound"


def table_of(rows, rot, gpu, **kw):
    t = torch.full((rows, rot // 2, 2), float("nan"), device=gpu)
    htpg.check(htpg.rope_table(t, rot, **kw), "htpg_rope_table")
    return t


@pytest.mark.parametrize("b,s,hq,hk,d,rot,half,norm,src,dst", [
    (1, 1, 32, 8, 128, 128, True, False, F32, F16),
    (1, 1, 1, 1, 8, 8, False, True, F16, F16),
    (2, 77, 24, 24, 64, 64, False, True, F32, F16),
    (3, 37, 20, 4, 80, 40, False, True, BF16, BF16),
    (2, 129, 6, 3, 72, 36, True, True, F32, F32),
    (2, 65, 5, 5, 40, 20, True, False, F16, F32),
    (4, 33, 12, 12, 128, 64, True, True, F32, BF16),
    (1, 300, 8, 2, 160, 160, True, True, BF16, F16),
    (1, 19, 3, 1, 512, 512, False, True, F32, F32),
    (2, 21, 3, 1, 510, 254, True, True, F16, BF16),
    (2, 21, 3, 1, 33, 30, False, True, F32, F16),      # odd head dims: nothing is 16-byte aligned
    (2, 21, 3, 1, 17, 2, True, True, F16, F16),
    (1, 50, 2, 2, 7, 0, True, True, F32, F32),         # no rotation
    (1, 4100, 9, 3, 64, 64, True, True, F32, F16),
])
@pytest.mark.parametrize("positions", [False, True])
def test_matches_fp64(gpu, b, s, hq, hk, d, rot, half, norm, src, dst, positions):
    g = torch.Generator(device=gpu).manual_seed(d * 1000 + s)
    rows = max(s, 64)
    packed = (torch.randn(b, s, (hq + 2 * hk) * d, generator=g, device=gpu) * 3).to(src)
    q, k, v = (t.unflatten(-1, (-1, d)) for t in packed.split([hq * d, hk * d, hk * d], -1))
    table = table_of(rows, rot, gpu, base=500.0) if rot else None
    pos = torch.randint(0, rows, (b, s), generator=g, device=gpu, dtype=torch.int32) if positions else None
    wq, wk = (1 + 0.3 * torch.randn(2, d, generator=g, device=gpu)).unbind(0) if norm else (None, None)
    outs = [torch.full((b, s, n, d), float("nan"), dtype=dst, device=gpu) for n in (hq, hk, hk)]
    prm = htpg.rope_params(q, k, v, *outs, rot_dim=rot, layout=int(half), table_rows=rows, eps=EPS)
    assert htpg.qkv_rope(prm, *outs, q, k, v, wq, wk, table, pos) == 0
    at = torch.arange(s, device=gpu).expand(b, s) if pos is None else pos
    close(outs[0], *rotated(q, table, at, rot, half, wq))
    close(outs[1], *rotated(k, table, at, rot, half, wk))
    assert torch.equal(outs[2], v.to(dst))


def test_strided_outputs_parts_and_in_place(gpu):
    g = torch.Generator(device=gpu).manual_seed(5)
    b, s, h, d = 2, 45, 6, 64
    x = torch.randn(b, s, h, d, generator=g, device=gpu)
    table, at = table_of(64, d, gpu), torch.arange(s, device=gpu).expand(b, s)
    want, size = rotated(x, table, at, d, False, None)
    # [batch][heads][tokens][dim], inside a larger buffer whose rest stays untouched
    big = torch.full((b, h, s + 3, d + 8), 7.0, dtype=F16, device=gpu)
    out = big[:, :, :s, :d].transpose(1, 2)
    prm = htpg.rope_params(x, None, None, out, None, None, d, 0, 64)
    assert htpg.qkv_rope(prm, out, None, None, x, None, None, table=table) == 0
    close(out, want, size)
    assert bool((big[:, :, s:] == 7).all()) and bool((big[..., d:] == 7).all())
    # tokens and heads exchanged in the input, two bytes off alignment; keys alone
    raw = torch.zeros(b * h * s * d + 1, dtype=F16, device=gpu)[1:].view(b, h, s, d).copy_(x.transpose(1, 2))
    k = raw.transpose(1, 2)
    out = torch.empty(b, s, h, d, dtype=F32, device=gpu)
    prm = htpg.rope_params(None, k, None, None, out, None, d, 1, 64)
    assert htpg.qkv_rope(prm, None, out, None, None, k, None, table=table) == 0
    close(out, *rotated(k, table, at, d, True, None))
    # in place
    for half in (0, 1):
        y = x.clone()
        w = torch.rand(d, generator=g, device=gpu)
        prm = htpg.rope_params(y, None, None, y, None, None, 32, half, 64)
        t = table_of(64, 32, gpu)
        assert htpg.qkv_rope(prm, y, None, None, y, None, None, q_weight=w, table=t) == 0
        close(y, *rotated(x, t, at, 32, bool(half), w))


def test_values_that_norms_meet(gpu):
    """Zero rows stay zero, huge and tiny rows keep their direction, NaN stays in its row."""
    d = 64
    g = torch.Generator(device=gpu).manual_seed(6)
    x = torch.randn(1, 6, 2, d, generator=g, device=gpu)
    x[0, 0] = 0
    x[0, 1] *= 1e15
    x[0, 2] *= 1e-18
    x[0, 3, 0, 5] = float("nan")
    w = torch.ones(d, device=gpu)
    table = table_of(8, d, gpu)
    out = torch.empty_like(x)
    prm = htpg.rope_params(x, None, None, out, None, None, d, 1, 8, eps=EPS)
    assert htpg.qkv_rope(prm, out, None, None, x, None, None, q_weight=w, table=table) == 0
    want, size = rotated(x, table, torch.arange(6, device=gpu)[None], d, True, w)
    assert bool((out[0, 0] == 0).all()) and bool(out[0, 3, 0].isnan().all())
    ok = torch.ones(6, 2, dtype=torch.bool, device=gpu)
    ok[3, 0] = False
    close(out[0][ok], want[0][ok], size[0][ok])


def test_positions_outside_the_table_are_nan_rows(gpu):
    x = torch.ones(1, 4, 3, 32, device=gpu)
    table = table_of(16, 32, gpu)
    pos = torch.tensor([[3, -1, 16, 2**31 - 1]], dtype=torch.int32, device=gpu)
    outs = [torch.zeros_like(x) for _ in range(3)]
    prm = htpg.rope_params(x, x, x, *outs, 32, 0, 16)
    assert htpg.qkv_rope(prm, *outs, x, x, x, table=table, positions=pos) == 0
    for o in outs[:2]:
        assert bool(o[0, 0].isfinite().all()) and bool(o[0, 1:].isnan().all())
    assert torch.equal(outs[2], x)


def test_other_stream_and_graph(gpu):
    d, s = 64, 200
    g = torch.Generator(device=gpu).manual_seed(8)
    x = torch.randn(1, s, 8, d, generator=g, device=gpu)
    table = table_of(256, d, gpu)
    out = torch.zeros(1, s, 8, d, dtype=F16, device=gpu)
    prm = htpg.rope_params(x, None, None, out, None, None, d, 1, 256)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            assert htpg.qkv_rope(prm, out, None, None, x, None, None, table=table, stream=side) == 0
    x.mul_(2)
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    close(out, *rotated(x, table, torch.arange(s, device=gpu)[None], d, True, None))


# ------------------------------------------------------------------ the table
def table_fp64(rows, rot, scaling, base, factor, original_rows, beta_fast, beta_slow):
    i = torch.arange(rot // 2, dtype=torch.float64)
    mult = 1.0
    if scaling == htpg.ROPE_NTK:
        base = base * factor ** (rot / (rot - 2))
    f = base ** (-2 * i / rot)
    if scaling == htpg.ROPE_LINEAR:
        f = f / factor
    if scaling == htpg.ROPE_YARN:
        c = lambda turns: rot / 2 * math.log(original_rows / (turns * 2 * math.pi)) / math.log(base)
        low, high = max(math.floor(c(beta_fast)), 0), min(math.ceil(c(beta_slow)), rot - 1)
        high = high if high > low else low + 0.001
        ramp = ((i - low) / (high - low)).clamp(0, 1)
        f = f / factor * ramp + f * (1 - ramp)
        mult = 0.1 * math.log(factor) + 1
    angle = torch.arange(rows, dtype=torch.float64)[:, None] * f
    return torch.stack([angle.cos(), angle.sin()], -1) * mult


@pytest.mark.parametrize("rows,rot,kw", [
    (1, 2, dict()), (131072, 8, dict(base=1e4)), (5000, 128, dict(base=1e6)),
    (4097, 64, dict(scaling=htpg.ROPE_LINEAR, factor=4.0)), (4097, 64, dict(scaling=htpg.ROPE_NTK, factor=8.0)),
    (9000, 128, dict(scaling=htpg.ROPE_YARN, factor=4.0, original_rows=2048)),
    (9000, 20, dict(scaling=htpg.ROPE_YARN, factor=40.0, original_rows=1, beta_fast=1.0)),
])
def test_table(gpu, rows, rot, kw):
    kw = {**dict(scaling=0, base=10000.0, factor=1.0, original_rows=0, beta_fast=32.0, beta_slow=1.0), **kw}
    got = table_of(rows, rot, gpu, **kw).cpu().double()
    # angles up to 2^17 in FP64 from a power and a product good to 2^-51: 2^-34; the store rounds by 2^-25 (values < 2)
    assert float((got - table_fp64(rows, rot, **kw)).abs().max()) <= 2.0**-24


@pytest.mark.parametrize("src", [F32, F16])
@pytest.mark.parametrize("d,rot,half", [(33, 30, 0), (33, 30, 1), (7, 2, 0), (510, 254, 1), (64, 64, 1)])
def test_positions_outside_the_table_at_any_head_dim(gpu, d, rot, half, src):
    """As above at sizes without vectors, and with a table that has no row."""
    x = torch.ones(2, 3, 2, d, device=gpu).to(src)
    table = table_of(16, rot, gpu)
    pos = torch.tensor([[3, -1, 16], [-2**31, 2**31 - 1, 15]], dtype=torch.int32, device=gpu)
    outs = [torch.zeros_like(x) for _ in range(3)]
    prm = htpg.rope_params(x, x, x, *outs, rot, half, 16)
    assert htpg.qkv_rope(prm, *outs, x, x, x, table=table, positions=pos) == 0
    inside = (pos >= 0) & (pos < 16)
    for o in outs[:2]:
        close(o[inside][:, None], *(y[inside][:, None] for y in rotated(x, table, pos.clamp(0, 15), rot, half, None)))
        assert bool(o[~inside].isnan().all())
    assert torch.equal(outs[2], x)
    prm = htpg.rope_params(x, x, x, *outs, rot, half, 0)
    assert htpg.qkv_rope(prm, *outs, x, x, x, table=table, positions=pos) == 0
    assert all(bool(o.isnan().all()) for o in outs[:2]) and torch.equal(outs[2], x)
