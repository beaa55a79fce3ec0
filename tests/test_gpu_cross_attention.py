"""Attention over an encoder's states (htpg_cross_attention) against a plain
implementation in FP64.

Bound of one output element, with w the row's weights relative to its largest
(largest 1) and W their sum:

  off <= ((p + 2 e) sum_j w_j |v_j| + f sum_j |v_j|) / W + h |out| + t,
  e = 2^-20 (1 + max_j (scale sum_d |q_d k_jd| + |bias_j|)).

p: a weight's rounding for the product with V, 2^-11 / 2^-8 (FP16 / BF16), and
2^-20 / 2^-15 with FP32 outputs (two parts); e: a score's FP32 error (products
are exact; the sum, the scaling and the exponential's argument and value are
good to a few 2^-23 of their size); f = 2^-24: FP16 weights below the normal
range; the products' sums add 2^-18 of sum_j w_j |v_j| (FP32 accumulation in
some order over up to 2^13 keys, errors of one sign at worst in 2^6 steps).  h:
the output's half ulp, t its smallest step."""
import math

import pytest
import torch

import htpg

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
INF = float("inf")
HALF_ULP = {F32: 2.0**-24, F16: 2.0**-11, BF16: 2.0**-8}


def reference(q, k, v, scale, lens=None, bias=None):
    """FP64 (out, sum w|v| / W, sum |v| / W, e) of every element; keys that take no part are left out."""
    b, n, h, d = q.shape
    group = h // k.shape[2]
    shape = (b, n, h, d)
    out, wv, av = (torch.zeros(shape, dtype=torch.float64, device=q.device) for _ in range(3))
    err = torch.zeros(b, n, h, 1, dtype=torch.float64, device=q.device)
    for i in range(b):
        m = k.shape[1] if lens is None else min(max(int(lens[i]), 0), k.shape[1])
        keep = torch.arange(m, device=q.device)
        if bias is not None:
            keep = keep[bias[i, :m] != -INF]
        if len(keep) == 0:
            continue
        for j in range(h):
            qq, kk, vv = q[i, :, j].double(), k[i, keep, j // group].double(), v[i, keep, j // group].double()
            s, size = qq @ kk.T * scale, qq.abs() @ kk.abs().T * scale
            if bias is not None:
                add = bias[i, keep].double()
                s, size = s + add, size + torch.where(add > -1e30, add.abs(), 0)  # lowest: no weight
            w = (s - s.amax(-1, keepdim=True)).exp()
            total = w.sum(-1, keepdim=True)
            out[i, :, j], wv[i, :, j], av[i, :, j] = w @ vv / total, w @ vv.abs() / total, vv.abs().sum(0) / total
            err[i, :, j] = 2.0**-20 * (1 + size.amax(-1, keepdim=True))
    return out, wv, av, err


def close(got, q, k, v, scale, lens=None, bias=None):
    want, wv, av, e = reference(q, k, v, scale, lens, bias)
    if got.dtype == F32:
        p, t = (2.0**-20 if q.dtype == F16 else 2.0**-15), 0.0
    else:
        p, t = HALF_ULP[q.dtype], 2.0**-24
    bound = (p + 2 * e + 2.0**-18) * wv + 2.0**-24 * av + HALF_ULP[got.dtype] * want.abs() * 1.01 + t + 1e-30
    off = (got.double() - want).abs()
    assert bool(torch.isfinite(got).all())
    assert bool((off <= bound).all()), f"off by {(off / bound).max().item():.2f} of the bound"


def call(q, k, v, dst, scale=None, lens=None, bias=None, out=None, **kw):
    scale = scale or 1 / math.sqrt(q.shape[3])
    out = torch.full(q.shape, float("nan"), dtype=dst, device=q.device) if out is None else out
    prm = htpg.attention_params(out, q, k, v, scale, **kw)
    assert htpg.cross_attention(prm, out, q, k, v, lens, bias) == 0
    assert htpg.check_device() == 0
    return out, scale


def inputs(gpu, b, n, m, h, hk, d, src, seed=0, sharp=1.0):
    g = torch.Generator(device=gpu).manual_seed(seed + 7919 * n + m)
    r = lambda *s: torch.randn(*s, generator=g, device=gpu)
    return (r(b, n, h, d) * sharp).to(src), r(b, m, hk, d).to(src), r(b, m, hk, d).to(src), g


TYPES = [(F16, F32), (F16, F16), (BF16, BF16), (BF16, F32)]


@pytest.mark.parametrize("src,dst", TYPES)
@pytest.mark.parametrize("b,n,m,h,hk,d", [
    (1, 1, 1, 1, 1, 8), (2, 1, 1500, 32, 8, 128), (3, 1, 77, 8, 8, 64), (5, 4, 333, 12, 2, 80), (1, 16, 4097, 4, 1, 160),
    (2, 17, 2, 3, 3, 72), (2, 127, 128, 4, 4, 64), (1, 128, 129, 4, 2, 128), (2, 129, 127, 2, 1, 96),
    (1, 256, 257, 3, 3, 40), (2, 300, 640, 2, 2, 192), (1, 513, 1000, 2, 1, 8), (1, 1000, 77, 5, 5, 64),
    (1, 65, 2500, 2, 2, 128), (3, 40, 5000, 1, 1, 64), (1, 2000, 16, 1, 1, 128),
    (2, 16, 300, 32, 8, 128), (1, 5, 200, 128, 1, 64), (1, 33, 150, 24, 3, 64), (1, 9, 100, 12, 2, 40), (1, 2, 70, 256, 1, 64),
])
def test_matches_fp64(gpu, b, n, m, h, hk, d, src, dst):
    q, k, v, _ = inputs(gpu, b, n, m, h, hk, d, src)
    out, scale = call(q, k, v, dst)
    close(out, q, k, v, scale)


@pytest.mark.parametrize("src,dst", TYPES)
@pytest.mark.parametrize("n,m,d", [(1, 300, 64), (3, 1030, 128), (140, 300, 64), (300, 77, 128), (129, 700, 160)])
def test_lengths_bias_and_what_masked_keys_hold(gpu, n, m, d, src, dst):
    b, h, hk = 7, 4, 2
    q, k, v, g = inputs(gpu, b, n, m, h, hk, d, src)
    lens = torch.tensor([m, 0, 1, m // 2, m + 9, -3, 65], dtype=torch.int32, device=gpu)
    bias = torch.randn(b, m, generator=g, device=gpu) * 2
    bias[torch.rand(b, m, generator=g, device=gpu) < 0.3] = -INF
    bias[3] = -INF                    # leaves nothing
    bias[4, : m - 1] = -INF           # the last key alone
    bias[4, m - 1] = 0.5
    bias[6, :64] = -INF
    bias[0, 5] = torch.finfo(F32).min  # the type's lowest value: no weight, but it takes part
    # what takes no part may hold anything
    dead = (torch.arange(m, device=gpu) >= lens[:, None].clamp(0, m)) | (bias == -INF)
    for bad in (float("nan"), INF, -INF):
        pick = dead & (torch.rand(b, m, generator=g, device=gpu) < 0.4)
        k[pick], v[pick] = bad, bad
    out, scale = call(q, k, v, dst, lens=lens, bias=bias)
    close(out, q, k, v, scale, lens, bias)
    assert bool((out[[1, 3, 5]] == 0).all())
    # lengths alone, and bias alone
    k2, v2 = torch.nan_to_num(k, 1.0, 2.0, 3.0), torch.nan_to_num(v, 1.0, 2.0, 3.0)
    out, _ = call(q, k2, v2, dst, lens=lens)
    close(out, q, k2, v2, scale, lens)
    out, _ = call(q, k, v2, dst, bias=torch.where(dead, -INF, bias))
    close(out, q, k, v2, scale, None, torch.where(dead, -INF, bias))


@pytest.mark.parametrize("n", [1, 8, 200])
def test_bias_all_lowest_value_is_uniform(gpu, n):
    q, k, v, _ = inputs(gpu, 2, n, 200, 2, 2, 64, F16)
    bias = torch.full((2, 200), torch.finfo(F32).min, device=gpu)
    out, _ = call(q, k, v, F32, bias=bias)
    want = v.double().mean(1, keepdim=True).expand(-1, n, -1, -1)
    assert float((out.double() - want).abs().max()) <= 1e-5


@pytest.mark.parametrize("n,m", [(1, 900), (200, 900)])
@pytest.mark.parametrize("src,dst", TYPES)
def test_sharp_rising_and_far_scores(gpu, n, m, src, dst):
    """Scores that grow along the keys, by little (the running maximum lags behind) and by a lot, and weights of one key."""
    q, k, v, _ = inputs(gpu, 1, n, m, 2, 2, 64, src)
    for step in (0.004, 0.05, 2.0):
        ramp = torch.arange(m, device=gpu, dtype=torch.float32)[None] * step
        for bias in (ramp, -ramp, ramp - 1e5):
            out, scale = call(q, k, v, dst, bias=bias)
            close(out, q, k, v, scale, None, bias)
    q = (q.float() * 30).to(src)
    out, scale = call(q, k, v, dst)
    close(out, q, k, v, scale)
    out, _ = call(q, k, v, dst, scale=1e-30)
    close(out, q, k, v, 1e-30)


@pytest.mark.parametrize("n", [1, 5, 150])
def test_nan_and_infinite_scores_stay_in_their_row(gpu, n):
    q, k, v, _ = inputs(gpu, 1, n, 200, 2, 1, 64, F16)
    q[0, 0, 0, 3] = float("nan")
    out = torch.zeros(1, n, 2, 64, device=gpu)
    prm = htpg.attention_params(out, q, k, v, 0.125)
    assert htpg.cross_attention(prm, out, q, k, v) == 0
    assert bool(out[0, 0, 0].isnan().all())
    q[0, 0, 0, 3] = 0
    keep = out.clone()
    keep[0, 0, 0] = 0
    assert bool(torch.isfinite(keep).all())


@pytest.mark.parametrize("n", [1, 200])
def test_layouts(gpu, n):
    """[batch][heads][tokens][dim] operands, a packed key/value projection, shared encoder states, padded outputs."""
    g = torch.Generator(device=gpu).manual_seed(3)
    b, m, h, hk, d = 3, 150, 4, 2, 64
    q = torch.randn(b, h, n, d, generator=g, device=gpu).half().transpose(1, 2)
    kv = torch.randn(b, m, 2 * hk * d + 8, generator=g, device=gpu).half()
    k, v = kv[..., :hk * d].unflatten(-1, (hk, d)), kv[..., hk * d:2 * hk * d].unflatten(-1, (hk, d))
    big = torch.full((b, n, h * d + 4), 5.0, device=gpu)
    out = big[..., :h * d].unflatten(-1, (h, d))
    out, scale = call(q, k, v, F32, out=out)
    close(out, q, k, v, scale)
    assert bool((big[..., h * d:] == 5).all())
    k1, v1 = k[:1].expand(b, -1, -1, -1), v[:1].expand(b, -1, -1, -1)
    bias = torch.randn(1, m, generator=g, device=gpu)
    out, _ = call(q, k1, v1, F16, bias=bias, bias_stride=0)
    close(out, q, k1, v1, scale, None, bias.expand(b, -1))
    # one copy of the queries for every head, and for every batch
    for qe in (q[:, :, :1].expand(-1, -1, h, -1), q[:1].expand(b, -1, -1, -1)):
        out, _ = call(qe, k, v, F16)
        close(out, qe, k, v, scale)
    # one batch, one head, strides of extents of one are not looked at
    q1 = q[:1, :, :1].as_strided((1, n, 1, d), (3, q.stride(1), 5, 1))
    k2 = k[:1, :, :1].as_strided((1, m, 1, d), (1, k.stride(1), 7, 1))
    v2 = v[:1, :, :1].as_strided((1, m, 1, d), (1, v.stride(1), 7, 1))
    out, _ = call(q1, k2, v2, F16)
    close(out, q1, k2, v2, scale)


def test_no_keys_gives_zeros(gpu):
    for n in (1, 200):
        q, k, v, _ = inputs(gpu, 2, n, 0, 4, 4, 64, F16)
        out, _ = call(q, k, v, F32)
        assert bool((out == 0).all())


@pytest.mark.parametrize("n,m", [(1, 5000), (100, 5000), (500, 300)])
def test_same_bits_every_time(gpu, n, m):
    q, k, v, _ = inputs(gpu, 1, n, m, 4, 2, 128, F16)
    first, _ = call(q, k, v, F32)
    for _ in range(5):
        again, _ = call(q, k, v, F32)
        assert torch.equal(first, again)


@pytest.mark.parametrize("n", [1, 150])
def test_other_streams_and_graph(gpu, n):
    q, k, v, _ = inputs(gpu, 2, n, 3000, 2, 2, 64, F16)
    side = [torch.cuda.Stream() for _ in range(3)]
    outs = [torch.empty(q.shape, device=gpu) for _ in side]
    prm = htpg.attention_params(outs[0], q, k, v, 0.125)
    torch.cuda.synchronize()
    for _ in range(4):  # several streams at once, each with its own scratch
        for st, o in zip(side, outs):
            assert htpg.cross_attention(prm, o, q, k, v, stream=st) == 0
    torch.cuda.synchronize()
    for o in outs:
        close(o, q, k, v, 0.125)
    graph = torch.cuda.CUDAGraph()
    out = torch.zeros_like(outs[0])
    with torch.cuda.graph(graph, stream=side[0]):
        assert htpg.cross_attention(prm, out, q, k, v, stream=side[0]) == 0
    q.mul_(0.5)
    # a larger call on that stream moves its scratch; the graph keeps what it captured
    big = inputs(gpu, 8, n, 6000, 4, 4, 128, F16, seed=1)
    o2 = torch.empty(big[0].shape, device=gpu)
    p2 = htpg.attention_params(o2, *big[:3], 0.1)
    torch.cuda.synchronize()
    assert htpg.cross_attention(p2, o2, *big[:3], stream=side[0]) == 0
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    close(out, q, k, v, 0.125)


def test_far_offsets(gpu):
    """Tokens whose element offsets pass 2^31: strided views over a large buffer."""
    b, m, h, d = 1, 300, 1, 64
    stride = 1 << 23  # 300 tokens x 2^23 elements: 5 GB
    buf = torch.empty((m - 1) * stride + d, dtype=F16, device=gpu)
    k = buf.as_strided((b, m, h, d), (0, stride, 0, 1))
    g = torch.Generator(device=gpu).manual_seed(2)
    k.copy_(torch.randn(b, m, h, d, generator=g, device=gpu).half())
    for n in (1, 140):
        q = torch.randn(b, n, h, d, generator=g, device=gpu).half()
        out, scale = call(q, k, k, F32)
        close(out, q, k.contiguous(), k.contiguous(), scale)
