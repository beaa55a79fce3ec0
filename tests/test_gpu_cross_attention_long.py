"""Attention with FP32 outputs over many keys, where what the tensor core's
sums lose (they round towards zero) would add up, against FP64.

Bound of one output element, with w the row's weights and W their sum:

  off <= (p + 2 e + a) sum_j w_j |v_j| / W + f sum_j |v_j| / W + 2^-24 |out|

p, e, f as with fewer keys (weights in two parts: 2^-20 for FP16, 2^-15 for BF16;
e = 2^-20 (1 + the row's largest sum of |products|); f = 2^-24).  a: the sums.  256
keys are 16 products of 16 keys, each in two parts, so 32 additions that lose at
most 2^-23 of the sum so far: 2^-18.  The sums of 256 keys are added to nearest:
at most 32 times 2^-24 for 8192 keys: 2^-19."""
import math

import pytest
import torch

import htpg

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
INF = float("inf")


def check(q, k, v, bias=None):
    b, n, h, d = q.shape
    group, scale = h // k.shape[2], 1 / math.sqrt(d)
    out = torch.full(q.shape, float("nan"), device=q.device)
    assert htpg.cross_attention(htpg.attention_params(out, q, k, v, scale), out, q, k, v, None, bias) == 0
    assert htpg.check_device() == 0
    p = 2.0**-20 if q.dtype == F16 else 2.0**-15
    worst = 0.0
    for i in range(b):
        keep = torch.arange(k.shape[1], device=q.device)
        if bias is not None:
            keep = keep[bias[i] != -INF]
        for j in range(h):
            qq, kk, vv = q[i, :, j].double(), k[i, keep, j // group].double(), v[i, keep, j // group].double()
            s, size = qq @ kk.T * scale, qq.abs() @ kk.abs().T * scale
            if bias is not None:
                s, size = s + bias[i, keep].double(), size + bias[i, keep].double().abs()
            w = (s - s.amax(-1, keepdim=True)).exp()
            total = w.sum(-1, keepdim=True)
            want = w @ vv / total
            e = 2.0**-20 * (1 + size.amax(-1, keepdim=True))
            bound = (p + 2 * e + 2.0**-18 + 2.0**-19) * (w @ vv.abs()) / total + 2.0**-24 * (vv.abs().sum(0) / total + want.abs())
            worst = max(worst, ((out[i, :, j].double() - want).abs() / bound).max().item())
    assert worst <= 1, f"off by {worst:.2f} of the bound"


def tensors(gpu, n, m, h, hk, d, src, b=1):
    g = torch.Generator(device=gpu).manual_seed(n + m + d)
    return [torch.randn(b, t, hh, d, generator=g, device=gpu).to(src) for t, hh in ((n, h), (m, hk), (m, hk))]


SHAPES = [
    (2000, 5000, 20, 20, 64),    # more units than SMs: whole ones, and a last round in key ranges
    (300, 8192, 4, 2, 128),      # few units, all in key ranges
    (2100, 1100, 20, 20, 160),   # one buffer of scores
    (1, 8192, 8, 2, 128),        # the single tokens' kernel
    (130, 257, 2, 2, 40),        # one key past the fourth tile
]


@pytest.mark.parametrize("src", [F16, BF16])
@pytest.mark.parametrize("n,m,h,hk,d", SHAPES)
def test_sums_of_one_sign(gpu, n, m, h, hk, d, src):
    """Small scores and positive values: every product adds, every lost bit shows."""
    q, k, v = tensors(gpu, n, m, h, hk, d, src)
    check(q * 0.05, k, v.abs() + 0.5)


@pytest.mark.parametrize("n,m,h,hk,d", SHAPES)
def test_scores_that_keep_rising(gpu, n, m, h, hk, d):
    """The largest score so far grows from tile to tile, so every sum is scaled down again and again."""
    q, k, v = tensors(gpu, n, m, h, hk, d, F16)
    q = q.abs()
    k = (k * 0.1 + torch.linspace(0, 60.0 / math.sqrt(d), m, device=gpu)[None, :, None, None]).half()
    check(q, k, v)


@pytest.mark.parametrize("n,m,h,hk,d", SHAPES)
def test_runs_of_masked_keys(gpu, n, m, h, hk, d):
    """Whole tiles without a key, at the front and between others; what they hold is never seen."""
    q, k, v = tensors(gpu, n, m, h, hk, d, F16)
    bias = torch.zeros(1, m, device=gpu)
    bias[:, :m // 3] = -INF
    bias[:, m // 2:m // 2 + m // 4] = -INF
    bias[:, 5::7] = -INF
    gone = bias[0] == -INF
    k[:, gone], v[:, gone] = float("nan"), INF
    check(q, k, v, bias)
