"""Key biases at the ends of their range (htpg_cross_attention): NaN, and values
so large that FP32 scores are whole numbers and coarser."""
import pytest
import torch

import htpg
from test_gpu_cross_attention import TYPES, call, close, inputs

pytestmark = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")


@pytest.mark.parametrize("src,dst", TYPES)
@pytest.mark.parametrize("n,m,d", [(1, 300, 64), (8, 1030, 128), (200, 300, 64), (129, 3000, 128), (150, 200, 192)])
def test_nan_bias_of_a_key_that_takes_part_is_nan(gpu, n, m, d, src, dst):
    """exp(NaN) is NaN: the batch's rows are.  A NaN past the length, like anything there, changes nothing."""
    b, h, hk = 6, 4, 2
    q, k, v, g = inputs(gpu, b, n, m, h, hk, d, src)
    bias = torch.randn(b, m, generator=g, device=gpu)
    lens = torch.tensor([m, m, m, m // 2, m, 1], dtype=torch.int32, device=gpu)
    bias[1, 3] = NAN
    bias[2] = NAN
    bias[3, m // 2:] = NAN
    bias[4] = -INF
    bias[4, m - 1] = NAN  # the only key, in the last tile
    bias[5, 1:] = NAN
    out = torch.zeros(q.shape, dtype=dst, device=gpu)
    prm = htpg.attention_params(out, q, k, v, 0.125)
    assert htpg.cross_attention(prm, out, q, k, v, lens, bias) == 0
    assert htpg.check_device() == 0
    assert bool(out[[1, 2, 4]].isnan().all())
    ok = [0, 3, 5]
    close(out[ok], q[ok], k[ok], v[ok], 0.125, lens[ok], torch.nan_to_num(bias[ok], nan=-INF))


@pytest.mark.parametrize("src,dst", TYPES)
@pytest.mark.parametrize("n,m", [(1, 640), (16, 640), (200, 640), (130, 4096)])
@pytest.mark.parametrize("far", [1e4, 1e6, 1.3e7, 2e7, 3e7, 5e7, 1e8, 1e9, 1e30])
@pytest.mark.parametrize("sign", [-1, 1])
def test_far_biases_keep_weights_in_range(gpu, n, m, src, dst, far, sign):
    """Every key's bias is far from zero, and rises along the keys by what its FP32 value can still show (at least 4)."""
    q, k, v, g = inputs(gpu, 1, n, m, 2, 2, 64, src)
    step = max(4.0, far * 2.0**-23)
    bias = (sign * far + step * torch.floor(torch.arange(m, device=gpu) / 64 * 2) / 2)[None].float()
    out, scale = call(q, k, v, dst, bias=bias)
    assert bool(out.isfinite().all())
    low, high = (getattr(v.double(), f)(1, keepdim=True) for f in ("amin", "amax"))  # an average of values
    slack = 2.0**-7 * v.abs().max().double()
    assert bool((out >= low - slack).all()) and bool((out <= high + slack).all())
    # keys in order of their bias: what is 60 below the last keys' has no weight
    seen = bias[0] >= bias[0, -1] - 60 - far * 2.0**-20
    close(out, q, k[:, seen], v[:, seen], scale, None, bias[:, seen])
