"""The block operators as the first CUDA work of a host thread."""
import threading

import pytest
import torch

import htpg

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,m", [(200, 77), (200, 3000), (1, 6000), (5, 0)])
@pytest.mark.parametrize("dst", [torch.float16, torch.float32])
def test_attention_first_in_a_thread(gpu, n, m, dst):
    g = torch.Generator(device=gpu).manual_seed(m)
    q, k = torch.randn(1, n, 4, 64, generator=g, device=gpu).half(), torch.randn(1, m, 2, 64, generator=g, device=gpu).half()
    want, out = (torch.full(q.shape, -1.0, dtype=dst, device=gpu) for _ in range(2))
    prm = htpg.attention_params(out, q, k, k, 0.125)
    stream = torch.cuda.Stream().cuda_stream
    htpg.check(htpg.cross_attention(prm, want, q, k, k))
    torch.cuda.synchronize()
    codes = []
    t = threading.Thread(target=lambda: codes.append(htpg.cross_attention(prm, out, q, k, k, stream=stream)))
    t.start()
    t.join()
    assert codes == [0]
    torch.cuda.synchronize()
    assert torch.equal(out, want)
