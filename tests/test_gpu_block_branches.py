"""Branches of the block operators that take particular sizes to reach, and the
example's block operator by operator."""
import os
import sys

import pytest
import torch

import htpg
from test_gpu_cross_attention import TYPES, call, close, inputs
from test_gpu_lora import close as lora_close
from test_gpu_rope import close as rope_close
from test_gpu_rope import rotated

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("src,dst", TYPES)
@pytest.mark.parametrize("n,m", [(1, 50), (20, 50), (130, 90)])
def test_more_batches_than_lengths_are_kept(gpu, n, m, src, dst):
    """The tiles keep 256 batches' lengths in shared memory and read the others'."""
    b = 300
    q, k, v, g = inputs(gpu, b, n, m, 1, 1, 40, src)
    lens = torch.randint(-1, m + 2, (b,), generator=g, device=gpu, dtype=torch.int32)
    lens[255:258] = torch.tensor([m, 0, 1], dtype=torch.int32)
    out, scale = call(q, k, v, dst, lens=lens)
    close(out, q, k, v, scale, lens)
    assert bool((out[256] == 0).all())


@pytest.mark.parametrize("src,dst", TYPES)
@pytest.mark.parametrize("d", [64, 128, 160])
@pytest.mark.parametrize("n,m", [(200, 4096), (1, 4096), (16, 3000)])
def test_key_ranges_beyond_a_short_length(gpu, n, m, d, src, dst):
    """Units are cut into ranges by kv_len: with short lengths some ranges hold no key, for some requests none does."""
    b, h, hk = 6, 4, 2
    q, k, v, g = inputs(gpu, b, n, m, h, hk, d, src)
    lens = torch.tensor([m, 1, 0, 65, 700, m - 1], dtype=torch.int32, device=gpu)
    out, scale = call(q, k, v, dst, lens=lens)
    close(out, q, k, v, scale, lens)
    assert bool((out[2] == 0).all())
    bias = torch.randn(b, m, generator=g, device=gpu)
    bias[0, :1000] = -float("inf")  # whole ranges masked
    bias[5, 70:] = -float("inf")
    out, _ = call(q, k, v, dst, lens=lens, bias=bias)
    close(out, q, k, v, scale, lens, bias)


@pytest.mark.parametrize("batch,tokens,text,heads,kv_heads,dim", [
    (3, 100, 77, 8, 8, 64), (2, 257, 130, 12, 4, 128), (5, 1, 33, 8, 2, 64)])
def test_example_operator_by_operator(gpu, batch, tokens, text, heads, kv_heads, dim):
    """What each operator of the example's block made of what it was given."""
    import cross_block
    block = cross_block.CrossBlock(batch, tokens, text, heads, kv_heads, dim)
    x, cond, lens, ids = cross_block.inputs(block)
    out = block.run(x, cond, lens, ids)
    adapters = block.ranks, block.scales
    base = torch.empty_like(block.q)
    htpg.check(htpg.w8a8_run(block.wq, base, x, channels=heads * dim))
    lora_close(block.q, base, x, ids, block.aq, block.bq, *adapters)
    for x32, x16, weight, n, hh in ((block.q, block.q16, block.q_weight, tokens, heads),
                                    (block.k, block.k16, block.k_weight, text, kv_heads)):
        at = torch.arange(n, device=gpu).expand(batch, n)
        rope_close(x16, *rotated(x32.view(batch, n, hh, dim), block.table, at, dim, True, weight))
    assert torch.equal(block.v16, block.v.view_as(block.v16).half())
    close(block.o, block.q16, block.k16, block.v16, dim**-0.5, lens)
    o = block.o.view(batch * tokens, heads * dim)
    htpg.check(htpg.w8a8_run(block.wo, base, o, channels=heads * dim))
    lora_close(out, base, o, ids, block.ao, block.bo, *adapters)


def test_captured_example_follows_its_inputs(gpu):
    """A captured block, replayed on inputs that changed, gives what a call gives."""
    import cross_block
    block = cross_block.CrossBlock(2, 64, 33, 8, 2, 64)
    args = cross_block.inputs(block)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):  # the linears' scratch belongs to the stream
        block.run(*args)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        block.run(*args)
    args[0].mul_(0.5)
    torch.cuda.synchronize()
    want = block.run(*args).clone()
    block.out.zero_()
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(block.out, want)
