"""The operators together as a user runs them: the example's block against the
same block in FP64."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))

# An activation row is rounded to 255 levels between its extremes: of k normal
# values (k <= 1536: extremes within 4 deviations) that is a step of at most
# 4 / 127 and an error of 4 / 127 / sqrt(12) = 0.91 % of the row's norm, and so
# of the product's.  Independent errors of the values and the second projection
# add to 1.3 %; those of q and k (0.91 % each, on scores of deviation about 1)
# change a weight by 1.3 % and the average of independent values by as much: 1.8 %.
TOLERANCE = 0.02


@pytest.mark.gpu
@pytest.mark.parametrize("batch,tokens,text,heads,kv_heads,dim", [
    (3, 100, 77, 8, 8, 64),
    (2, 257, 130, 12, 4, 128),
    (5, 1, 33, 8, 2, 64),     # one token each
])
def test_block_matches_fp64(batch, tokens, text, heads, kv_heads, dim):
    import cross_block
    block = cross_block.CrossBlock(batch, tokens, text, heads, kv_heads, dim)
    args = cross_block.inputs(block)
    ref = block.plain(*args)
    out = block.run(*args).clone()
    assert float((out - ref).norm() / ref.norm()) < TOLERANCE
    # a request without text: its attention is zero, and so is its update
    args[2][0] = 0
    out = block.run(*args)
    assert torch.equal(out[:tokens], torch.zeros_like(out[:tokens]))
