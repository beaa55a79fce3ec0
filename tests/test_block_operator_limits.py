"""More refusals of the transformer-block operators, made on the host before the
device is touched (like those of test_block_operators.py)."""
import ctypes

import pytest

import htpg
from test_block_operators import A16, LORA, _attn


def lora(lib, **change):
    p = htpg.LoraParams(**{**LORA, **{k: v for k, v in change.items() if k in LORA}})
    a = dict.fromkeys(("out", "base", "x", "ids", "a", "b", "ranks", "scales"), A16)
    a.update({k: v for k, v in change.items() if k in ("out", "base")})
    return lib.htpg_lora_run(ctypes.byref(p), *a.values(), None)


def test_lora_base_in_place_has_the_output_rows(lib):
    """out[i] at i * ldo and base[i] at i * ldb of one buffer: rows would be overwritten before they are read."""
    assert lora(lib, ldb=96, ldo=104) == htpg.EARGS
    assert lora(lib, ldb=104, ldo=96) == htpg.EARGS
    assert lora(lib, ldb=0, ldo=104) == htpg.EARGS      # dense base


BIG = 2**31 - 1


@pytest.mark.parametrize("name", ["m", "k", "n"])
def test_lora_sizes_whose_index_arithmetic_would_wrap(lib, name):
    """Sizes are rounded up to whole tiles in 32 bits."""
    dense = dict(ldx=0, ldb=0, ldo=0)
    for size in ((BIG, 2**30 + 1) if name == "m" else (BIG - 7, 2**30 + 8)):
        assert lora(lib, **dense, **{name: size}) == htpg.ECAPACITY


@pytest.mark.parametrize("name", ["q_len", "kv_len"])
def test_attention_lengths_whose_index_arithmetic_would_wrap(lib, name):
    for size in (BIG, 2**30 + 1):
        p = _attn(**{name: size})
        args = dict.fromkeys(("out", "q", "k", "v"), A16)
        assert lib.htpg_cross_attention(ctypes.byref(p), *args.values(), None, None, None) == htpg.ECAPACITY
