"""More refusals of the transformer-block operators, made on the host before the
device is touched (like those of test_block_operators.py)."""
import ctypes

import pytest

import htpg
from test_block_operators import A16, LORA


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
