"""What the Python entry points of the transformer-block operators refuse
because the library would read or write past a tensor (htpg.py).  Every refusal
comes before the library is called, so these run without a GPU."""
import pytest
import torch

import htpg

F32, F16 = torch.float32, torch.float16


def lora(m=5, k=64, n=96, adapters=2, rank=8):
    """out, base, x, a, b that fit together."""
    z = torch.zeros
    return dict(out=z(m, n), base=z(m, n), x=z(m, k), a=z(adapters, rank, k, dtype=F16), b=z(adapters, n, rank, dtype=F16))


@pytest.mark.parametrize("name", ["out", "base", "x"])
@pytest.mark.parametrize("dtype", [F16, torch.bfloat16, torch.float64, torch.int32])
def test_lora_activations_are_fp32(name, dtype):
    t = lora()
    assert htpg.lora_params(**t).m == 5
    t[name] = t[name].to(dtype)
    with pytest.raises(ValueError, match="FP32"):
        htpg.lora_params(**t)


@pytest.mark.parametrize("name", ["out", "base", "x"])
def test_lora_rows_that_are_one_row_are_refused(name):
    """A row stride of 0 means dense to the library: m rows would be read where there is one."""
    t = lora()
    t[name] = t[name][:1].expand(5, -1)
    with pytest.raises(ValueError, match="own"):
        htpg.lora_params(**t)
    t = lora()
    t[name] = t[name].as_strided(t[name].shape, (8, 1))  # rows that overlap
    with pytest.raises(ValueError, match="own"):
        htpg.lora_params(**t)
    one = lora(m=1)  # of a single row the stride is not looked at
    one[name] = one[name].as_strided(one[name].shape, (0, 1))
    assert htpg.lora_params(**one).m == 1
