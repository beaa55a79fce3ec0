"""What the Python entry points of the transformer-block operators refuse
because the library would read or write past a tensor (htpg.py).  Every refusal
comes before the library is called, so they run without a GPU."""
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


# ------------------------------------------------------------------ arrays of one call
# Each entry: the array's name, its type and how many elements the call reads.
I32 = torch.int32


class Reached(Exception):
    """The library was called: nothing was refused."""


@pytest.fixture
def reached(monkeypatch):
    """A library whose functions raise Reached, and host tensors that pass for device ones."""
    def function(*_):
        raise Reached

    class Lib:
        def __getattr__(self, name):
            return function
    monkeypatch.setattr(htpg, "lib", Lib)
    monkeypatch.setattr(htpg, "stream_ptr", lambda stream: 0)
    monkeypatch.setattr(htpg, "_on_device", lambda t: True)


def _rope(**change):
    q, k, t = torch.zeros(2, 3, 4, 64), torch.zeros(2, 3, 2, 64), torch.zeros
    prm = htpg.rope_params(q, k, k, q, k, k, 32, htpg.ROPE_HALF, 16)
    arrays = dict(q_weight=t(64), k_weight=t(64), table=t(16, 16, 2), positions=t(2, 3, dtype=I32))
    return htpg.qkv_rope(prm, q, k, k, q, k, k, **{**arrays, **change})


def _attn(**change):
    q, k, t = torch.zeros(2, 3, 4, 64, dtype=F16), torch.zeros(2, 7, 2, 64, dtype=F16), torch.zeros
    prm = htpg.attention_params(q, q, k, k, 0.125, bias_stride=change.pop("bias_stride", None))
    return htpg.cross_attention(prm, q, q, k, k, **{**dict(kv_lens=t(2, dtype=I32), key_bias=t(2, 7)), **change})


def _lora(**change):
    t = lora(adapters=3)
    z = torch.zeros
    arrays = dict(row_adapter=z(5, dtype=I32), ranks=z(3, dtype=I32), scales=z(3))
    a = {**arrays, **change}
    return htpg.lora_run(htpg.lora_params(**t), t["out"], t["base"], t["x"], a["row_adapter"], t["a"], t["b"], a["ranks"],
                         a["scales"])


ARRAYS = [(_rope, "q_weight", F32, 64), (_rope, "k_weight", F32, 64), (_rope, "table", F32, 16 * 32),
          (_rope, "positions", I32, 6), (_attn, "kv_lens", I32, 2), (_attn, "key_bias", F32, 14),
          (_lora, "row_adapter", I32, 5), (_lora, "ranks", I32, 3), (_lora, "scales", F32, 3)]


@pytest.mark.parametrize("call,name,dtype,n", ARRAYS)
def test_arrays_of_a_call(reached, call, name, dtype, n):
    z = torch.zeros
    with pytest.raises(Reached):  # as it should be, and longer
        call()
    with pytest.raises(Reached):
        call(**{name: z(n + 3, dtype=dtype) if name != "key_bias" else z(3, 7)})
    for other in (torch.int64, F16, torch.float64, I32 if dtype == F32 else F32):
        with pytest.raises(ValueError, match=name):
            call(**{name: z(n, dtype=other)})
    with pytest.raises(ValueError, match=name):  # one too few
        call(**{name: z(n - 1, dtype=dtype)})
    with pytest.raises(ValueError, match=name):  # not dense
        call(**{name: z(2 * n, dtype=dtype)[::2]})


@pytest.mark.parametrize("call,name", [(c, n) for c, n, *_ in ARRAYS if c is not _lora])
def test_arrays_that_may_be_left_out(reached, call, name):
    with pytest.raises(Reached):
        call(**{name: None})


def test_positions_of_one_sequence_for_a_batch(reached):
    with pytest.raises(ValueError, match="positions"):
        _rope(positions=torch.zeros(1, 3, dtype=I32))
    with pytest.raises(ValueError, match="positions"):  # [1][seq] expanded has no memory for the second
        _rope(positions=torch.zeros(1, 3, dtype=I32).expand(2, -1))


def test_key_bias_rows(reached):
    """Rows at bias_stride: shared, padded, and too short for the batch or the keys."""
    big = torch.zeros(2, 16)
    for good, stride in ((torch.zeros(1, 7), 0), (torch.zeros(7), 0), (big[:, :7], 16), (torch.zeros(2, 7), None),
                         (torch.zeros(1, 7).expand(2, -1), 0)):
        with pytest.raises(Reached):
            _attn(key_bias=good, bias_stride=stride)
    for bad, stride in ((torch.zeros(1, 7), None), (torch.zeros(1, 7).expand(2, -1), None), (torch.zeros(2, 7), 16),
                        (torch.zeros(1, 6), 0), (torch.zeros(2, 7), -7)):
        with pytest.raises(ValueError, match="key_bias"):
            _attn(key_bias=bad, bias_stride=stride)


def test_rope_table_buffer(reached):
    with pytest.raises(Reached):
        htpg.rope_table(torch.zeros(16, 32, 2), 64)
    for bad in (torch.zeros(16, 31, 2), torch.zeros(16, 32, 2, dtype=torch.float64), torch.zeros(16, 32, 4)[..., :2]):
        with pytest.raises(ValueError, match="table"):
            htpg.rope_table(bad, 64)


@pytest.mark.parametrize("call", [_rope, _attn, _lora])
def test_host_tensors_are_refused(call):
    with pytest.raises(ValueError, match="host"):
        call()
