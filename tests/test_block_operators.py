"""The transformer-block operators' argument checks (htpg_rope_table,
htpg_qkv_rope, htpg_cross_attention, htpg_lora_run).  Every refusal is made on
the host before the device is touched, so these run without a GPU; addresses
stand for device memory that is never read."""
import ctypes

import pytest
import torch

import htpg

A16 = 1 << 20  # an aligned address
NAN, INF = float("nan"), float("inf")


def test_structs_match_the_header():
    assert ctypes.sizeof(htpg.RopeScaling) == 40
    assert ctypes.sizeof(htpg.RopeParams) == 48 + 18 * 8
    assert ctypes.sizeof(htpg.AttentionParams) == 40 + 13 * 8
    assert ctypes.sizeof(htpg.LoraParams) == 24 + 3 * 8


TABLE = dict(scaling=htpg.ROPE_YARN, original_rows=4096, base=1e4, factor=4.0, beta_fast=32.0, beta_slow=1.0)


@pytest.mark.parametrize("change,rows,rot,table,code", [
    (dict(scaling=4), 8, 64, A16, htpg.EARGS), (dict(scaling=-1), 8, 64, A16, htpg.EARGS),
    (dict(base=1.0), 8, 64, A16, htpg.EARGS), (dict(base=NAN), 8, 64, A16, htpg.EARGS),
    (dict(base=INF), 8, 64, A16, htpg.EARGS), (dict(factor=0.5), 8, 64, A16, htpg.EARGS),
    (dict(factor=NAN), 8, 64, A16, htpg.EARGS), (dict(original_rows=0), 8, 64, A16, htpg.EARGS),
    (dict(beta_fast=0.0), 8, 64, A16, htpg.EARGS), (dict(beta_slow=64.0), 8, 64, A16, htpg.EARGS),
    (dict(scaling=htpg.ROPE_NTK), 8, 2, A16, htpg.EARGS), ({}, -1, 64, A16, htpg.EARGS),
    ({}, 8, 63, A16, htpg.EARGS), ({}, 8, 0, A16, htpg.EARGS), ({}, 8, 64, None, htpg.EARGS),
    ({}, 8, 64, A16 + 4, htpg.ECONTROL), ({}, 0, 64, A16, htpg.OK),
])
def test_rope_table_refusals(lib, change, rows, rot, table, code):
    s = htpg.RopeScaling(**{**TABLE, **change})
    assert lib.htpg_rope_table(table, rows, rot, ctypes.byref(s), None) == code


ROPE = dict(in_type=htpg.TYPE_F32, out_type=htpg.TYPE_F16, batch=2, seq=3, q_heads=4, kv_heads=2, head_dim=64,
            rot_dim=64, layout=1, table_rows=16, eps=1e-6, reserved=0)


@pytest.mark.parametrize("change,ptrs,code", [
    (dict(in_type=2), {}, htpg.EARGS), (dict(out_type=8), {}, htpg.EARGS), (dict(batch=-1), {}, htpg.EARGS),
    (dict(seq=-1), {}, htpg.EARGS), (dict(reserved=1), {}, htpg.EARGS), (dict(q_heads=0), {}, htpg.EARGS),
    (dict(kv_heads=0), {}, htpg.EARGS), (dict(head_dim=0), {}, htpg.EARGS), (dict(rot_dim=63), {}, htpg.EARGS),
    (dict(rot_dim=-2), {}, htpg.EARGS), (dict(layout=2), {}, htpg.EARGS), (dict(eps=-1.0), {}, htpg.EARGS),
    (dict(eps=NAN), {}, htpg.EARGS), (dict(table_rows=-1), {}, htpg.EARGS),
    (dict(head_dim=514), {}, htpg.ECAPACITY), (dict(rot_dim=66), {}, htpg.ECAPACITY),
    (dict(seq=17), {}, htpg.ECAPACITY),  # no positions: tokens past the table
    ({}, dict(q=None), htpg.EARGS), ({}, dict(k_out=None), htpg.EARGS), ({}, dict(table=None), htpg.EARGS),
    ({}, dict(q=None, q_out=None, k=None, k_out=None, v=None, v_out=None), htpg.EARGS),
    ({}, dict(q=A16 + 2), htpg.ECONTROL), ({}, dict(v_out=A16 + 1), htpg.ECONTROL),
    ({}, dict(q_weight=A16 + 2), htpg.ECONTROL), ({}, dict(table=A16 + 4), htpg.ECONTROL),
    (dict(batch=0), {}, htpg.OK), (dict(seq=0), {}, htpg.OK),
])
def test_qkv_rope_refusals(lib, change, ptrs, code):
    p = htpg.RopeParams(**{**ROPE, **change})
    a = {**dict.fromkeys(("q_out", "k_out", "v_out", "q", "k", "v", "q_weight", "k_weight", "table"), A16),
         "positions": None, **ptrs}
    assert lib.htpg_qkv_rope(ctypes.byref(p), *a.values(), None) == code
    assert lib.htpg_qkv_rope(None, *a.values(), None) == htpg.EARGS


def _attn(**change):
    p = htpg.AttentionParams(**{**dict(type=htpg.TYPE_F16, out_type=htpg.TYPE_F32, batch=2, q_len=3, kv_len=5,
                                       q_heads=4, kv_heads=2, head_dim=64, scale=0.125, reserved=0, bias_stride=5),
                                **{k: v for k, v in change.items() if not k.endswith("_stride")}})
    for name, s in (("q", (768, 256, 64)), ("k", (640, 128, 64)), ("v", (640, 128, 64)), ("out", (768, 256, 64))):
        getattr(p, name + "_stride")[:] = change.get(name + "_stride", s)
    return p


@pytest.mark.parametrize("change,ptrs,code", [
    (dict(type=htpg.TYPE_F32), {}, htpg.EARGS), (dict(out_type=htpg.TYPE_BF16), {}, htpg.EARGS),
    (dict(reserved=1), {}, htpg.EARGS), (dict(batch=-1), {}, htpg.EARGS), (dict(q_len=-1), {}, htpg.EARGS),
    (dict(kv_len=-1), {}, htpg.EARGS), (dict(q_heads=0), {}, htpg.EARGS), (dict(kv_heads=0), {}, htpg.EARGS),
    (dict(head_dim=0), {}, htpg.EARGS), (dict(scale=0.0), {}, htpg.EARGS), (dict(scale=-1.0), {}, htpg.EARGS),
    (dict(scale=NAN), {}, htpg.EARGS), (dict(scale=INF), {}, htpg.EARGS),
    (dict(kv_heads=3), {}, htpg.ECAPACITY), (dict(head_dim=60), {}, htpg.ECAPACITY),
    (dict(head_dim=200), {}, htpg.ECAPACITY),
    ({}, dict(out=None), htpg.EARGS), ({}, dict(q=None), htpg.EARGS), ({}, dict(k=None), htpg.EARGS),
    ({}, dict(v=None), htpg.EARGS),
    ({}, dict(q=A16 + 8), htpg.ECONTROL), ({}, dict(out=A16 + 4), htpg.ECONTROL), ({}, dict(lens=A16 + 2), htpg.ECONTROL),
    ({}, dict(bias=A16 + 1), htpg.ECONTROL),
    (dict(q_stride=(768, 260, 64)), {}, htpg.ECONTROL), (dict(k_stride=(640, 128, 68)), {}, htpg.ECONTROL),
    (dict(v_stride=(644, 128, 64)), {}, htpg.ECONTROL), (dict(out_stride=(768, 258, 64)), {}, htpg.ECONTROL),
    (dict(q_stride=(768, -256, 64)), {}, htpg.ECONTROL), (dict(k_stride=(-640, 128, 64)), {}, htpg.ECONTROL),
    (dict(v_stride=(640, 128, -64)), {}, htpg.ECONTROL), (dict(k_stride=(640, 0, 64)), {}, htpg.ECONTROL),
    (dict(q_stride=(1 << 38, 256, 64)), {}, htpg.ECONTROL), (dict(out_stride=(0, 256, 64)), {}, htpg.ECONTROL),
    (dict(out_stride=(768, 256, 0)), {}, htpg.ECONTROL),
    (dict(batch=0), {}, htpg.OK), (dict(q_len=0), {}, htpg.OK),
])
def test_cross_attention_refusals(lib, change, ptrs, code):
    p = _attn(**change)
    a = {**dict.fromkeys(("out", "q", "k", "v"), A16), "lens": None, "bias": None, **ptrs}
    assert lib.htpg_cross_attention(ctypes.byref(p), *a.values(), None) == code
    assert lib.htpg_cross_attention(None, *a.values(), None) == htpg.EARGS


LORA = dict(type=htpg.TYPE_F16, m=4, k=64, n=96, adapters=2, max_rank=16, ldx=64, ldb=96, ldo=96)


@pytest.mark.parametrize("change,ptrs,code", [
    (dict(type=htpg.TYPE_F32), {}, htpg.EARGS), (dict(m=-1), {}, htpg.EARGS), (dict(k=0), {}, htpg.EARGS),
    (dict(n=0), {}, htpg.EARGS), (dict(adapters=0), {}, htpg.EARGS), (dict(max_rank=0), {}, htpg.EARGS),
    (dict(ldx=-4), {}, htpg.EARGS), (dict(ldx=60), {}, htpg.EARGS), (dict(ldo=92), {}, htpg.EARGS),
    (dict(ldb=92), {}, htpg.EARGS), (dict(k=60), {}, htpg.ECAPACITY), (dict(n=100), {}, htpg.ECAPACITY),
    (dict(max_rank=12), {}, htpg.ECAPACITY), (dict(max_rank=136), {}, htpg.ECAPACITY),
    (dict(ldx=66), {}, htpg.ECONTROL), (dict(ldo=98), {}, htpg.ECONTROL), (dict(ldb=98), {}, htpg.ECONTROL),
    *[({}, {n: None}, htpg.EARGS) for n in ("out", "x", "ids", "a", "b", "ranks", "scales")],
    *[({}, {n: A16 + 8}, htpg.ECONTROL) for n in ("out", "base", "x", "a", "b")],
    *[({}, {n: A16 + 2}, htpg.ECONTROL) for n in ("ids", "ranks", "scales")],
    (dict(m=0), {}, htpg.OK),
])
def test_lora_refusals(lib, change, ptrs, code):
    p = htpg.LoraParams(**{**LORA, **change})
    a = {**dict.fromkeys(("out", "base", "x", "ids", "a", "b", "ranks", "scales"), A16), **ptrs}
    assert lib.htpg_lora_run(ctypes.byref(p), *a.values(), None) == code
    assert lib.htpg_lora_run(None, *a.values(), None) == htpg.EARGS


def test_parameter_builders_refuse_what_does_not_fit():
    t = torch.zeros
    q, k = t(2, 3, 4, 64), t(2, 3, 2, 64)
    with pytest.raises(ValueError):
        htpg.rope_params(q, k, k, q, None, k, 64, 0, 16)
    with pytest.raises(ValueError):
        htpg.rope_params(q, k, t(2, 3, 1, 64), q, k, t(2, 3, 1, 64), 64, 0, 16)
    with pytest.raises(ValueError):
        htpg.rope_params(q.double(), None, None, q.double(), None, None, 64, 0, 16)
    with pytest.raises(ValueError):
        htpg.rope_params(q.transpose(2, 3), None, None, q.transpose(2, 3), None, None, 64, 0, 16)
    with pytest.raises(ValueError):
        htpg.attention_params(q, q, k, t(2, 4, 2, 64), 1.0)
    x, a, b, o = t(5, 64), t(2, 8, 64), t(2, 96, 8), t(5, 96)
    with pytest.raises(ValueError):
        htpg.lora_params(o, None, x, a, t(2, 96, 16))
    with pytest.raises(ValueError):
        htpg.lora_params(o, None, t(64, 5).t(), a, b)
    with pytest.raises(ValueError):
        htpg.lora_params(o, None, x, a.transpose(1, 2).contiguous().transpose(1, 2), b)
    assert htpg.lora_params(o, None, x, a.half(), b.half()).max_rank == 8
