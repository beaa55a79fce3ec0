"""Cases for the operators of a text-conditioned transformer block: the
per-head norm and rotation of the projected queries, keys and values
(qkv_rope), attention over an encoder's states (cross_attention), and low-rank
adapters of many requests beside a shared projection (lora_run).

`run` computes a case in plain torch operations, or, with `own` set, through
the library's entry points.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6
INF = float("inf")


def listed():
    return [
        # qkv_rope: one token of one request in an LLM decode step, far into a
        # long context; plain rotation, the packed projection's row in FP32
        dict(name="rope 1 token", op="rope", batch=1, seq=1, heads=32, kv_heads=8, dim=128, rot=128, half=True,
             norm=False, positions=True, rows=32768, src="f32", dst="f16"),
        # a ragged prompt batch: grouped heads, half of each head rotated
        dict(name="rope 3x1111 partial", op="rope", batch=3, seq=1111, heads=20, kv_heads=4, dim=80, rot=40,
             half=False, norm=True, positions=True, rows=8192, src="bf16", dst="bf16"),
        # one image's tokens (4096 of hidden 1536): norm + rotation of the packed QKV rows
        dict(name="rope 4096x24x64", op="rope", batch=1, seq=4096, heads=24, kv_heads=24, dim=64, rot=64, half=False,
             norm=True, positions=False, rows=4096, src="f32", dst="f16"),
        # four images of 4096 tokens, 128-wide heads
        dict(name="rope 16384x12x128", op="rope", batch=4, seq=4096, heads=12, kv_heads=12, dim=128, rot=128,
             half=True, norm=True, positions=False, rows=4096, src="f32", dst="f16"),
        # cross_attention: one new token of each of 16 requests over its own
        # encoder states (ragged lengths), grouped heads
        dict(name="attn 16x1 over 1500", op="attn", batch=16, q=1, kv=1500, heads=32, kv_heads=8, dim=128,
             lens=True, bias=False, src="f16", dst="f32"),
        # two images' tokens over a text prompt of up to 77 tokens
        dict(name="attn 2x4096 over 77", op="attn", batch=2, q=4096, kv=77, heads=24, kv_heads=24, dim=64, lens=True,
             bias=False, src="f16", dst="f32"),
        # odd sizes, narrow heads, weighted and masked prompt tokens
        dict(name="attn 3x1001 over 333", op="attn", batch=3, q=1001, kv=333, heads=8, kv_heads=8, dim=40, lens=False,
             bias=True, src="f16", dst="f16"),
        # four images' worth of tokens in one sequence over a long prompt
        dict(name="attn 16384 over 512", op="attn", batch=1, q=16384, kv=512, heads=12, kv_heads=12, dim=128,
             lens=False, bias=False, src="bf16", dst="bf16"),
        # four images over another image's 4096 tokens
        dict(name="attn 4x4096 over 4096", op="attn", batch=4, q=4096, kv=4096, heads=12, kv_heads=12, dim=128,
             lens=False, bias=False, src="f16", dst="f16"),
        # lora_run: four single-token requests, each with its own adapter, at
        # the LLM up projection
        dict(name="lora 4x4096x14336", op="lora", m=4, k=4096, n=14336, adapters=4, rank=16, ragged=False, mixed=True,
             src="f16"),
        # a batch of prompts in any order, adapters of different ranks, some rows without one
        dict(name="lora 1000x1536x1536", op="lora", m=1000, k=1536, n=1536, adapters=6, rank=32, ragged=True,
             mixed=True, src="f16"),
        # four images, each with its own adapter, at the MLP's first linear
        dict(name="lora 16384x1536x6144", op="lora", m=16384, k=1536, n=6144, adapters=4, rank=64, ragged=False,
             mixed=False, src="f16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "attn", "lora"])
    while True:
        if op == "rope":
            dim = rng.choice([40, 64, 72, 80, 96, 128, 160])
            kv_heads = rng.choice([1, 2, 4, 8, 12])
            c = dict(op=op, batch=rng.choice([1, 1, 2, 3, 4, 16]), seq=_log(rng, 1, 16384),
                     heads=kv_heads * rng.choice([1, 2, 4]), kv_heads=kv_heads, dim=dim,
                     rot=rng.choice([dim, dim, dim // 2]), half=rng.random() < 0.5, norm=rng.random() < 0.6,
                     positions=rng.random() < 0.5, rows=16384, **dict(zip(("src", "dst"), rng.choice(
                         [("f32", "f16"), ("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "bf16")]))))
            if c["batch"] * c["seq"] * (c["heads"] + 2 * kv_heads) * dim <= 16384 * 36 * 128:
                return c
        elif op == "attn":
            kv_heads = rng.choice([1, 2, 4, 8, 12, 24])
            c = dict(op=op, batch=rng.choice([1, 2, 3, 4, 16]), q=1 if rng.random() < 0.25 else _log(rng, 1, 16384),
                     kv=_log(rng, 1, 8192), heads=kv_heads * rng.choice([1, 1, 2, 4]), kv_heads=kv_heads,
                     dim=rng.choice([40, 64, 72, 80, 96, 128, 160]), lens=rng.random() < 0.4, bias=rng.random() < 0.3,
                     **dict(zip(("src", "dst"), rng.choice([("f16", "f32"), ("f16", "f16"), ("bf16", "bf16")]))))
            if c["batch"] * c["heads"] * c["q"] * c["kv"] <= 4 * 12 * 4096 * 4096 and \
                    c["batch"] * c["heads"] * c["q"] * c["kv"] * c["dim"] <= 4 * 12 * 4096 * 4096 * 128 and \
                    c["batch"] * max(c["q"], c["kv"]) * c["heads"] * c["dim"] <= 1 << 27:
                return c
        else:
            k, n = rng.choice([(1536, 1536), (1536, 4608), (1536, 6144), (6144, 1536), (1152, 4608), (4096, 14336),
                               (14336, 4096), (32 * rng.randint(4, 90), 32 * rng.randint(4, 90))])
            c = dict(op=op, m=_log(rng, 1, 16384), k=k, n=n, adapters=rng.choice([1, 2, 4, 7, 16]),
                     rank=rng.choice([8, 16, 32, 64, 128]), ragged=rng.random() < 0.4, mixed=rng.random() < 0.5,
                     src=rng.choice(["f16", "bf16"]))
            if c["m"] * (k + n) <= 16384 * 7680 and c["m"] * c["adapters"] * c["rank"] * (k + n) <= 16384 * 256 * 7680:
                return c


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def _outliers(x, g):
    """Activations as projections give them: half a per cent of entries 20 times larger."""
    return torch.where(torch.rand(x.shape, generator=g, device="cuda") < 0.005, x * 20, x)


def _prepare_rope(c, g):
    b, s, h, hk, d = c["batch"], c["seq"], c["heads"], c["kv_heads"], c["dim"]
    packed = _outliers(_randn(g, b, s, (h + 2 * hk) * d), g).to(DTYPES[c["src"]])
    st = {"q": packed[..., :h * d].view(b, s, h, d), "k": packed[..., h * d:(h + hk) * d].view(b, s, hk, d),
          "v": packed[..., (h + hk) * d:].view(b, s, hk, d)}
    # cosines and sines of positions x frequencies, stretched by 4 for a long context
    freq = 10000.0 ** (-torch.arange(0, c["rot"], 2, dtype=torch.float64, device="cuda") / c["rot"])
    angle = torch.arange(c["rows"], dtype=torch.float64, device="cuda")[:, None] / 4 * freq
    st["table"] = torch.stack([angle.cos(), angle.sin()], -1).float().contiguous()
    st["pos"] = torch.randint(0, c["rows"], (b, s), generator=g, device="cuda",
                              dtype=torch.int32) if c["positions"] else None
    st["wq"] = 1 + 0.2 * _randn(g, d) if c["norm"] else None
    st["wk"] = 1 + 0.2 * _randn(g, d) if c["norm"] else None
    if own:  # what a program keeps: output buffers and the call's parameters
        out = DTYPES[c["dst"]]
        st["out"] = [torch.empty(b, s, n, d, dtype=out, device="cuda") for n in (h, hk, hk)]
        st["prm"] = _htpg().rope_params(st["q"], st["k"], st["v"], *st["out"], rot_dim=c["rot"],
                                        layout=1 if c["half"] else 0, table_rows=c["rows"], eps=EPS)
    return st


def _prepare_attn(c, g):
    b, q, kv, h, hk, d, t = c["batch"], c["q"], c["kv"], c["heads"], c["kv_heads"], c["dim"], DTYPES[c["src"]]
    # normed and rotated queries and keys; each head's norm weight sets how sharp it is
    sharp = 0.5 + 2.5 * torch.rand(h, 1, generator=g, device="cuda")
    st = {"q": (_randn(g, b, q, h, d) * sharp).to(t), "k": _randn(g, b, kv, hk, d, dtype=t),
          "v": _randn(g, b, kv, hk, d, dtype=t), "lens": None, "bias": None, "scale": 1 / math.sqrt(d)}
    if c["lens"]:  # between half full and full, as prompts padded to the longest
        st["lens"] = torch.randint((kv + 1) // 2, kv + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
    if c["bias"]:  # log weights of the prompt's tokens; one in eight takes no part
        u = torch.rand(b, kv, generator=g, device="cuda")
        st["bias"] = torch.where(u < 0.125, torch.full_like(u, -INF), torch.where(u > 0.8, _randn(g, b, kv), 0 * u))
    if own:
        st["out"] = torch.empty(b, q, h, d, dtype=DTYPES[c["dst"]], device="cuda")
        st["prm"] = _htpg().attention_params(st["out"], st["q"], st["k"], st["v"], scale=st["scale"])
    return st


def _prepare_lora(c, g):
    m, k, n, ad, r, t = c["m"], c["k"], c["n"], c["adapters"], c["rank"], DTYPES[c["src"]]
    st = {"x": _outliers(_randn(g, m, k), g), "base": _randn(g, m, n),
          "a": (_randn(g, ad, r, k) / math.sqrt(k)).to(t), "b": (0.3 * _randn(g, ad, n, r)).to(t),
          "scales": 0.5 + torch.rand(ad, generator=g, device="cuda")}
    if c["ragged"]:
        st["ranks"] = torch.randint(1, r + 1, (ad,), generator=g, device="cuda", dtype=torch.int32)
    else:
        st["ranks"] = torch.full((ad,), r, dtype=torch.int32, device="cuda")
    if c["mixed"]:  # any order; with several adapters, -1: a request without one
        st["ids"] = torch.randint(-1 if ad > 4 else 0, ad, (m,), generator=g, device="cuda", dtype=torch.int32)
    else:  # whole requests one after another
        st["ids"] = (torch.arange(m, device="cuda") * ad // m).to(torch.int32)
    if own:
        st["out"] = torch.empty(m, n, device="cuda")
        st["prm"] = _htpg().lora_params(st["out"], st["base"], st["x"], st["a"], st["b"])
    return st


def _htpg():
    at = os.path.join(os.getcwd(), "htp-ops-lib-sd.cpp_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import htpg
    return htpg


def prepare(case, seed):
    state = {"rope": _prepare_rope, "attn": _prepare_attn, "lora": _prepare_lora}[case["op"]](case, _gen(seed))
    state["case"] = case
    if own:
        state["htpg"] = _htpg()
    return state


# ------------------------------------------------------------------ one pass
def _rope_part(x, w, st, rotated, out):
    c = st["case"]
    x = x.float()
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
    if rotated:
        r = c["rot"]
        cs = st["table"][:c["seq"]] if st["pos"] is None else st["table"][st["pos"].long()]
        cos, sin = cs[..., None, :, 0], cs[..., None, :, 1]
        y = torch.empty_like(x)
        if c["half"]:
            first, second = slice(0, r // 2), slice(r // 2, r)
        else:
            first, second = slice(0, r, 2), slice(1, r, 2)
        y[..., first] = x[..., first] * cos - x[..., second] * sin
        y[..., second] = x[..., first] * sin + x[..., second] * cos
        y[..., r:] = x[..., r:]
        x = y
    return x.to(out)


def _rope(st):
    out = DTYPES[st["case"]["dst"]]
    return [_rope_part(st["q"], st["wq"], st, True, out), _rope_part(st["k"], st["wk"], st, True, out),
            _rope_part(st["v"], None, st, False, out)]


def _allowed(st, b, kv):
    """[b][kv]: the keys that take part."""
    ok = torch.ones(b, kv, dtype=torch.bool, device="cuda")
    if st["lens"] is not None:
        ok = ok & (torch.arange(kv, device="cuda") < st["lens"][:, None])
    if st["bias"] is not None:
        ok = ok & (st["bias"] > -INF)
    return ok


def _attn(st):
    c = st["case"]
    group = c["heads"] // c["kv_heads"]
    q = st["q"].float().transpose(1, 2)
    k = st["k"].float().transpose(1, 2).repeat_interleave(group, 1)
    v = st["v"].float().transpose(1, 2).repeat_interleave(group, 1)
    s = (q @ k.transpose(2, 3)) * st["scale"]
    if st["bias"] is not None:
        s = s + st["bias"][:, None, None, :]
    if st["lens"] is not None or st["bias"] is not None:
        ok = _allowed(st, c["batch"], c["kv"])
        s = torch.where(ok[:, None, None, :], s, -INF)
        v = torch.where(ok[:, None, :, None], v, 0)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top > -INF, top, 0))
    total = p.sum(-1, keepdim=True)
    o = torch.where(total > 0, (p @ v) / total, 0)  # no key takes part: zeros
    return o.transpose(1, 2).to(DTYPES[c["dst"]])


def _lora(st):
    c = st["case"]
    ad, r = c["adapters"], c["rank"]
    live = torch.arange(r, device="cuda") < st["ranks"][:, None]  # [ad][r]
    a = torch.where(live[:, :, None], st["a"].float(), 0).reshape(ad * r, c["k"])
    b = torch.where(live[:, None, :], st["b"].float(), 0).transpose(1, 2).reshape(ad * r, c["n"])
    mine = st["ids"][:, None] == torch.arange(ad, device="cuda").repeat_interleave(r)
    t = torch.where(mine, (st["x"] @ a.t()) * st["scales"].repeat_interleave(r), 0)
    return st["base"] + t @ b


def _own_rope(st):
    h = st["htpg"]
    h.check(h.qkv_rope(st["prm"], *st["out"], st["q"], st["k"], st["v"], st["wq"], st["wk"], st["table"], st["pos"]),
            "htpg_qkv_rope")
    return st["out"]


def _own_attn(st):
    h = st["htpg"]
    h.check(h.cross_attention(st["prm"], st["out"], st["q"], st["k"], st["v"], st["lens"], st["bias"]),
            "htpg_cross_attention")
    return st["out"]


def _own_lora(st):
    h = st["htpg"]
    h.check(h.lora_run(st["prm"], st["out"], st["base"], st["x"], st["ids"], st["a"], st["b"], st["ranks"],
                       st["scales"]), "htpg_lora_run")
    return st["out"]


def run(state):
    if own:
        return {"rope": _own_rope, "attn": _own_attn, "lora": _own_lora}[state["case"]["op"]](state)
    return {"rope": _rope, "attn": _attn, "lora": _lora}[state["case"]["op"]](state)


# ------------------------------------------------------------------ what a pass needs
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def work(case):
    c = case
    if c["op"] == "rope":
        elements = c["batch"] * c["seq"] * (c["heads"] + 2 * c["kv_heads"]) * c["dim"]
        used = min(c["rows"], c["batch"] * c["seq"]) if c["positions"] else c["seq"]
        return {"bytes": elements * (SIZE[c["src"]] + SIZE[c["dst"]]) + used * c["rot"] * 4, "flops": elements * 6}
    if c["op"] == "attn":
        rows = c["batch"] * c["q"] * c["heads"] * c["dim"]
        keys = c["kv"] * (0.75 if c["lens"] else 1)
        moved = rows * (SIZE[c["src"]] + SIZE[c["dst"]]) + 2 * c["batch"] * keys * c["kv_heads"] * c["dim"] * 2
        return {"bytes": moved + (4 * c["batch"] * c["kv"] if c["bias"] else 0), "flops": 4 * rows * keys}
    rank = (c["rank"] + 1) / 2 if c["ragged"] else c["rank"]
    used = min(c["adapters"], c["m"])
    return {"bytes": 4 * c["m"] * (c["k"] + 2 * c["n"] + 1) + 2 * used * rank * (c["k"] + c["n"]),
            "flops": 2 * c["m"] * rank * (c["k"] + c["n"])}


# ------------------------------------------------------------------ 64 bits
def _exact_rope(c, st):
    d, r = c["dim"], c["rot"]
    outs = []
    for name, weight in (("q", "wq"), ("k", "wk"), ("v", None)):
        x = st[name].double()
        if weight and st[weight] is not None:
            x = x / (x.pow(2).sum(-1, keepdim=True) / d + EPS).sqrt() * st[weight].double()
        if name != "v":
            pos = torch.arange(c["seq"], device="cuda").expand(c["batch"], -1) if st["pos"] is None else st["pos"]
            cs = torch.view_as_complex(st["table"].double())[pos.long()][:, :, None]
            head = x[..., :r]
            if c["half"]:
                z = torch.complex(head[..., :r // 2].contiguous(), head[..., r // 2:].contiguous()) * cs
                head = torch.cat([z.real, z.imag], -1)
            else:
                head = torch.view_as_real(torch.view_as_complex(head.unflatten(-1, (-1, 2)).contiguous()) * cs).flatten(-2)
            x = torch.cat([head, x[..., r:]], -1)
        outs.append(x)
    return outs


def _exact_attn(c, st):
    group = c["heads"] // c["kv_heads"]
    out = torch.zeros(c["batch"], c["q"], c["heads"], c["dim"], dtype=torch.float64, device="cuda")
    for i in range(c["batch"]):
        n = c["kv"] if st["lens"] is None else int(st["lens"][i])
        keep = torch.arange(n, device="cuda")
        if st["bias"] is not None:
            keep = keep[st["bias"][i, :n] != -INF]
        if not len(keep):
            continue
        for h in range(c["heads"]):
            k, v = st["k"][i, keep, h // group].double(), st["v"][i, keep, h // group].double()
            s = st["q"][i, :, h].double() @ k.T * st["scale"]
            if st["bias"] is not None:
                s += st["bias"][i, keep].double()
            out[i, :, h] = torch.softmax(s, -1) @ v
    return out


def _exact_lora(c, st):
    out = st["base"].double()
    for j in range(c["adapters"]):
        rows, r = torch.nonzero(st["ids"] == j)[:, 0], int(st["ranks"][j])
        t = st["x"][rows].double() @ st["a"][j, :r].double().T
        out[rows] += float(st["scales"][j]) * (t @ st["b"][j, :, :r].double().T)
    return out


def exact(case, seed):
    state = prepare(case, seed)
    return {"rope": _exact_rope, "attn": _exact_attn, "lora": _exact_lora}[case["op"]](case, state)
