"""A text-conditioned attention block on one GPU, from the library's operators:

    q = W_q x, k = W_k c, v = W_v c        W8A8 projections (htpg_w8a8_run)
    q, out += adapters of each request     htpg_lora_run, in place
    q, k: RMS norm per head, positions     htpg_qkv_rope, FP32 -> FP16
    attention over the text's states       htpg_cross_attention, masked by length
    out = W_o attention                    W8A8

    python examples/cross_block.py         # builds, runs, compares with FP64, times it

Every request of the batch has its own text length and its own adapter (or
none).  All calls go to the current stream and allocate nothing after the first
one there, so the block can be captured in a CUDA graph (done here for the timing;
the graph takes scratch of its own for attention and adapters)."""
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "htp-ops-lib-sd.cpp_b200"))
import htpg  # noqa: E402


def quantised(n, k, gen):
    """A W8A8 weight: the library's handle and the FP64 matrix it stands for."""
    w = torch.randint(-127, 128, (n, k), generator=gen, dtype=torch.int32).to(torch.int8).numpy()
    sw = np.full(n, 1.0 / (73.3 * k ** 0.5), np.float32)  # 73.3: such codes' root mean square
    blob = torch.from_numpy(htpg.pack_w8a8_constants(w, sw)).cuda()
    return htpg.w8a8_weights(blob, k, n), torch.from_numpy(w * np.float64(sw[0])).cuda()


class CrossBlock:
    """The block's weights, adapters and buffers for `batch` requests of `tokens` queries over `text` states."""

    def __init__(self, batch, tokens, text, heads, kv_heads, dim, adapters=2, max_rank=16, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.batch, self.tokens, self.text, self.heads, self.kv_heads, self.dim = batch, tokens, text, heads, kv_heads, dim
        c, ckv = heads * dim, kv_heads * dim
        (self.wq, self.wq64), (self.wk, self.wk64), (self.wv, self.wv64), (self.wo, self.wo64) = (
            quantised(n, c, g) for n in (c, ckv, ckv, c))
        rnd = lambda *s: torch.randn(*s, generator=g).cuda()  # noqa: E731
        self.aq, self.bq, self.ao, self.bo = ((rnd(*s) / s[-1] ** 0.5).half() for s in (
            (adapters, max_rank, c), (adapters, c, max_rank), (adapters, max_rank, c), (adapters, c, max_rank)))
        self.ranks = torch.tensor([max_rank - 8 * (i % 2) for i in range(adapters)], dtype=torch.int32).cuda()
        self.scales = torch.full((adapters,), 0.5).cuda()
        self.q_weight, self.k_weight = 1 + 0.1 * rnd(dim), 1 + 0.1 * rnd(dim)
        self.table = torch.empty(max(tokens, text), dim // 2, 2, device="cuda")
        htpg.check(htpg.rope_table(self.table, dim), "rope_table")
        new = lambda dtype, *s: torch.empty(*s, dtype=dtype, device="cuda")  # noqa: E731
        f32, f16 = torch.float32, torch.float16
        self.q, self.k, self.v = new(f32, batch * tokens, c), new(f32, batch * text, ckv), new(f32, batch * text, ckv)
        self.q16, self.k16 = new(f16, batch, tokens, heads, dim), new(f16, batch, text, kv_heads, dim)
        self.v16 = new(f16, batch, text, kv_heads, dim)
        self.o = new(f32, batch, tokens, heads, dim)
        self.out = new(f32, batch * tokens, c)

    def run(self, x, cond, kv_lens, row_adapter):
        """x [batch * tokens][heads * dim], cond [batch * text][heads * dim] FP32 -> the attention's update of x."""
        b, t, s, h, hk, d = self.batch, self.tokens, self.text, self.heads, self.kv_heads, self.dim
        check = htpg.check
        check(htpg.w8a8_run(self.wq, self.q, x, channels=h * d), "w8a8_run")
        check(htpg.w8a8_run(self.wk, self.k, cond, channels=hk * d), "w8a8_run")
        check(htpg.w8a8_run(self.wv, self.v, cond, channels=hk * d), "w8a8_run")
        check(htpg.lora_run(htpg.lora_params(self.q, self.q, x, self.aq, self.bq), self.q, self.q, x, row_adapter,
                            self.aq, self.bq, self.ranks, self.scales), "lora_run")
        q, k, v = self.q.view(b, t, h, d), self.k.view(b, s, hk, d), self.v.view(b, s, hk, d)
        n = self.table.shape[0]
        check(htpg.qkv_rope(htpg.rope_params(q, None, None, self.q16, None, None, d, htpg.ROPE_HALF, n),
                            self.q16, None, None, q, None, None, self.q_weight, None, self.table), "qkv_rope")
        check(htpg.qkv_rope(htpg.rope_params(None, k, v, None, self.k16, self.v16, d, htpg.ROPE_HALF, n),
                            None, self.k16, self.v16, None, k, v, None, self.k_weight, self.table), "qkv_rope")
        check(htpg.cross_attention(htpg.attention_params(self.o, self.q16, self.k16, self.v16, d ** -0.5), self.o,
                                   self.q16, self.k16, self.v16, kv_lens), "cross_attention")
        o = self.o.view(b * t, h * d)
        check(htpg.w8a8_run(self.wo, self.out, o, channels=h * d), "w8a8_run")
        check(htpg.lora_run(htpg.lora_params(self.out, self.out, o, self.ao, self.bo), self.out, self.out, o,
                            row_adapter, self.ao, self.bo, self.ranks, self.scales), "lora_run")
        return self.out

    def plain(self, x, cond, kv_lens, row_adapter):
        """The same in FP64."""
        b, t, s, h, hk, d = self.batch, self.tokens, self.text, self.heads, self.kv_heads, self.dim
        x, cond = x.double(), cond.double()

        def adapt(y, x, a, bb):
            for i, r in enumerate(self.ranks.tolist()):
                rows = row_adapter == i
                y[rows] += self.scales[i].double() * (x[rows] @ a[i, :r].double().T) @ bb[i, :, :r].double().T
            return y

        def turn(y, weight):
            y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + 1e-6) * weight.double()
            cs = self.table[:y.shape[1]].double()[:, None]
            a, c = y[..., :d // 2], y[..., d // 2:]
            return torch.cat([a * cs[..., 0] - c * cs[..., 1], a * cs[..., 1] + c * cs[..., 0]], -1)

        q = turn(adapt(x @ self.wq64.T, x, self.aq, self.bq).view(b, t, h, d), self.q_weight)
        k = turn((cond @ self.wk64.T).view(b, s, hk, d), self.k_weight).repeat_interleave(h // hk, 2)
        v = (cond @ self.wv64.T).view(b, s, hk, d).repeat_interleave(h // hk, 2)
        score = torch.einsum("bthd,bshd->bhts", q, k) * d ** -0.5
        gone = torch.arange(s, device="cuda")[None, :] >= kv_lens[:, None]
        p = torch.softmax(score.masked_fill(gone[:, None, None], -torch.inf), -1).nan_to_num(0.0)
        o = torch.einsum("bhts,bshd->bthd", p, v).reshape(b * t, h * d)
        return adapt(o @ self.wo64.T, o, self.ao, self.bo)


def inputs(block, seed=1):
    g = torch.Generator().manual_seed(seed)
    c = block.heads * block.dim
    x, cond = torch.randn(block.batch * block.tokens, c, generator=g), torch.randn(block.batch * block.text, c, generator=g)
    lens = torch.randint(1, block.text + 1, (block.batch,), generator=g, dtype=torch.int32)
    ids = torch.arange(block.batch, dtype=torch.int32) % (len(block.ranks) + 1) - 1  # -1: no adapter
    return x.cuda(), cond.cuda(), lens.cuda(), ids.repeat_interleave(block.tokens).cuda()


def main():
    block = CrossBlock(batch=4, tokens=1024, text=77, heads=24, kv_heads=24, dim=64)
    args = inputs(block)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        for _ in range(3):
            out = block.run(*args)
    stream.synchronize()
    ref = block.plain(*args)
    print(f"relative RMS error against FP64 (INT8 activations): {float((out - ref).norm() / ref.norm()):.4f}")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        block.run(*args)
    a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    for _ in range(5):
        graph.replay()
    a.record()
    for _ in range(50):
        graph.replay()
    b.record()
    torch.cuda.synchronize()
    print(f"{block.batch} x {block.tokens} queries over {block.text} states, {block.heads} heads of {block.dim}: "
          f"{a.elapsed_time(b) / 50 * 1000:.1f} us a block")


if __name__ == "__main__":
    main()
