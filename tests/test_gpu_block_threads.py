"""The block operators in several host threads: as a thread's first CUDA work,
and beside a thread that clears the scratch after a launch gave up."""
import threading

import pytest
import torch

import htpg

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,m", [(200, 77), (200, 3000), (1, 6000), (5, 0)])
@pytest.mark.parametrize("dst", [torch.float16, torch.float32])
def test_attention_first_in_a_thread(gpu, n, m, dst):
    g = torch.Generator(device=gpu).manual_seed(m)
    r = lambda *s: torch.randn(*s, generator=g, device=gpu).half()
    q, k = r(1, n, 4, 64), r(1, m, 2, 64)
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


def test_clearing_the_scratch_waits_for_launches(gpu):
    """Counters and partial sums are cleared between calls, not between the launches of one."""
    g = torch.Generator(device=gpu).manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g, device=gpu)
    a, b = (r(2, 16, 1536) / 40).half(), r(2, 1536, 16).half()
    ranks, scales = torch.full((2,), 16, dtype=torch.int32, device=gpu), torch.ones(2, device=gpu)
    q, k = r(1, 1, 4, 64).half(), r(1, 6000, 2, 64).half()
    jobs, failed = [], []
    for i in range(3):
        m = 8 + 700 * i
        x, base = r(m, 1536), r(m, 1536)
        ids = torch.randint(0, 2, (m,), generator=g, device=gpu, dtype=torch.int32)
        out, att = torch.empty_like(base), torch.empty(q.shape, device=gpu)
        lora, attn = htpg.lora_params(out, base, x, a, b), htpg.attention_params(att, q, k, k, 0.125)

        def call(stream=None, lora=lora, attn=attn, out=out, base=base, x=x, ids=ids, att=att):
            return (htpg.lora_run(lora, out, base, x, ids, a, b, ranks, scales, stream=stream) or
                    htpg.cross_attention(attn, att, q, k, k, stream=stream))
        assert call() == 0
        torch.cuda.synchronize()
        jobs.append((call, out, att, out.clone(), att.clone(), torch.cuda.Stream().cuda_stream))

    def work(call, stream):
        for _ in range(200):
            code = call(stream)
            if code:
                failed.append(code)

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(j[0], j[5])) for j in jobs]
    for t in threads:
        t.start()
    for _ in range(50):
        htpg.check(htpg.lib().htpg_debug_simulate_abort(0))
        assert htpg.check_device() == htpg.EWATCHDOG
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed and htpg.check_device() == 0
    for _, out, att, want, want_att, _ in jobs:
        assert torch.equal(out, want) and torch.equal(att, want_att)
