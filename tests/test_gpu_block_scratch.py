"""The block operators' scratch: graphs captured on one stream, forked captures,
streams that come and go and threads' default streams run at once without
sharing it, and what they held is used again.

Every result is compared bit for bit with the same call alone: the operators
add in an order that does not depend on timing."""
import ctypes
import gc
import threading

import pytest
import torch

import htpg

pytestmark = pytest.mark.gpu

F16, F32 = torch.float16, torch.float32
PER_THREAD = 2  # cudaStreamPerThread


class Call:
    """One operator that needs scratch, with inputs of its own."""

    def __init__(self, kind, gpu, seed, scale=1):
        g = torch.Generator(device=gpu).manual_seed(seed)
        r = lambda *s: torch.randn(*s, generator=g, device=gpu)
        self.kind = kind
        if kind == "lora":
            m, k, n = 24 * scale, 1536, 1536
            self.args = (r(m, n), r(m, k), torch.randint(-1, 3, (m,), generator=g, device=gpu, dtype=torch.int32),
                         (r(3, 16, k) / 40).to(F16), r(3, n, 16).to(F16),
                         torch.full((3,), 16, dtype=torch.int32, device=gpu), torch.ones(3, device=gpu))
            self.out = torch.empty(m, n, device=gpu)
            base, x, _, a, b, _, _ = self.args
            self.prm = htpg.lora_params(self.out, base, x, a, b)
        else:  # one row over several ranges of keys; tiles over several ranges, FP32 sums in scratch
            n, m = (1, 6000 * scale) if kind == "few" else (200 * scale, 3000)
            self.args = (r(1, n, 4, 64).to(F16), r(1, m, 2, 64).to(F16), r(1, m, 2, 64).to(F16))
            self.out = torch.empty(1, n, 4, 64, device=gpu)
            self.prm = htpg.attention_params(self.out, *self.args, 0.125)

    def __call__(self, stream=None):
        if self.kind == "lora":
            base, *rest = self.args
            rc = htpg.lora_run(self.prm, self.out, base, *rest, stream=stream)
        else:
            rc = htpg.cross_attention(self.prm, self.out, *self.args, stream=stream)
        assert rc == 0, (rc, htpg.lib().htpg_last_cuda_error())

    def alone(self):
        torch.cuda.synchronize()
        self()
        torch.cuda.synchronize()
        return self.out.clone()


def scratch():
    size, blocks = ctypes.c_size_t(0), ctypes.c_int(0)
    htpg.check(htpg.lib().htpg_debug_op_scratch(ctypes.byref(size), ctypes.byref(blocks)))
    return size.value, blocks.value


def capture(stream, *calls):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        for c in calls:
            c(stream)
    return graph


KINDS = ["lora", "few", "tiles"]


@pytest.mark.parametrize("kind", KINDS)
def test_capture_on_a_stream_without_a_call_before(gpu, kind):
    c = Call(kind, gpu, 1, scale=2)
    want = c.alone()
    graph = capture(torch.cuda.Stream(), c)
    c.out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(c.out, want)


@pytest.mark.parametrize("kind", KINDS)
def test_graphs_of_one_stream_and_the_stream_itself_at_once(gpu, kind):
    own = torch.cuda.Stream()
    calls = [Call(kind, gpu, s, scale) for s, scale in ((1, 1), (2, 1), (3, 2))]
    want = [c.alone() for c in calls]
    eager = Call(kind, gpu, 4)
    want_eager = eager.alone()
    graphs = [capture(own, *[c] * 8) for c in calls]
    sides = [torch.cuda.Stream() for _ in graphs]
    for _ in range(20):
        for c in (*calls, eager):
            c.out.zero_()
        torch.cuda.synchronize()
        for graph, side in zip(graphs, sides):
            with torch.cuda.stream(side):
                graph.replay()
        for _ in range(8):
            eager(own)
        torch.cuda.synchronize()
        for c, w in zip((*calls, eager), (*want, want_eager)):
            assert torch.equal(c.out, w)


@pytest.mark.parametrize("kind", KINDS)
def test_branches_of_one_capture(gpu, kind):
    main, side = torch.cuda.Stream(), torch.cuda.Stream()
    a, b = Call(kind, gpu, 5), Call(kind, gpu, 6)
    want = a.alone(), b.alone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=main):
        side.wait_stream(main)
        for _ in range(8):
            a(main)
            b(side)
        main.wait_stream(side)
    for _ in range(20):
        a.out.zero_(), b.out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(a.out, want[0]) and torch.equal(b.out, want[1])


def test_a_larger_call_in_the_same_capture(gpu):
    small, large = Call("lora", gpu, 7), Call("lora", gpu, 8, scale=64)
    want = small.alone(), large.alone()
    graph = capture(torch.cuda.Stream(), small, large, small)
    small.out.zero_(), large.out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(small.out, want[0]) and torch.equal(large.out, want[1])


def test_blocks_of_graphs_that_are_gone_are_used_again(gpu):
    c = Call("lora", gpu, 9)
    want = c.alone()
    stream = torch.cuda.Stream()
    sizes = []
    for _ in range(6):
        graph = capture(stream, c)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(c.out, want)
        sizes.append(scratch())
        del graph
        gc.collect()
        torch.cuda.synchronize()
    assert len(set(sizes[1:])) == 1


def test_streams_that_come_and_go(gpu):
    """Handles are reused: a new stream has no block of the one before, and blocks do not pile up without end."""
    rt = torch.cuda.cudart()
    c = Call("lora", gpu, 10)
    want = c.alone()
    for _ in range(300):
        handle = ctypes.c_void_p()
        assert int(rt.cudaStreamCreate(ctypes.addressof(handle))) == 0
        c.out.zero_()
        torch.cuda.synchronize()
        for _ in range(4):
            c(handle.value)
        assert int(rt.cudaStreamDestroy(handle.value)) == 0  # its work goes on
        torch.cuda.synchronize()
        assert torch.equal(c.out, want)
    # 128 streams' at most, and some that wait for the next user
    assert scratch()[1] <= 140


@pytest.mark.parametrize("kind", KINDS)
def test_threads_with_their_own_default_stream(gpu, kind):
    calls = [Call(kind, gpu, 20 + i) for i in range(3)]
    want = [c.alone() for c in calls]
    failed = []

    def work(c):
        try:
            for _ in range(100):
                c(PER_THREAD)
        except BaseException as e:  # noqa: BLE001
            failed.append(e)

    for _ in range(4):
        for c in calls:
            c.out.zero_()
        torch.cuda.synchronize()
        threads = [threading.Thread(target=work, args=(c,)) for c in calls]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        torch.cuda.synchronize()
        assert not failed
        for c, w in zip(calls, want):
            assert torch.equal(c.out, w)


def test_after_a_launch_that_gave_up_graphs_start_from_zero_counters(gpu):
    calls = [Call(k, gpu, 30) for k in KINDS]
    want = [c.alone() for c in calls]
    graph = capture(torch.cuda.Stream(), *calls)
    graph.replay()
    torch.cuda.synchronize()
    htpg.check(htpg.lib().htpg_debug_simulate_abort(0xFF))
    assert htpg.check_device() == htpg.EWATCHDOG and htpg.check_device() == 0
    for c in calls:
        c.out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    for c, w in zip(calls, want):
        assert torch.equal(c.out, w)


def test_capture_while_another_thread_needs_more(gpu):
    """Scratch grows on one stream while another thread captures (torch captures for all threads)."""
    a = Call("lora", gpu, 31)
    want = a.alone()
    big = [Call("lora", gpu, 32 + i, scale=100 * (i + 1)) for i in range(3)]
    streams = [torch.cuda.Stream() for _ in range(3)]
    wants = [b.alone() for b in big]
    for b in big:
        b.out.zero_()
    stream, failed = torch.cuda.Stream(), []
    torch.cuda.synchronize()

    def grow():
        try:
            for b, st in zip(big, streams):
                b(st)
        except BaseException as e:  # noqa: BLE001
            failed.append(e)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        a(stream)
        t = threading.Thread(target=grow)
        t.start()
        t.join()
        a(stream)
    assert not failed
    a.out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(a.out, want)
    for b, w in zip(big, wants):
        assert torch.equal(b.out, w)
