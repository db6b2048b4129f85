"""pagedAttention on several streams, from several threads and in graph replays, where the kernel itself joins the parts of a unit.

That happens for batches of up to eight workgroups a unit on average (a request and key head), whose units are longer than
eight tiles of 32 tokens: there workgroups count themselves in, in numbers that calls share.
"""
import threading

import pytest
import torch

import blockedAttention
from blockedattention_amd import capi
from test_gpu_paged_attention import Batch

pytestmark = pytest.mark.gpu


class Call:
    """A batch on the GPU, called as often as wanted."""

    def __init__(self, dev, seed, dtype=torch.float16, dim=64, lens=None):
        g = torch.Generator().manual_seed(seed)
        self.lens = torch.randint(300, 700, (40,), generator=g).tolist() if lens is None else lens
        b = Batch(self.lens, 4, 2, dim, 16, dtype, seed=seed)
        # four workgroups a compute unit at most, fewer for more dimensions
        assert 4 * torch.cuda.get_device_properties(dev).multi_processor_count <= 8 * 4 * len(self.lens)
        self.ref, self.bound = b.expect(0.125)
        self.q, self.k, self.v, self.table = b.q.to(dev), b.k.to(dev), b.v.to(dev), b.table.to(dev)
        self.n = torch.tensor(self.lens, device=dev)

    def __call__(self):
        return blockedAttention.pagedAttention(self.q, self.k, self.v, self.table, self.n, 0.125)

    def right(self, out):
        return bool(((out.double().cpu() - self.ref).abs() <= self.bound).all())


@pytest.fixture(scope="module")
def calls(dev):
    return [Call(dev, seed, dtype, dim) for seed, dtype, dim in ((1, torch.float16, 64), (2, torch.bfloat16, 128), (3, torch.float16, 128), (4, torch.bfloat16, 64))]


def test_several_streams_in_flight(dev, calls):
    want = [c() for c in calls]
    assert all(c.right(w) for c, w in zip(calls, want))
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    got = [[] for _ in calls]
    for _ in range(25):
        for c, s, g in zip(calls, streams, got):
            with torch.cuda.stream(s):
                g.append(c())
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert all(torch.equal(x, w) for x in g)


def test_threads_on_one_stream_and_on_their_own(dev, calls):
    want = [c() for c in calls]
    torch.cuda.synchronize()
    for own in (False, True):
        got, errors = [[] for _ in calls], []

        def work(i, stream):
            try:
                with torch.cuda.stream(stream):
                    for _ in range(25):
                        got[i].append(calls[i]())
            except Exception as e:  # noqa: BLE001
                errors.append(e)

        shared = torch.cuda.Stream()
        threads = [threading.Thread(target=work, args=(i, torch.cuda.Stream() if own else shared)) for i in range(len(calls))]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        torch.cuda.synchronize()
        assert not errors
        for w, g in zip(want, got):
            assert len(g) == 25 and all(torch.equal(x, w) for x in g)


def test_replays_beside_eager_calls(dev, calls):
    """A graph of two calls, replayed with other lengths each time, while other calls run on another stream."""
    a, b, other = calls[0], calls[1], calls[2]
    side = torch.cuda.Stream()
    wanted_other = other()
    a(), b()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = a(), b()
    g = torch.Generator().manual_seed(7)
    first = [c.n.clone() for c in (a, b)]
    for step in range(6):
        for c, n in zip((a, b), first):
            c.n.copy_(n if step in (0, 5) else (n * torch.rand(40, generator=g).to(dev)).long())
        want = [c() for c in (a, b)]
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            beside = [other() for _ in range(6)]
        graph.replay()
        eager = a()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1]) and torch.equal(eager, want[0]), step
        assert all(torch.equal(x, wanted_other) for x in beside), step
    assert a.right(outs[0]) and b.right(outs[1])


def test_counters_are_zero_after_every_call(dev, calls):
    counters = capi.paged_counters(dev)
    for _ in range(3):
        for c in calls:
            out = torch.full_like(c.q, float("nan"))
            capi.paged_attention(capi.paged_cache(c.k, c.v), c.q, c.table, c.n, out, 0.125, 0, counters)
            assert (counters == 0).all()
            assert torch.equal(out, c())
