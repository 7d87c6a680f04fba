"""Attention over the 8-bit cache in captured graphs and on several streams: calls that overlap on the GPU have workspaces of their own, so every result is, bit for bit, that of
the call alone.  Sequences are long enough that several CTAs share an item and meet in the workspace."""
from ctypes import addressof, c_void_p

import pytest
import torch

from dinoml_v2_b200 import kernels

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


class _Call:
    """One attention call and its result alone.  `new`: rows of each sequence (None: one each, through the kernel of few rows; hundreds go through that of many)."""

    def __init__(self, seed, lengths, new=None, heads=8, kv_heads=2, dim=128, block=64, dtype=torch.bfloat16):
        g = torch.Generator(device=DEV)
        g.manual_seed(seed)
        need = [-(-n // block) for n in lengths]
        self.cache = kernels.kv_cache(sum(need), kv_heads, block, dim)
        for x, scale in zip(self.cache[:2], self.cache[2:]):
            x.copy_((torch.randn(x.shape, device=DEV, generator=g) * 40).round().clamp(-127, 127))
            scale.copy_(torch.rand(scale.shape, device=DEV, generator=g) / 40)
        order = torch.randperm(sum(need), device=DEV, generator=g).tolist()
        self.table = _ints([[order.pop() for _ in range(n)] + [-1] * (max(need) - n) for n in need])
        self.lengths = _ints(lengths)
        self.starts = None if new is None else _ints([sum(new[:i]) for i in range(len(new) + 1)])
        self.q = torch.randn(len(lengths) if new is None else sum(new), heads, dim, device=DEV, generator=g).to(dtype)
        self.out = torch.empty_like(self.q)
        self.want = kernels.kv_cache_attention(self.q, self.cache, self.table, self.lengths, self.starts)
        assert torch.isfinite(self.want).all() and bool(self.want.any())

    def run(self, stream=None):
        kernels.kv_cache_attention(self.q, self.cache, self.table, self.lengths, self.starts, out=self.out, stream=stream)

    def check(self):
        assert torch.equal(self.out, self.want)
        self.out.zero_()


def _captured(stream, call, repeats=1):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        for _ in range(repeats):
            call.run()
    return graph


def _calls(kind):
    if kind == "few":
        return [_Call(1, [9000, 70, 900]), _Call(2, [20000]), _Call(3, [4000] * 6)]
    if kind == "many":
        return [_Call(1, [3000, 900], [500, 300]), _Call(2, [5000], [700]), _Call(3, [1500] * 4, [200, 90, 300, 40])]
    return [_Call(1, [9000, 70, 900]), _Call(2, [5000, 8000], [700, 1]), _Call(3, [1500] * 4, [200, 1, 1, 40], dim=64)]


@pytest.mark.parametrize("kind", ["few", "many", "both"])
def test_graphs_of_one_stream_side_by_side(kind):
    """Graphs captured on one stream, replayed on two others beside one another and beside calls on the stream of their capture."""
    a, b, eager = _calls(kind)
    side, left, right = (torch.cuda.Stream() for _ in range(3))
    graphs = [_captured(side, call, 3) for call in (a, b)]
    torch.cuda.synchronize()
    for _ in range(20):
        for _ in range(5):
            for graph, stream in zip(graphs, (left, right)):
                with torch.cuda.stream(stream):
                    graph.replay()
            eager.run(side)
        torch.cuda.synchronize()
        for call in (a, b, eager):
            call.check()
    assert kernels.device_status() == 0


@pytest.mark.parametrize("kind", ["few", "many", "both"])
def test_streams_side_by_side(kind):
    calls = _calls(kind)
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    for _ in range(20):
        for _ in range(5):
            for call, stream in zip(calls, streams):
                call.run(stream)
        torch.cuda.synchronize()
        for call in calls:
            call.check()
    assert kernels.device_status() == 0


def test_branches_of_one_capture():
    a, b, c = _calls("both")
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        other.wait_stream(side)
        for _ in range(3):
            a.run()
            c.run()
            with torch.cuda.stream(other):
                b.run()
        side.wait_stream(other)
    for _ in range(20):
        graph.replay()
        torch.cuda.synchronize()
        for call in (a, b, c):
            call.check()
    assert kernels.device_status() == 0


def test_graphs_that_are_gone_give_their_memory_back():
    call = _Call(2, [5000], [700])
    side = torch.cuda.Stream()
    free = []
    for i in range(24):
        graph = _captured(side, call)
        graph.replay()
        torch.cuda.synchronize()
        call.check()
        graph.reset()
        del graph
        if i % 8 == 7:
            torch.cuda.synchronize()
            free.append(torch.cuda.mem_get_info()[0])
    assert free[0] - free[-1] < 32 << 20, free               # a set of this call is 39 MB
    assert kernels.device_status() == 0


def test_streams_that_are_released_give_their_memory_back():
    call = _Call(2, [5000], [700])
    free = []
    for i in range(24):
        handle = c_void_p()
        assert int(torch.cuda.cudart().cudaStreamCreate(addressof(handle))) == 0
        stream = torch.cuda.ExternalStream(handle.value)
        for _ in range(2):
            call.run(stream)
        kernels.release_stream(stream)
        call.check()
        assert int(torch.cuda.cudart().cudaStreamDestroy(handle.value)) == 0
        if i % 8 == 7:
            free.append(torch.cuda.mem_get_info()[0])
    assert free[0] - free[-1] < 32 << 20, free               # a set of this call is 39 MB
    assert kernels.device_status() == 0
