"""Scratch memory of the sequence operators: calls that may run at the same time share none, whatever
stream a graph is replayed on.  The operators have a fixed order of sums, so results are compared
bit for bit."""

import ctypes
import gc
import threading

import pytest
import torch

import oxide_hip as ox
from test_gpu_muon import matrix
from test_gpu_recurrence import gates, make

pytestmark = pytest.mark.gpu
F32 = torch.float32


class Calls:
    """One set of the operators' calls with more than one launch, on operands of its own."""

    def __init__(self, module, dev, seed):
        self.module = module
        self.u, self.g = make((1, 3000, 24), F32, dev, seed), gates((1, 3000, 24), F32, dev, seed + 1)
        self.x, self.w = make((600, 700), F32, dev, seed + 2), make((700,), F32, dev, seed + 3)
        self.q = torch.rsqrt(self.x.square().mean(1))
        self.v = torch.from_numpy(matrix((300, 310), seed + 4)).to(dev)
        self.outs = [torch.empty_like(t) for t in (self.u, self.u, self.u, self.x, self.w, self.v)]
        self.run()
        torch.cuda.synchronize()
        self.want = [t.clone() for t in self.outs]

    def run(self, stream=None):
        h, du, dg, dx, dw, o = self.outs
        m = self.module
        m.gated_recurrence_forward(self.u, self.g, h, stream=stream)
        m.gated_recurrence_backward(self.u, self.u, self.g, h, du, dg, stream=stream)
        m.rms_norm_backward(self.x, self.x, self.w, self.q, dx, dw, stream=stream)
        m.orthogonalize(self.v, o, stream=stream)

    def clear(self):
        for t in self.outs:
            t.zero_()

    def check(self):
        for a, b in zip(self.outs, self.want):
            assert torch.equal(a, b)


def recorded(monkeypatch):
    """The scratch ranges that calls take from now on."""
    ranges, whole = [], ox.StreamWorkspaces.ptr_bytes

    def noting(self, nbytes, stream):
        got = whole(self, nbytes, stream)
        if got[0] is not None:
            ranges.append((got[0], got[0] + got[1]))
        return got

    monkeypatch.setattr(ox.StreamWorkspaces, "ptr_bytes", noting)
    return ranges


def apart(a, b):
    return all(x1 <= y0 or y1 <= x0 for x0, x1 in a for y0, y1 in b)


def test_graphs_of_one_stream_on_several(dev, monkeypatch):
    """Two graphs captured on one stream and replayed on two, beside eager calls on the first."""
    module = ox.load_kernels(0)
    sets = [Calls(module, dev, 10 * i) for i in range(3)]
    one, two, three = (torch.cuda.Stream() for _ in range(3))
    ranges, graphs, parts = recorded(monkeypatch), [], []
    for calls in sets[:2]:
        graphs.append(ox.HipGraphExec.capture(one, lambda: calls.run(one)))
        parts.append(ranges[:])
        ranges.clear()
    sets[2].run(one)
    parts.append(ranges[:])
    assert all(len(p) == 4 for p in parts)
    for i in range(3):
        assert all(apart(parts[i], parts[j]) for j in range(i))
    for _ in range(5):
        for calls in sets:
            calls.clear()
        torch.cuda.synchronize()
        for _ in range(10):
            graphs[0].launch(two)
            graphs[1].launch(three)
            sets[2].run(one)
        torch.cuda.synchronize()
        for calls in sets:
            calls.check()


def test_a_stream_says_whether_it_is_captured(dev):
    one, two, said = torch.cuda.Stream(), torch.cuda.Stream(), []

    def ask():
        for s in (one, two):
            out = ctypes.c_int(7)
            ox.check(ox.lib().oxh_stream_is_capturing(s.cuda_stream, ctypes.byref(out)))
            said.append(out.value)

    ask()
    with torch.cuda.stream(one):
        x = torch.zeros(8, device=dev)
        graph = ox.HipGraphExec.capture(one, lambda: (x.add_(1), ask()))
    ask()
    assert said == [0, 0, 1, 0, 0, 0]
    del graph


def test_scratch_lives_with_its_graph(dev, monkeypatch):
    """What a graph's launches write is nobody else's until the graph goes, and is given back then."""
    module = ox.load_kernels(0)
    calls, stream = Calls(module, dev, 5), torch.cuda.Stream()
    ranges = recorded(monkeypatch)
    graph = ox.HipGraphExec.capture(stream, lambda: calls.run(stream))
    mine = ranges[:]
    with torch.cuda.stream(stream):
        others = [torch.full((n,), 3, dtype=torch.uint8, device=dev)
                  for p in mine for n in [p[1] - p[0]] * 4]
    assert apart(mine, [(t.data_ptr(), t.data_ptr() + t.numel()) for t in others])
    for _ in range(3):
        calls.clear()
        torch.cuda.synchronize()
        graph.launch(torch.cuda.current_stream())
        torch.cuda.synchronize()
        calls.check()
        assert all((t == 3).all() for t in others)
    held = torch.cuda.memory_allocated()
    del graph
    gc.collect()
    assert held - torch.cuda.memory_allocated() >= max(b - a for a, b in mine)


def test_calls_of_one_graph_share_scratch(dev, monkeypatch):
    """Recorded calls on one stream run in their order, so a graph of many takes no more than the
    largest and the smaller ones before it."""
    module = ox.load_kernels(0)
    calls, stream = Calls(module, dev, 7), torch.cuda.Stream()
    ranges = recorded(monkeypatch)

    def several():
        for _ in range(10):
            calls.run(stream)

    start = torch.cuda.memory_allocated()
    graph = ox.HipGraphExec.capture(stream, several)
    used = torch.cuda.memory_allocated() - start
    assert len(ranges) == 40 and used <= sum(b - a for a, b in set(ranges)) + 4 * 512
    assert len(set(ranges)) <= 4 and len(set(ranges[4:])) == 1
    calls.clear()
    torch.cuda.synchronize()
    graph.launch(torch.cuda.current_stream())
    torch.cuda.synchronize()
    calls.check()


def test_graphs_of_torch(dev, monkeypatch):
    """Captures by ``torch.cuda.graph``, which all use one stream: scratch of each graph's pool, free
    for its later allocations, and of no other graph."""
    module = ox.load_kernels(0)
    sets, graphs, ranges, parts = [], [], recorded(monkeypatch), []
    for i in range(2):
        calls, graph = Calls(module, dev, 20 + 10 * i), torch.cuda.CUDAGraph()
        ranges.clear()
        with torch.cuda.graph(graph):
            for _ in range(2):
                calls.run()
                calls.u.add_(torch.zeros_like(calls.u) * 2)
        parts.append(ranges[:])
        sets.append(calls)
        graphs.append(graph)
    assert len(parts[0]) == len(parts[1]) == 8 and apart(*parts)
    assert module._sequence_ws._kept == []
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(4):
        for calls in sets:
            calls.clear()
        torch.cuda.synchronize()
        for _ in range(5):
            for graph, stream in zip(graphs, streams):
                with torch.cuda.stream(stream):
                    graph.replay()
            eager = Calls(module, dev, 50)
        torch.cuda.synchronize()
        eager.check()
        for calls in sets:
            calls.check()


def test_outgrown_buffers_are_given_back(dev):
    """A stream's buffer for eager calls is one, at most 64 MB larger than the largest call's."""
    ws, stream = ox.StreamWorkspaces(), torch.cuda.Stream()
    start = torch.cuda.memory_allocated()
    for size in (1 << 10, 1 << 20, 300 << 20, (300 << 20) + 1):
        _, got = ws.ptr_bytes(size, stream.cuda_stream)
        assert size <= got <= size + (64 << 20)
        assert torch.cuda.memory_allocated() - start <= got + 512
    torch.cuda.synchronize()


def test_threads_on_one_stream(dev):
    """Host threads that call one module on one stream, each with operands of its own."""
    module = ox.load_kernels(0)
    sets = [Calls(module, dev, 60 + 10 * i) for i in range(4)]
    stream, wrong = torch.cuda.Stream(), []

    def work(calls):
        try:
            for _ in range(20):
                calls.run(stream)
        except Exception as error:  # noqa: BLE001 - reported below
            wrong.append(error)

    for _ in range(3):
        for calls in sets:
            calls.clear()
        torch.cuda.synchronize()
        threads = [threading.Thread(target=work, args=(calls,)) for calls in sets]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        torch.cuda.synchronize()
        assert not wrong
        for calls in sets:
            calls.check()


def test_graphs_that_end_during_a_capture(dev):
    """No wait is made while another graph is captured: its scratch is freed with that one, or with
    the next that ends."""
    module = ox.load_kernels(0)
    calls, stream = Calls(module, dev, 9), torch.cuda.Stream()
    capture = lambda: ox.HipGraphExec.capture(stream, lambda: calls.run(stream))  # noqa: E731
    start, first = torch.cuda.memory_allocated(), [capture()]
    other = torch.cuda.Stream()
    with torch.cuda.stream(other):
        x = torch.zeros(8, device=dev)
        second = ox.HipGraphExec.capture(other, lambda: (first.clear(), x.add_(1)))
    assert torch.cuda.memory_allocated() > start + 512
    del second
    gc.collect()
    assert torch.cuda.memory_allocated() <= start + 512  # x
    first.append(capture())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        first.clear()
        x.add_(1)
    assert len(ox._unfreed) == 1
    graph.replay()
    third = capture()
    del third
    gc.collect()
    assert ox._unfreed == []
    torch.cuda.synchronize()
    assert float(x[0]) == 1
