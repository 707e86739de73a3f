"""A ChunkPlan on streams other than the one that was current when it was made.

Its tables are uploaded asynchronously there: a first use elsewhere has to wait for the
upload, and a plan that is dropped must not give its tables' memory back before the
last call on another stream has read them."""
import struct

import pytest
import torch

from dllm_serve_amd import _capi
from dllm_serve_amd.layers.attention import ChunkPlan, chunk_attention

SCALE = 128 ** -0.5


class _Stream:
    def __init__(self, handle):
        self.cuda_stream, self.waited = handle, []

    def wait_event(self, event):
        self.waited.append(event)


class _Tables:
    def __init__(self):
        self.streams = []

    def record_stream(self, stream):
        self.streams.append(stream)


def _streams_of(plan):
    return struct.unpack(f"={len(plan._packed) // 8}q", plan._packed)[10 + 6 * len(plan.groups):]


def test_other_streams_wait_once(monkeypatch):
    plan = ChunkPlan([1, 2], [300, 0], [[1, 0], []], "cpu")
    own, other = _Stream(5), _Stream(7)
    plan._ready, plan._tables, plan._streams = object(), _Tables(), (own.cuda_stream,)
    plan._packed = plan._pack()
    now, capturing = [own], [False]
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: now[0])
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing[0])
    plan._join()
    assert own.waited == [] and plan._tables.streams == []
    now[0] = other
    for _ in range(2):
        plan._join()
        assert other.waited == [plan._ready] and plan._tables.streams == [other]
        assert _streams_of(plan) == (5, 7)
    # a captured stream cannot wait for an event from outside its graph
    now[0], capturing[0] = _Stream(9), True
    plan._join()
    assert now[0].waited == [] and _streams_of(plan) == (5, 7)
    # the list of streams stays short; a forgotten one waits again
    capturing[0] = False
    for h in range(100, 100 + plan._STREAMS):
        now[0] = _Stream(h)
        plan._join()
        assert now[0].waited == [plan._ready]
    assert len(_streams_of(plan)) == plan._STREAMS and 7 not in _streams_of(plan)
    now[0] = other
    plan._join()
    assert other.waited == [plan._ready] * 2


def _inputs(dev, lens, Hq, Hkv, pages, seed):
    g = torch.Generator().manual_seed(seed)
    n = sum(lens)
    x = [torch.randn(n, h, 128, generator=g).bfloat16().to(dev) for h in (Hq, Hkv, Hkv)]
    return x + [torch.randn(pages, 256, Hkv, 128, generator=g).bfloat16().to(dev) for _ in range(2)]


def _busy(a, n=24):
    """Work of some ten milliseconds on the current stream."""
    for _ in range(n):
        a = torch.mm(a, a)
    return a


@pytest.mark.gpu
@pytest.mark.parametrize("native", [True, False])
def test_first_use_on_another_stream(dev, native, monkeypatch):
    """The upload is queued behind other work; the call's stream is idle."""
    if not native:
        monkeypatch.setattr(_capi, "native", None)
    lens, cached, tables = [3, 40, 1], [700, 0, 300], [[4, 1, 6], [], [2, 0]]
    x = _inputs(dev, lens, 4, 2, 7, 41)
    want = chunk_attention(*x, ChunkPlan(lens, cached, tables, dev, mask_block=1), SCALE)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    big = torch.randn(8192, 8192, device=dev, dtype=torch.bfloat16) * 0.01
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.cuda.stream(a):
            keep = _busy(big)
            plan = ChunkPlan(lens, cached, tables, dev, mask_block=1)
        with torch.cuda.stream(b):
            outs = [chunk_attention(*x, plan, SCALE) for _ in range(3)]
        torch.cuda.synchronize()
        assert all(torch.equal(o, want) for o in outs)
        assert _streams_of(plan) == (a.cuda_stream, b.cuda_stream)
    del keep


@pytest.mark.gpu
def test_plan_dropped_while_another_stream_still_needs_it(dev):
    lens, cached, tables = [5, 33], [600, 20], [[3, 0, 5], [1]]
    x = _inputs(dev, lens, 4, 2, 6, 42)
    want = chunk_attention(*x, ChunkPlan(lens, cached, tables, dev, mask_block=1), SCALE)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    big = torch.randn(8192, 8192, device=dev, dtype=torch.bfloat16) * 0.01
    torch.cuda.synchronize()
    with torch.cuda.stream(a):
        plan = ChunkPlan(lens, cached, tables, dev, mask_block=1)
        size, at = plan._tables.numel(), plan._tables.data_ptr()
    with torch.cuda.stream(b):
        keep = _busy(big)
        out = chunk_attention(*x, plan, SCALE)
        del plan
    with torch.cuda.stream(a):
        # what the plan's stream allocates next, of the same size; zeros are lengths of zero
        fresh = [torch.zeros(size, dtype=torch.int32, device=dev) for _ in range(4)]
    assert all(t.data_ptr() != at for t in fresh)
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    del keep


@pytest.mark.gpu
def test_one_plan_in_two_graphs_and_eager(dev):
    lens, cached, tables = [1, 1], [2500, 900], [list(range(10)), [10, 11, 12, 13]]
    x = _inputs(dev, lens, 7, 1, 14, 43)
    with torch.cuda.stream(torch.cuda.Stream()):
        plan = ChunkPlan(lens, cached, tables, dev, mask_block=1)
    want = chunk_attention(*x, plan, SCALE)
    graphs, outs = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(chunk_attention(*x, plan, SCALE))
    for i in range(6):
        outs[i % 2].zero_()
        graphs[i % 2].replay()
        assert torch.equal(chunk_attention(*x, plan, SCALE), want)
        torch.cuda.synchronize()
        assert torch.equal(outs[i % 2], want)
