"""A step whose tables the host builds has run before it is captured: inside a capture
the upload would be replayed from pinned memory that has been given to something else."""
import pytest
import torch

from dllm_serve_amd import _capi
from dllm_serve_amd.engine.kv_cache import quantized_pages
from dllm_serve_amd.engine.sequence import PageAllocator, Sequence, prepare_step
from dllm_serve_amd.layers.attention import Attention
from dllm_serve_amd.sparse.state import SparseConfig
from dllm_serve_amd.utils.context import get_context, reset_context

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def _step_of_reuse(dev):
    cfg = SparseConfig(enabled=True, default_block_len=32, retention_ratio=0.9, pool_kernel=3, delay_step=1,
                       head_select=True)
    seqs = [Sequence([1] * n, 64, 126336, cfg, device=dev) for n in (200, 400)]
    alloc = PageAllocator([5, 2, 7, 0, 3])
    for s in seqs:
        alloc.allocate(s)
        s.advance()
        s.advance()
    g = torch.Generator().manual_seed(51)
    x = [torch.randn(64, h * 128, generator=g).to(BF16).to(dev) for h in (8, 2, 2)]
    return seqs, x


def _layer(dev, quantised):
    attn = Attention(8, 128, 128 ** -0.5, 2, causal=False)
    if quantised:
        attn.k_cache, attn.v_cache = quantized_pages(8, 2, device=dev), quantized_pages(8, 2, device=dev)
    else:
        attn.k_cache, attn.v_cache = torch.zeros(2, 8, 256, 2, 128, dtype=BF16, device=dev)
    return attn


def test_uploads_inside_a_capture_are_refused(dev):
    seqs, x = _step_of_reuse(dev)
    bf16, pages = _layer(dev, False), _layer(dev, True)
    y = torch.zeros(4, device=dev)

    def capture(layer, match):
        graph = torch.cuda.CUDAGraph()
        y.zero_()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            y.add_(1)
            with pytest.raises(RuntimeError, match=match):
                layer(*x)
        graph.replay()
        torch.cuda.synchronize()
        assert (y == 1).all()

    prepare_step(seqs, dev)
    for layer in (bf16, pages):
        capture(layer, "before the capture")
    # the plan is there, its page table is not
    bf16(*x)
    capture(pages, "page table, before the capture")
    reset_context()


@pytest.mark.parametrize("quantised", [False, True])
def test_after_one_forward_the_step_is_captured(dev, quantised):
    seqs, x = _step_of_reuse(dev)
    layer = _layer(dev, quantised)
    if quantised:
        for t in (layer.k_cache, layer.v_cache):
            t.copy_(torch.randint(0, 120, t.shape, dtype=torch.uint8, device=dev))
    else:
        for t in (layer.k_cache, layer.v_cache):
            t.normal_()
    prepare_step(seqs, dev)
    want = layer(*x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer(*x)
    for _ in range(3):
        out.zero_()
        graph.replay()
        assert torch.equal(layer(*x), want)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    reset_context()


def test_pages_follow_the_slot_mapping(dev):
    """8-bit pages that the block table does not name: state 2 reads the rows of the slot
    mapping, as it does with a bf16 cache."""
    seqs, x = _step_of_reuse(dev)
    layer = _layer(dev, True)
    for t in (layer.k_cache, layer.v_cache):
        t.copy_(torch.randint(0, 120, t.shape, dtype=torch.uint8, device=dev))
    prepare_step(seqs, dev)
    want = layer(*x)
    moved = [4, 6, 1]  # the sequences' pages 5 | 2, 7 elsewhere
    for t in (layer.k_cache, layer.v_cache):
        t[moved] = t[[5, 2, 7]]
        t[[5, 2, 7]] = 0
    reset_context()
    prepare_step(seqs, dev)
    ctx = get_context()
    to = dict(zip([5, 2, 7], moved))
    ctx.slot_mapping = [torch.tensor([to[s // 256] * 256 + s % 256 for s in m.tolist()], dtype=torch.int32, device=dev)
                        for m in ctx.slot_mapping]
    assert torch.equal(layer(*x), want)
    reset_context()


def test_a_step_over_pages_takes_one_workspace(dev):
    seqs, x = _step_of_reuse(dev)
    layer = _layer(dev, True)
    prepare_step(seqs, dev)
    want = layer(*x)
    plan = get_context()._dllm_plan
    assert list(plan._args) == [(8, 2, 128, "pages")]
    other = _layer(dev, True)       # another layer with the checked caches of the first
    other.k_cache, other.v_cache = layer.k_cache, layer.v_cache
    assert torch.equal(other(*x), want) and len(plan._args) == 1
    # a bf16 layer in the same step has its own
    _layer(dev, False)(*x)
    assert set(plan._args) == {(8, 2, 128, "pages"), (8, 2, 128)}
    assert torch.equal(layer(*x), want)
    # caches that are rebound are checked again
    layer.k_cache = torch.zeros(8, 2, 100, dtype=torch.uint8, device=dev)
    with pytest.raises(ValueError, match="k_cache"):
        layer(*x)
    reset_context()


@pytest.mark.parametrize("with_dense", [False, True])
def test_state_2_over_pages_is_one_native_call(dev, with_dense, monkeypatch):
    """The same bits as the Python form; other layouts and caches are left to it."""
    seqs, x = _step_of_reuse(dev)
    if with_dense:  # a sequence without a cache in the same step
        seqs.insert(1, Sequence([3] * 90, 38, 126336, None, device=dev))
        g = torch.Generator().manual_seed(52)
        x = [torch.randn(192, h * 128, generator=g).to(BF16).to(dev) for h in (8, 2, 2)]
    layer = _layer(dev, True)
    for t in (layer.k_cache, layer.v_cache):
        t.copy_(torch.randint(0, 120, t.shape, dtype=torch.uint8, device=dev))
    prepare_step(seqs, dev)
    with monkeypatch.context() as m:
        m.setattr(_capi, "native", None)
        want = layer(*x)
    reset_context()
    prepare_step(seqs, dev)
    assert torch.equal(layer(*x), want)       # builds the plan
    plan = get_context()._dllm_plan
    with monkeypatch.context() as m:
        def python_form(*a):
            raise AssertionError("the Python form ran")
        m.setattr(Attention, "_mixed_sparse_dense_attention", python_form)
        assert torch.equal(layer(*x), want)
        three = [t.view(t.shape[0], -1, 128) for t in x]
        assert torch.equal(layer(*three), want)
        # in a graph too
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = layer(*x)
        for _ in range(3):
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)
    packed = plan._packed[(8, 2, 128, "pages")]
    call = lambda kc, vc: _capi.native.attn(*x, kc, vc, packed, float(layer.scale))  # noqa: E731
    assert torch.equal(call(layer.k_cache, layer.v_cache), want)
    bf16 = torch.zeros(8, 256, 2, 128, dtype=BF16, device=dev)
    for kc, vc in ((bf16, bf16), (layer.k_cache, bf16), (layer.k_cache[:, :1], layer.v_cache), (layer.k_cache, None),
                   (layer.k_cache[:0], layer.v_cache[:0]), (layer.k_cache.cpu(), layer.v_cache.cpu())):
        assert call(kc, vc) is None
    reset_context()
