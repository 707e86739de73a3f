"""The layer over 8-bit pages: the rows that the selection keeps are quantised as they
are copied, and the reuse steps attend over the pages.

What is stored is compared bit for bit with the oracle's row format applied to the
rows that the same selection keeps in a bf16 cache (which other tests pin); outputs of
the reuse step with the formula in 64 bits over the rows as the pages hold them."""
import numpy as np
import pytest
import torch

from oracle import chunk, quant
from test_gpu_chunk import check

from dllm_serve_amd import _capi
from dllm_serve_amd.engine.device_step import DeviceStepState, install_context
from dllm_serve_amd.engine.kv_cache import allocate_kv_cache, quantized_pages
from dllm_serve_amd.engine.sequence import PageAllocator, Sequence, prepare_step, slot_mapping_for
from dllm_serve_amd.layers.attention import Attention
from dllm_serve_amd.sparse.state import SparseConfig
from dllm_serve_amd.utils.context import get_context, reset_context

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
MASK = 126336


def _np(t):
    return t.detach().double().cpu().numpy()


def _quantised(cache, slots, heads):
    """Pages with the rows that a bf16 cache holds in these slots."""
    pages = np.zeros((cache.shape[0], heads, quant.RECORD), dtype=np.uint8)
    quant.store(_np(cache.view(-1, heads, 128))[slots], pages, slots)
    return pages


@pytest.mark.parametrize("n_tok,keep,Hq,Hkv,head_select", [
    (264, 116, 4, 4, True), (264, 116, 14, 2, True), (200, 20, 4, 2, False),
    (3000, 1500, 2, 2, True), (2500, 2400, 4, 2, False), (20000, 900, 2, 1, True), (20000, 9000, 2, 1, True)])
def test_selection_quantises_what_it_stores(dev, n_tok, keep, Hq, Hkv, head_select):
    g = torch.Generator().manual_seed(n_tok + keep)
    q, k, v = (torch.randn(n_tok, h, 128, generator=g).to(BF16).to(dev) for h in (Hq, Hkv, Hkv))
    bs, bl = n_tok // 2, 32
    pages = -(-keep // 256) + 2
    slots = torch.randperm(pages * 256, generator=g)[:keep].to(torch.int32)
    slots[keep // 2] = -1          # outside: left out
    slots[keep // 3] = pages * 256
    jobs = torch.tensor([[0, n_tok, bs, bl, keep, 0, int(head_select), 3]], dtype=torch.int32, device=dev)
    ws = torch.empty(_capi.select_workspace_size(1, n_tok - bl, Hq, Hkv, 128), dtype=torch.uint8, device=dev)
    kc, vc = (torch.zeros(pages, 256, Hkv, 128, dtype=BF16, device=dev) for _ in range(2))
    k8, v8 = quantized_pages(pages, Hkv, device=dev), quantized_pages(pages, Hkv, device=dev)
    idx = [torch.full((1, Hkv, keep), -1, dtype=torch.int64, device=dev) for _ in range(2)]
    for a, b, i in ((kc, vc, idx[0]), (k8, v8, idx[1])):
        _capi.select_kv_store(q, k, v, jobs, 1, n_tok - bl, keep, np.float32(128 ** 0.5), a, b, slots.to(dev), i, ws)
    assert torch.equal(*idx)
    ok = [s for s in slots.tolist() if 0 <= s < pages * 256]
    assert np.array_equal(k8.cpu().numpy(), _quantised(kc, ok, Hkv))
    assert np.array_equal(v8.cpu().numpy(), _quantised(vc, ok, Hkv))


def _batch(dev, head_select):
    cfg = [SparseConfig(enabled=True, default_block_len=32, retention_ratio=r, pool_kernel=3, delay_step=1,
                        head_select=head_select) for r in (0.5, 0.9)]
    seqs = [Sequence([1] * 100, 64, MASK, None, device=dev), Sequence([2] * 200, 64, MASK, cfg[0], device=dev),
            Sequence([3] * 400, 64, MASK, cfg[1], device=dev)]
    alloc = PageAllocator([5, 2, 7, 0, 3])
    for s in (seqs[2], seqs[1]):
        alloc.allocate(s)
    return seqs


def _rows(n, h, g, dev):
    return torch.randn(n, h * 128, generator=g).to(BF16).to(dev)


@pytest.mark.parametrize("Hq,Hkv,head_select", [(8, 8, True), (28, 4, False)])
def test_three_steps(dev, Hq, Hkv, head_select):
    full, attn = (Attention(Hq, 128, 128 ** -0.5, Hkv, causal=False) for _ in range(2))
    full.k_cache, full.v_cache = torch.zeros(2, 8, 256, Hkv, 128, dtype=BF16, device=dev)
    attn.k_cache, attn.v_cache = allocate_kv_cache(attn, 1, Hkv, 128, device=dev, num_blocks=8, quantized=True)[:, 0]
    assert attn.k_cache.dtype == torch.uint8 and attn.k_cache.shape == (8, Hkv, _capi.PAGE_BYTES)
    seqs = _batch(dev, head_select)
    g = torch.Generator().manual_seed(31)
    for step in range(4):
        prepare_step(seqs, dev)
        lens = [164, 264, 464] if step < 2 else [164, 32, 32]
        n = sum(lens)
        q, k, v = _rows(n, Hq, g, dev), _rows(n, Hkv, g, dev), _rows(n, Hkv, g, dev)
        out, ref = attn(q, k, v), full(q, k, v)
        at = n if step < 2 else lens[0]
        assert torch.equal(out[:at], ref[:at])       # full attention does not read the cache
        if step == 1:
            slots = [s for x in seqs[1:] for s in slot_mapping_for(x)]
            for a, b in ((full.k_cache, attn.k_cache), (full.v_cache, attn.v_cache)):
                assert np.array_equal(b.cpu().numpy(), _quantised(a, slots, Hkv))
        if step >= 2:
            for s, L in zip(seqs[1:], lens[1:]):
                rows = slot_mapping_for(s)
                held = [quant.load(c.cpu().numpy(), rows) for c in (attn.k_cache, attn.v_cache)]
                x = [_np(t[at:at + L]).reshape(L, -1, 128) for t in (q, k, v)]
                check(out[at:at + L], *chunk.attend(*x, *held, 128 ** -0.5), L + len(rows), f"step {step}")
                at += L
        reset_context()
        for s in seqs:
            s.advance()


@pytest.mark.parametrize("Hq,Hkv", [(4, 4), (14, 2)])
def test_device_plan_and_graph(dev, Hq, Hkv):
    """Tables built on the device give the host plan's bits; captured steps replay them."""
    attn = Attention(Hq, 128, 128 ** -0.5, Hkv, causal=False)
    attn.k_cache, attn.v_cache = quantized_pages(8, Hkv, device=dev), quantized_pages(8, Hkv, device=dev)
    seqs = _batch(dev, True)
    ds = DeviceStepState(seqs, dev, 464)
    g = torch.Generator().manual_seed(32)
    for step in range(3):
        n = [892, 892, 228][step]
        q, k, v = _rows(n, Hq, g, dev), _rows(n, Hkv, g, dev), _rows(n, Hkv, g, dev)
        prepare_step(seqs, dev)
        want = attn(q, k, v)
        pages = attn.k_cache.clone(), attn.v_cache.clone()
        reset_context()
        install_context(seqs, ds.build(seqs))
        assert torch.equal(attn(q, k, v), want)
        assert torch.equal(attn.k_cache, pages[0]) and torch.equal(attn.v_cache, pages[1])
        if step:
            gr = torch.cuda.CUDAGraph()
            torch.cuda.synchronize()
            with torch.cuda.graph(gr):
                install_context(seqs, ds.build(seqs))
                out = attn(q, k, v)
            for _ in range(3):
                q.copy_(_rows(n, Hq, g, dev))
                gr.replay()
                torch.cuda.synchronize()
                got = out.clone()
                got_pages = attn.k_cache.clone()
                prepare_step(seqs, dev)
                assert torch.equal(attn(q, k, v), got) and torch.equal(attn.k_cache, got_pages)
        reset_context()
        ds.advance()
        for s in seqs:
            s.advance()


def test_what_the_layer_refuses(dev):
    attn = Attention(4, 128, 128 ** -0.5, 4, causal=False)
    attn.k_cache, attn.v_cache = quantized_pages(8, 2, device=dev), quantized_pages(8, 2, device=dev)
    seqs = _batch(dev, True)
    g = torch.Generator().manual_seed(33)
    for s in seqs:
        s.advance()
    prepare_step(seqs, dev)
    with pytest.raises(ValueError, match="KV heads"):
        attn(_rows(892, 4, g, dev), _rows(892, 4, g, dev), _rows(892, 4, g, dev))
    reset_context()
    for s in seqs:
        s.advance()
    attn.k_cache, attn.v_cache = quantized_pages(8, 4, device=dev), quantized_pages(8, 4, device=dev)
    prepare_step(seqs, dev)
    x = _rows(228, 4, g, dev)
    attn(x, x, x)
    del get_context()._dllm_plan
    tables = [s.block_table for s in seqs]
    seqs[2].block_table = seqs[2].block_table[:1]    # 388 kept rows
    with pytest.raises(ValueError, match="pages"):
        attn(x, x, x)
    seqs[2].block_table = tables[2]
    reset_context()
