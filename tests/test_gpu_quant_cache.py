"""store_kvcache / load_kvcache over 8-bit pages: codes, scale bytes and the values
read back are bit-exact against the oracle's row format."""
import numpy as np
import pytest
import torch

from oracle import quant
from dllm_serve_amd.engine.kv_cache import quantized_pages
from dllm_serve_amd.layers.attention import load_kvcache, store_kvcache

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def _np(t):
    return t.detach().double().cpu().numpy()


def _same(a, b):
    return np.array_equal(a, b, equal_nan=True)


def _rows(n, h, seed, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, h, 128, generator=g) * torch.exp(spread * torch.randn(n, h, 1, generator=g))
    return x.to(BF16)


@pytest.mark.parametrize("n,heads,pages", [(1, 1, 1), (3, 4, 2), (33, 4, 3), (257, 5, 3), (700, 32, 4)])
def test_store_then_load(dev, n, heads, pages):
    g = torch.Generator().manual_seed(n)
    k, v = _rows(n, heads, 1), _rows(n, heads, 2)
    slots = torch.randperm(pages * 256, generator=g)[:n].to(torch.int32)
    kc, vc = quantized_pages(pages, heads, device=dev), quantized_pages(pages, heads, device=dev)
    kc.random_(0, 256)  # what was there before stays around the rows
    want_k, want_v = kc.cpu().numpy().copy(), vc.cpu().numpy().copy()
    store_kvcache(k.to(dev), v.to(dev), kc, vc, slots.to(dev))
    quant.store(_np(k), want_k, slots.numpy())
    quant.store(_np(v), want_v, slots.numpy())
    assert np.array_equal(kc.cpu().numpy(), want_k) and np.array_equal(vc.cpu().numpy(), want_v)
    ko, vo = torch.zeros_like(k, device=dev), torch.zeros_like(v, device=dev)
    back = slots.flip(0).contiguous()
    load_kvcache(ko, vo, kc, vc, back.to(dev))
    assert _same(_np(ko), quant.load(want_k, back.numpy())) and _same(_np(vo), quant.load(want_v, back.numpy()))


def test_every_bf16_magnitude(dev):
    """Rows led by each bf16 value (subnormal, normal, largest), the rest at every distance below it."""
    bits = torch.arange(0, 0x7F80, 1, dtype=torch.int32)
    lead = bits.to(torch.int16).view(BF16)
    n = lead.numel()
    g = torch.Generator().manual_seed(0)
    lower = torch.rand(n, 127, generator=g) * bits[:, None].float()  # bit patterns below the lead's
    x = torch.cat([bits[:, None], lower.to(torch.int32)], 1)
    x = (x | (torch.randint(0, 2, x.shape, generator=g, dtype=torch.int32) << 15)).to(torch.int16).view(BF16).view(n, 1, 128)
    pages = -(-n // 256)
    kc, vc = quantized_pages(pages, 1, device=dev), quantized_pages(pages, 1, device=dev)
    slots = torch.arange(n, dtype=torch.int32)
    store_kvcache(x.to(dev), x.flip(0).contiguous().to(dev), kc, vc, slots.to(dev))
    codes, scale = quant.quantise(_np(x)[:, 0])
    got = kc.cpu().numpy().reshape(pages, quant.RECORD)
    assert np.array_equal(got[:, :256 * 128].reshape(-1, 128)[:n], codes)
    assert np.array_equal(got[:, 256 * 128:].reshape(-1)[:n], scale)
    ko, vo = torch.empty_like(x, device=dev), torch.empty_like(x, device=dev)
    load_kvcache(ko, vo, kc, vc, slots.to(dev))
    want = quant.dequantise(codes, scale)
    assert _same(_np(ko)[:, 0], want) and _same(_np(vo)[:, 0], want[::-1])


def test_nan_and_infinities(dev):
    x = _rows(8, 4, 5, 0.0)
    x[0, 0, 3] = float("nan")
    x[1, 1, 7] = float("inf")
    x[2, 2, 127] = float("-inf")
    x[3, 3] = float("nan")
    x[4, 0] = 0.0
    kc, vc = quantized_pages(1, 4, device=dev), quantized_pages(1, 4, device=dev)
    slots = torch.arange(8, dtype=torch.int32, device=dev)
    store_kvcache(x.to(dev), x.to(dev), kc, vc, slots)
    ko, vo = torch.empty_like(x, device=dev), torch.empty_like(x, device=dev)
    load_kvcache(ko, vo, kc, vc, slots)
    codes, scale = quant.quantise(_np(x))
    want = quant.dequantise(codes, scale)
    assert _same(_np(ko), want) and _same(_np(vo), want)
    assert np.isnan(want[3, 3]).all() and (want[4, 0] == 0).all()


def test_slots_outside_are_skipped(dev):
    x = _rows(6, 2, 9, 0.0)
    kc, vc = quantized_pages(1, 2, device=dev), quantized_pages(1, 2, device=dev)
    slots = torch.tensor([-1, 3, 256, 2**31 - 1, -2**31, 255], dtype=torch.int32, device=dev)
    store_kvcache(x.to(dev), x.to(dev), kc, vc, slots)
    want = np.zeros((1, 2, quant.RECORD), dtype=np.uint8)
    quant.store(_np(x), want, slots.cpu().numpy())
    assert np.array_equal(kc.cpu().numpy(), want)
    ko, vo = torch.full_like(x, 7.0, device=dev), torch.full_like(x, 8.0, device=dev)
    load_kvcache(ko, vo, kc, vc, slots)
    assert (ko[[0, 2, 3, 4]] == 7).all() and (vo[[0, 2, 3, 4]] == 8).all()
    assert _same(_np(ko[[1, 5]]), quant.load(want, [3, 255]))


def test_unwritten_rows_read_as_zeros(dev):
    kc, vc = quantized_pages(1, 2, device=dev), quantized_pages(1, 2, device=dev)
    ko, vo = torch.ones(4, 2, 128, dtype=BF16, device=dev), torch.ones(4, 2, 128, dtype=BF16, device=dev)
    load_kvcache(ko, vo, kc, vc, torch.arange(4, dtype=torch.int32, device=dev))
    assert (ko == 0).all() and (vo == 0).all()


@pytest.mark.parametrize("width,offset", [(3 * 256, 256), (3 * 256 + 4, 2), (3 * 256 + 1, 1)])
def test_strided_rows(dev, width, offset):
    """Column slices of a fused projection, 16-byte aligned or not."""
    buf = torch.zeros(20, width, dtype=BF16, device=dev)
    x = _rows(20, 2, 3, 0.5).to(dev)
    k = buf[:, offset:offset + 256].view(20, 2, 128)
    k.copy_(x)
    kc, vc = quantized_pages(1, 2, device=dev), quantized_pages(1, 2, device=dev)
    slots = torch.arange(20, dtype=torch.int32, device=dev)
    store_kvcache(k, x, kc, vc, slots)
    assert torch.equal(kc, vc)
    out = torch.full((20, width), 5.0, dtype=BF16, device=dev)
    ko = out[:, offset:offset + 256].view(20, 2, 128)
    vo = torch.empty_like(x)
    load_kvcache(ko, vo, kc, vc, slots)
    assert torch.equal(ko, vo)
    assert (out[:, :offset] == 5).all() and (out[:, offset + 256:] == 5).all()


def test_empty_and_another_stream(dev):
    kc, vc = quantized_pages(2, 2, device=dev), quantized_pages(2, 2, device=dev)
    e = torch.empty(0, 2, 128, dtype=BF16, device=dev)
    store_kvcache(e, e, kc, vc, torch.empty(0, dtype=torch.int32, device=dev))
    x = _rows(300, 2, 4, 0.0).to(dev)
    slots = torch.arange(300, dtype=torch.int32, device=dev)
    ko, vo = torch.empty_like(x), torch.empty_like(x)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        store_kvcache(x, x, kc, vc, slots)
        load_kvcache(ko, vo, kc, vc, slots)
    s.synchronize()
    codes, scale = quant.quantise(_np(x))
    assert _same(_np(ko), quant.dequantise(codes, scale)) and torch.equal(ko, vo)
