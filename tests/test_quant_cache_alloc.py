"""Sizing and binding of the cache in 8-bit pages, on the CPU."""
import pytest
import torch
from torch import nn

from dllm_serve_amd.engine.kv_cache import allocate_kv_cache, block_bytes, kv_cache_blocks
from dllm_serve_amd.layers.attention import Attention


def test_sizes():
    """33024 bytes a page and KV head against 65536 in bf16."""
    assert block_bytes(32, 32, 128, quantized=True) == 2 * 32 * 32 * 33024
    assert block_bytes(28, 4, 128, world_size=2, quantized=True) == 2 * 28 * 2 * 33024
    GiB = 1 << 30
    plain, quant = (kv_cache_blocks(288 * GiB, 0, 0, 0, 0.9, 32, 32, 128, quantized=b) for b in (False, True))
    assert plain < quant <= 2 * plain


def test_binding():
    m = nn.ModuleList([Attention(8, 128, 128 ** -0.5, 4, causal=False) for _ in range(2)])
    cache = allocate_kv_cache(m, 2, 4, 128, device="cpu", num_blocks=3, quantized=True)
    assert cache.shape == (2, 2, 3, 4, 33024) and cache.dtype == torch.uint8 and int(cache.sum()) == 0
    for i, a in enumerate(m):
        assert a.k_cache.shape == (3, 4, 33024) and a.k_cache.data_ptr() == cache[0, i].data_ptr()
        assert a.v_cache.data_ptr() == cache[1, i].data_ptr()
    with pytest.raises(ValueError, match="128"):
        allocate_kv_cache(nn.Module(), 2, 4, 64, device="cpu", num_blocks=3, quantized=True)
