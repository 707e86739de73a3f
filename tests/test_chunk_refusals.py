"""What the 8-bit cache and the chunk attention refuse, without a GPU."""
import ctypes

import pytest
import torch

from dllm_serve_amd import _capi
from dllm_serve_amd.engine.kv_cache import quantized_pages
from dllm_serve_amd.layers.attention import ChunkPlan, chunk_attention, load_kvcache, store_kvcache

BF16 = torch.bfloat16
FAKE = ctypes.c_void_p(4096)
ODD = ctypes.c_void_p(4104)


def _err(rc):
    return rc, _capi.load().dllm_last_error().decode()


def _paged(**kw):
    a = dict(q=FAKE, k=FAKE, v=FAKE, o=FAKE, cu=FAKE, ids=None, n_seg=1, max_q=1, max_cached=64, tq=0, tc=0, kc=FAKE, vc=FAKE, kind=1,
             pages=4, table=FAKE, max_pages=1, lens=FAKE, mask=1, Hq=4, Hkv=2, D=128, qs=512, ks=256, vs=256, os=512,
             scale=0.1, ws=None, ws_bytes=0, stream=None)
    a.update(kw)
    return _err(_capi.load().dllm_attn_chunk_paged_fwd(*a.values()))


@pytest.mark.parametrize("change,code,text", [
    (dict(D=64), "UNSUPPORTED", "head_dim"),
    (dict(Hq=5), "INVALID_ARG", "multiple"),
    (dict(q=None), "INVALID_ARG", "null"),
    (dict(k=ODD), "INVALID_ARG", "aligned"),
    (dict(qs=516), "INVALID_ARG", "multiples of 8"),
    (dict(ks=128), "INVALID_ARG", "smaller"),
    (dict(n_seg=-1), "INVALID_ARG", "negative"),
    (dict(mask=-1), "INVALID_ARG", "negative"),
    (dict(tq=-1), "INVALID_ARG", "negative"),
    (dict(tc=-1), "INVALID_ARG", "negative"),
    (dict(n_seg=70000, max_pages=1, max_cached=0), "INVALID_ARG", "too large"),
    (dict(kind=2), "INVALID_ARG", "cache type"),
    (dict(scale=0.0), "INVALID_ARG", "softmax_scale"),
    (dict(scale=-1.0), "INVALID_ARG", "softmax_scale"),
    (dict(scale=float("nan")), "INVALID_ARG", "softmax_scale"),
    (dict(scale=float("inf")), "INVALID_ARG", "softmax_scale"),
    (dict(cu=None), "INVALID_ARG", "null"),
    (dict(lens=None), "INVALID_ARG", "null"),
    (dict(kc=None), "INVALID_ARG", "null cache"),
    (dict(table=None), "INVALID_ARG", "page table"),
    (dict(max_pages=0), "INVALID_ARG", "page table"),
    (dict(vc=ODD), "INVALID_ARG", "aligned"),
    (dict(pages=-1), "INVALID_ARG", "pages"),
    (dict(pages=(1 << 23) + 1), "INVALID_ARG", "pages"),
    (dict(n_seg=1 << 20, max_pages=1 << 12), "INVALID_ARG", "table"),
    (dict(max_q=1 << 30), "UNSUPPORTED", ""),
    (dict(max_cached=2**31 - 2), "UNSUPPORTED", ""),
    (dict(max_q=1 << 22), "UNSUPPORTED", "4 GiB"),
    (dict(max_cached=100000, max_pages=400), "WORKSPACE", "workspace"),
    (dict(max_cached=100000, max_pages=400, ws=ODD, ws_bytes=1 << 30), "INVALID_ARG", "aligned"),
])
def test_c_entry_refuses(change, code, text):
    rc, msg = _paged(**change)
    assert rc == getattr(_capi, "DLLM_ERR_" + code) and text in msg, (rc, msg)


def test_c_entry_with_nothing_to_do():
    assert _paged(n_seg=0)[0] == 0 and _paged(max_q=0)[0] == 0
    assert _capi.chunk_workspace_size(0, 1, 100000, 4, 2, 128) == 0
    assert _capi.chunk_workspace_size(1, 1, 100000, 5, 2, 128) == 0
    assert _capi.chunk_workspace_size(1, 1, 0, 4, 2, 128) == 0
    assert _capi.chunk_workspace_size(1, 1, 100000, 4, 2, 128) > 0
    with pytest.raises(RuntimeError, match="unsupported sizes"):
        _capi.chunk_launch_shape(1, 1, 10, 4, 2, 64)


def test_c_cache_entries_refuse():
    lib = _capi.load()
    for fn in (lib.dllm_store_kvcache_fp8, lib.dllm_load_kvcache_fp8):
        def call(k=FAKE, ks=256, v=FAKE, vs=256, kp=FAKE, vp=FAKE, pages=4, slots=FAKE, n=3, H=2, D=128):
            return _err(fn(k, ks, v, vs, kp, vp, pages, slots, n, H, D, None))
        assert call(D=64)[0] == _capi.DLLM_ERR_UNSUPPORTED
        assert call(n=-1)[0] == _capi.DLLM_ERR_INVALID_ARG
        assert call(H=0)[0] == _capi.DLLM_ERR_INVALID_ARG
        assert call(pages=(1 << 23) + 1)[0] == _capi.DLLM_ERR_INVALID_ARG
        assert call(ks=255)[0] == _capi.DLLM_ERR_INVALID_ARG
        assert call(kp=ODD)[0] == _capi.DLLM_ERR_INVALID_ARG
        assert call(slots=None)[0] == _capi.DLLM_ERR_INVALID_ARG
        assert call(n=2**31 - 1, H=2)[0] == _capi.DLLM_ERR_UNSUPPORTED
        assert call(n=0)[0] == 0 and call(pages=0)[0] == 0
    assert lib.dllm_quant_page_bytes(128) == _capi.PAGE_BYTES and lib.dllm_quant_page_bytes(64) == 0


def test_store_and_load_refuse():
    x = torch.zeros(4, 2, 128, dtype=BF16)
    kc, vc = quantized_pages(2, 2), quantized_pages(2, 2)
    slots = torch.zeros(4, dtype=torch.int32)
    for fn in (store_kvcache, load_kvcache):
        with pytest.raises(RuntimeError, match="GPU"):
            fn(x, x, kc, vc, slots)
        with pytest.raises(AssertionError):
            fn(x, x, kc, vc, slots[:3])
        with pytest.raises(AssertionError):
            fn(x.float(), x.float(), kc, vc, slots)
        with pytest.raises(AssertionError):
            fn(x, x[:3], kc, vc, slots)
        with pytest.raises(ValueError, match="pages of 3"):
            fn(x, x, quantized_pages(2, 3), quantized_pages(2, 3), slots)
        with pytest.raises(ValueError, match="v_cache"):
            fn(x, x, kc, torch.zeros(2, 256, 2, 128, dtype=BF16), slots)
        with pytest.raises(ValueError, match="k_cache"):
            fn(x, x, kc[:, :, :-256], vc, slots)
    with pytest.raises(ValueError, match="128"):
        quantized_pages(2, 2, 64)


def test_plan_refuses():
    ChunkPlan([1, 0], [256, 0], [[3], []], "cpu")
    ChunkPlan([1], [256], [[3, -1]], "cpu")  # pages past the cached rows are not read
    with pytest.raises(ValueError, match="block tables"):
        ChunkPlan([1, 1], [256], [[3], []], "cpu")
    with pytest.raises(ValueError, match="negative"):
        ChunkPlan([-1], [256], [[3]], "cpu")
    with pytest.raises(ValueError, match="negative"):
        ChunkPlan([1], [256], [[3]], "cpu", mask_block=-2)
    with pytest.raises(ValueError, match="2 pages"):
        ChunkPlan([1], [257], [[3]], "cpu")
    with pytest.raises(ValueError, match="pages"):
        ChunkPlan([1], [257], [[3, -1]], "cpu")
    with pytest.raises(ValueError, match="int32"):
        ChunkPlan([2**31], [0], [[]], "cpu")


def test_chunk_attention_refuses():
    q, k = torch.zeros(3, 4, 128, dtype=BF16), torch.zeros(3, 2, 128, dtype=BF16)
    kc = quantized_pages(2, 2)
    plan = ChunkPlan([3], [4], [[0]], "cpu")
    with pytest.raises(RuntimeError, match="GPU only"):
        chunk_attention(q, k, k, kc, kc, plan, 0.1)
    with pytest.raises(TypeError, match="bf16"):
        chunk_attention(q.float(), k, k, kc, kc, plan, 0.1)
    with pytest.raises(ValueError, match="heads"):
        chunk_attention(q[:, :3], k, k, kc, kc, plan, 0.1)
    with pytest.raises(ValueError, match="must be"):
        chunk_attention(torch.zeros(3, 4, 64, dtype=BF16), k, k, kc, kc, plan, 0.1)
    with pytest.raises(ValueError, match="contiguous heads"):
        chunk_attention(q.transpose(0, 1).contiguous().transpose(0, 1), k, k, kc, kc, plan, 0.1)


def test_quantising_selection_refuses():
    lib = _capi.load()

    def call(pages=4, kp=FAKE, ws=FAKE, ws_bytes=1 << 30, D=128):
        return _err(lib.dllm_select_kv_store_fp8(FAKE, FAKE, FAKE, 300, 512, 256, 256, FAKE, 1, 268, 100, 4, 2, D, 11.3,
                                                 kp, FAKE, pages, FAKE, 100, None, ws, ws_bytes, None))
    assert call(D=64)[0] == _capi.DLLM_ERR_UNSUPPORTED
    assert call(pages=-1)[0] == _capi.DLLM_ERR_INVALID_ARG
    assert call(pages=(1 << 23) + 1)[0] == _capi.DLLM_ERR_INVALID_ARG
    assert call(kp=ODD)[0] == _capi.DLLM_ERR_INVALID_ARG
    assert call(kp=None)[0] == _capi.DLLM_ERR_INVALID_ARG
    assert call(ws_bytes=16)[0] == _capi.DLLM_ERR_WORKSPACE
