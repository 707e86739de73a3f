"""Sizes that one call of the 8-bit cache copies cannot launch are refused before they are tried."""
import ctypes

import pytest

from dllm_serve_amd import _capi

FAKE = ctypes.c_void_p(4096)


@pytest.mark.parametrize("n,H", [(1 << 28, 1), (1 << 23, 32), ((1 << 28) - 128, 1), (1 << 29, 2), (2**31 - 1, 1)])
def test_more_rows_than_a_launch_has_threads(n, H):
    lib = _capi.load()
    for fn in (lib.dllm_store_kvcache_fp8, lib.dllm_load_kvcache_fp8):
        rc = fn(FAKE, 128 * H, FAKE, 128 * H, FAKE, FAKE, 4, FAKE, n, H, 128, None)
        assert rc == _capi.DLLM_ERR_UNSUPPORTED and b"in one call" in lib.dllm_last_error()
