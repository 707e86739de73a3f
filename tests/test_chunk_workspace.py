"""The workspace of the chunk attention stays bounded for batches that mix long and short
sequences: from the sizes alone, no GPU."""
import random

import pytest

from dllm_serve_amd import _capi

GIB = 1 << 30


def _sizes(lens, cached, Hq, Hkv, totals=True):
    a = (len(lens), max(lens), max(cached), Hq, Hkv, 128) + ((sum(lens), sum(cached)) if totals else ())
    return _capi.chunk_workspace_size(*a), _capi.chunk_launch_shape(*a)


@pytest.mark.parametrize("Hq,Hkv", [(32, 32), (28, 4)])
@pytest.mark.parametrize("totals", [True, False])
@pytest.mark.parametrize("lens,cached", [
    # a piece of a long prompt among single tokens
    ([2048] + [1] * 63, [131072] + [500] * 63),
    ([512] + [1] * 31, [30000] + [500] * 31),
    # one long sequence among very many single tokens, and among blocks
    ([1] * 4096, [131072] + [1000] * 4095),
    ([32] * 1024, [131072] + [1000] * 1023),
    ([1] * 60000, [200] * 60000),
])
def test_mixed_batches(lens, cached, Hq, Hkv, totals):
    ws, shape = _sizes(lens, cached, Hq, Hkv, totals)
    assert ws <= GIB and shape["grid"] > 0
    parts = ws // (shape["rows"] * 130 * 4)
    assert parts <= shape["grid"] and (ws > 0) == (shape["n_split"] > 1)


def test_batches_that_fit_are_launched_at_once():
    for lens, cached in (([1] * 256, [131072] + [1000] * 255), ([32] * 2, [5000] * 2)):
        ws, shape = _sizes(lens, cached, 28, 4)
        assert shape["n_split"] > 1
        rows = -(-max(lens) * 7 // shape["rows"]) * shape["rows"]
        assert ws == len(lens) * 4 * rows * shape["n_split"] * 130 * 4


def test_any_sizes():
    rng = random.Random(5)
    for _ in range(3000):
        n, Hkv = int(2 ** rng.uniform(0, 15)), rng.choice([1, 2, 4, 8, 32])
        L, C = int(2 ** rng.uniform(0, 13)), int(2 ** rng.uniform(0, 20))
        g = rng.choice([1, 2, 7, 8])
        tq, tc = rng.choice([(0, 0), (rng.randint(L, n * L), rng.randint(C, n * C))])
        a = (n, L, C, g * Hkv, Hkv, 128, tq, tc)
        ws, shape = _capi.chunk_workspace_size(*a), _capi.chunk_launch_shape(*a)
        # parts of a segment's rows where the longest split that the kernel takes sets them
        least = -(-C // 15872) * Hkv * -(-L * g // shape["rows"]) * shape["rows"] * 520
        assert ws <= max(GIB, least if shape["rows"] < 128 else 0), a
        assert 0 < shape["grid"] <= (1 << 22) + 32
        if shape["rows"] < 128:
            assert -(-C // shape["n_split"]) <= 15872
