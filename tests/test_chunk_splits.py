"""How the chunk attention's keys are dealt to workgroups: nearly equal batches get nearly the
same parts.  From the sizes alone, no GPU."""
import random

import pytest

from dllm_serve_amd import _capi


def _parts(lens, cached, Hq, Hkv):
    return _capi.chunk_launch_shape(len(lens), max(lens), max(cached), Hq, Hkv, 128, sum(lens), sum(cached))["n_split"]


@pytest.mark.parametrize("lens,cached,Hq,Hkv", [
    ([1] * 8, 1000, 28, 4), ([4] * 2, 900, 28, 4), ([1], 1000, 32, 32), ([1] * 2, 2000, 32, 32), ([1] * 32, 2000, 28, 4),
    ([1] * 16, 4000, 28, 4), ([32] * 3, 1000, 28, 4), ([1] * 40, 3000, 28, 4), ([1] * 5, 3565, 32, 32), ([8] * 8, 3000, 28, 4),
])
def test_a_row_less_is_at_most_a_part_more_or_less(lens, cached, Hq, Hkv):
    n = len(lens)
    equal = _parts(lens, [cached] * n, Hq, Hkv)
    for less in (1, 2, 31, cached // 20):
        assert abs(_parts(lens, [cached] * (n - 1) + [cached - less] if n > 1 else [cached - less], Hq, Hkv) - equal) <= 1
    # the same total without the longest sequence: given by a caller that knows no more
    total = sum([cached] * n) - 1
    shape = _capi.chunk_launch_shape(n, max(lens), cached, Hq, Hkv, 128, sum(lens), total)
    assert abs(shape["n_split"] - equal) <= 1


def test_the_parts_change_step_by_step():
    """One cached row less at a time, from equal lengths down to a single long sequence: the parts
    of the longest one change by a step of what rounding them to four tiles makes."""
    rng = random.Random(9)
    for _ in range(60):
        n, L, Hkv = rng.randint(2, 40), rng.choice([1, 1, 1, 4, 32]), rng.choice([4, 8, 32])
        g, top = rng.choice([1, 7]), int(2 ** rng.uniform(9, 14))
        tiles = -(-top // 32)
        last = None
        for total in range(n * top, top, -max(1, n * top // 4000)):
            p = _capi.chunk_launch_shape(n, L, top, g * Hkv, Hkv, 128, n * L, total)
            if p["rows"] == 128:
                break
            # part lengths, rounded to four tiles, from the parts: a range
            lo, hi = -(-tiles // p["n_split"]), tiles // max(1, p["n_split"] - 1) if p["n_split"] > 1 else 10**9
            if last is not None and not (p["n_split"] == 1 or last[2] == 1):
                assert lo <= last[1] + 8 + last[1] // 8 and last[0] <= hi + 8 + hi // 8, (n, L, g, Hkv, top, total, p, last)
            last = lo, hi, p["n_split"]
