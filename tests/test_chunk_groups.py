"""Which sequences a ChunkPlan launches together, and its tables, without a GPU."""
import random
import struct

import pytest

from dllm_serve_amd import _capi
from dllm_serve_amd.layers.attention import ChunkPlan


def _plan(lens, cached):
    return ChunkPlan(lens, cached, [list(range(7, 7 + -(-n // 256))) for n in cached], "cpu", mask_block=1)


@pytest.mark.parametrize("lens,cached,groups", [
    ([], 0, []),
    ([0, 0], 300, [2]),
    ([5], 9, [1]),
    ([1] * 40, 3000, [40]),
    ([32] * 8, 3000, [8]),
    ([2048] + [1] * 31, 2000, [1, 31]),
    ([1] * 31 + [2048], 2000, [1, 31]),
    ([2048, 1], 2000, [2]),              # one short sequence is not worth a launch
    ([256, 1, 1], 2000, [1, 2]),
    ([256, 1, 1], 100, [3]),             # nor are few keys
    ([64] + [1] * 4, 2000, [5]),         # nor a few tokens beside a block
    ([64] + [1] * 8, 2000, [1, 8]),
    ([128] + [8] * 40, 2000, [41]),      # a sixteenth is not less than one
    ([130] + [8] * 40, 2000, [1, 40]),
    ([2048, 0, 100, 1, 1, 90] + [1] * 10, 1000, [1, 2, 13]),
    ([40, 0, 300, 1, 200, 260], 700, [6]),
    ([300, 0, 0, 0, 0], 2000, [5]),
])
def test_groups(lens, cached, groups):
    plan = _plan(lens, [cached] * len(lens))
    assert [g[1] for g in plan.groups] == groups
    at = 0
    for first, n, max_q, max_cached, total_q, total_cached in plan.groups:
        assert first == at
        at += n
    assert at == plan.n_seg == len(lens)


def test_every_sequence_is_in_one_group():
    rng = random.Random(3)
    for _ in range(200):
        lens = [int(2 ** rng.uniform(0, rng.choice([1, 5, 11]))) * rng.randint(0, 3) for _ in range(rng.randint(1, 60))]
        cached = [rng.randint(0, 3000) for _ in lens]
        plan = _plan(lens, cached)
        order = plan._tables[2 * plan.n_seg + 1:3 * plan.n_seg + 1].tolist()
        assert sorted(order) == list(range(len(lens)))
        assert (plan._seg_ids is None) == (order == sorted(order))
        assert plan.cached_lens.tolist() == [cached[b] for b in order]
        table = plan.block_tables.view(plan.n_seg, plan.max_pages).tolist() if plan.max_pages else [[]] * plan.n_seg
        for i, b in enumerate(order):
            need = -(-cached[b] // 256)
            assert table[i][:need] == list(range(7, 7 + need))
        for first, n, max_q, max_cached, total_q, total_cached in plan.groups:
            q, c = [lens[b] for b in order[first:first + n]], [cached[b] for b in order[first:first + n]]
            assert (max_q, max_cached, total_q, total_cached) == (max(q), max(c), sum(q), sum(c))
            # nothing far shorter is left in a group beside it
            short = [x for x in q if 0 < x * 16 < max_q]
            assert len(short) < 2 or len(short) * max_q * (max_q + max_cached) < 1 << 20
        packed = struct.unpack(f"={len(plan._packed) // 8}q", plan._packed)
        assert packed[2] == len(plan.groups) and packed[10:] == tuple(x for g in plan.groups for x in g)


def test_workspace_of_a_piece_among_tokens():
    """What the piece and the tokens need by themselves."""
    lens, cached = [2048] + [1] * 63, [131072] + [500] * 63
    for Hq, Hkv in ((32, 32), (28, 4)):
        need = [_capi.chunk_workspace_size(n, mq, mc, Hq, Hkv, 128, tq, tc) for _, n, mq, mc, tq, tc in _plan(lens, cached).groups]
        assert len(need) == 2 and max(need) < 64 << 20
