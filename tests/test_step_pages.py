"""What a step's plan does with the sequences' pages, without a GPU."""
import pytest
import torch

from dllm_serve_amd import _capi
from dllm_serve_amd.engine.sequence import PageAllocator, Sequence, prepare_step
from dllm_serve_amd.layers.attention import StepPlan
from dllm_serve_amd.sparse.state import SparseConfig
from dllm_serve_amd.utils.context import get_context, reset_context

CPU = torch.device("cpu")


class _Pages(list):
    """A block table that counts how often it is read as a whole."""
    reads = 0

    def __iter__(self):
        self.reads += 1
        return super().__iter__()

    def __getitem__(self, i):
        self.reads += isinstance(i, slice)
        return super().__getitem__(i)


def _reuse_step(prompts=(200, 400, 900)):
    cfg = SparseConfig(enabled=True, default_block_len=32, retention_ratio=0.9, pool_kernel=3, delay_step=1,
                       head_select=True)
    seqs = [Sequence([1] * n, 64, 126336, cfg, device="cpu") for n in prompts]
    alloc = PageAllocator([5, 2, 7, 0, 3, 9, 4, 1, 6, 8])
    for s in reversed(seqs):
        s.block_table = _Pages()
        alloc.allocate(s)
        s.advance()
        s.advance()
    prepare_step(seqs, "cpu")
    for s in seqs:
        s.block_table.reads = 0
    return seqs


def test_a_plan_without_8_bit_pages_leaves_the_block_tables_alone():
    seqs = _reuse_step()
    plan = StepPlan(get_context(), CPU)
    assert plan.n_cached == 3 and all(s.block_table.reads == 0 for s in seqs)
    reset_context()


def test_page_tables():
    seqs = _reuse_step()
    plan = StepPlan(get_context(), CPU)
    table, lens = plan.page_tables()
    assert lens.tolist() == [s.current_sparse_token for s in seqs]
    for s, row in zip(seqs, table.tolist()):
        need = -(-s.current_sparse_token // 256)
        assert row[:need] == list(s.block_table)[:need]
    again = plan.page_tables()
    assert again[0] is table and again[1] is lens
    reset_context()


def test_page_tables_refuse_too_few_pages():
    seqs = _reuse_step()
    plan = StepPlan(get_context(), CPU)
    seqs[2].block_table = list(seqs[2].block_table)[:2]
    with pytest.raises(ValueError, match="rows in 2 pages"):
        plan.page_tables()
    reset_context()


def test_pages_are_those_of_the_slot_mapping():
    """Other pages than the block table's, rows of a page in another order, no block table."""
    seqs = _reuse_step()
    ctx = get_context()
    rows = [s.current_sparse_token for s in seqs]
    pages = [[20, 11], [12, 30], [14, 13, 21, 40]]
    want = [p[:-(-n // 256)] for p, n in zip(pages, rows)]
    maps = [[p[r // 256] * 256 + r % 256 for r in range(n)] for p, n in zip(pages, rows)]
    maps[1] = torch.tensor(maps[1], dtype=torch.int32)
    maps[2][:256] = maps[2][:256][::-1]
    del seqs[0].block_table
    ctx.slot_mapping = maps
    table, lens = StepPlan(ctx, CPU).page_tables()
    assert lens.tolist() == rows
    assert [row[:len(w)] for row, w in zip(table.tolist(), want)] == want
    reset_context()


@pytest.mark.parametrize("change", ["starts in a page", "gap", "two pages", "row twice", "outside"])
def test_mappings_that_pages_cannot_be_read_by(change):
    seqs = _reuse_step((400,))
    ctx = get_context()
    n = seqs[0].current_sparse_token
    assert 256 < n < 500
    m = [5 * 256 + r if r < 256 else 7 * 256 + r - 256 for r in range(n)]
    if change == "starts in a page":
        m = [x + 1 for x in m]
    elif change == "gap":
        m[-1] += 1
    elif change == "two pages":
        m[10], m[300] = m[300], m[10]
    elif change == "row twice":
        m[10] = m[11]
    else:
        m[0] = -1
    ctx.slot_mapping = [m]
    with pytest.raises(ValueError, match="one cache page"):
        StepPlan(ctx, CPU).page_tables()
    reset_context()


def test_a_plan_of_device_tables_needs_block_tables():
    seqs = _reuse_step()
    plan = StepPlan(get_context(), CPU)
    plan._cached_seqs = None  # as StepPlan.from_device leaves it
    with pytest.raises(ValueError, match="block tables"):
        plan.page_tables()
    reset_context()


def test_workspace_of_the_attention_that_runs():
    """Over 8-bit pages the other attention's workspace is not allocated."""
    _reuse_step((200, 400, 1500))
    plan = StepPlan(get_context(), CPU)
    sizes = {p: _capi.chunk_workspace_size(3, plan.max_q_cached, plan.max_keep_cached, 2, 2, 128, plan.rows_cached,
                                           plan.keeps_cached)
             if p else _capi.block_cached_workspace_size(3, plan.max_q_cached, plan.max_keys_cached, 2, 2, 128)
             for p in (True, False)}
    assert sizes[True] > 0 and sizes[False] > 0
    a = plan.launch_args(2, 2, 128, True)
    assert a["ws_bytes"] == sizes[True] and a is plan.launch_args(2, 2, 128, True)
    assert [t.numel() for t in plan._ws.values()] == [sizes[True]]
    assert plan.launch_args(2, 2, 128)["ws_bytes"] == sizes[False]
    assert sorted(t.numel() for t in plan._ws.values()) == sorted(sizes.values())
    assert plan.launch_args(2, 2, 128, True) is a
    reset_context()
