"""What a step's plan does with the sequences' pages, without a GPU."""
import pytest
import torch

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


def test_page_tables_refuse():
    seqs = _reuse_step()
    plan = StepPlan(get_context(), CPU)
    seqs[2].block_table = list(seqs[2].block_table)[:2]
    with pytest.raises(ValueError, match="rows in 2 pages"):
        plan.page_tables()
    del seqs[1].block_table
    with pytest.raises(ValueError, match="block tables"):
        plan.page_tables()
    reset_context()
