"""chunk_attention against the formula in 64 bits, at the lengths, masks and layouts
where it can go wrong.

The bound of an output, from the roundings the kernels make: the result in bf16 (2^-8
of it), every probability in bf16 (2^-8, in the numerator and in the row sum alike:
2^-8 * sum p |v - o|), the scores in f32 (relative change of a probability at most
twice the error of its score, which is 140 roundings of 2^-23 of sum |q k| and the
exponential's 2^-20), and the f32 sums over the keys."""
import numpy as np
import pytest
import torch

from oracle import chunk, quant
from dllm_serve_amd import _capi
from dllm_serve_amd.engine.kv_cache import quantized_pages
from dllm_serve_amd.layers.attention import ChunkPlan, chunk_attention, load_kvcache, store_kvcache

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
SCALE = 128 ** -0.5


def _np(t):
    return t.detach().double().cpu().numpy()


def check(out, ref, spread, reach, keys, what=""):
    o = _np(out).reshape(ref.shape)
    assert np.array_equal(np.isnan(o), np.isnan(ref)), what
    ok = np.isfinite(ref)
    assert np.array_equal(o[~ok & ~np.isnan(ref)], ref[~ok & ~np.isnan(ref)]), what
    with np.errstate(invalid="ignore"):
        p = 2.0 ** -8 + 2 * (140 * 2.0 ** -23 * reach[..., None] + 2.0 ** -20)
        tol = 2.0 ** -8 * np.abs(ref) + 1.05 * p * (spread + np.abs(ref)) + (keys / 16 + 40) * 2.0 ** -23 * spread + 1e-30
        bad = np.abs(o - ref) > tol
    assert not (bad & ok).any(), f"{what}: worst {np.nanmax(np.where(ok, np.abs(o - ref) / tol, 0)):.2f} of the bound"


class Batch:
    """New rows, a paged cache of the wanted kind and the cached rows as float64."""

    def __init__(self, dev, lens, cached, Hq, Hkv, bits, seed=0, spare=2, kv_scale=1.0):
        g = torch.Generator().manual_seed(seed)
        self.dev, self.lens, self.cached, self.Hkv, self.bits = dev, lens, cached, Hkv, bits
        n = sum(lens)

        def normal(*s):
            return (kv_scale * torch.randn(*s, generator=g)).to(BF16)

        self.q, self.k, self.v = normal(n, Hq, 128), normal(n, Hkv, 128), normal(n, Hkv, 128)
        need = [-(-c // 256) for c in cached]
        self.pages = sum(need) + spare
        perm = torch.randperm(self.pages, generator=g).tolist()
        self.tables = [perm[sum(need[:b]):sum(need[:b + 1])] for b in range(len(lens))]
        rows = self.pages * 256
        if bits == 8:
            self.kc, self.vc = quantized_pages(self.pages, Hkv, device=dev), quantized_pages(self.pages, Hkv, device=dev)
            slots = torch.arange(rows, dtype=torch.int32, device=dev)
            store_kvcache(normal(rows, Hkv, 128).to(dev), normal(rows, Hkv, 128).to(dev), self.kc, self.vc, slots)
        else:
            self.kc = normal(self.pages, 256, Hkv, 128).to(dev)
            self.vc = normal(self.pages, 256, Hkv, 128).to(dev)

    def slots(self, b):
        r = np.arange(self.cached[b])
        return np.array(self.tables[b] or [0])[r // 256] * 256 + r % 256

    def cache_rows(self, pages, b):
        s = self.slots(b)
        if self.bits == 8:
            return quant.load(pages.cpu().numpy(), s)
        return _np(pages.view(-1, self.Hkv, 128))[s]

    def run(self, mask_block=0, scale=SCALE):
        plan = ChunkPlan(self.lens, self.cached, self.tables, self.dev, mask_block=mask_block)
        d = self.dev
        return chunk_attention(self.q.to(d), self.k.to(d), self.v.to(d), self.kc, self.vc, plan, scale)

    def verify(self, out, mask_block=0, scale=SCALE, keep=None):
        r0 = 0
        for b, L in enumerate(self.lens):
            x = [_np(t[r0:r0 + L]) for t in (self.q, self.k, self.v)]
            kc, vc = self.cache_rows(self.kc, b), self.cache_rows(self.vc, b)
            ref, spread, reach = chunk.attend(*x, kc, vc, scale, mask_block, None if keep is None else keep[b])
            check(out[r0:r0 + L], ref, spread, reach, L + self.cached[b], f"sequence {b}")
            r0 += L


SHAPES = [
    # lens, cached, Hq, Hkv, mask_block
    ([1], [0], 2, 2, 1),
    ([1], [1], 2, 2, 1),
    ([1, 1, 1], [31, 32, 33], 4, 2, 1),
    ([1, 1], [255, 257], 7, 1, 0),
    ([1], [1500], 7, 1, 1),
    ([2, 3], [64, 700], 2, 1, 1),
    ([16, 17], [5, 300], 2, 2, 0),
    ([32, 5, 33], [129, 0, 256], 4, 2, 4),
    ([0, 7, 0, 40], [300, 13, 0, 100], 4, 4, 1),
    ([65], [90], 7, 1, 32),
    ([130, 9], [40, 512], 2, 1, 1),
    ([300], [0], 2, 2, 1),
    ([129], [77], 3, 1, 33),
    ([260, 70], [511, 0], 4, 4, 0),
    ([100, 20], [1500, 0], 2, 1, 1),   # many rows, keys split, a short sequence beside a long one
    ([520], [700], 2, 1, 16),          # the new rows' own tiles are split as well
    # more than 1024 rows of a KV head: tiles of 128 rows
    ([65], [90], 16, 1, 32),
    ([70, 9, 0], [40, 512, 3], 16, 1, 1),
    ([65, 1, 80], [700, 0, 1500], 16, 1, 1),
    ([300], [0], 4, 1, 0),
    ([130], [64], 14, 1, 5),
    ([66], [4200], 16, 1, 1),
    # parts of a row joined in several rounds
    ([1], [33000], 2, 1, 1),
    # one block of 17 to 32 rows, whole and in parts
    ([17], [500], 2, 2, 1),
    ([8, 6], [2000, 1500], 4, 1, 4),
]


def _forms(n):
    """Query heads per KV head with which n new rows take the rows form, and the tile form."""
    return 2, -(-1032 // n)


def test_the_shapes_take_both_forms():
    rows = {_capi.chunk_launch_shape(len(a), max(a), max(b), Hq, Hkv, 128, sum(a), sum(b))["rows"]
            for a, b, Hq, Hkv, _ in SHAPES}
    assert rows == {16, 32, 128}
    shape = _capi.chunk_launch_shape(3, 80, 1500, 16, 1, 128, 146, 2200)
    assert shape["rows"] == 128 and shape["n_split"] > 1


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("lens,cached,Hq,Hkv,mask_block", SHAPES)
def test_against_the_formula(dev, lens, cached, Hq, Hkv, mask_block, bits):
    b = Batch(dev, lens, cached, Hq, Hkv, bits, seed=len(lens) + sum(lens) + sum(cached))
    b.verify(b.run(mask_block), mask_block)


@pytest.mark.parametrize("bits", [8, 16])
def test_one_token_of_a_long_cache_is_split(dev, bits):
    shape = _capi.chunk_launch_shape(1, 1, 9000, 7, 1, 128)
    assert shape["n_split"] > 8
    b = Batch(dev, [1], [9000], 7, 1, bits, seed=3)
    b.verify(b.run(1), 1)


@pytest.mark.parametrize("bits", [8, 16])
def test_ragged_batch_whose_short_sequences_leave_splits_empty(dev, bits):
    b = Batch(dev, [1, 1, 2], [3000, 0, 40], 4, 2, bits, seed=4)
    b.verify(b.run(1), 1)


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("g", _forms(70))
def test_large_scores(dev, bits, g):
    """Scores of hundreds: the maximum moves, most probabilities vanish."""
    b = Batch(dev, [70, 1], [300, 600], g, 1, bits, seed=5, kv_scale=4.0)
    b.verify(b.run(1, scale=0.5), 1, scale=0.5)


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("cached", [70, 600])
@pytest.mark.parametrize("L,g", [(5, 1), (40, 1), (140, 1), (70, 15), (130, 9)])
def test_nan_and_infinity_reach_only_the_rows_that_see_them(dev, bits, L, g, cached):
    b = Batch(dev, [L], [cached], 2 * g, 2, bits, seed=6)
    b.v[L - 1, 0, 3] = float("nan")
    b.v[L - 2, 1, 9] = float("inf")
    b.k[L - 1, 1, 0] = float("nan")
    b.k[L - 2, 0, :] = float("inf")
    out = b.run(1)
    ref_rows = slice(0, L - 2)
    assert torch.isfinite(out[ref_rows]).all()
    x = [_np(t) for t in (b.q, b.k, b.v)]
    ref, spread, reach = chunk.attend(*x, b.cache_rows(b.kc, 0), b.cache_rows(b.vc, 0), SCALE, 1)
    check(out[ref_rows], ref[ref_rows], spread[ref_rows], reach[ref_rows], L + cached)
    o = _np(out).reshape(ref.shape)
    assert np.isnan(o[L - 1]).all(axis=-1)[g:].all()   # a NaN score
    assert (o[L - 2, g:, 9] == np.inf).all() and np.isnan(o[L - 1, g:, 9]).all()


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("g", _forms(20))
def test_stale_rows_behind_the_cached_length(dev, bits, g):
    """The rest of the last page holds NaN: it takes no part."""
    b = Batch(dev, [1, 20], [40, 300], 2 * g, 2, bits, seed=7)
    want = [b.run(m) for m in (0, 1)]
    for s, c in enumerate(b.cached):
        page, row = b.tables[s][-1], c % 256
        for t in (b.kc, b.vc):
            if bits == 8:
                t[page, :, row * 128:256 * 128] = 0x7F
                t[page, :, 256 * 128 + row:] = 255
            else:
                t[page, row:] = float("nan")
    assert all(torch.equal(b.run(m), w) for m, w in zip((0, 1), want))


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("g", _forms(20))
def test_pages_outside_the_cache_are_left_out(dev, bits, g):
    b = Batch(dev, [20, 1], [600, 520], g, 1, bits, seed=8)
    plan = ChunkPlan(b.lens, b.cached, b.tables, dev, mask_block=1)
    # a table that lost a page after the plan was made, as a runner's bug would
    t = plan.block_tables.view(2, plan.max_pages)
    t[0, 1] = -1
    t[1, 0] = b.pages
    t[1, 2] = 2**31 - 1
    out = chunk_attention(b.q.to(dev), b.k.to(dev), b.v.to(dev), b.kc, b.vc, plan, SCALE)
    keep = [np.ones(600, bool), np.zeros(520, bool)]
    keep[0][256:512] = False
    keep[1][256:512] = True
    b.verify(out, 1, keep=keep)


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("g", _forms(33))
def test_empty_cache_and_no_sequences(dev, bits, g):
    b = Batch(dev, [5, 33], [0, 0], 2 * g, 2, bits, seed=9, spare=0)
    assert b.kc.shape[0] == 0
    b.verify(b.run(1), 1)
    b = Batch(dev, [], [], 2, 2, bits, seed=9)
    assert b.run(1).shape == (0, 256)


@pytest.mark.parametrize("bits", [8, 16])
def test_layouts(dev, bits):
    """Column slices of one fused projection, two- and three-dimensional."""
    b = Batch(dev, [9, 50], [100, 3], 4, 2, bits, seed=10)
    want = b.run(1)
    fused = torch.cat([b.q.flatten(1), b.k.flatten(1), b.v.flatten(1), torch.zeros(59, 8, dtype=BF16)], 1).to(dev)
    q, k, v = fused[:, :512], fused[:, 512:768], fused[:, 768:1024]
    plan = ChunkPlan(b.lens, b.cached, b.tables, dev, mask_block=1)
    assert torch.equal(chunk_attention(q, k, v, b.kc, b.vc, plan, SCALE), want)
    assert torch.equal(chunk_attention(q.view(59, 4, 128), k.view(59, 2, 128), v, b.kc, b.vc, plan, SCALE), want)


def test_rows_outside_the_segments_stay(dev):
    """The C entry point writes the segments' rows only."""
    b = Batch(dev, [3, 4], [10, 300], 2, 2, 8, seed=11)
    plan = ChunkPlan(b.lens, b.cached, b.tables, dev, mask_block=1)
    o = torch.full((9, 256), 3.0, dtype=BF16, device=dev)
    ws = torch.empty(max(1, _capi.chunk_workspace_size(2, 4, 300, 2, 2, 128)), dtype=torch.uint8, device=dev)
    q, k, v = (torch.cat([t, t[:2]]).to(dev) for t in (b.q, b.k, b.v))
    cu, lens, tables = plan._args
    _capi.attn_chunk_paged_fwd_raw(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), cu, None, 2, 4, 300,
                                   7, 310, b.kc.data_ptr(), b.vc.data_ptr(), _capi.CACHE_FP8, b.pages, tables, plan.max_pages,
                                   lens, 1, 2, 2, 128, 256, 256, 256, 256, SCALE, ws.data_ptr(), ws.numel(),
                                   _capi._stream(dev))
    assert (o[7:] == 3).all()
    b.verify(o[:7], 1)


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("lens,cached", [([1, 1, 9], [700, 40, 5]), ([32, 3, 8], [300, 9, 0]), ([150, 2, 70], [600, 8, 20])])
def test_some_sequences_of_a_packed_batch(dev, bits, lens, cached):
    """Segment ids: the sequences of a launch in another order, one of them not in it."""
    b = Batch(dev, lens, cached, 4, 2, bits, seed=12)
    ids = [2, 0]
    plan = ChunkPlan([lens[i] for i in ids], [cached[i] for i in ids], [b.tables[i] for i in ids], dev)
    cu = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device=dev)
    seg = torch.tensor(ids, dtype=torch.int32, device=dev)
    q, k, v = b.q.to(dev), b.k.to(dev), b.v.to(dev)
    o = torch.full_like(q, 5.0)
    ws = torch.empty(max(16, _capi.chunk_workspace_size(2, plan.max_q, plan.max_cached, 4, 2, 128)), dtype=torch.uint8,
                     device=dev)
    kind = _capi.CACHE_FP8 if bits == 8 else _capi.CACHE_BF16
    _, n, tables = plan._args
    _capi.attn_chunk_paged_fwd_raw(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), cu.data_ptr(), seg.data_ptr(),
                                   2, plan.max_q, plan.max_cached, 0, 0, b.kc.data_ptr(), b.vc.data_ptr(), kind, b.pages,
                                   tables, plan.max_pages, n, 0, 4, 2, 128, 512, 256, 256, 512, SCALE, ws.data_ptr(),
                                   ws.numel(), _capi._stream(dev))
    assert (o[lens[0]:lens[0] + lens[1]] == 5).all()
    o[lens[0]:lens[0] + lens[1]] = b.run(0).view(-1, 4, 128)[lens[0]:lens[0] + lens[1]]
    b.verify(o, 0)


@pytest.mark.parametrize("bits", [8, 16])
def test_native_and_python_calls_agree(dev, bits, monkeypatch):
    b = Batch(dev, [1, 30], [2500, 90], 14, 2, bits, seed=17)
    want = b.run(1)
    pages = quantized_pages(1, 2, device=dev), quantized_pages(1, 2, device=dev)
    slots = torch.arange(31, dtype=torch.int32, device=dev)
    store_kvcache(b.k.to(dev), b.v.to(dev), *pages, slots)
    back = [torch.empty_like(b.k, device=dev) for _ in range(2)]
    load_kvcache(*back, *pages, slots)
    monkeypatch.setattr(_capi, "native", None)
    assert torch.equal(b.run(1), want)
    again = quantized_pages(1, 2, device=dev), quantized_pages(1, 2, device=dev)
    store_kvcache(b.k.to(dev), b.v.to(dev), *again, slots)
    assert all(torch.equal(x, y) for x, y in zip(pages, again))
    out = [torch.empty_like(b.k, device=dev) for _ in range(2)]
    load_kvcache(*out, *pages, slots)
    assert all(torch.equal(x, y) for x, y in zip(back, out))


@pytest.mark.parametrize("bits", [8, 16])
def test_captured_graph_replays(dev, bits):
    """Captured and replayed, with eager calls of the same plan between the replays."""
    b = Batch(dev, [1, 1], [2500, 900], 7, 1, bits, seed=13)
    plan = ChunkPlan(b.lens, b.cached, b.tables, dev, mask_block=1)
    q, k, v = b.q.to(dev), b.k.to(dev), b.v.to(dev)
    want = chunk_attention(q, k, v, b.kc, b.vc, plan, SCALE)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(chunk_attention(q, k, v, b.kc, b.vc, plan, SCALE))
        graphs.append(gr)
    for i in range(4):
        outs[i % 2].zero_()
        graphs[i % 2].replay()
        assert torch.equal(chunk_attention(q, k, v, b.kc, b.vc, plan, SCALE), want)
        torch.cuda.synchronize()
        assert torch.equal(outs[i % 2], want)
    q2 = torch.flip(q, [0]).contiguous()
    q.copy_(q2)
    graphs[0].replay()
    assert torch.equal(outs[0], chunk_attention(q, k, v, b.kc, b.vc, plan, SCALE))


def test_two_streams_at_once(dev):
    b = Batch(dev, [1], [6000], 7, 1, 8, seed=14)
    plan = ChunkPlan(b.lens, b.cached, b.tables, dev, mask_block=1)
    q, k, v = b.q.to(dev), b.k.to(dev), b.v.to(dev)
    want = chunk_attention(q, k, v, b.kc, b.vc, plan, SCALE)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(20):
        for s, o in zip(streams, outs):
            with torch.cuda.stream(s):
                o.append(chunk_attention(q, k, v, b.kc, b.vc, plan, SCALE))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for o in outs for x in o)


def test_same_inputs_same_bits(dev):
    b = Batch(dev, [1, 30, 200], [4000, 600, 90], 4, 2, 8, seed=15)
    first = b.run(1)
    assert all(torch.equal(b.run(1), first) for _ in range(3))


@pytest.mark.parametrize("mask_block", [1, 8])
def test_a_prompt_in_chunks_is_the_prompt_at_once(dev, mask_block):
    """Prefill in chunks, each stored (8-bit) and attended over the pages, then single tokens:
    every step against the formula over the rows as the cache holds them."""
    Hq, Hkv, D, total = 4, 2, 128, 330
    g = torch.Generator().manual_seed(16)
    q, k, v = (torch.randn(total, h, D, generator=g).to(BF16) for h in (Hq, Hkv, Hkv))
    kc, vc = quantized_pages(3, Hkv, device=dev), quantized_pages(3, Hkv, device=dev)
    table, at = [2, 0], 0
    for L in (96, 120, 104, 1, 8, 1):
        x = [t[at:at + L].to(dev) for t in (q, k, v)]
        plan = ChunkPlan([L], [at], [table], dev, mask_block=mask_block)
        pos = torch.arange(at, at + L)
        slots = (torch.tensor(table)[pos // 256] * 256 + pos % 256).to(torch.int32).to(dev)
        store_kvcache(x[1], x[2], kc, vc, slots)
        out = chunk_attention(*x, kc, vc, plan, SCALE)
        held = [_np(t[:at]) for t in (k, v)]
        held = [quant.dequantise(*quant.quantise(t)) if at else t for t in held]
        ref = chunk.attend(*[_np(t[at:at + L]) for t in (q, k, v)], *held, SCALE, mask_block)
        check(out, *ref, at + L, f"chunk at {at}")
        at += L
    ko, vo = torch.empty(at, Hkv, D, dtype=BF16, device=dev), torch.empty(at, Hkv, D, dtype=BF16, device=dev)
    pos = torch.arange(at)
    load_kvcache(ko, vo, kc, vc, (torch.tensor(table)[pos // 256] * 256 + pos % 256).to(torch.int32).to(dev))
    assert np.array_equal(_np(ko), quant.dequantise(*quant.quantise(_np(k[:at]))))
    assert np.array_equal(_np(vo), quant.dequantise(*quant.quantise(_np(v[:at]))))


@pytest.mark.parametrize("bits", [8, 16])
def test_pieces_are_launched_longest_first(dev, bits, monkeypatch):
    """512 rows and more: the sequences in another order, here over several turns of the
    order of the M tiles, both sides of the native call, from a graph as well."""
    b = Batch(dev, [40, 0, 300, 1, 200, 260], [10, 5, 0, 520, 700, 30], 48, 48, bits, seed=21)
    plan = ChunkPlan(b.lens, b.cached, b.tables, dev, mask_block=1)
    assert plan._seg_ids is not None and plan.cached_lens.tolist() == [700, 520, 0, 30, 10, 5]
    shape = _capi.chunk_launch_shape(6, plan.max_q, plan.max_cached, 48, 48, 128, plan.total_rows, plan.total_cached)
    assert shape["rows"] == 128 and shape["n_split"] == 1 and shape["grid"] > 512
    want = b.run(1)
    b.verify(want, 1)
    b.verify(b.run(0), 0)
    q, k, v = b.q.to(dev), b.k.to(dev), b.v.to(dev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = chunk_attention(q, k, v, b.kc, b.vc, plan, SCALE)
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert torch.equal(chunk_attention(q, k, v, b.kc, b.vc, plan, SCALE), want)
    monkeypatch.setattr(_capi, "native", None)
    assert torch.equal(b.run(1), want)


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("len_,cached,g", [(1, 1500, 4), (3, 33000, 2), (100, 1500, 2), (66, 4200, 16), (5, 20, 2)])
def test_nan_rows_of_q(dev, bits, len_, cached, g):
    """A NaN in q is a NaN in its row of o, however many parts the keys are in, and in no other."""
    b = Batch(dev, [len_], [cached], g, 1, bits, seed=22)
    want = b.run(1)
    b.q[len_ - 1, g - 1, 5] = float("nan")
    out = b.run(1).view(len_, g, 128)
    assert out[len_ - 1, g - 1].isnan().all()
    out[len_ - 1, g - 1] = want.view(len_, g, 128)[len_ - 1, g - 1]
    assert torch.equal(out.view_as(want), want)


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("len_,g", [(1, 4), (100, 2), (66, 16)])
def test_nan_keys_of_one_part(dev, bits, len_, g):
    """A whole page of NaN keys, all that some part sees: every row is NaN."""
    b = Batch(dev, [len_], [4200], g, 1, bits, seed=23)
    page = b.tables[0][5]
    if bits == 8:
        b.kc[page, :, :256 * 128] = 0x7F
    else:
        b.kc[page] = float("nan")
    assert b.run(1).isnan().all()


def test_plans_are_made_before_a_capture(dev):
    x = torch.zeros(4, device=dev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x += 1
        with pytest.raises(RuntimeError, match="before the capture"):
            ChunkPlan([1], [0], [[]], dev)
    graph.replay()
    torch.cuda.synchronize()
    assert (x == 1).all()


@pytest.mark.parametrize("bits", [8, 16])
def test_pages_beyond_4_gib(dev, bits):
    """The last pages of a cache whose byte offsets do not fit 32 bits: the same bits as from a small one."""
    lens, cached = [1, 40], [300, 700]
    small = [Batch(dev, lens, cached, g, 1, bits, seed=24) for g in _forms(40)]
    b = small[0]
    pages = 4 * 2**30 // (_capi.PAGE_BYTES if bits == 8 else 256 * 256) + 64
    far = pages - b.pages
    if bits == 8:
        kc, vc = (torch.empty(pages, 1, _capi.PAGE_BYTES, dtype=torch.uint8, device=dev) for _ in range(2))
    else:
        kc, vc = (torch.empty(pages, 256, 1, 128, dtype=BF16, device=dev) for _ in range(2))
    for s in small:
        kc[far:], vc[far:] = s.kc, s.vc
        plan = ChunkPlan(lens, cached, [[p + far for p in t] for t in s.tables], dev, mask_block=1)
        out = chunk_attention(s.q.to(dev), s.k.to(dev), s.v.to(dev), kc, vc, plan, SCALE)
        assert torch.equal(out, s.run(1))
    k, v = b.k.to(dev), b.v.to(dev)
    slots = torch.arange(41, dtype=torch.int32, device=dev) * 100 + far * 256
    store_kvcache(k, v, kc, vc, slots)
    store_kvcache(k, v, b.kc, b.vc, slots - far * 256)
    # slots past the end are left out of both
    back, want = ([torch.zeros_like(k) for _ in range(2)] for _ in range(2))
    load_kvcache(*back, kc, vc, slots)
    load_kvcache(*want, b.kc, b.vc, slots - far * 256)
    assert all(torch.equal(x, y) for x, y in zip(back, want)) and back[0].any()
