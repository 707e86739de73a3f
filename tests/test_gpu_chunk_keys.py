"""chunk_attention with keys that decide the output one by one, so that a key, tile, part
or page that is left out, read from elsewhere, joined twice or seen too early shows,
however many keys there are.

Every key is a code of random signs, 6 c.  A row of q is the sum of two keys' codes: the
two have one and the same score, 6 (128 + c_a c_b) / sqrt(128), and every other key's is 6 c_u
(c_a + c_b) / sqrt(128), whose standard deviation is 6 sqrt(256 + 2 c_a c_b) / sqrt(128).  With
partners of c_a c_b >= -10 and 2^32 pairs of a row and a key (6.3 standard deviations) the
others lie 10 below at least, and 37 on the average, so together they weigh below 1e-3 of
a value of at most 6.  The output is (V_a + V_b) / 2, up to the rounding of the two
probabilities to bf16 (2^-8 each, in the product and in the sum, which may be made against
different maxima) and of the result (2^-8)."""
import pytest
import torch

from dllm_serve_amd import _capi
from dllm_serve_amd.engine.kv_cache import quantized_pages
from dllm_serve_amd.layers.attention import ChunkPlan, chunk_attention, load_kvcache, store_kvcache

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
SCALE = 128 ** -0.5


class Marked:
    """Sequences whose keys are codes.  With `share` they have the same pages."""

    def __init__(self, dev, lens, cached, Hq, Hkv, bits, seed, share=False, mask_block=1):
        self.g = torch.Generator(device=dev).manual_seed(seed)
        self.dev, self.lens, self.cached, self.Hq, self.Hkv, self.mask_block = dev, lens, cached, Hq, Hkv, mask_block
        need = [-(-c // 256) for c in cached]
        pages = (max(need) if share else sum(need)) + 2
        perm = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
        self.tables = [perm[:n] if share else perm[sum(need[:b]):sum(need[:b + 1])] for b, n in enumerate(need)]
        rows = pages * 256
        self.n = sum(lens)
        signs = torch.randint(0, 2, (rows + self.n, Hkv, 128), generator=self.g, device=dev, dtype=torch.int8)
        self.codes = (2 * signs - 1).to(BF16)
        values = torch.randn(rows + self.n, Hkv, 128, generator=self.g, device=dev).to(BF16)
        keys = self.codes * 6
        self.k, self.v = keys[rows:].contiguous(), values[rows:].contiguous()
        if bits == 8:
            self.kc, self.vc = quantized_pages(pages, Hkv, device=dev), quantized_pages(pages, Hkv, device=dev)
            slots = torch.arange(rows, dtype=torch.int32, device=dev)
            store_kvcache(keys[:rows], values[:rows], self.kc, self.vc, slots)
            held = torch.empty_like(keys[:rows])
            load_kvcache(held, values[:rows], self.kc, self.vc, slots)
            assert torch.equal(held, keys[:rows])
        else:
            self.kc, self.vc = (t[:rows].contiguous().view(pages, 256, Hkv, 128) for t in (keys, values))
        self.values = values
        self.new0 = rows
        # per row of q: its sequence's page table, cached rows, new rows and those it sees
        width = max(1, max(need))
        tab = torch.zeros(len(lens), width, dtype=torch.int64)
        for b, t in enumerate(self.tables):
            tab[b, :len(t)] = torch.tensor(t, dtype=torch.int64)
        self.tab = tab.to(dev)
        per_row = [(b, cached[b], sum(lens[:b]), L, self.sees(cached[b], L, t)) for b, L in enumerate(lens) for t in range(L)]
        self.row = torch.tensor(per_row, dtype=torch.int64).t().to(dev)  # [5, rows]
        self.plan = ChunkPlan(lens, cached, self.tables, dev, mask_block=mask_block)
        self.bits = bits

    def attend(self, q):
        return chunk_attention(q, self.k, self.v, self.kc, self.vc, self.plan, SCALE).view(self.n, self.Hq, 128).float()

    def sees(self, n, L, t):
        b = self.mask_block
        return L if b == 0 else min(L, ((n + t) // b + 1) * b - n)

    def shape(self):
        p = self.plan
        return _capi.chunk_launch_shape(p.n_seg, p.max_q, p.max_cached, self.Hq, self.Hkv, 128, p.total_rows, p.total_cached)

    def at(self, key):
        """Rows of codes / values of keys [rows, Hq] (counted over cached, then new rows)."""
        b, n, r0, _, _ = (x[:, None] for x in self.row)
        old = key.clamp(max=self.tab.shape[1] * 256 - 1)
        slot = self.tab[b.expand_as(key), old // 256] * 256 + old % 256
        return torch.where(key < n, slot, self.new0 + r0 + key - n)

    def of(self, rows, key):
        head = torch.arange(self.Hq, device=self.dev) // (self.Hq // self.Hkv)
        return rows[self.at(key), head[None, :].expand_as(key)].float()

    def rand(self, high):
        """Integers below high [rows, Hq] (at least 1)."""
        return (torch.rand(high.shape, generator=self.g, device=self.dev) * high).long().clamp(max=high - 1)

    def partner(self, a, pick):
        """Of eight picks, those whose code is nearest to that of key a."""
        ca, best, dot = self.of(self.codes, a), None, None
        for _ in range(8):
            b = pick()
            d = (ca * self.of(self.codes, b)).sum(-1)
            best = b if best is None else torch.where(d > dot, b, best)
            dot = d if dot is None else torch.maximum(d, dot)
        return best

    def check(self, a, b):
        q = (self.of(self.codes, a) + self.of(self.codes, b)).to(BF16)
        o = self.attend(q)
        va, vb = self.of(self.values, a), self.of(self.values, b)
        ref = 0.5 * (va + vb)
        tol = 2.0 ** -8 * ref.abs() + 1.05 * 2.0 ** -8 * (va.abs() + vb.abs()) + 6e-3
        bad = ~((o - ref).abs() <= tol)
        if bad.any():
            r, h, d = bad.nonzero()[0].tolist()
            raise AssertionError(f"row {r} head {h} d {d}: {o[r, h, d]} for {ref[r, h, d]}, keys {a[r, h]} and {b[r, h]}; "
                                 f"{int(bad.any(-1).sum())} rows differ")

    def seen(self):
        return (self.row[1] + self.row[4])[:, None].expand(-1, self.Hq)

    def pair(self, a):
        """Row r's two keys: a and another one that it sees."""
        n = self.seen()
        self.check(a, self.partner(a, lambda: (a + 1 + self.rand((n - 1).clamp(min=1))) % n))

    def all_of(self, keys):
        """Every key of `keys` (of each KV head) decides some row."""
        keys, per = torch.as_tensor(keys, dtype=torch.int64, device=self.dev), self.n * (self.Hq // self.Hkv)
        g = self.Hq // self.Hkv
        r = torch.arange(self.n, device=self.dev)[:, None] * g + torch.arange(self.Hq, device=self.dev)[None, :] % g
        for i in range(0, len(keys), per):
            self.pair(torch.minimum(keys[(i + r) % len(keys)], self.seen() - 1))

    def anywhere(self, times):
        for _ in range(times):
            self.pair(self.rand(self.seen()))

    def hidden(self, times):
        """A new row that row r does not see, and one that it sees: the latter alone counts."""
        _, n, _, L, see = (x[:, None].expand(-1, self.Hq) for x in self.row)
        for _ in range(times):
            b = n + torch.where(see < L, see + self.rand((L - see).clamp(min=1)), self.rand(L))
            a = self.partner(b, lambda: self.rand(n + see))
            # rows that see all of their sequence's rows are an ordinary pair
            sees_b = (b - n < see)[..., None]
            va, vb = self.of(self.values, a), self.of(self.values, b)
            q = (self.of(self.codes, a) + self.of(self.codes, b)).to(BF16)
            o = self.attend(q)
            ref = torch.where(sees_b, 0.5 * (va + vb), va)
            tol = 2.0 ** -8 * ref.abs() + 1.05 * 2.0 ** -8 * (va.abs() + vb.abs()) + 6e-3
            assert ((o - ref).abs() <= tol).all()


# ---- runs of segments ----------------------------------------------------------------
# Batches whose parts need more than the workspace's limit are launched in several runs.

RUNS = [
    # one long sequence among single tokens: rows form, parts set by the page ids of a split
    ([1] * 1100, [300, 5] * 200 + [16200] + [40, 0, 256] * 233, 64, 64, 16),
    # a piece of a prompt among single tokens: tile form
    ([1] * 20 + [520] + [1] * 44, [300] * 10 + [0] * 10 + [20000] + [700] * 44, 28, 4, 128),
]


class OneCall(Marked):
    """All sequences in one call of the C entry point, where a plan may launch some apart."""

    def attend(self, q):
        p, (cu, lens, tables) = self.plan, self.plan._args
        o = torch.full((self.n, self.Hq * 128), float("nan"), dtype=BF16, device=self.dev)
        need = _capi.chunk_workspace_size(p.n_seg, p.max_q, p.max_cached, self.Hq, self.Hkv, 128, p.total_rows, p.total_cached)
        ws = torch.empty(max(need, 16), dtype=torch.uint8, device=self.dev)
        rows = (self.Hq * 128, self.Hkv * 128, self.Hkv * 128, self.Hq * 128)
        _capi.attn_chunk_paged_fwd_raw(
            q.data_ptr(), self.k.data_ptr(), self.v.data_ptr(), o.data_ptr(), cu, p._seg_ids, p.n_seg, p.max_q,
            p.max_cached, p.total_rows, p.total_cached, self.kc.data_ptr(), self.vc.data_ptr(),
            _capi.CACHE_FP8 if self.bits == 8 else _capi.CACHE_BF16, self.kc.shape[0], tables, p.max_pages, lens,
            self.mask_block, self.Hq, self.Hkv, 128, *rows, SCALE, ws.data_ptr(), need, _capi._stream(self.dev))
        return o.view(self.n, self.Hq, 128).float()


@pytest.mark.parametrize("lens,cached,Hq,Hkv,rows", RUNS)
def test_segments_in_runs(dev, lens, cached, Hq, Hkv, rows):
    b = OneCall(dev, lens, cached, Hq, Hkv, 8, seed=61, share=True)
    shape, p = b.shape(), b.plan
    ws = _capi.chunk_workspace_size(p.n_seg, p.max_q, p.max_cached, Hq, Hkv, 128, p.total_rows, p.total_cached)
    a_segment = Hkv * -(-p.max_q * Hq // Hkv // rows) * shape["n_split"]
    assert shape["rows"] == rows and 0 < ws <= 1 << 30 and shape["n_split"] > 1
    assert p.n_seg * a_segment > ws // (rows * 520) >= a_segment  # several runs, one segment or more each
    b.anywhere(12)
    b.hidden(4)


# ---- every tile, page, part and round ---------------------------------------------------

def _borders(n, L):
    """First and last key of every run of 32 cached rows (tiles, pages, parts and rounds of
    parts begin and end there) and of every 32 new rows."""
    out = [x for i in range(0, n, 32) for x in (i, min(i + 31, n - 1))]
    return out + [n + x for i in range(0, L, 32) for x in (i, min(i + 31, L - 1))]


CASES = [
    # lens, cached, Hq, Hkv, mask_block, shared pages, rows of a workgroup, parts
    # parts of a row joined in three rounds, and the same of two rows of 16
    ([1], [33000], 16, 1, 1, False, 16, range(100, 200)),
    ([2], [33000], 16, 1, 1, False, 32, range(100, 200)),
    ([1], [131071], 8, 1, 1, False, 16, range(200, 300)),
    # parts as long as a workgroup's page ids reach (15872 rows): whole, one row more, three
    ([1] * 16, [31744] * 16, 16, 16, 1, True, 16, [2]),
    ([1] * 16, [31745] * 16, 16, 16, 1, True, 16, [3]),
    ([20] * 16, [33000] * 16, 16, 16, 4, True, 32, [3]),
    # one part, page ids fetched again every 64 pages
    ([100] * 16, [17000] * 16, 32, 32, 1, True, 128, [1]),
    ([70] * 16, [33100] * 16, 32, 32, 0, True, 128, [1]),
    # parts of new and cached tiles, of cached pages that begin inside a part
    ([66], [4200], 16, 1, 1, False, 128, range(10, 100)),
    ([600, 530], [40000, 1000], 8, 2, 32, False, 128, range(2, 200)),
    ([300], [2500], 8, 1, 0, False, 128, range(2, 100)),
    # few keys, ragged, several M tiles, eight wavefronts and four
    ([1], [900], 4, 4, 1, False, 16, range(2, 20)),
    ([1], [511], 32, 32, 1, False, 16, [1]),
    ([1, 3, 1], [1, 700, 4000], 14, 2, 1, False, 32, range(2, 100)),
    ([1] * 32, [512 + 97 * i for i in range(32)], 28, 4, 1, False, 16, range(2, 20)),
    ([32] * 4, [608, 1216, 90, 0], 4, 4, 0, False, 32, range(1, 20)),
    ([32] * 16, [384 + 56 * i for i in range(16)], 28, 4, 0, False, 32, [1]),
    ([9, 40], [255, 257], 14, 2, 4, False, 32, [1]),
    ([260, 70], [511, 0], 4, 4, 33, False, 32, range(1, 20)),
]


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("lens,cached,Hq,Hkv,mask_block,share,rows,parts", CASES)
def test_every_key_counts_once(dev, lens, cached, Hq, Hkv, mask_block, share, rows, parts, bits):
    b = Marked(dev, lens, cached, Hq, Hkv, bits, seed=62 + len(lens) + max(cached), share=share, mask_block=mask_block)
    shape = b.shape()
    assert shape["rows"] == rows and shape["n_split"] in parts, shape
    longest = max(range(len(lens)), key=lambda i: cached[i])
    b.all_of(_borders(cached[longest], lens[longest]))
    b.anywhere(6)
    if mask_block:
        b.hidden(4)


# ---- long and short new rows in one plan ---------------------------------------------------

MIXED = [
    # lens, cached, Hq, Hkv, mask_block, sequences of every launch
    ([1] * 20 + [520] + [1] * 44, [300] * 10 + [0] * 10 + [2000] + [700] * 44, 28, 4, 1, [1, 64]),
    # three launches, sequences without new rows, another order
    ([1, 0, 700, 2, 40, 1, 600, 0, 33] + [1] * 20, [50, 9, 800, 31, 0, 2000, 0, 0, 7] + [90 + i for i in range(20)], 8, 2, 4,
     [2, 2, 25]),
    # too few rows for an order of their own
    ([64] + [1] * 10, [500] + [1900] * 10, 14, 2, 1, [1, 10]),
    ([3, 400, 0, 1], [10, 20, 30, 5], 4, 2, 0, [4]),
]


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("lens,cached,Hq,Hkv,mask_block,groups", MIXED)
def test_short_among_long(dev, lens, cached, Hq, Hkv, mask_block, groups, bits, monkeypatch):
    b = Marked(dev, lens, cached, Hq, Hkv, bits, seed=64, mask_block=mask_block)
    assert [g[1] for g in b.plan.groups] == groups
    b.anywhere(12)
    if mask_block:
        b.hidden(4)
    # the Python form, a graph and, launched at once, the C entry point
    q = torch.randn(b.n, Hq, 128, generator=b.g, device=dev).to(BF16)
    want = chunk_attention(q, b.k, b.v, b.kc, b.vc, b.plan, SCALE)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = chunk_attention(q, b.k, b.v, b.kc, b.vc, b.plan, SCALE)
    for _ in range(3):
        out.zero_()
        graph.replay()
        assert torch.equal(chunk_attention(q, b.k, b.v, b.kc, b.vc, b.plan, SCALE), want)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    with monkeypatch.context() as m:
        m.setattr(_capi, "native", None)
        assert torch.equal(chunk_attention(q, b.k, b.v, b.kc, b.vc, b.plan, SCALE), want)
    once = OneCall(dev, lens, cached, Hq, Hkv, bits, seed=64, mask_block=mask_block)
    once.anywhere(4)
