"""Drop-in ``Attention`` layer and KV-cache helpers on the gfx950 kernels.

Interface of dllmserve/layers/attention.py (``Attention(num_heads,
head_dim, scale, num_kv_heads, causal)``, ``.forward(q, k, v)``,
``store_kvcache``, ``load_kvcache``, the ``k_cache`` / ``v_cache`` /
``layer_id`` attributes a model runner binds).  The diffusion branch
(attention.py:150-306) is reproduced per sequence:

* cache state 0 or no SparseConfig: full bidirectional attention over the
  sequence's rows (K3a);
* state 1: full attention (K3a), and the top-n_keep non-block rows of every
  KV head (``head_select``) or of all heads are written to the sequence's
  cache slots (K5/K6 fused with K1);
* state 2: the block rows attend to [cached rows ; block rows] (K3b), read
  straight from the paged cache by slot, without the reference's gather and
  concatenation copies.

A cache of 8-bit pages (engine.kv_cache, ``quantized=True``) is written by the
same selection, its rows quantised on the way, and state 2 then attends over
the pages.  ``chunk_attention`` is the same attention for callers with their
own tables: chunks of any length over 8-bit or bf16 pages, bidirectional,
causal or causal between blocks.

Per step the layer builds one launch plan from ``context.seqs`` (host
integers only, no device synchronisation) and caches it on the Context, so
the 32 layers of a forward reuse it.  Every kernel runs on the caller's
current HIP stream; nothing falls back to the CPU.
"""
from __future__ import annotations

import contextlib
import os
import struct
import weakref

import numpy as np
import torch
from torch import nn

from .. import _capi
from ..sparse.state import keep_count
from ..utils.context import get_context


def _token_rows(t: torch.Tensor, heads: int, head_dim: int, name: str):
    """(t, rows, token stride in elements) of q/k/v given as [rows, heads *
    head_dim] or [rows, heads, head_dim] with contiguous heads; any other
    shape goes through the reference's ``view(-1, heads, head_dim)``."""
    sh = t.shape
    if len(sh) == 2 and sh[1] == heads * head_dim:
        st = t.stride()
        if st[1] != 1:
            raise ValueError(f"{name} must have contiguous heads; got shape {tuple(sh)} strides {st}")
        return t, sh[0], st[0]
    if len(sh) != 3 or sh[1] != heads or sh[2] != head_dim:
        t = t.view(-1, heads, head_dim)
        sh = t.shape
    st = t.stride()
    if st[2] != 1 or st[1] != head_dim:
        raise ValueError(f"{name} must be [rows, heads, head_dim] with contiguous heads; got shape "
                         f"{tuple(sh)} strides {st}")
    return t, sh[0], st[0]


def _slot_tensor(slot_mapping, device) -> torch.Tensor:
    if not isinstance(slot_mapping, torch.Tensor):
        slot_mapping = torch.tensor(list(slot_mapping), dtype=torch.int32)
    if slot_mapping.dtype != torch.int32 or slot_mapping.device != device or not slot_mapping.is_contiguous():
        slot_mapping = slot_mapping.to(device=device, dtype=torch.int32).contiguous()
    return slot_mapping


def store_kvcache(key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                  slot_mapping: torch.Tensor) -> None:
    """k_cache.flat[slot_mapping[i], :] = key[i], same for value (attention.py:33-50).
    With 8-bit pages (quantized_pages) the rows are quantised as they are written."""
    if k_cache.dtype == torch.uint8 or v_cache.dtype == torch.uint8:
        _quant_copy(_capi.store_kvcache_fp8, key, value, k_cache, v_cache, slot_mapping)
        return
    N, num_heads, head_dim = key.shape
    D = num_heads * head_dim
    assert key.stride(-1) == 1 and value.stride(-1) == 1
    assert key.stride(1) == head_dim and value.stride(1) == head_dim
    assert k_cache.stride(1) == D and v_cache.stride(1) == D
    if slot_mapping.numel() != N:
        print(f"Warning: slot_mapping.numel {slot_mapping.numel()} != N {N}")
    assert slot_mapping.numel() == N
    assert k_cache.is_contiguous() and v_cache.is_contiguous(), "KV cache must be contiguous"
    assert key.dtype == value.dtype == k_cache.dtype == v_cache.dtype == torch.bfloat16, "bf16 tensors expected"
    slot = _slot_tensor(slot_mapping, key.device)
    _capi.store_kvcache(key, value, k_cache, v_cache, slot, N, D)


def load_kvcache(key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                 slot_mapping: torch.Tensor) -> None:
    """key[i] = k_cache.flat[slot_mapping[i], :], same for value (attention.py:77-92).
    From 8-bit pages the rows come back as the bf16 values they stand for."""
    if k_cache.dtype == torch.uint8 or v_cache.dtype == torch.uint8:
        _quant_copy(_capi.load_kvcache_fp8, key, value, k_cache, v_cache, slot_mapping)
        return
    N, num_heads, head_dim = key.shape
    D = num_heads * head_dim
    assert key.stride(-1) == 1 and value.stride(-1) == 1
    assert key.stride(1) == head_dim and value.stride(1) == head_dim
    assert k_cache.stride(1) == D and v_cache.stride(1) == D
    assert slot_mapping.numel() == N
    assert k_cache.is_contiguous() and v_cache.is_contiguous(), "KV cache must be contiguous"
    assert key.dtype == value.dtype == k_cache.dtype == v_cache.dtype == torch.bfloat16, "bf16 tensors expected"
    slot = _slot_tensor(slot_mapping, key.device)
    _capi.load_kvcache(key, value, k_cache, v_cache, slot, N, D)


def _check_pages(k_cache: torch.Tensor, v_cache: torch.Tensor, device) -> int:
    """Check a pair of 8-bit caches and return their KV heads."""
    for t, n in ((k_cache, "k_cache"), (v_cache, "v_cache")):
        if (t.dtype != torch.uint8 or t.dim() != 3 or t.shape[2] != _capi.PAGE_BYTES or not t.is_contiguous()
                or t.device != device or t.shape[1] != k_cache.shape[1]):
            raise ValueError(f"{n} must be contiguous 8-bit pages, uint8 [num_pages, KV heads, {_capi.PAGE_BYTES}] on "
                             f"{device}; got {t.dtype} {tuple(t.shape)} on {t.device}")
    return k_cache.shape[1]


def _on_device(device: torch.device):
    """Makes `device` current where it is not: a launch on another device's stream fails."""
    if device.type != "cuda" or device.index is None or device.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(device)


def _quant_copy(copy, key, value, k_cache, v_cache, slot_mapping) -> None:
    if _capi.native is not None and _capi.native.quant_copy(key, value, k_cache, v_cache, slot_mapping,
                                                            copy is _capi.store_kvcache_fp8):
        return
    N, num_heads, head_dim = key.shape
    assert value.shape == key.shape and value.device == key.device
    assert key.stride(-1) == 1 and value.stride(-1) == 1
    assert key.stride(1) == head_dim and value.stride(1) == head_dim
    assert slot_mapping.numel() == N
    assert key.dtype == value.dtype == torch.bfloat16, "bf16 tensors expected"
    if _check_pages(k_cache, v_cache, key.device) != num_heads:
        raise ValueError(f"rows of {num_heads} KV heads, pages of {k_cache.shape[1]}")
    slot = _slot_tensor(slot_mapping, key.device)
    with _on_device(key.device):
        copy(key, value, k_cache, v_cache, slot, N, num_heads, head_dim)


class ChunkPlan:
    """Launch tables of one step's chunk attention, shared by its layers.

    Sequence b feeds ``seqlens[b]`` new rows behind ``cached_lens[b]`` rows in the
    256-row cache pages ``block_tables[b]`` (host integers; more pages than
    needed are fine).  ``mask_block`` 0: the new rows see each other; b >= 1:
    a row sees the rows up to the end of its own block of b positions
    (1: causal), positions counted from the first cached row: behind a cache that
    holds a selection of the rows, n cached rows do not end at position n, and
    only 0 and 1 mean what they say.  The tables are
    uploaded with one asynchronous copy on the stream that is current; nothing
    synchronises the host.  The first call on any other stream makes that stream
    wait for the upload, and a plan may be dropped while calls are in flight.  A plan
    for a captured graph is made before the capture, has to have arrived by then
    (torch.cuda.graph synchronises) and to live as long as the graph, which holds its
    addresses.

    ``cached_lens`` and ``block_tables`` are in the order of the launches, which is
    the sequences' own unless they feed _SORT_ROWS rows together: then those with
    the most keys come first, so that no long workgroup starts when the others end.

    A launch takes the form, grid and workspace of its longest new rows, so short
    sequences among long ones go into one of their own (``groups``)."""

    # The order costs a dependent load at the start of every workgroup, which only
    # pieces of prompts are long enough not to feel.
    _SORT_ROWS = 512

    def __init__(self, seqlens, cached_lens, block_tables, device, mask_block: int = 0):
        seqlens, cached = [int(n) for n in seqlens], [int(n) for n in cached_lens]
        tables = [[int(p) for p in t] for t in block_tables]
        if not (len(seqlens) == len(cached) == len(tables)):
            raise ValueError(f"{len(seqlens)} sequences, {len(cached)} cached lengths, {len(tables)} block tables")
        if any(n < 0 for n in seqlens + cached) or not 0 <= mask_block < 2**31:
            raise ValueError("lengths and mask_block must not be negative (nor mask_block exceed int32)")
        need = [-(-n // _capi.PAGE_ROWS) for n in cached]
        for b, (t, n) in enumerate(zip(tables, need)):
            if len(t) < n or any(p < 0 for p in t[:n]):
                raise ValueError(f"sequence {b}: {cached[b]} cached rows need {n} pages, block table {t[:n]}")
        self.device = torch.device(device)
        if self.device.type == "cuda" and self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        _not_captured("make the ChunkPlan", self.device)
        self.n_seg = B = len(seqlens)
        self.total_rows, self.total_cached = sum(seqlens), sum(cached)
        self.max_q, self.max_cached = max(seqlens, default=0), max(cached, default=0)
        self.max_pages = W = max(need, default=0)
        self.max_page = max((p for t, n in zip(tables, need) for p in t[:n]), default=-1)
        self.mask_block = int(mask_block)
        order, self.groups = [], []
        for members in self._cut(seqlens, cached):
            if self.total_rows >= self._SORT_ROWS:
                members.sort(key=lambda b: -(seqlens[b] + cached[b]))  # stable
            # first sequence in the order, sequences, longest new rows and cache, sums of both
            q, c = [seqlens[b] for b in members], [cached[b] for b in members]
            self.groups.append((len(order), len(members), max(q), max(c), sum(q), sum(c)))
            order += members
        flat = np.full(3 * B + 1 + B * W, -1, dtype=np.int64)
        flat[0] = 0
        flat[1:B + 1] = np.cumsum(seqlens)
        flat[B + 1:2 * B + 1] = [cached[b] for b in order]
        flat[2 * B + 1:3 * B + 1] = order
        for i, b in enumerate(order):
            flat[3 * B + 1 + i * W:3 * B + 1 + i * W + need[b]] = tables[b][:need[b]]
        if flat.max() >= 2**31:
            raise ValueError("chunk tables exceed int32")
        host = torch.from_numpy(flat.astype(np.int32))
        if self.device.type == "cuda":
            host = host.pin_memory()
        self._tables = dev = host.to(self.device, non_blocking=True)
        self._ready, self._streams = None, ()  # the upload's event, the streams that are behind it
        if self.device.type == "cuda":
            stream = torch.cuda.current_stream(self.device)
            self._ready = torch.cuda.Event()
            self._ready.record(stream)
            self._streams = (stream.cuda_stream,)
        self.cu, self.cached_lens, self.block_tables = dev[:B + 1], dev[B + 1:2 * B + 1], dev[3 * B + 1:]
        self._seg_ids = None if order == sorted(order) else dev[2 * B + 1:].data_ptr()
        self._args = (self.cu.data_ptr(), self.cached_lens.data_ptr(), self.block_tables.data_ptr())
        self._packed = self._pack()

    @staticmethod
    def _cut(seqlens, cached) -> list:
        """The sequences (indices, in order) of every launch.

        Those with under a sixteenth of the longest one's new rows are launched apart where
        there are two or more and they would waste enough: their number times the rows
        of the longest times the keys that there may be, 2^20 or more.  One launch / two, in us,
        28/4 heads, beside single tokens behind 2000: 2048 rows behind 6000 and 31 of them 1470 / 260,
        2 301 / 251, 512 behind 3000 and 16 189 / 59, 256 behind 500 and 2 62 / 31, 64 behind 1000 and 8 26 / 25,
        but 4 20 / 23; 256 rows and two tokens, all behind 100, 18 / 24."""
        out, rest = [], list(range(len(seqlens)))
        while rest:
            most = max(seqlens[b] for b in rest)
            short = [b for b in rest if seqlens[b] * 16 < most]
            n = sum(seqlens[b] > 0 for b in short)
            if n < 2 or n * most * (most + max(cached[b] for b in rest)) < 1 << 20:
                short = []
            apart = set(short)
            out.append([b for b in rest if b not in apart])
            rest = short
        return out

    _STREAMS = 16  # streams remembered; one that was forgotten waits once more

    def _pack(self) -> bytes:
        """The plan for the native form (csrc/native.cpp, ChunkTables), its launches, the streams behind it."""
        groups = [x for g in self.groups for x in g]
        return struct.pack(
            f"={10 + len(groups) + len(self._streams)}q", -1 if self.device.index is None else self.device.index,
            self.total_rows, len(self.groups), self.max_pages, self.max_page, self.mask_block, *self._args,
            self._seg_ids or 0, *groups, *self._streams)

    def _join(self) -> None:
        """Puts the device's current stream behind the upload, and the tables' memory
        behind what that stream will have read of it when the plan is dropped.  (A stream
        that is being captured cannot wait for an event from outside its graph.)"""
        stream = torch.cuda.current_stream(self.device)
        if stream.cuda_stream in self._streams or torch.cuda.is_current_stream_capturing():
            return
        stream.wait_event(self._ready)
        self._tables.record_stream(stream)
        self._streams = (self._streams + (stream.cuda_stream,))[-self._STREAMS:]
        self._packed = self._pack()


def chunk_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                    plan: ChunkPlan, softmax_scale: float) -> torch.Tensor:
    """Attention of every sequence's new rows over its cached rows and over
    each other (see ChunkPlan), [rows, Hq * 128].

    q / k / v are the new rows of all sequences, packed, as
    [rows, heads * 128] or [rows, heads, 128] with contiguous heads, bf16.  The
    caches are 8-bit pages (quantized_pages) or bf16 [num_pages, 256, Hkv,
    128]; the new rows are read from k / v, so they may be stored before or after."""
    D = 128
    if _capi.native is not None:
        o = _capi.native.chunk(q, k, v, k_cache, v_cache, plan._packed, float(softmax_scale))
        if o is not None:
            return o
    for t, n in ((q, "q"), (k, "k"), (v, "v")):
        if t.dtype != torch.bfloat16:
            raise TypeError(f"bf16 {n} expected, got {t.dtype}")
        if t.dim() not in (2, 3) or t.numel() != t.shape[0] * (t.shape[1] if t.dim() == 2 else t.shape[1] * D) \
                or t.dim() == 2 and t.shape[1] % D:
            raise ValueError(f"{n} must be [rows, heads * 128] or [rows, heads, 128]; got {tuple(t.shape)}")
    heads = [t.shape[1] // D if t.dim() == 2 else t.shape[1] for t in (q, k, v)]
    Hq, Hkv = heads[0], heads[1]
    if heads[2] != Hkv or Hkv == 0 or Hq == 0 or Hq % Hkv:
        raise ValueError(f"{heads[0]} / {heads[1]} / {heads[2]} heads of q / k / v")
    q, nq, q_st = _token_rows(q, Hq, D, "q")
    k, nk, k_st = _token_rows(k, Hkv, D, "k")
    v, nv, v_st = _token_rows(v, Hkv, D, "v")
    dev = q.device
    if not (q.is_cuda and k.is_cuda and v.is_cuda):
        raise RuntimeError("chunk_attention runs on the GPU only (no CPU fallback)")
    if k.device != dev or v.device != dev or plan.device != dev:
        raise ValueError(f"q / k / v and the plan are on {q.device} / {k.device} / {v.device} / {plan.device}")
    if not (nq == nk == nv == plan.total_rows):
        raise ValueError(f"q / k / v have {nq} / {nk} / {nv} rows, the plan's sequences feed {plan.total_rows}")
    if k_cache.dtype == torch.uint8:
        if _check_pages(k_cache, v_cache, dev) != Hkv:
            raise ValueError(f"k / v of {Hkv} KV heads, pages of {k_cache.shape[1]}")
        kind, pages = _capi.CACHE_FP8, min(k_cache.shape[0], v_cache.shape[0])
    else:
        for t, n in ((k_cache, "k_cache"), (v_cache, "v_cache")):
            if (t.dtype != torch.bfloat16 or not t.is_contiguous() or t.device != dev or t.dim() != 4
                    or tuple(t.shape[1:]) != (_capi.PAGE_ROWS, Hkv, D)):
                raise ValueError(f"{n} must be contiguous bf16 [num_pages, {_capi.PAGE_ROWS}, {Hkv}, {D}] or 8-bit "
                                 f"pages on {dev}; got {t.dtype} {tuple(t.shape)} on {t.device}")
        kind, pages = _capi.CACHE_BF16, min(k_cache.shape[0], v_cache.shape[0])
    if plan.max_page >= pages:
        raise ValueError(f"a block table names page {plan.max_page} of a cache of {pages}")
    with _on_device(dev):
        plan._join()
        o = torch.empty(nq, Hq * D, dtype=torch.bfloat16, device=dev)
        need = max((_capi.chunk_workspace_size(n, mq, mc, Hq, Hkv, D, tq, tc) for _, n, mq, mc, tq, tc in plan.groups),
                   default=0)
        # from the allocator at every call: a plan may be used on several streams and in several graphs
        ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        cu, lens, tables = plan._args
        for first, n, mq, mc, tq, tc in plan.groups if nq else ():
            _capi.attn_chunk_paged_fwd_raw(
                q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), cu if plan._seg_ids else cu + 4 * first,
                plan._seg_ids + 4 * first if plan._seg_ids else None, n, mq, mc, tq, tc, k_cache.data_ptr(),
                v_cache.data_ptr(), kind, pages, tables + 4 * first * plan.max_pages, plan.max_pages, lens + 4 * first,
                plan.mask_block, Hq, Hkv, D, q_st, k_st, v_st, o.stride(0), float(softmax_scale),
                None if ws is None else ws.data_ptr(), need, _capi._stream(dev))
    return o


class StepLayout:
    """Host integers of one diffusion step: per-sequence mode (0 full, 1 full
    + select-and-store, 2 block vs cache, -1 unrecognised), fed rows, block
    span and n_keep, and the launch sizes derived from them (attention.py:
    168-265, sequence.py:99-152).  No tensors are created."""

    def __init__(self, seqs):
        if not seqs:
            raise ValueError("diffusion context has no sequences")
        rows, modes, spans, keeps, cfgs = [], [], [], [], []
        for seq in seqs:
            cfg = seq.sparse_state.config if seq.sparse_state is not None else None
            cfgs.append((bool(cfg.head_select), int(cfg.pool_kernel)) if cfg is not None else (False, 1))
            st = seq.sparse_state
            N = seq.num_tokens
            if st is None or st.is_full_attention:
                modes.append(0)
                rows.append(N)
                spans.append((0, 0))
                keeps.append(0)
            elif st.should_compute_cache:
                bs, bl = st.block_span(seq.num_prompt_tokens, N)
                bl = max(0, min(bl, N - bs)) if bs < N else 0
                if bl == 0:
                    raise ValueError(f"sequence {seq.seq_id}: cache state 1 with an empty block "
                                     f"(block start {bs}, {N} tokens)")
                modes.append(1)
                rows.append(N)
                spans.append((bs, bl))
                keeps.append(keep_count(N - bl, st.retention_ratio))
            elif st.should_reuse_cache:
                bs, bl_raw = st.compute_block_boundaries(seq.num_prompt_tokens, N)
                if bl_raw < 0:  # the reference's torch.arange(bs, bs + bl) raises here too
                    raise RuntimeError(f"sequence {seq.seq_id}: block {st.current_block_idx} starts at {bs}, "
                                       f"past the {N} tokens of the sequence")
                bl = bl_raw
                modes.append(2)
                rows.append(bl)
                spans.append((bs, bl))
                keeps.append(seq.current_sparse_token)
            else:
                modes.append(-1)  # unrecognised state: rows stay zero (outputs = zeros_like(q))
                rows.append(N)
                spans.append((0, 0))
                keeps.append(0)
        self.modes, self.rows, self.spans, self.keeps = modes, rows, spans, keeps
        self.cfgs = cfgs  # (head_select, pool_kernel) per sequence; selection jobs carry their own
        self.n_seq = len(seqs)
        self.total_rows = int(sum(rows))
        self.cu = np.zeros(self.n_seq + 1, dtype=np.int64)
        self.cu[1:] = np.cumsum(rows)
        self.any_skipped = any(m == -1 for m in modes)
        # longest first (ties by index): with the XCD interleave of the dense
        # kernel, long segments then start early and short ones fill the tail
        # (16 ragged Dream GQA segments: 3-12 % faster than batch order)
        self.dense = sorted((i for i, m in enumerate(modes) if m in (0, 1)), key=lambda i: (-rows[i], i))
        self.jobs_idx = [i for i, m in enumerate(modes) if m == 1]
        self.cached = [i for i, m in enumerate(modes) if m == 2]
        self.n_dense = len(self.dense)
        self.max_q_dense = max((rows[i] for i in self.dense), default=0)
        self.n_job = len(self.jobs_idx)
        self.max_kc = max((rows[i] - spans[i][1] for i in self.jobs_idx), default=0)
        self.max_keep = max((keeps[i] for i in self.jobs_idx), default=0)
        self.max_blk = max((spans[i][1] for i in self.jobs_idx), default=0)
        self.n_cached = len(self.cached)
        self.max_q_cached = max((rows[i] for i in self.cached), default=0)
        self.max_keys_cached = max((rows[i] + keeps[i] for i in self.cached), default=0)
        self.max_keep_cached = max((keeps[i] for i in self.cached), default=0)
        self.rows_cached = sum(rows[i] for i in self.cached)
        self.keeps_cached = sum(keeps[i] for i in self.cached)
        self.total_slots = sum(keeps[i] for i in self.cached + self.jobs_idx)
        # a launch over every sequence in batch order gets no id table: the
        # kernels then read a segment's offsets one dependent load earlier
        self.dense_identity = self.dense == list(range(self.n_seq))
        self.cached_identity = self.cached == list(range(self.n_seq))

    def signature(self) -> tuple:
        """Everything a captured step's launches depend on."""
        return (tuple(self.modes), tuple(self.rows), tuple(self.keeps), tuple(s[1] for s in self.spans),
                tuple(self.cfgs[i] for i in self.jobs_idx))


def _not_captured(what: str, device: torch.device) -> None:
    """Refuses an upload of tables inside a capture: the graph's replays would copy from
    pinned memory that has long been given to something else."""
    if device.type == "cuda":
        with _on_device(device):
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError(f"{what} before the capture")


class StepPlan:
    """Launch tables of one diffusion forward (shared by all layers).

    ``StepPlan(context, device, ...)`` builds them from host integers of
    ``context.seqs`` and uploads them with one asynchronous copy (not inside
    a capture: a forward of the same Context has to come before it);
    ``StepPlan.from_device`` wraps tables the device-side builder wrote.
    Its layers and the graphs captured from it share its workspaces: they run
    one after another."""

    _SCALARS = ("n_seq", "total_rows", "any_skipped", "n_dense", "max_q_dense", "n_job", "max_kc", "max_keep",
                "max_blk", "n_cached", "max_q_cached", "max_keys_cached", "max_keep_cached", "rows_cached",
                "keeps_cached", "dense_identity", "cached_identity")

    def __init__(self, context, device: torch.device, num_kv_heads: int = 0, head_dim: int = 0, num_heads: int = 0,
                 layout: StepLayout | None = None):
        _not_captured("run the step's forward once, which builds its plan,", device)
        seqs = context.seqs
        lay = layout if layout is not None else StepLayout(seqs)
        self._take(lay, device)
        rows, spans, keeps, cu = lay.rows, lay.spans, lay.keeps, lay.cu
        dense, jobs_idx, cached = lay.dense, lay.jobs_idx, lay.cached

        # slots of sparse sequences: state-2 sequences first (contiguous, so
        # slot_off below brackets each of them), then state-1 sequences
        slot_mapping = context.slot_mapping if context.slot_mapping is not None else []
        slot_parts, slot_base = [], {}
        off = 0
        for i in cached + jobs_idx:
            if i >= len(slot_mapping):
                raise ValueError(f"context.slot_mapping has no entry for sequence index {i}")
            sm = slot_mapping[i]
            n = sm.numel() if isinstance(sm, torch.Tensor) else len(sm)
            if n != keeps[i]:
                print(f"Warning: slot_mapping.numel {n} != N {keeps[i]}")
            assert n == keeps[i]
            slot_base[i] = off
            off += n
            slot_parts.append(_slot_tensor(sm, device))
        self.slots = torch.cat(slot_parts) if slot_parts else torch.zeros(1, dtype=torch.int32, device=device)

        # selection jobs: row0, n_tok, blk_start, blk_len, n_keep, slot_off, head_select, pool_k
        jobs = np.zeros((max(1, self.n_job), _capi.JOB_COLS), dtype=np.int64)
        for r, i in enumerate(jobs_idx):
            bs, bl = spans[i]
            hs, pk = lay.cfgs[i]
            jobs[r] = (cu[i], rows[i], bs, bl, keeps[i], slot_base[i], int(hs), pk)

        # cached (state 2) segments: slot offsets indexed by position in `cached`
        slot_off = np.zeros(self.n_cached + 1, dtype=np.int64)
        for r, i in enumerate(cached):
            slot_off[r] = slot_base[i]
            slot_off[r + 1] = slot_base[i] + keeps[i]

        # one asynchronous host->device copy (from pinned memory) of every int32 table
        parts = [cu, np.array(dense or [0]), np.array(cached or [0]), slot_off, jobs.reshape(-1)]
        flat = np.concatenate([p.astype(np.int64) for p in parts])
        if flat.size and (flat.max() >= 2**31 or flat.min() < -(2**31)):
            raise ValueError("step tables exceed int32")
        host = torch.from_numpy(flat.astype(np.int32))
        if device.type == "cuda":
            host = host.pin_memory()
        dev = host.to(device, non_blocking=True)
        o = 0
        self.cu = dev[o:o + cu.size]; o += cu.size
        self.dense_ids = dev[o:o + max(1, len(dense))]; o += max(1, len(dense))
        self.cached_ids = dev[o:o + max(1, len(cached))]; o += max(1, len(cached))
        self.slot_off = dev[o:o + slot_off.size]; o += slot_off.size
        self.jobs = dev[o:o + jobs.size]
        # what page_tables() needs, which only 8-bit pages call
        self._cached_seqs = [(seqs[i], keeps[i], slot_mapping[i]) for i in cached]

    def _take(self, lay: StepLayout, device) -> None:
        self.device = device
        for k in self._SCALARS:
            setattr(self, k, getattr(lay, k))
        self._ws = {}
        self._args = {}
        self._packed = {}
        self.last_idx = None
        self._cached_seqs = self._block_tables = None
        self._pages = None

    @classmethod
    def from_device(cls, lay: StepLayout, device, cu, dense_ids, cached_ids, slot_off, jobs, slots,
                    block_tables=None) -> "StepPlan":
        """Plan over tables already on the device (written by dllm_step_build).
        block_tables: int32 [n_seq, max_pages], the cache pages of every
        sequence (needed with 8-bit pages)."""
        self = cls.__new__(cls)
        self._take(lay, device)
        self._block_tables = block_tables
        self.cu, self.dense_ids, self.cached_ids = cu, dense_ids, cached_ids
        self.slot_off, self.jobs, self.slots = slot_off, jobs, slots
        return self

    def workspace(self, key, nbytes: int) -> torch.Tensor | None:
        """A device buffer of at least ``nbytes`` kept under ``key`` for the
        step.  A larger request under the same key replaces (and frees) the
        earlier buffer, so a caller that keeps an address must key by
        everything the size depends on."""
        if nbytes <= 0:
            return None
        t = self._ws.get(key)
        if t is None or t.numel() < nbytes:
            t = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
            self._ws[key] = t
        return t

    def page_tables(self):
        """(page table [n_cached, max_pages], cached lengths [n_cached]) of the
        state-2 sequences on the device, int32: what attention over 8-bit
        pages reads instead of the slot lists.

        A host-built plan's pages are those of context.slot_mapping, every 256th
        slot's.  The lists must name whole pages, the last one from row 0 on, in any
        order inside a page; lists and CPU tensors are checked, device tensors are
        not (that would wait for the GPU)."""
        if self._pages is None:
            t = self._block_tables
            if t is None:
                t = self._pages_of_slots()
            elif not self.cached_identity:
                t = t.index_select(0, self.cached_ids)
            self._pages = t, self.slot_off[1:] - self.slot_off[:-1]
        return self._pages

    def _pages_of_slots(self) -> torch.Tensor:
        if self._cached_seqs is None:
            raise ValueError("8-bit pages need the sequences' block tables on the device")
        _not_captured("run the step's forward over 8-bit pages once, which uploads its page table,", self.device)
        R = _capi.PAGE_ROWS
        width = max(1, -(-self.max_keep_cached // R))
        at = torch.zeros(self.n_cached, width, dtype=torch.int64)  # past a sequence's pages: not read
        base = 0
        for r, (seq, keep, slots) in enumerate(self._cached_seqs):
            need = -(-keep // R)
            pages = getattr(seq, "block_table", None)
            if pages is not None and len(pages) < need:
                raise ValueError(f"cached sequence {r}: {keep} rows in {len(pages)} pages")
            if not (isinstance(slots, torch.Tensor) and slots.is_cuda):
                a = np.asarray(slots, dtype=np.int64).reshape(-1)
                for j in range(0, keep, R):
                    run = np.sort(a[j:j + R])
                    if run[0] % R or not np.array_equal(run, run[0] + np.arange(run.size)):
                        raise ValueError(f"cached sequence {r}: slots {j} .. {j + run.size - 1} of its slot_mapping are not "
                                         f"the rows of one cache page from row 0 on, which 8-bit pages are read by")
            at[r, :need] = base + R * torch.arange(need)
            base += keep
        if base == 0:
            return torch.full((self.n_cached, width), -1, dtype=torch.int32, device=self.device)
        if self.device.type == "cuda":
            at = at.pin_memory()
        at = at.to(self.device, non_blocking=True)
        return (self.slots.index_select(0, at.view(-1)) >> 8).view(self.n_cached, width)

    def launch_args(self, Hq: int, Hkv: int, D: int, pages: bool = False) -> dict:
        """Device addresses of the step's tables and the workspace of its
        attention over cached rows (K3b, or with ``pages`` the one over 8-bit
        pages) for one head shape, computed once per step for all layers.  The
        workspace is keyed by the head shape and held in the returned dict, so
        the address cached here stays valid while the plan lives, whatever other
        head shapes later ask for."""
        key = (Hq, Hkv, D, "pages") if pages else (Hq, Hkv, D)
        a = self._args.get(key)
        if a is None:
            need = 0
            if self.n_cached and pages:
                need = _capi.chunk_workspace_size(self.n_cached, self.max_q_cached, self.max_keep_cached, Hq, Hkv, D,
                                                  self.rows_cached, self.keeps_cached)
            elif self.n_cached:
                need = _capi.block_cached_workspace_size(self.n_cached, self.max_q_cached, self.max_keys_cached, Hq,
                                                         Hkv, D)
            ws = self.workspace(("cached",) + key, need)
            a = dict(cu=self.cu.data_ptr(), slots=self.slots.data_ptr(), slot_off=self.slot_off.data_ptr(),
                     dense_ids=None if self.dense_identity else self.dense_ids.data_ptr(),
                     cached_ids=None if self.cached_identity else self.cached_ids.data_ptr(),
                     ws=None if ws is None else ws.data_ptr(), ws_bytes=0 if ws is None else ws.numel(),
                     ws_tensor=ws)
            if not (self.any_skipped or self.n_job) and self.device.type == "cuda":
                # the step's launches for the native form (csrc/native.cpp, PlanArgs and PageArgs)
                dev = self.device.index if self.device.index is not None else torch.cuda.current_device()
                packed = struct.pack(
                    "=17q", dev, self.total_rows, Hq, Hkv, D, self.n_dense, self.max_q_dense, a["cu"],
                    a["dense_ids"] or 0, self.n_cached, self.max_q_cached, self.max_keys_cached, a["cached_ids"] or 0,
                    a["slots"], a["slot_off"], a["ws"] or 0, a["ws_bytes"])
                if pages:
                    table, lens = self.page_tables()
                    packed += struct.pack("=6q", self.max_keep_cached, self.rows_cached, self.keeps_cached,
                                          table.data_ptr(), table.shape[1], lens.data_ptr())
                self._packed[key] = packed
            self._args[key] = a
        return a


class Attention(nn.Module):
    """Drop-in for dllmserve.layers.attention.Attention (attention.py:95-119)."""

    keep_indices = os.environ.get("DLLM_KEEP_SELECT_INDICES", "0") == "1"

    def __init__(self, num_heads, head_dim, scale, num_kv_heads, causal=True):
        super().__init__()
        self.num_heads = num_heads
        self.head_dim = head_dim
        self.scale = scale
        self.num_kv_heads = num_kv_heads
        self.causal = causal
        self.k_cache = self.v_cache = torch.tensor([])
        self.layer_id = None
        self.last_select_indices = None
        # (weak references, addresses, sizes, device, result) of the last bound
        # cache that passed _check_cache: weak, so that a cache the runner
        # drops or re-sizes is freed at once, not kept alive by this check
        self._cache_ok = None

    def forward(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> torch.Tensor:
        # q/k/v as [rows, heads * head_dim] or [rows, heads, head_dim] are used
        # without the reference's view (attention.py:108-110); other shapes
        # take that view
        context = get_context()
        if context.is_diffusion:
            # a step whose plan is built and that only attends: one native call
            plan = getattr(context, "_dllm_plan", None)
            if plan is not None:
                o = self._native_attention(plan, q, k, v)
                if o is not None:
                    return o
            return self._mixed_sparse_dense_attention(q, k, v, context)
        raise NotImplementedError(
            "only the diffusion branch (context.is_diffusion=True) is provided; the autoregressive "
            "prefill/decode branch of the reference is unused by diffusion models")

    def _native_attention(self, plan, q, k, v):
        """The step's attention through the native form, or None (see csrc/native.cpp)."""
        key = (self.num_heads, self.num_kv_heads, self.head_dim)
        packed = plan._packed.get(key) or plan._packed.get(key + ("pages",))
        if packed is None or _capi.native is None:
            return None
        return _capi.native.attn(q, k, v, self.k_cache, self.v_cache, packed, float(self.scale))

    def _plan(self, context, device) -> StepPlan:
        plan = getattr(context, "_dllm_plan", None)
        if plan is None or plan.device != device:
            plan = StepPlan(context, device, self.num_kv_heads, self.head_dim, self.num_heads)
            context._dllm_plan = plan
        return plan

    def _check_cache(self, device) -> tuple:
        """Check the bound cache and return (k address, v address, slots).
        The kernels address it as flat bf16 rows of Hkv * head_dim elements on
        q's device (the checks store_kvcache makes, attention.py:42-47); a
        cache that passed keeps passing while the same tensors keep their
        addresses and sizes."""
        kc, vc = self.k_cache, self.v_cache
        key = (kc.data_ptr(), vc.data_ptr(), kc.numel(), vc.numel(), device)
        ok = self._cache_ok
        if ok is not None and ok[0]() is kc and ok[1]() is vc and ok[2:7] == key:
            return ok[7]
        if kc.dtype == torch.uint8:
            if _check_pages(kc, vc, device) != self.num_kv_heads or self.head_dim != 128:
                raise ValueError(f"8-bit pages of {kc.shape[1]} KV heads of 128, the layer has {self.num_kv_heads} of "
                                 f"{self.head_dim}")
            res = (kc.data_ptr(), vc.data_ptr(), min(kc.shape[0], vc.shape[0]) * _capi.PAGE_ROWS)
            self._cache_ok = (weakref.ref(kc), weakref.ref(vc)) + key + (res,)
            return res
        for t, n in ((kc, "k_cache"), (vc, "v_cache")):
            if (t.dtype != torch.bfloat16 or not t.is_contiguous() or t.device != device or t.dim() < 2
                    or tuple(t.shape[-2:]) != (self.num_kv_heads, self.head_dim)):
                raise ValueError(f"{n} must be a contiguous bf16 tensor [..., {self.num_kv_heads}, {self.head_dim}] "
                                 f"on {device}; got {t.dtype} {tuple(t.shape)} on {t.device}")
        res = (kc.data_ptr(), vc.data_ptr(), min(kc.numel(), vc.numel()) // (self.num_kv_heads * self.head_dim))
        self._cache_ok = (weakref.ref(kc), weakref.ref(vc)) + key + (res,)
        return res

    def _mixed_sparse_dense_attention(self, q, k, v, context):
        Hq, Hkv, D = self.num_heads, self.num_kv_heads, self.head_dim
        q, nq, q_st = _token_rows(q, Hq, D, "q")
        k, nk, k_st = _token_rows(k, Hkv, D, "k")
        v, nv, v_st = _token_rows(v, Hkv, D, "v")
        if q.dtype != torch.bfloat16 or k.dtype != torch.bfloat16 or v.dtype != torch.bfloat16:
            raise TypeError(f"bf16 q/k/v expected, got {q.dtype}/{k.dtype}/{v.dtype}")
        if not (q.is_cuda and k.is_cuda and v.is_cuda):
            raise RuntimeError("Attention runs on the GPU only (no CPU fallback)")
        if not (k.get_device() == v.get_device() == q.get_device()):
            raise ValueError(f"q/k/v are on different devices: {q.device}/{k.device}/{v.device}")
        dev = q.device
        plan = self._plan(context, dev)
        if nq != plan.total_rows or nk != plan.total_rows or nv != plan.total_rows:
            raise ValueError(f"q/k/v have {nq}/{nk}/{nv} rows, the step's sequences feed {plan.total_rows}")
        known = len(plan._args)
        args = plan.launch_args(Hq, Hkv, D, bool(plan.n_cached) and self.k_cache.dtype == torch.uint8)
        first = len(plan._args) > known
        if first:  # the step's first layer of this shape: its launch arguments exist only now
            o = self._native_attention(plan, q, k, v)
            if o is not None:
                return o
        o = torch.zeros_like(q) if plan.any_skipped else torch.empty_like(q)
        o_st = o.stride(0)
        stream = _capi._stream(dev)
        qp, kp, vp, op = q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr()

        if plan.n_dense:
            _capi.attn_varlen_fwd_raw(qp, kp, vp, op, args["cu"], args["dense_ids"], plan.n_dense, plan.max_q_dense,
                                      Hq, Hkv, D, q_st, k_st, v_st, o_st, float(self.scale), stream)

        if plan.n_job:
            if not (self.k_cache.numel() and self.v_cache.numel()):
                raise RuntimeError("cache state 1 needs k_cache/v_cache bound to this layer")
            self._check_cache(dev)
            ws = plan.workspace("select", _capi.select_workspace_size(plan.n_job, plan.max_kc, Hq, Hkv, D))
            idx = None
            if self.keep_indices:
                idx = torch.full((plan.n_job, Hkv, plan.max_keep), -1, dtype=torch.int64, device=dev)
            q3 = q if q.dim() == 3 else q.view(-1, Hq, D)
            k3 = k if k.dim() == 3 else k.view(-1, Hkv, D)
            v3 = v if v.dim() == 3 else v.view(-1, Hkv, D)
            _capi.select_kv_store(q3, k3, v3, plan.jobs, plan.n_job, plan.max_kc, plan.max_keep, np.float32(D ** 0.5),
                                  self.k_cache, self.v_cache, plan.slots, idx, ws)
            self.last_select_indices = idx

        if plan.n_cached:
            if not (self.k_cache.numel() and self.v_cache.numel()):
                raise RuntimeError("cache state 2 needs k_cache/v_cache bound to this layer")
            kc, vc, cache_slots = self._check_cache(dev)
            if self.k_cache.dtype == torch.uint8:
                self._attend_pages(plan, args, qp, kp, vp, op, kc, vc, cache_slots, q_st, k_st, v_st, o_st, stream)
                return o if o.dim() == 2 else o.view(-1, Hq * D)
            _capi.attn_block_cached_fwd_raw(qp, kp, vp, op, args["cu"], args["cached_ids"], plan.n_cached,
                                            plan.max_q_cached, plan.max_keys_cached, kc, vc, cache_slots,
                                            args["slots"], args["slot_off"], Hq, Hkv, D, q_st, k_st, v_st, o_st,
                                            float(self.scale), args["ws"], args["ws_bytes"], stream)
        return o if o.dim() == 2 else o.view(-1, Hq * D)

    def _attend_pages(self, plan, args, qp, kp, vp, op, kc, vc, cache_slots, q_st, k_st, v_st, o_st, stream) -> None:
        """The state-2 sequences' blocks against their cached rows in 8-bit pages and against themselves."""
        Hq, Hkv, D = self.num_heads, self.num_kv_heads, self.head_dim
        table, lens = plan.page_tables()
        _capi.attn_chunk_paged_fwd_raw(qp, kp, vp, op, args["cu"], args["cached_ids"], plan.n_cached,
                                       plan.max_q_cached, plan.max_keep_cached, plan.rows_cached, plan.keeps_cached,
                                       kc, vc, _capi.CACHE_FP8, cache_slots // _capi.PAGE_ROWS, table.data_ptr(),
                                       table.shape[1], lens.data_ptr(), 0, Hq, Hkv, D, q_st, k_st, v_st, o_st,
                                       float(self.scale), args["ws"], args["ws_bytes"], stream)
