"""The checks of test_gpu_chunk_keys on the CPU: they pass the formula, and fail it with one
mistake planted at a time."""
import pytest
import torch

import test_gpu_chunk_keys as keys

N = 1700


def _formula(weight=lambda row, n_keys: torch.ones(n_keys), order=lambda key: key, hide=True):
    """chunk_attention in 64 bits; weight: how often a row's keys count, order: which key is read."""
    def attend(q, k, v, kc, vc, plan, scale):
        m, cur = attend.of, 0
        g = m.Hq // m.Hkv
        out = torch.zeros(m.n, m.Hq, 128, dtype=torch.float64)
        for b, (L, n) in enumerate(zip(m.lens, m.cached)):
            slots = torch.tensor([m.tables[b][r // 256] * 256 + r % 256 for r in range(n)], dtype=torch.int64)
            kk, vv = (torch.cat([c.view(-1, m.Hkv, 128)[slots], x[cur:cur + L]]).double()[order(torch.arange(n + L))]
                      for c, x in ((kc, k), (vc, v)))
            for t in range(L):
                see = n + (m.sees(n, L, t) if hide else L)
                for h in range(m.Hq):
                    s = kk[:see, h // g] @ q[cur + t, h].double() * scale
                    p = torch.exp(s - s.max()) * weight(t, n + L)[:see].double()
                    out[cur + t, h] = p @ vv[:see, h // g] / p.sum()
            cur += L
        return out.to(torch.bfloat16).view(m.n, -1)
    return attend


def _run(monkeypatch, **planted):
    m = keys.Marked("cpu", [4], [N], 16, 2, 16, seed=63)
    attend = _formula(**planted)
    attend.of = m
    monkeypatch.setattr(keys, "chunk_attention", attend)
    m.all_of(keys._borders(N, 4))
    m.hidden(2)


def test_the_formula_passes(monkeypatch):
    _run(monkeypatch)


def _times(lo, hi, w):
    def weight(row, n):
        x = torch.ones(n)
        x[lo:hi] = w
        return x
    return weight


def _moved(key):
    key = key.clone()
    key[256:288] += 32
    return key


@pytest.mark.parametrize("planted", [
    dict(weight=_times(1696, 1700, 0)),       # the last tile of the cache left out
    dict(weight=_times(1535, 1536, 0)),       # one row
    dict(weight=_times(256, 512, 2)),         # a part joined twice
    dict(weight=_times(1703, 1704, 0)),       # a new row that only the last row sees
    dict(order=_moved),                       # a tile read from the next one's place
    dict(hide=False),                         # new rows seen too early
])
def test_one_mistake_fails(monkeypatch, planted):
    with pytest.raises(AssertionError):
        _run(monkeypatch, **planted)
