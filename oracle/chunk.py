"""Attention of a chunk of new rows over cached rows and over itself, in float64.

New row t of a sequence with n cached rows stands at position n + t.  It sees the
cached rows and, of the L new ones, all (mask_block 0) or those whose position lies
before the end of its own block of mask_block positions.  Scores that are NaN make the
row NaN; rows whose scores are all -infinity are zeros.
"""
from __future__ import annotations

import numpy as np


def visible(n: int, L: int, t: int, mask_block: int) -> int:
    return L if mask_block == 0 else min(L, ((n + t) // mask_block + 1) * mask_block - n)


def attend(q, k, v, kc, vc, scale: float, mask_block: int = 0, keep=None):
    """q [L, Hq, D], k / v [L, Hkv, D], kc / vc [n, Hkv, D]; keep: which cached
    rows take part.  Returns (o, spread, reach) of [L, Hq, D], [L, Hq, D] and [L, Hq]:
    the outputs, sum_u p_u |v_u| and max_u sum_d |q_d k_ud| * scale, which an error
    bound of a computation in fewer bits needs."""
    q, k, v, kc, vc = (np.asarray(x, dtype=np.float64) for x in (q, k, v, kc, vc))
    L, Hq, D = q.shape
    n, g = kc.shape[0], Hq // k.shape[1]
    rows = np.arange(n) if keep is None else np.nonzero(keep)[0]
    o, spread, reach = np.zeros((L, Hq, D)), np.zeros((L, Hq, D)), np.zeros((L, Hq))
    for t in range(L):
        see = visible(n, L, t, mask_block)
        for h in range(Hq):
            kk = np.concatenate([kc[rows, h // g], k[:see, h // g]])
            vv = np.concatenate([vc[rows, h // g], v[:see, h // g]])
            with np.errstate(invalid="ignore", over="ignore"):
                s = kk @ q[t, h] * scale
                top = s.max() if not np.isnan(s).any() else np.nan
                if top == -np.inf:
                    continue
                p = np.exp(s - top)
                p /= p.sum()
                o[t, h] = p @ vv
                spread[t, h] = p @ np.abs(vv)
                reach[t, h] = (np.abs(kk) @ np.abs(q[t, h])).max() * scale
    return o, spread, reach
