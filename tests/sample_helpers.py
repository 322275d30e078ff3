"""ca_sample's definition in 64 bits, row by row, for its tests."""
from __future__ import annotations

import numpy as np

STEP = 2.0 ** -44  # weights are whole numbers of these


def sample_ref(row, u, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, dead=()):
    """(token, prob, slack) of one row of fp32 values: `slack` is how far, as a
    weight, the nearest border is from the number that decides on it."""
    x = np.asarray(row, dtype=np.float64).copy()
    x[np.isnan(x)] = -np.inf
    for i in dead:
        if 0 <= i < len(x):
            x[i] = -np.inf
    m = x.max()
    if m == -np.inf:
        return 0, 0.0, np.inf
    with np.errstate(invalid="ignore"):
        one = np.where(x == m, 1.0, np.exp(x - m))
        slack = np.inf
        if not temperature > 0:
            token = int(np.argmax(x == m))
        else:
            t = float(np.float32(temperature))
            w = np.where(x == m, 1.0, np.where(x == -np.inf, 0.0, np.exp((x - m) / t)))
            order = np.lexsort((np.arange(len(x)), -x))  # value descending, index ascending
            ws = w[order]
            keep = np.ones(len(x), dtype=bool)
            if top_k > 0:
                keep[top_k:] = False
            if top_p < 1:
                p = max(float(np.float32(top_p)), 0.0)
                before = np.concatenate([[0.0], np.cumsum(ws)[:-1]])
                need = p * ws[keep].sum()
                # Entries of no weight may be kept or not: they are never drawn.
                real = keep & (ws > 4 * STEP)
                real[0] = False
                if real.any():
                    slack = min(slack, np.abs(before[real] - need).min())
                keep &= before < need
            if min_p > 0:
                least = min(float(np.float32(min_p)), 1.0)
                slack = min(slack, np.abs(ws[1:] - least)[ws[1:] != ws[0]].min(initial=np.inf))
                keep &= ws >= least
            keep[0] = True
            kept = np.zeros(len(x), dtype=bool)
            kept[order[keep]] = True
            cum = np.cumsum(np.where(kept, w, 0.0))
            u = float(np.float32(u))
            u = min(u, 1 - 2.0 ** -24) if u >= 0 else 0.0
            target = u * cum[-1]
            token = int(np.argmax(cum > target))
            if u > 0:
                slack = min(slack, np.abs(cum - target).min())
        return token, float(one[token] / one.sum()), slack
