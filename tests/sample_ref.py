"""The choice of lc_sample in float64 (numpy only, from the formulas in include/lucciola_attn.h)."""
from __future__ import annotations

import numpy as np

NONE = 0xffffffff


def choose(x, rand, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, margin): the choice for the logits x (float64), and how far, as a share of the
    weight, the draw and the top-p cut stay from a border at least."""
    x = np.where(x > -1e30, x, -np.inf)
    order = np.argsort(-x, kind="stable")
    order = order[x[order] > -np.inf]
    if len(order) == 0:
        return NONE, 1.0
    if not temperature > 0:
        return int(order[0]), 1.0
    top = x[order]
    with np.errstate(all="ignore"):
        w = np.exp(np.where(top == top[0], 0.0, (top - top[0]) / temperature))
    if top_k > 0:
        w = w[:top_k]
    margin = 1.0
    if top_p < 1:
        c = np.cumsum(w)
        need = top_p * c[-1]
        margin = np.abs(c - need).min() / c[-1]
        w = w[:max(1, int((c < need).sum()) + 1)]
    if min_p > 0:
        w = w[:max(1, int((w >= min_p).sum()))]
    c = np.cumsum(w)
    goal = rand * c[-1]
    if goal > 0:
        margin = min(margin, np.abs(c - goal).min() / c[-1])
    at = min(int((c <= goal).sum()) if goal > 0 else 0, len(w) - 1)
    while w[at] == 0:  # rand at its upper end
        at -= 1
    return int(order[at]), margin
