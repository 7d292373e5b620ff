"""One token a row from its logits and a given number, in float64 (the definition that ``cdb_sample`` follows)."""

from __future__ import annotations

import math

import numpy as np


def order(logits: np.ndarray) -> np.ndarray:
    """Tokens that can be drawn: larger logits first, the lower index among equals; -inf and NaN left out."""

    x = np.asarray(logits, dtype=np.float64)
    x = np.where(np.isnan(x), -np.inf, x) + 0.0
    idx = np.argsort(-x, kind="stable")
    return idx[x[idx] > -np.inf]


def kept(logits: np.ndarray, temperature: float = 1.0, top_k: int = 0, top_p: float = 1.0,
         min_p: float = 0.0) -> tuple[np.ndarray, np.ndarray]:
    """(tokens, weights) that the filters keep, in the order of ``order``."""

    x = np.asarray(logits, dtype=np.float64)
    idx = order(x)
    if idx.size == 0 or not temperature > 0:
        return idx[:1], np.ones(min(idx.size, 1))
    if 0 < top_k:
        idx = idx[:top_k]
    top = x[idx[0]]
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(x[idx] == top, 1.0, 0.0 if math.isinf(top) else np.exp((x[idx] - top) / temperature))
    if top_p < 1:
        before = np.cumsum(w) - w
        n = max(1, int((before < top_p * w.sum()).sum()))
        idx, w = idx[:n], w[:n]
    n = int((w >= min(min_p, 1.0)).sum())
    return idx[:n], w[:n]


def draw(logits: np.ndarray, u: float, temperature: float = 1.0, top_k: int = 0, top_p: float = 1.0,
         min_p: float = 0.0) -> tuple[int, float]:
    """(token, log-probability); (-1, -inf) where nothing can be drawn."""

    idx, w = kept(logits, temperature, top_k, top_p, min_p)
    if idx.size == 0:
        return -1, -math.inf
    by_index = np.argsort(idx)
    idx, w = idx[by_index], w[by_index]
    run = np.cumsum(w)
    u = min(max(u, 0.0), 1.0)
    n = min(int(np.searchsorted(run, u * run[-1], side="right")), int(np.flatnonzero(w).max()))
    return int(idx[n]), math.log(w[n] / run[-1])
