"""Oracle: the 8-bit paged KV cache and attention over it (numpy; no reference counterpart).

The cache is kept here by position, not by layout: codes as the values they stand for before scaling,
one exponent a tile of 16 tokens and KV head. Codes and exponents follow the definition exactly, with the
rotation in fp32 (each product and sum rounded once); attention is computed in 64 bits.
"""

from __future__ import annotations

import numpy as np

TILE = 16


def rotate(x: np.ndarray, bias: np.ndarray | None, cos: np.ndarray | None, sin: np.ndarray | None,
           positions: np.ndarray, style: int) -> np.ndarray:
    """fp32 x [tokens, heads, D] (+ bias [heads, D]), rotated."""

    x = np.asarray(x, np.float32)
    if bias is not None:
        x = x + np.asarray(bias, np.float32)
    if style == 0:
        return x
    c, s = cos[positions][:, None, :], sin[positions][:, None, :]
    out = np.empty_like(x)
    half = x.shape[-1] // 2
    a, b = (slice(0, half), slice(half, None)) if style == 1 else (slice(0, None, 2), slice(1, None, 2))
    with np.errstate(invalid="ignore", over="ignore"):
        out[..., a] = x[..., a] * c - x[..., b] * s
        out[..., b] = x[..., b] * c + x[..., a] * s
    return out


def round_e4m3(x: np.ndarray) -> np.ndarray:
    """|x| <= 448 rounded to e4m3, ties to even; infinities and NaN give NaN."""

    x = np.asarray(x, np.float64)
    finite = np.isfinite(x)
    y = np.where(finite, x, 0.0)
    _, e = np.frexp(np.maximum(np.abs(y), 2.0 ** -6))
    step = np.ldexp(1.0, e - 4)
    return np.where(finite, np.rint(y / step) * step, np.nan)


def tile_exponent(x: np.ndarray) -> int:
    """The exponent of the smallest power of two (2**-126 at least) that brings x's finite values within 448."""

    a = np.abs(np.asarray(x, np.float64))
    a = a[np.isfinite(a)]
    top = float(a.max(initial=0.0))
    if top == 0.0:
        return -126
    m, e = np.frexp(top)  # top = m * 2**e, 448 = 0.875 * 2**9
    return max(int(e) - (9 if m <= 0.875 else 8), -126)


class Cache:
    """Codes [layers, 2, tiles, Hkv, 16, D] and exponents [layers, 2, tiles, Hkv]; tile = slot // 16."""

    def __init__(self, codes: np.ndarray, exponents: np.ndarray) -> None:
        self.codes, self.exponents = codes.astype(np.float64), exponents.astype(np.int64)

    def append(self, layer: int, slot: int, k: np.ndarray, v: np.ndarray, steps: np.ndarray | None = None) -> None:
        """Tokens k, v [n, Hkv, D] (fp32) of one tile, the first at ``slot`` and the others ``steps`` (0, ..) behind
        it; consecutive without."""

        tile, off = slot // TILE, slot % TILE
        at = off + (np.arange(len(k)) if steps is None else steps)
        assert at[0] == off and at[-1] < TILE
        for plane, x in enumerate((k, v)):
            for h in range(x.shape[1]):
                code, old = self.codes[layer, plane, tile, h], self.exponents[layer, plane, tile, h]
                new = tile_exponent(x[:, h])
                if off:
                    new = max(new, old)
                    if new != old:
                        code[:off] = round_e4m3(np.ldexp(code[:off], old - new))
                code[at] = round_e4m3(np.ldexp(x[:, h].astype(np.float64), -new))
                self.exponents[layer, plane, tile, h] = new

    def write(self, layer: int, rows: np.ndarray, k: np.ndarray, v: np.ndarray) -> None:
        """A batch of tokens at slots ``rows`` (negative: left out), a tile's tokens next to each other."""

        t = 0
        while t < len(rows):
            if rows[t] < 0:
                t += 1
                continue
            run, n = [0], 1
            while t + n < len(rows) and rows[t] % TILE + n < TILE and rows[t + n] in (rows[t] + n, -1):
                run += [n] if rows[t + n] >= 0 else []
                n += 1
            steps = np.array(run)
            self.append(layer, int(rows[t]), k[t + steps], v[t + steps], steps)
            t += n

    def values(self, layer: int, plane: int, slots: np.ndarray) -> np.ndarray:
        """[len(slots), Hkv, D] in 64 bits."""

        tile, off = slots // TILE, slots % TILE
        e = self.exponents[layer, plane][tile]  # [n, Hkv]
        return np.ldexp(self.codes[layer, plane][tile, :, off], e[..., None])


def attend(q: np.ndarray, k: np.ndarray, v: np.ndarray, end: np.ndarray, scale: float, round_off: float,
           score_off: float, prob_off: float, floor: float = 0.0, top_off: float = 0.0
           ) -> tuple[np.ndarray, np.ndarray]:
    """Attention of q [n, H, D] over k, v [tokens, Hkv, D] in 64 bits, query i over keys 0..end[i], and a bound on
    what a computation may be off by whose scores are off by at most
    d = scale * sum_d (score_off |q_d| + top_off max|q|) |k_d|,
    whose probabilities and sums are off by the relative ``prob_off`` besides, and whose results are rounded by
    the relative ``round_off``; ``floor`` is what each probability may be off by at any size, the largest being 1.

    Scores off by at most d move each p_i / sum(p) by a factor within exp(+-2 d); so
    |error| <= round_off |o| + (1 + round_off) (exp(2 d + prob_off) - 1) sum_i p_i |v_i| + floor sum_i |v_i|.
    """

    n, heads, dim = q.shape
    group = heads // k.shape[1]
    out, bound = np.zeros((n, heads, dim)), np.zeros((n, heads, dim))
    for h in range(heads):
        kh, vh = k[:, h // group], v[:, h // group]
        s = q[:, h] @ kh.T * scale
        size = np.abs(q[:, h])
        mass = (score_off * size + top_off * size.max(1, keepdims=True)) @ np.abs(kh).T * scale
        seen = np.arange(len(kh))[None, :] <= end[:, None]
        for i in range(n):
            ks = seen[i]
            p = np.exp(s[i, ks] - s[i, ks].max())
            p /= p.sum()
            o = p @ vh[ks]
            d = mass[i, ks].max()
            out[i, h] = o
            bound[i, h] = round_off * np.abs(o) + (1 + round_off) * np.expm1(2 * d + prob_off) * (p @ np.abs(vh[ks]))
            bound[i, h] += floor * np.abs(vh[ks]).sum(0)
    return out, bound
