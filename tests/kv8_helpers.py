"""Inputs, layout and oracle calls shared by the 8-bit KV cache tests."""

from __future__ import annotations

import numpy as np
import torch

from continuous_depth_batching_amd import kv8
from oracle import kv8 as oracle

TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
SEED_SCALES = (118, 124)  # scale bytes of a pool in use


def rope_tables(dim: int, positions: int) -> tuple[np.ndarray, np.ndarray]:
    f = np.arange(positions)[:, None] * 10000.0 ** (-np.arange(0, dim, 2) / dim)[None, :]
    return np.cos(f).astype(np.float32), np.sin(f).astype(np.float32)


def pack(codes: np.ndarray, block_size: int) -> torch.Tensor:
    """Oracle codes [layers, 2, tiles, Hkv, 16, D] in the pool's layout."""

    layers, _, tiles, heads, _, dim = codes.shape
    x = torch.from_numpy(codes).float().to(torch.float8_e4m3fn).view(torch.uint8)
    nt = block_size // 16
    x = x.view(layers, 2, tiles // nt, nt, heads, 16, dim).permute(0, 1, 2, 4, 3, 5, 6)
    k = x[:, 0].unflatten(-1, (dim // 16, 16)).transpose(-3, -2).flatten(-3)
    v = x[:, 1].unflatten(-2, (4, 4)).transpose(-2, -1).flatten(-3)
    return torch.stack([k, v], dim=1).contiguous().view(torch.float8_e4m3fn)


def unpack(pool: kv8.Kv8Pool) -> tuple[np.ndarray, np.ndarray]:
    """The pool's codes [layers, 2, tiles, Hkv, 16, D] (as values) and exponents [layers, 2, tiles, Hkv]."""

    dim = pool.head_dim
    x = pool.codes.cpu().float()
    k = x[:, 0].unflatten(-1, (dim // 16, 16, 16)).transpose(-3, -2).flatten(-2)
    v = x[:, 1].unflatten(-1, (4, dim, 4)).transpose(-2, -1).flatten(-3, -2)
    y = torch.stack([k, v], dim=1).permute(0, 1, 2, 4, 3, 5, 6).flatten(2, 3)
    e = pool.scales.cpu().int().permute(0, 1, 2, 4, 3).flatten(2, 3) - 127
    return y.numpy().astype(np.float64), e.numpy()


def random_pool(rng: np.random.Generator, layers: int, blocks: int, block_size: int, heads: int, dim: int,
                device: str, *, nan_codes: bool = False) -> tuple[kv8.Kv8Pool, oracle.Cache]:
    """A pool in use and its oracle; with ``nan_codes`` a sprinkling of NaN codes over all of it."""

    tiles = blocks * (block_size // 16)
    codes = oracle.round_e4m3(np.clip(rng.standard_normal((layers, 2, tiles, heads, 16, dim)) * 90, -448, 448))
    if nan_codes:
        codes[rng.random(codes.shape) < 0.02] = np.nan
    bytes_ = rng.integers(*SEED_SCALES, size=(layers, 2, tiles, heads))
    nt = block_size // 16
    scales = torch.from_numpy(bytes_.astype(np.uint8)).view(layers, 2, blocks, nt, heads).transpose(3, 4).contiguous()
    pool = kv8.Kv8Pool(pack(codes, block_size).to(device), scales.to(device))
    return pool, oracle.Cache(codes, bytes_ - 127)


def tables(rng: np.random.Generator, tokens: np.ndarray, block_size: int, spare: int = 2
           ) -> tuple[np.ndarray, int]:
    """A block table of randomly placed blocks for ``tokens`` tokens a row, and the pool's block count."""

    blocks = -(-np.asarray(tokens) // block_size)
    perm = rng.permutation(int(blocks.sum()) + spare).astype(np.int32)
    table = np.full((len(blocks), max(1, int(blocks.max()) + 1)), -1, dtype=np.int32)
    at = 0
    for s, n in enumerate(blocks):
        table[s, :n] = perm[at:at + n]
        at += int(n)
    return table, int(blocks.sum()) + spare


def slots(table_row: np.ndarray, positions: np.ndarray, block_size: int) -> np.ndarray:
    return table_row[positions // block_size].astype(np.int64) * block_size + positions % block_size


def values(rng: np.random.Generator, dtype: str, *shape: int, std: float = 1.0) -> torch.Tensor:
    return torch.from_numpy(rng.standard_normal(shape, dtype=np.float32) * np.float32(std)).to(TYPES[dtype])


def same_cache(pool: kv8.Kv8Pool, cache: oracle.Cache) -> None:
    codes, exponents = unpack(pool)
    np.testing.assert_array_equal(exponents, cache.exponents)
    np.testing.assert_array_equal(codes, cache.codes)  # NaN equals NaN here


def close(got: torch.Tensor, want: np.ndarray, bound: np.ndarray) -> None:
    g = got.detach().cpu().double().numpy()
    np.testing.assert_array_equal(np.isnan(g), np.isnan(want))
    ok = np.isnan(want) | (np.abs(g - want) <= bound)
    assert ok.all(), f"{(~ok).sum()} of {ok.size} off, worst {np.nanmax(np.abs(g - want) / bound):.3g} of the bound"
