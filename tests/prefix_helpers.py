"""Batches of rows that share prefixes, and their attention in float64."""

from __future__ import annotations

import math
from types import SimpleNamespace

import numpy as np
import torch

from continuous_depth_batching_amd import ops


def make(group, lengths, own, *, heads=8, kv=4, dim=64, dtype=torch.bfloat16, rope=1, bias=False, block=16, layers=2,
         layer0=0, padding=(), seed=0, device="cuda", extra_blocks=3, scale_q=1.0, shuffle_rows=False, dead=float("nan")):
    """Rows ``b`` of group ``group[b]`` with ``own[b]`` >= 1 tokens of their own, the new one among them. Slots of the
    pool that hold no token of a row are ``dead``."""

    rng = np.random.default_rng(seed)
    gen = torch.Generator().manual_seed(seed)
    group, lengths, own = (np.asarray(a, dtype=np.int64) for a in (group, lengths, own))
    rows = group.size
    start = np.where(group >= 0, lengths[group] if lengths.size else 0, 0)
    pos = start + own - 1
    need, shared = -(-(pos + 1) // block), start // block
    held = -(-lengths // block)
    total = int(held.sum() + (need - shared).sum()) + extra_blocks
    ids = rng.permutation(total)
    at = np.concatenate([[0], np.cumsum(held)])
    used = int(at[-1])
    width = int(need.max(initial=1)) + 1
    table = np.full((rows, width), -1, dtype=np.int64)
    pool = torch.full((layers, 2, total * block, kv, dim), dead)
    layer = np.where(group >= 0, group, np.arange(rows)) % (layers - layer0)

    def randn(*shape):
        return torch.randn(*shape, generator=gen)

    for n, length in enumerate(lengths):
        if length and (group == n).any():
            slots = (ids[at[n] + np.arange(length) // block] * block + np.arange(length) % block)
            l = layer0 + int(layer[np.flatnonzero(group == n)[0]])
            pool[l][:, slots] = randn(2, int(length), kv, dim)
    for b in range(rows):
        s, n = int(shared[b]), int(need[b])
        if group[b] >= 0:
            table[b, :s] = ids[at[group[b]]:at[group[b]] + s]
        table[b, s:n] = ids[used:used + n - s]
        used += n - s
        l, tail = layer0 + int(layer[b]), int(start[b] % block)
        if tail:  # the row's copy of the block in which the prefix ends
            of = int(ids[at[group[b] + 1] - 1]) * block
            pool[l][:, table[b, s] * block + np.arange(tail)] = pool[l][:, of + np.arange(tail)]
        t = np.arange(int(start[b]), int(pos[b]))
        if t.size:
            pool[l][:, table[b, t // block] * block + t % block] = randn(2, t.size, kv, dim)
    fused = randn(rows, (heads + 2 * kv) * dim)
    fused[:, :heads * dim] *= scale_q
    fused = fused.to(dtype).to(device)
    q, k, v = fused.split([heads * dim, kv * dim, kv * dim], dim=1)
    table_row = None
    if shuffle_rows:
        table_row = rng.permutation(rows + 2)[:rows]
        spread = np.full((rows + 2, width), -1, dtype=np.int64)
        spread[table_row] = table
        table = spread
    seq = pos.copy()
    seq[list(padding)] = -1
    cos = sin = None
    if rope:
        inv = 10000.0 ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
        ang = torch.arange(int(pos.max(initial=0)) + 1, dtype=torch.float64)[:, None] * inv
        cos, sin = ang.cos().float().to(device), ang.sin().float().to(device)

    def ints(a):
        return None if a is None else torch.as_tensor(np.asarray(a), dtype=torch.int32).to(device)

    plan = ops.prefix_decode_plan(group, lengths, num_heads=heads, num_kv_heads=kv)
    nbytes = ops.prefix_decode_workspace_bytes(plan, heads, kv, dim, int(own.max(initial=1)))
    return SimpleNamespace(
        q=q.view(rows, heads, dim), k=k.view(rows, kv, dim), v=v.view(rows, kv, dim), pool=pool.to(dtype).to(device),
        block=block, layer=ints(layer), layer0=layer0, table=ints(table), table_row=ints(table_row), seq=ints(seq),
        cos=cos, sin=sin, rope=rope, q_bias=(0.2 * randn(heads, dim)).to(dtype).to(device) if bias else None,
        k_bias=(0.2 * randn(kv, dim)).to(dtype).to(device) if bias else None, host_plan=plan, plan=plan.to(device),
        workspace=torch.empty(nbytes, dtype=torch.uint8, device=device), scale=dim ** -0.5, start=start,
        group=group, lengths=lengths)


def call(s, out=None, plan=None, workspace=None):
    out = torch.empty(s.q.shape, dtype=s.q.dtype, device=s.q.device) if out is None else out
    return ops.prefix_decode_attention_raw(
        s.q, s.k, s.v, ops.KVPoolView(s.pool, s.block), s.layer, s.layer0, s.table, s.table_row, s.seq, s.cos, s.sin,
        s.rope, s.q_bias, s.k_bias, plan or s.plan, out, workspace if workspace is not None else s.workspace, s.scale)


def turned(x, bias, s):
    """[rows, heads, D] float64 on the host: x + bias, rotated to the rows' positions."""

    x = x.double().cpu()
    if bias is not None:
        x = x + bias.double().cpu()
    if not s.rope:
        return x
    p = s.seq.cpu().long().clamp(min=0)
    c, n = s.cos.double().cpu()[p][:, None], s.sin.double().cpu()[p][:, None]
    h = x.shape[-1] // 2
    y = torch.empty_like(x)
    a, b = (slice(0, h), slice(h, None)) if s.rope == 1 else (slice(0, None, 2), slice(1, None, 2))
    y[..., a] = x[..., a] * c - x[..., b] * n
    y[..., b] = x[..., b] * c + x[..., a] * n
    return y


def check(s, out, before):
    """Outputs and cache after a call, against the pool ``before`` it; bounds from the roundings that are made.

    Keys: fp32 rotation (3 roundings of terms up to |a| + |b|), one rounding to storage. Scores: queries in two bf16
    parts leave 2^-16 of an element, fp32 sums D + 3 roundings of 2^-24 of the terms' sizes; an error d of the scores
    (in log2) changes weights, and with them the result, by at most 2 ln2 d of the mean |v|, P in two bf16 parts by
    2 * 2^-16 of it. Sums of n weights: n / 4 + 64 roundings. The result is rounded once."""

    low = s.q.dtype is torch.bfloat16
    half = torch.finfo(s.q.dtype).eps / 2
    rows, heads, dim = s.q.shape
    kv = s.k.shape[1]
    q = turned(s.q, s.q_bias, s)
    k = turned(s.k, s.k_bias, s)
    size = turned(s.k.abs(), None if s.k_bias is None else s.k_bias.abs(), SimpleNamespace(
        seq=s.seq, rope=s.rope, cos=None if s.cos is None else s.cos.abs(),
        sin=None if s.sin is None else -s.sin.abs()))
    size2 = turned(s.k.abs(), None if s.k_bias is None else s.k_bias.abs(), SimpleNamespace(
        seq=s.seq, rope=s.rope, cos=None if s.cos is None else s.cos.abs(),
        sin=None if s.sin is None else s.sin.abs())).abs()
    size = torch.maximum(size.abs(), size2)
    pool, was, out = s.pool.cpu(), before.cpu(), out.double().cpu()
    table, layer, seq = s.table.cpu().numpy(), s.layer.cpu().numpy(), s.seq.cpu().numpy()
    trow = np.arange(rows) if s.table_row is None else s.table_row.cpu().numpy()
    changed = was.clone()
    for b in range(rows):
        p = int(seq[b])
        if p < 0:
            assert (out[b] == 0).all()
            continue
        l = s.layer0 + int(layer[b])
        t = np.arange(p + 1)
        slots = torch.from_numpy(table[trow[b], t // s.block].astype(np.int64) * s.block + t % s.block)
        new = pool[l][:, slots[-1]].double()
        assert ((new[0] - k[b]).abs() <= half * k[b].abs() + 2.0 ** -21 * size[b]).all(), b
        assert torch.equal(pool[l][1, slots[-1]], s.v[b].cpu())
        changed[l][:, slots[-1]] = pool[l][:, slots[-1]]
        keys, values = pool[l][0, slots].double(), pool[l][1, slots].double()
        qb = q[b].view(kv, heads // kv, dim)
        score = torch.matmul(qb, keys.permute(1, 2, 0)) * (s.scale * math.log2(math.e))
        terms = torch.matmul(qb.abs(), keys.abs().permute(1, 2, 0)).amax(-1, keepdim=True) * s.scale * 1.4427
        w = torch.softmax(score * math.log(2.0), dim=-1)
        want = torch.matmul(w, values.transpose(0, 1))
        mean = torch.matmul(w, values.abs().transpose(0, 1))
        d = terms * ((2.0 ** -16 if low else 0.0) + (dim + 8) * 2.0 ** -24) + score.abs().amax(-1, True) * 2.0 ** -22
        slack = 2 * math.log(2.0) * d * (1 + d) + (2.0 ** -15 if low else 0.0) + (p / 4 + 64) * 2.0 ** -24
        bound = half * want.abs() + slack * mean * (1 + half)
        err = (out[b].view_as(want) - want).abs()
        assert (err <= bound).all(), (b, p, float((err / bound).max()))
    same = (pool == changed) | (pool.isnan() & changed.isnan())
    assert same.all(), "a slot changed that holds no new token"
