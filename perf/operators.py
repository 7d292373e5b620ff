"""Timed cases of the operators around an 8-bit paged KV cache.

The cache holds keys and values in tiles of 16 tokens of one KV head: e4m3 codes and one power-of-two
scale a tile, kept as its biased exponent (a byte b stands for 2 ** (b - 127)), keys and values apart:

* codes   ``[layers, 2, blocks, kv heads, block / 16, 16 * dim]``; a key tile lies as
  ``[dim / 16][16 tokens][16]``, a value tile as ``[4][dim][4 tokens]``;
* scales  ``[layers, 2, blocks, kv heads, block / 16]``.

A tile's scale is the smallest power of two that keeps its largest finite magnitude within 448. Tokens
appended to a tile that holds earlier ones keep the larger of both scales, and where it grows the earlier
codes are rounded again; a tile written from its first token starts anew. Codes behind the last written
token stay as they are. Rotations are computed in fp32 and not rounded before they are coded.

Four operators:

* ``decode``   one new token a row: rotate, append to the cache, attend over all of the row's tokens;
* ``prefill``  causal attention of prompt chunks over [cached | new] tokens already in the cache;
* ``write``    rotation and quantising cache write of prompt chunks (or of a decode batch's tokens);
* ``layout``   block tables, slot maps and attention tiles from the requests' cached and new lengths.

Lengths are spread evenly over the logarithm of a range, in an order drawn from the seed, so a case's work
does not depend on the seed.
"""

import math

import numpy as np
import torch

own = False

DEV = "cuda"
TILE = 16
QUERIES = 128  # query tokens of one attention tile
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
FP8 = torch.float8_e4m3fn


def listed():
    return [
        # The tail of a generation: one sequence left, bound by latency.
        dict(name="decode_row1", kind="decode", dtype="bf16", heads=16, kv=16, dim=128, rope=1, bias=False, rows=1,
             lo=900, hi=900, block=16, layers=1),
        # The headline decode launch: 256 sequences mid-way through their lengths, rows at two loop depths.
        dict(name="decode_rows256", kind="decode", dtype="bf16", heads=16, kv=16, dim=128, rope=1, bias=False, rows=256,
             lo=32, hi=2048, block=16, layers=2),
        # Few sequences with long histories and query heads that share a KV head.
        dict(name="decode_shared_long", kind="decode", dtype="bf16", heads=32, kv=8, dim=128, rope=1, bias=False,
             rows=21, lo=4096, hi=32768, block=64, layers=1),
        # A small fp32 batch of narrow heads.
        dict(name="decode_f32", kind="decode", dtype="f32", heads=12, kv=12, dim=64, rope=2, bias=True, rows=33, lo=5,
             hi=1500, block=32, layers=1),
        # The first prefill batch: fresh prompts of all lengths under an 8192-token budget.
        dict(name="prefill_fresh", kind="prefill", dtype="bf16", heads=16, kv=16, dim=128, seqs=24, lo=24, hi=1300,
             past=0, block=16),
        # Chunks of long prompts: a few new tokens after a long cached history.
        dict(name="prefill_history", kind="prefill", dtype="bf16", heads=16, kv=16, dim=128, seqs=4, lo=100, hi=128,
             past=16000, block=16),
        # Two long documents, query heads sharing KV heads.
        dict(name="prefill_long", kind="prefill", dtype="bf16", heads=32, kv=8, dim=128, seqs=2, lo=6000, hi=8190,
             past=0, block=64),
        # The cache write of the first prefill batch.
        dict(name="write_fresh", kind="write", dtype="bf16", heads=16, kv=16, dim=128, rope=1, bias=False, seqs=24,
             lo=24, hi=1300, past=0, block=16),
        # One new token of each of 61 sequences, most of them into a tile that holds earlier tokens.
        dict(name="write_tokens61", kind="write", dtype="bf16", heads=16, kv=16, dim=128, rope=1, bias=False, seqs=61,
             lo=1, hi=1, past=777, block=16),
        # Chunks that start inside a tile, at the wide shape with interleaved rotation and biases, in fp32.
        dict(name="write_wide_f32", kind="write", dtype="f32", heads=55, kv=55, dim=96, rope=2, bias=True, seqs=5,
             lo=37, hi=900, past=133, block=32),
        # The layout of one prefill batch.
        dict(name="layout_prompts", kind="layout", seqs=24, lo=24, hi=1300, past=0, block=16),
        # Chunked prompts and single tokens of many requests together.
        dict(name="layout_many", kind="layout", seqs=1000, lo=1, hi=1024, past=4000, block=16),
    ]


def _spread(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["decode", "decode", "prefill", "prefill", "write", "layout"])
    block = rng.choice([16, 16, 32, 64])
    if kind == "layout":
        hi = _spread(rng, 1, 2000)
        seqs = max(1, min(_spread(rng, 1, 1000), 150_000 // hi))
        return dict(kind=kind, seqs=seqs, lo=_spread(rng, 1, hi), hi=hi, past=rng.choice([0, _spread(rng, 1, 4000)]),
                    block=block)
    dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
    heads, kv = rng.choice([(16, 16), (16, 16), (55, 55), (32, 8), (12, 12), (28, 4), (8, 1), (5, 5)])
    dim = 96 if heads == 55 else rng.choice([64, 96, 128, 128, 128])
    rope, bias = rng.choice([(1, False), (2, True), (1, True), (0, False)])
    shape = dict(kind=kind, dtype=dtype, heads=heads, kv=kv, dim=dim)
    if kind == "decode":
        hi = _spread(rng, 16, 16000)
        rows = max(1, min(_spread(rng, 1, 320), 1_500_000 // (hi * max(kv, 4))))
        return dict(shape, rope=rope, bias=bias, rows=rows, lo=_spread(rng, 1, hi), hi=hi, block=block,
                    layers=rng.choice([1, 2]))
    if kind == "prefill":
        past = rng.choice([0, 0, _spread(rng, 1, 16000)])
        hi = _spread(rng, 1, 8000 if past == 0 else 2000 if past < 2000 else 256)
        seqs = max(1, min(_spread(rng, 1, 24), 60_000_000 // (hi * (past + hi) * max(1, heads // 16))))
        return dict(shape, seqs=seqs, lo=_spread(rng, 1, hi), hi=hi, past=past, block=block)
    hi = _spread(rng, 1, 1500)
    seqs = max(1, min(_spread(rng, 1, 100), 5000 // hi))
    return dict(shape, rope=rope, bias=bias, seqs=seqs, lo=_spread(rng, 1, hi), hi=hi,
                past=rng.choice([0, _spread(rng, 1, 4000)]), block=block)


# -- inputs ------------------------------------------------------------------------------------------------------


def _lengths(n, lo, hi):
    q = (np.arange(n) + 0.5) / n
    return np.clip(np.rint(lo * (hi / lo) ** q), lo, hi).astype(np.int64)


def _generators(seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    return np.random.default_rng(seed), gen


def _normal(gen, dtype, *shape, std=1.0):
    return torch.empty(shape, dtype=torch.float32, device=DEV).normal_(0.0, std, generator=gen).to(dtype)


def _dev(a, dtype=np.int32):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=dtype)).to(DEV)


def _tables(rng, tokens, block):
    """A block table of randomly placed blocks for sequences of ``tokens`` tokens, and the block count."""
    blocks = -(-tokens // block)
    total = int(blocks.sum())
    perm = rng.permutation(total).astype(np.int32)
    table = np.full((tokens.size, max(1, int(blocks.max()))), -1, dtype=np.int32)
    at = 0
    for s, n in enumerate(blocks):
        table[s, :n] = perm[at:at + n]
        at += int(n)
    return table, total


def _pool(gen, case, layers, blocks):
    """A cache in use: codes over most of their range, values of a few units."""
    shape = (layers, 2, blocks, case["kv"], case["block"] // TILE)
    codes = _normal(gen, torch.float32, *shape, TILE * case["dim"], std=90.0)
    scales = torch.randint(127 - 7, 127 - 4, shape, generator=gen, device=DEV, dtype=torch.uint8)
    return codes.clamp_(-448.0, 448.0).to(FP8), scales


def _rope(case, positions):
    """fp32 cos/sin [positions, dim / 2]; the split-half tables hold bf16 values."""
    if not case["rope"]:
        return None, None
    base = 10000.0 if case["rope"] == 1 else 50000.0
    inv = base ** (-torch.arange(0, case["dim"], 2, dtype=torch.float64, device=DEV) / case["dim"])
    f = torch.arange(positions, dtype=torch.float64, device=DEV)[:, None] * inv[None, :]
    cos, sin = f.cos().float(), f.sin().float()
    if case["rope"] == 1:
        cos, sin = cos.bfloat16().float(), sin.bfloat16().float()
    return cos.contiguous(), sin.contiguous()


def _biases(gen, case):
    dt = TYPES[case["dtype"]]
    if not case["bias"]:
        return None, None
    return _normal(gen, dt, case["heads"], case["dim"], std=0.1), _normal(gen, dt, case["kv"], case["dim"], std=0.1)


def _qkv(gen, case, tokens):
    """q, k and v [tokens, heads, dim] as column slices of one fused projection's output."""
    h, g, d = case["heads"], case["kv"], case["dim"]
    fused = _normal(gen, TYPES[case["dtype"]], tokens, (h + 2 * g) * d)
    q, k, v = fused.split([h * d, g * d, g * d], dim=1)
    return q.view(tokens, h, d), k.view(tokens, g, d), v.view(tokens, g, d)


def prepare(case, seed):
    rng, gen = _generators(seed)
    s = dict(case=case, kind=case["kind"], keep={})
    if case["kind"] == "layout":
        lens = rng.permutation(_lengths(case["seqs"], case["lo"], case["hi"]))
        past = rng.integers(case["past"] // 2, case["past"] + 1, size=case["seqs"])
        held, need = -(-past // case["block"]), -(-(past + lens) // case["block"])
        total = int(need.sum())
        perm = rng.permutation(total + 7).astype(np.int32)
        table = np.full((case["seqs"] + 3, -(-(case["past"] + case["hi"]) // case["block"]) + 2), -1, dtype=np.int32)
        order = rng.permutation(case["seqs"] + 3)[:case["seqs"]]
        at = 0
        for r, n in zip(order, held):
            table[r, :n] = perm[at:at + n]
            at += int(n)
        s.update(past=_dev(past), lens=_dev(lens), table=_dev(table), table_row=_dev(order), free=_dev(perm[at:]),
                 tokens=int(lens.sum()), tiles=int((-(-lens // QUERIES)).sum()) + 5)
        return s
    if case["kind"] == "decode":
        contexts = rng.permutation(_lengths(case["rows"], case["lo"], case["hi"]))
        table, blocks = _tables(rng, contexts, case["block"])
        s["codes"], s["scales"] = _pool(gen, case, case["layers"], blocks)
        s["q"], s["k"], s["v"] = _qkv(gen, case, case["rows"])
        s.update(layer=_dev(rng.integers(0, case["layers"], size=case["rows"])), table=_dev(table),
                 position=_dev(contexts - 1), longest=int(contexts.max()))
        s["cos"], s["sin"] = _rope(case, s["longest"])
        s["q_bias"], s["k_bias"] = _biases(gen, case)
        return s
    lens = rng.permutation(_lengths(case["seqs"], case["lo"], case["hi"]))
    past = np.full_like(lens, case["past"])
    table, blocks = _tables(rng, past + lens, case["block"])
    s["codes"], s["scales"] = _pool(gen, case, 1, blocks)
    pos = np.concatenate([np.arange(p, p + n) for p, n in zip(past, lens)])
    seq = np.repeat(np.arange(lens.size), lens)
    s.update(table=_dev(table), past=_dev(past), cu=_dev(np.concatenate([[0], np.cumsum(lens)])),
             position=_dev(pos), longest=int((past + lens).max()), most=int(lens.max()))
    if case["kind"] == "write":
        rows = table[seq, pos // case["block"]].astype(np.int64) * case["block"] + pos % case["block"]
        s.update(rows=_dev(rows, np.int64), written=int(np.unique(rows // TILE).size))
        s["q"], s["k"], s["v"] = _qkv(gen, case, pos.size)
        s["cos"], s["sin"] = _rope(case, s["longest"])
        s["q_bias"], s["k_bias"] = _biases(gen, case)
        return s
    # Attention tiles of 128 query tokens, longest key range first.
    first = np.concatenate([np.arange(0, n, QUERIES) for n in lens])
    tile_seq = np.repeat(np.arange(lens.size), -(-lens // QUERIES))
    end = past[tile_seq] + np.minimum(first + QUERIES, lens[tile_seq])
    order = np.argsort(-end, kind="stable")
    s["q"] = _normal(gen, TYPES[case["dtype"]], pos.size, case["heads"], case["dim"])
    s.update(seq=_dev(seq), table_row=_dev(np.arange(lens.size)), tile_seq=_dev(tile_seq[order]),
             tile_q0=_dev(first[order]))
    return s


# -- plain forms -------------------------------------------------------------------------------------------------


def _rotate(x, bias, cos, sin, positions, style):
    """x [tokens, heads, dim] + bias, rotated, in fp32."""
    x = x.float()
    if bias is not None:
        x = x + bias.float()
    if style == 0:
        return x
    c, n = cos[positions.long()][:, None, :], sin[positions.long()][:, None, :]
    if style == 1:
        lo, hi = x.chunk(2, dim=-1)
        return torch.cat([lo * c - hi * n, hi * c + lo * n], dim=-1)
    even, odd = x[..., 0::2], x[..., 1::2]
    return torch.stack([even * c - odd * n, odd * c + even * n], dim=-1).flatten(-2)


def _exponent(amax):
    """The biased exponent of a tile's scale."""
    bits = amax.contiguous().view(torch.int32)
    return ((bits >> 23) - 8 + ((bits & 0x7FFFFF) > 0x600000)).clamp(1, 254)


def _power(biased):
    """2 ** (biased - 127) in fp32, for exponents of normal numbers."""
    return (biased.clamp(1, 254) << 23).view(torch.float32)


def _unpack(tiles, dim):
    """[..., 2, heads, 16 * dim] bytes of key and value tiles -> fp32 codes [..., 2, heads, 16 tokens, dim]."""
    x = tiles.view(FP8).float()
    k = x[..., 0, :, :].unflatten(-1, (dim // 16, TILE, 16)).transpose(-3, -2).flatten(-2)
    v = x[..., 1, :, :].unflatten(-1, (4, dim, 4)).transpose(-2, -1).flatten(-3, -2)
    return torch.stack([k, v], dim=-4)


def _pack(x, dim):
    """fp32 codes [..., 2, heads, 16 tokens, dim] -> bytes of the tiles."""
    k = x[..., 0, :, :, :].unflatten(-1, (dim // 16, 16)).transpose(-3, -2).flatten(-3)
    v = x[..., 1, :, :, :].unflatten(-2, (4, 4)).transpose(-2, -1).flatten(-3)
    return torch.stack([k, v], dim=-3).to(FP8).view(torch.uint8)


def _append(codes, scales, tiles, layers, new, mask):
    """Put the tokens ``new`` [tiles, 2, heads, 16, dim], where ``mask`` [tiles, 16] holds, into tiles of the cache."""
    nt, dim = codes.shape[4], new.shape[-1]
    raw = codes.view(torch.uint8)
    at = (layers, slice(None), tiles // nt, slice(None), tiles % nt)
    old, was = raw[at], scales[at].int()
    here = mask[:, None, None, :, None]
    amax = torch.where(here & torch.isfinite(new), new.abs(), 0.0).amax(dim=(-2, -1))
    need = _exponent(amax)
    start = mask.int().argmax(dim=1)
    now = torch.where((start == 0)[:, None, None], need, torch.maximum(need, was))
    held = torch.arange(TILE, device=mask.device)[None, :] < start[:, None]
    kept = _unpack(old, dim)
    again = kept * torch.where(start[:, None, None] > 0, _power(127 + was - now), 1.0)[..., None, None]
    fresh = new * _power(254 - now)[..., None, None]
    value = torch.where(here, fresh, torch.where(held[:, None, None, :, None], again, kept))
    raw[at] = _pack(value, dim)
    scales[at] = now.to(torch.uint8)


def _gather(codes, scales, layers, table, dim):
    """fp32 keys and values [rows, 2, heads, tokens, dim] of the blocks in ``table`` [rows, blocks]."""
    at = (layers[:, None], slice(None), table.clamp(min=0).long())
    x = _unpack(codes.view(torch.uint8)[at].permute(0, 1, 4, 2, 3, 5), dim)  # [rows, blocks, tiles, 2, heads, 16, dim]
    x = x * _power(scales[at].int()).permute(0, 1, 4, 2, 3)[..., None, None]
    return x.permute(0, 3, 4, 1, 2, 5, 6).flatten(3, 5)


def _softmax_rows(score):
    top = score.amax(dim=-1, keepdim=True)
    p = torch.exp(score - top)
    return p, p.sum(dim=-1, keepdim=True)


def _plain_decode(s):
    case, dim = s["case"], s["case"]["dim"]
    rows, group = case["rows"], case["heads"] // case["kv"]
    position = s["position"].long()
    q = _rotate(s["q"], s["q_bias"], s["cos"], s["sin"], position, case["rope"])
    k = _rotate(s["k"], s["k_bias"], s["cos"], s["sin"], position, case["rope"])
    offset = position % TILE
    mask = torch.arange(TILE, device=DEV)[None, :] == offset[:, None]
    new = torch.stack([k, s["v"].float()], dim=1)[:, :, :, None, :].expand(-1, -1, -1, TILE, -1)
    tile = s["table"].gather(1, (position // case["block"])[:, None])[:, 0].long() * (case["block"] // TILE)
    _append(s["codes"], s["scales"], tile + position % case["block"] // TILE, s["layer"].long(), new, mask)
    kv = _gather(s["codes"], s["scales"], s["layer"].long(), s["table"], dim)
    seen = torch.arange(kv.shape[3], device=DEV)[None, :] <= position[:, None]
    q = q.view(rows, case["kv"], group, dim)
    score = torch.matmul(q, kv[:, 0].transpose(-1, -2)) * dim ** -0.5
    p, total = _softmax_rows(score.masked_fill(~seen[:, None, None, :], -math.inf))
    out = torch.matmul(p, kv[:, 1].masked_fill(~seen[:, None, :, None], 0.0)) / total
    return out.view(rows, case["heads"], dim).to(TYPES[case["dtype"]]), s["codes"], s["scales"]


def _plain_prefill(s):
    case, dim = s["case"], s["case"]["dim"]
    seqs, most, group = case["seqs"], s["most"], case["heads"] // case["kv"]
    kv = _gather(s["codes"], s["scales"], torch.zeros(seqs, dtype=torch.long, device=DEV), s["table"], dim)
    seq = s["seq"].long()
    index = s["position"].long() - s["past"].long()[seq]  # of the query in its chunk
    q = torch.zeros((seqs, most, case["heads"], dim), device=DEV)
    q[seq, index] = s["q"].float()
    q = q.view(seqs, most, case["kv"], group, dim).permute(0, 2, 3, 1, 4)
    keys = torch.arange(kv.shape[3], device=DEV)
    end = s["past"].long()[:, None] + torch.arange(most, device=DEV)[None, :]
    seen = keys <= end[..., None]
    live = keys < (s["past"] + s["cu"].diff())[:, None]
    score = torch.matmul(q, kv[:, 0, :, None].transpose(-1, -2)).mul_(dim ** -0.5)
    p, total = _softmax_rows(score.masked_fill_(~seen[:, None, None], -math.inf))
    out = torch.matmul(p, kv[:, 1].masked_fill(~live[:, None, :, None], 0.0)[:, :, None]) / total
    return out.permute(0, 3, 1, 2, 4).flatten(2, 3)[seq, index].to(TYPES[case["dtype"]])


def _plain_write(s):
    case, dim = s["case"], s["case"]["dim"]
    position = s["position"]
    q = _rotate(s["q"], s["q_bias"], s["cos"], s["sin"], position, case["rope"])
    k = _rotate(s["k"], s["k_bias"], s["cos"], s["sin"], position, case["rope"])
    # The tokens of one tile follow each other: number the tiles, and lay the tokens out in them.
    tile, offset = s["rows"] // TILE, s["rows"] % TILE
    number = torch.cat([tile.new_zeros(1), (tile[1:] != tile[:-1]).long()]).cumsum(0)
    tiles = tile.new_zeros(s["written"]).index_copy(0, number, tile)
    mask = torch.zeros((s["written"], TILE), dtype=torch.bool, device=DEV)
    mask[number, offset] = True
    new = torch.zeros((s["written"], 2, case["kv"], TILE, dim), device=DEV)
    new[number, 0, :, offset] = k
    new[number, 1, :, offset] = s["v"].float()
    _append(s["codes"], s["scales"], tiles, torch.zeros_like(tiles), new, mask)
    return q.to(TYPES[case["dtype"]]), s["codes"], s["scales"]


def _plain_layout(s):
    block, tokens, tiles = s["case"]["block"], s["tokens"], s["tiles"]
    past, lens, row = s["past"].long(), s["lens"].long(), s["table_row"].long()
    seqs, width = past.numel(), s["table"].shape[1]
    cu = torch.cat([lens.new_zeros(1), lens.cumsum(0)])
    held, need = (past + block - 1) // block, (past + lens + block - 1) // block
    taken = torch.cat([lens.new_zeros(1), (need - held).cumsum(0)])
    # New blocks in request order, from the front of the free list.
    column = torch.arange(width, device=DEV)[None, :]
    fresh = (column >= held[:, None]) & (column < need[:, None])
    from_free = s["free"][(taken[:-1, None] + column - held[:, None]).clamp(0, s["free"].numel() - 1)]
    table = torch.where(fresh, from_free, s["table"][row])
    s["table"][row] = table
    # Slots of the tokens.
    at = torch.arange(tokens, device=DEV)
    seq = torch.searchsorted(cu, at, right=True) - 1
    position = past[seq] + at - cu[seq]
    slots = table[seq, position // block].long() * block + position % block
    # Tiles of 128 query tokens, longest key range first, in request order among equals.
    count = (lens + QUERIES - 1) // QUERIES
    upto = torch.cat([lens.new_zeros(1), count.cumsum(0)])
    at = torch.arange(tiles, device=DEV)
    tseq = (torch.searchsorted(upto, at, right=True) - 1).clamp(max=seqs - 1)
    first = (at - upto[tseq]) * QUERIES
    real = at < upto[-1]
    end = torch.where(real, past[tseq] + torch.minimum(first + QUERIES, lens[tseq]), -1)
    order = torch.sort(end, descending=True, stable=True).indices
    tile_seq = torch.where(real, tseq, -1)[order]
    tile_q0 = torch.where(real, first, 0)[order]
    counts = torch.stack([cu[-1], upto[-1], taken[-1], torch.zeros_like(cu[-1])])
    return [cu.int(), position.int(), slots, tile_seq.int(), tile_q0.int(), counts.int(), s["table"]]


# -- the framework's calls ---------------------------------------------------------------------------------------


def _own_decode(s):
    from continuous_depth_batching_amd import kv8

    case, keep = s["case"], s["keep"]
    if not keep:
        nbytes = kv8.decode_workspace_bytes(case["rows"], case["heads"], case["kv"], case["dim"], s["longest"])
        keep.update(pool=kv8.Kv8Pool(s["codes"], s["scales"]),
                    workspace=torch.empty(nbytes, dtype=torch.uint8, device=DEV))
    out = torch.empty_like(s["q"], memory_format=torch.contiguous_format)
    kv8.decode_attention_raw(s["q"], s["k"], s["v"], keep["pool"], s["layer"], 0, s["table"], None, s["position"],
                             s["cos"], s["sin"], case["rope"], s["q_bias"], s["k_bias"], out, keep["workspace"],
                             case["dim"] ** -0.5)
    return out, s["codes"], s["scales"]


def _own_prefill(s):
    from continuous_depth_batching_amd import kv8

    case, keep = s["case"], s["keep"]
    if not keep:
        splits = kv8.prefill_splits(s["tile_seq"].numel(), case["heads"], case["kv"], s["longest"])
        nbytes = kv8.prefill_workspace_bytes(s["tile_seq"].numel(), splits, case["heads"], case["dim"])
        keep.update(pool=kv8.Kv8Pool(s["codes"], s["scales"]), splits=splits,
                    workspace=torch.empty(nbytes, dtype=torch.uint8, device=DEV))
    out = torch.empty_like(s["q"])
    kv8.prefill_attention_raw(s["q"], keep["pool"], 0, s["table"], s["table_row"], s["cu"], s["past"], s["tile_seq"],
                              s["tile_q0"], out, case["dim"] ** -0.5, keep["splits"], keep["workspace"])
    return out


def _own_write(s):
    from continuous_depth_batching_amd import kv8

    case, keep = s["case"], s["keep"]
    if not keep:
        keep["pool"] = kv8.Kv8Pool(s["codes"], s["scales"])
    q_out = torch.empty_like(s["q"], memory_format=torch.contiguous_format)
    kv8.write_raw(s["q"], s["k"], s["v"], q_out, keep["pool"], 0, s["rows"], s["position"], s["cos"], s["sin"],
                  case["rope"], s["q_bias"], s["k_bias"])
    return q_out, s["codes"], s["scales"]


def _own_layout(s):
    from continuous_depth_batching_amd import kv8

    out = kv8.BatchLayout.allocate(s["past"].numel(), s["tokens"], s["tiles"], s["past"].device)
    kv8.batch_layout_raw(s["past"], s["lens"], s["table"], s["table_row"], s["free"], s["case"]["block"], out)
    return [out.cu_q, out.positions, out.rows, out.tile_seq, out.tile_q0, out.counts, s["table"]]


def run(s):
    kind = s["kind"]
    if own:
        calls = {"decode": _own_decode, "prefill": _own_prefill, "write": _own_write, "layout": _own_layout}
        return calls[kind](s)
    plain = {"decode": _plain_decode, "prefill": _plain_prefill, "write": _plain_write, "layout": _plain_layout}
    return plain[kind](s)


def work(case):
    lens = _lengths(case.get("seqs", case.get("rows")), case["lo"], case["hi"])
    if case["kind"] == "layout":
        past = case["past"] * 3 // 4  # the middle of its range
        blocks = int((-(-(past + lens) // case["block"])).sum()) - lens.size * -(-past // case["block"])
        tokens, tiles = int(lens.sum()), int((-(-lens // QUERIES)).sum())
        return dict(bytes=12 * tokens + 8 * tiles + 16 * lens.size + 8 * blocks, flops=0)
    h, g, d, e = case["heads"], case["kv"], case["dim"], 2 if case["dtype"] == "bf16" else 4
    token = 2 * g * (d + 1 / TILE) + 4 / case["block"]  # codes, scales and table entry of a cached token
    if case["kind"] == "decode":
        read = int(lens.sum()) * token + case["rows"] * (2 * h + 2 * g) * d * e
        return dict(bytes=read + case["rows"] * 2 * g * (d + 1), flops=4 * int(lens.sum()) * h * d)
    tokens = int(lens.sum())
    if case["kind"] == "prefill":
        seen = int((lens * case["past"] + lens * (lens + 1) // 2).sum())
        cached = tokens + case["seqs"] * case["past"]
        return dict(bytes=2 * tokens * h * d * e + cached * token, flops=4 * seen * h * d)
    return dict(bytes=tokens * ((2 * h + 2 * g) * d * e + 2 * g * (d + 1 / TILE) + 12), flops=0)


# -- the definition in 64 bits -----------------------------------------------------------------------------------


def _exact_turn(x, bias, s, positions):
    x = x.double()
    if bias is not None:
        x = x + bias.double()
    style, d = s["case"]["rope"], x.shape[-1]
    if style == 0:
        return x
    c, n = s["cos"].double()[positions][:, None], s["sin"].double()[positions][:, None]
    a, b = (slice(0, d // 2), slice(d // 2, d)) if style == 1 else (slice(0, d, 2), slice(1, d, 2))
    y = torch.empty_like(x)
    y[..., a] = x[..., a] * c - x[..., b] * n
    y[..., b] = x[..., b] * c + x[..., a] * n
    return y


def _exact_round(x):
    """x rounded to e4m3, ties to even, in 64 bits (|x| <= 448)."""
    step = torch.exp2(torch.frexp(x.abs().clamp(min=2.0 ** -6)).exponent.double() - 4)
    return torch.round(x / step) * step


def _exact_scale(amax):
    m, e = torch.frexp(amax)  # amax = m * 2 ** e with m in [0.5, 1)
    e = torch.where(m > 0.875, e - 8, e - 9).clamp(min=-126)
    return torch.where(amax > 0, e, -126)


def _exact_places(dim):
    """Where token t's element i lies in a key tile and in a value tile: two [16, dim] tables."""
    t, i = torch.arange(TILE, device=DEV)[:, None], torch.arange(dim, device=DEV)[None, :]
    return (i // 16) * 256 + t * 16 + i % 16, (t // 4) * dim * 4 + i * 4 + t % 4


def _exact_put(codes, exps, layer, plane, tile, offset, values, place):
    """Append values [heads, n, dim] at ``offset`` of one tile; codes 64-bit, exps the scales' exponents."""
    nt = codes.shape[4]
    where = (layer, plane, tile // nt, slice(None), tile % nt)
    held, was = codes[where][:, place], exps[where]
    n = values.shape[1]
    now = _exact_scale(values.abs().amax(dim=(1, 2)))
    if offset:
        now = torch.maximum(now, was)
        held[:, :offset] = _exact_round(held[:, :offset] * torch.exp2((was - now).double())[:, None, None])
    held[:, offset:offset + n] = _exact_round(values * torch.exp2(-now.double())[:, None, None])
    flat = codes[where]
    flat[:, place.flatten()] = held.flatten(1)
    codes[where] = flat
    exps[where] = now


def _exact_sequence(codes, exps, layer, blocks, tokens, dim):
    """Keys and values [heads, tokens, dim] of one sequence."""
    both = []
    for plane, place in enumerate(_exact_places(dim)):
        c = codes[layer, plane, blocks]  # [blocks, heads, tiles, 16 * dim]
        x = c[..., place].double() * torch.exp2(exps[layer, plane, blocks].double())[..., None, None]
        both.append(x.transpose(0, 1).flatten(1, 3)[:, :tokens])
    return both


def _exact_attend(q, k, v, scale, end):
    """q [heads, n, dim] over k, v [kv heads, tokens, dim]; query i sees keys up to end[i]."""
    g = q.shape[0] // k.shape[0]
    score = torch.matmul(q.unflatten(0, (-1, g)), k[:, None].transpose(-1, -2)) * scale
    score = score.masked_fill(torch.arange(k.shape[1], device=DEV)[None, :] > end[:, None], -math.inf)
    return torch.matmul(torch.softmax(score, dim=-1), v[:, None]).flatten(0, 1)


def exact(case, seed):
    if case["kind"] == "layout":
        return None
    s = prepare(case, seed)
    dim, block = case["dim"], case["block"]
    if case["kind"] == "prefill":
        cu, past, out = s["cu"].tolist(), s["past"].tolist(), []
        codes, exps = s["codes"].float(), s["scales"].int() - 127
        for i in range(case["seqs"]):
            n, p = cu[i + 1] - cu[i], past[i]
            blocks = s["table"][i, :-(-(p + n) // block)].long()
            k, v = _exact_sequence(codes, exps, 0, blocks, p + n, dim)
            q = s["q"][cu[i]:cu[i + 1]].double().transpose(0, 1)
            end = p + torch.arange(n, device=DEV)
            out.append(torch.cat([_exact_attend(q[:, a:a + 1024], k, v, dim ** -0.5, end[a:a + 1024])
                                  for a in range(0, n, 1024)], dim=1))
        return torch.cat(out, dim=1).transpose(0, 1)
    position = s["position"].long()
    k = _exact_turn(s["k"], s["k_bias"], s, position)
    q = _exact_turn(s["q"], s["q_bias"], s, position)
    codes, exps = s["codes"].double(), s["scales"].int() - 127
    places = _exact_places(dim)
    if case["kind"] == "write":
        rows = s["rows"].tolist()
        starts = [t for t in range(len(rows)) if t == 0 or rows[t] // TILE != rows[t - 1] // TILE] + [len(rows)]
        for a, b in zip(starts, starts[1:]):
            for plane, x in enumerate((k, s["v"].double())):
                _exact_put(codes, exps, 0, plane, rows[a] // TILE, rows[a] % TILE, x[a:b].transpose(0, 1),
                           places[plane])
        return q, codes, None
    out, layers = [], s["layer"].tolist()
    for b, p in enumerate(position.tolist()):
        tile = int(s["table"][b, p // block]) * (block // TILE) + p % block // TILE
        for plane, x in enumerate((k, s["v"].double())):
            _exact_put(codes, exps, layers[b], plane, tile, p % TILE, x[b][:, None], places[plane])
        blocks = s["table"][b, :p // block + 1].long()
        keys, values = _exact_sequence(codes, exps, layers[b], blocks, p + 1, dim)
        out.append(_exact_attend(q[b][:, None], keys, values, dim ** -0.5, position[b:b + 1])[:, 0])
    return torch.stack(out), codes, None
