"""Timed cases of the operators that draw many answers from one prompt.

Two operators:

* ``prefix``  decode attention of a batch whose rows share prompts: one new token a row, rotated and
  appended to the paged cache of its row and loop depth, then attention over all of the row's tokens.
  Rows of a group begin with the same tokens, held once in the cache. Where a prefix ends inside a block,
  each row holds that block's tokens in a block of its own;
* ``sample``  one token a row from its logits and a given random number: temperature, the ``top_k``
  largest, the smallest set of the largest that holds ``top_p`` of what these weigh, and none below
  ``min_p`` times the largest; then the first token, in the order of the vocabulary, at which the running
  weight passes the random number's share of the total, and the logarithm of its share.

Lengths are spread evenly over the logarithm of a range, in an order drawn from the seed, so a case's work
does not depend on the seed.
"""

import math

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # Eight answers to one question, a few tokens in: bound by latency.
        dict(name="prefix_row8", kind="prefix", dtype="bf16", heads=16, kv=16, dim=128, rope=1, bias=False, groups=1,
             rows=8, plo=900, phi=900, lo=3, hi=60, block=16, layers=1),
        # A full batch of answers to one prompt, rows at two loop depths, which is two groups.
        dict(name="prefix_rows256", kind="prefix", dtype="bf16", heads=16, kv=16, dim=128, rope=1, bias=False,
             groups=2, rows=128, plo=2048, phi=2048, lo=32, hi=512, block=16, layers=2),
        # Sixteen prompts of all lengths, sixteen answers each.
        dict(name="prefix_prompts16", kind="prefix", dtype="bf16", heads=16, kv=16, dim=128, rope=1, bias=False,
             groups=16, rows=16, plo=300, phi=4000, lo=16, hi=600, block=16, layers=1),
        # One long document under every question, query heads that share KV heads.
        dict(name="prefix_document", kind="prefix", dtype="bf16", heads=32, kv=8, dim=128, rope=1, bias=False,
             groups=1, rows=64, plo=32000, phi=32000, lo=16, hi=400, block=64, layers=1),
        # The wide shape with interleaved rotation and biases; prefixes end inside a block.
        dict(name="prefix_wide", kind="prefix", dtype="bf16", heads=55, kv=55, dim=96, rope=2, bias=True, groups=3,
             rows=33, plo=411, phi=1777, lo=7, hi=300, block=32, layers=1),
        # A small fp32 batch of narrow heads.
        dict(name="prefix_f32", kind="prefix", dtype="f32", heads=12, kv=12, dim=64, rope=2, bias=True, groups=3,
             rows=11, plo=130, phi=701, lo=5, hi=250, block=32, layers=1),
        # The tail of a generation: one sequence left, all filters on.
        dict(name="sample_row1", kind="sample", dtype="bf16", rows=1, vocab=49152, spread=2.5, masked=0.0,
             mix="filters"),
        # A full batch whose requests ask for different things, greedy ones among them.
        dict(name="sample_rows256", kind="sample", dtype="bf16", rows=256, vocab=49152, spread=2.5, masked=0.0,
             mix="mixed"),
        # Plain sampling, no filter: every token can be drawn.
        dict(name="sample_all", kind="sample", dtype="bf16", rows=128, vocab=65536, spread=2.0, masked=0.0,
             mix="temperature"),
        # Nucleus sampling of flat distributions, from fp32 logits: the nucleus holds many tokens.
        dict(name="sample_nucleus_flat", kind="sample", dtype="f32", rows=64, vocab=65536, spread=1.0, masked=0.0,
             mix="top_p"),
        # Constrained decoding: a grammar leaves a part of an odd vocabulary.
        dict(name="sample_masked", kind="sample", dtype="bf16", rows=33, vocab=32771, spread=3.0, masked=0.9,
             mix="filters"),
        # A large vocabulary in fp32.
        dict(name="sample_wide_f32", kind="sample", dtype="f32", rows=256, vocab=131072, spread=2.5, masked=0.0,
             mix="mixed"),
    ]


def _spread(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    if rng.random() < 0.5:
        vocab = _spread(rng, 50, 131072)
        rows = max(1, min(_spread(rng, 1, 512), 12_000_000 // vocab))
        return dict(kind="sample", dtype=rng.choice(["bf16", "bf16", "f32"]), rows=rows, vocab=vocab,
                    spread=rng.choice([0.5, 1.0, 2.0, 2.5, 3.0, 5.0]), masked=rng.choice([0.0, 0.0, 0.4, 0.97]),
                    mix=rng.choice(["mixed", "filters", "temperature", "top_k", "top_p", "min_p"]))
    heads, kv = rng.choice([(16, 16), (16, 16), (55, 55), (32, 8), (12, 12), (28, 4), (8, 1), (5, 5)])
    dim = 96 if heads == 55 else rng.choice([64, 96, 128, 128, 128])
    rope, bias = rng.choice([(1, False), (2, True), (1, True), (0, False)])
    groups = _spread(rng, 1, 24)
    rows = max(1, min(_spread(rng, 1, 256), 256 // groups))
    phi = max(1, min(_spread(rng, 1, 30000), 4_000_000 // (groups * rows * max(kv, 4)), 400_000 // (groups * kv)))
    hi = max(1, min(_spread(rng, 1, 1000), 450_000 // (groups * rows * max(kv, 4))))
    return dict(kind="prefix", dtype=rng.choice(["bf16", "bf16", "bf16", "f32"]), heads=heads, kv=kv, dim=dim,
                rope=rope, bias=bias, groups=groups, rows=rows, plo=_spread(rng, 1, phi), phi=phi,
                lo=_spread(rng, 1, hi), hi=hi, block=rng.choice([16, 16, 32, 64]), layers=rng.choice([1, 1, 2]))


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


def _prepare_prefix(case, seed):
    rng, gen = _generators(seed)
    block, h, g, d = case["block"], case["heads"], case["kv"], case["dim"]
    dt, rows = TYPES[case["dtype"]], case["groups"] * case["rows"]
    # The groups' rows lie scattered over the batch.
    group = rng.permutation(np.repeat(np.arange(case["groups"]), case["rows"]))
    lengths = _lengths(case["groups"], case["plo"], case["phi"])
    start = lengths[group]
    tokens = rng.permutation(_lengths(rows, case["lo"], case["hi"]))
    position = start + tokens - 1  # of the new token
    shared, need = start // block, -(-(position + 1) // block)
    held = -(-lengths // block)
    total = int(held.sum() + (-(-tokens // block) + 1).sum())  # whatever lengths meet, a few blocks stay free
    ids = rng.permutation(total).astype(np.int64)
    at = np.concatenate([[0], np.cumsum(held)])
    own_at = at[-1] + np.concatenate([[0], np.cumsum(need - shared)])
    table = np.full((rows, int(need.max())), -1, dtype=np.int64)
    for r in range(rows):
        n = int(shared[r])
        table[r, :n] = ids[at[group[r]]:at[group[r]] + n]
        table[r, n:need[r]] = ids[own_at[r]:own_at[r + 1]]
    pool = _normal(gen, dt, case["layers"], 2, total * block, g, d)
    # A block in which a prefix ends: each row has its own copy of the prefix's tokens.
    tails = [r for r in range(rows) if start[r] % block]
    if tails:
        of = np.concatenate([np.arange(start[r] % block) + ids[at[group[r] + 1] - 1] * block for r in tails])
        to = np.concatenate([np.arange(start[r] % block) + table[r, shared[r]] * block for r in tails])
        pool[:, :, _dev(to, np.int64)] = pool[:, :, _dev(of, np.int64)]
    fused = _normal(gen, dt, rows, (h + 2 * g) * d)  # one projection's output
    q, k, v = fused.split([h * d, g * d, g * d], dim=1)
    cos, sin = _rope(case, int(position.max()) + 1)
    biases = (_normal(gen, dt, h, d, std=0.1), _normal(gen, dt, g, d, std=0.1)) if case["bias"] else (None, None)
    return dict(case=case, keep={}, pool=pool, table=_dev(table), position=_dev(position), start=_dev(start),
                group=group, lengths=lengths, layer=_dev(group % case["layers"]), most=int((position - start).max()) + 1,
                q=q.view(rows, h, d), k=k.view(rows, g, d), v=v.view(rows, g, d), cos=cos, sin=sin,
                q_bias=biases[0], k_bias=biases[1])


def _choice(rng, rows, values, dtype=np.float32):
    return _dev(rng.choice(np.asarray(values, dtype=dtype), size=rows), dtype)


def _prepare_sample(case, seed):
    rng, gen = _generators(seed)
    rows, vocab, mix = case["rows"], case["vocab"], case["mix"]
    # Most tokens are about as unlikely as each other, a few stand out.
    logits = _normal(gen, torch.float32, rows, vocab, std=case["spread"])
    best = torch.randint(0, vocab, (rows, 12), generator=gen, device=DEV)
    logits.scatter_add_(1, best, _normal(gen, torch.float32, rows, 12, std=2.0) + 3.0 * case["spread"])
    if case["masked"]:
        out = torch.rand((rows, vocab), generator=gen, device=DEV) < case["masked"]
        out[torch.arange(rows, device=DEV), best[:, 0]] = False
        logits.masked_fill_(out, -math.inf)
    s = dict(case=case, keep={}, logits=logits.to(TYPES[case["dtype"]]),
             uniform=torch.rand(rows, generator=gen, device=DEV, dtype=torch.float64),
             temperature=None, top_k=None, top_p=None, min_p=None)
    if mix == "mixed":
        s.update(temperature=_choice(rng, rows, [0.0, 0.3, 0.6, 0.7, 1.0, 1.0, 1.5]),
                 top_k=_choice(rng, rows, [0, 0, 1, 20, 50, 50, 1000], np.int32),
                 top_p=_choice(rng, rows, [1.0, 1.0, 0.5, 0.8, 0.9, 0.95, 0.99]),
                 min_p=_choice(rng, rows, [0.0, 0.0, 0.02, 0.05, 0.1]))
    elif mix == "filters":
        s.update(temperature=_choice(rng, rows, [0.6, 0.7, 1.0]), top_k=_choice(rng, rows, [20, 40, 50], np.int32),
                 top_p=_choice(rng, rows, [0.8, 0.9, 0.95]), min_p=_choice(rng, rows, [0.0, 0.05]))
    elif mix == "temperature":
        s.update(temperature=_choice(rng, rows, [0.7, 1.0]))
    elif mix == "top_k":
        s.update(top_k=_choice(rng, rows, [1, 2, 40, 500, 5000], np.int32))
    elif mix == "top_p":
        s.update(temperature=_choice(rng, rows, [0.8, 1.0]), top_p=_choice(rng, rows, [0.5, 0.9, 0.95, 0.99]))
    elif mix == "min_p":
        s.update(temperature=_choice(rng, rows, [1.0, 1.5]), min_p=_choice(rng, rows, [0.01, 0.05, 0.2]))
    return s


def prepare(case, seed):
    return _prepare_prefix(case, seed) if case["kind"] == "prefix" else _prepare_sample(case, seed)


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


def _plain_prefix(s):
    case, pool, dim, block = s["case"], s["pool"], s["case"]["dim"], s["case"]["block"]
    rows, kv, group = s["q"].shape[0], case["kv"], case["heads"] // case["kv"]
    position, start, layer, table = s["position"].long(), s["start"].long(), s["layer"].long(), s["table"].long()
    q = _rotate(s["q"], s["q_bias"], s["cos"], s["sin"], position, case["rope"]).view(rows, kv, group, dim)
    k = _rotate(s["k"], s["k_bias"], s["cos"], s["sin"], position, case["rope"])
    slot = table.gather(1, (position // block)[:, None])[:, 0] * block + position % block
    pool[layer, 0, slot] = k.to(pool.dtype)
    pool[layer, 1, slot] = s["v"]
    # Each row's own tokens.
    at = start[:, None] + torch.arange(s["most"], device=DEV)[None, :]
    seen = at <= position[:, None]
    slots = table.gather(1, (at // block).clamp(max=table.shape[1] - 1)).clamp(min=0) * block + at % block
    keys = pool[layer[:, None], 0, slots].float().permute(0, 2, 3, 1)  # [rows, kv, dim, tokens]
    score = torch.matmul(q, keys).mul_(dim ** -0.5).masked_fill_(~seen[:, None, None, :], -math.inf)
    top = score.amax(dim=-1, keepdim=True)
    # The tokens of each prefix, for all rows that begin with them.
    members = [torch.from_numpy(np.flatnonzero(s["group"] == n)).to(DEV) for n in range(len(s["lengths"]))]
    shared, values = [], []
    for rows_of, length in zip(members, s["lengths"].tolist()):
        at = torch.arange(length, device=DEV)
        slots = table[rows_of[0], at // block] * block + at % block
        k0, v0 = (pool[layer[rows_of[:1]], plane, slots].float() for plane in (0, 1))  # [tokens, kv, dim]
        x = torch.matmul(q[rows_of].transpose(0, 1).flatten(1, 2), k0.permute(1, 2, 0)).mul_(dim ** -0.5)
        x = x.unflatten(1, (-1, group)).transpose(0, 1)  # [rows, kv, group, tokens]
        top[rows_of] = torch.maximum(top[rows_of], x.amax(dim=-1, keepdim=True))
        shared.append(x)
        values.append(v0)
    p = torch.exp(score - top)
    total = p.sum(dim=-1, keepdim=True)
    at = start[:, None] + torch.arange(s["most"], device=DEV)[None, :]
    slots = table.gather(1, (at // block).clamp(max=table.shape[1] - 1)).clamp(min=0) * block + at % block
    own_values = pool[layer[:, None], 1, slots].float().masked_fill(~seen[:, :, None, None], 0.0)
    out = torch.matmul(p, own_values.transpose(1, 2))
    for rows_of, x, v0 in zip(members, shared, values):
        p = torch.exp(x - top[rows_of])
        total[rows_of] += p.sum(dim=-1, keepdim=True)
        o = torch.matmul(p.transpose(0, 1).flatten(1, 2), v0.transpose(0, 1))
        out[rows_of] += o.unflatten(1, (-1, group)).transpose(0, 1)
    return (out / total).view(rows, case["heads"], dim).to(pool.dtype), pool


def _plain_sample(s):
    # In 64 bits throughout: a weight's last bits decide on which side of a border the random number falls.
    x = s["logits"].double()
    rows, vocab = x.shape
    ones = torch.ones(rows, 1, device=DEV, dtype=torch.float64)
    temperature = ones if s["temperature"] is None else s["temperature"].double()[:, None]
    order = torch.sort(x, dim=1, descending=True, stable=True)
    top = order.values[:, :1]
    scaled = (order.values - top) / temperature
    weight = torch.where(temperature > 0, torch.exp(scaled), (order.indices == order.indices[:, :1]).double())
    place = torch.arange(vocab, device=DEV)[None, :]
    if s["top_k"] is not None:
        k = s["top_k"].long()[:, None]
        weight = torch.where((k > 0) & (place >= k), 0.0, weight)
    if s["top_p"] is not None:
        p = s["top_p"].double()[:, None]
        before = torch.cumsum(weight, dim=1) - weight
        goal = p * weight.sum(dim=1, keepdim=True)
        weight = torch.where((p < 1) & (before >= goal) & (place > 0), 0.0, weight)
    if s["min_p"] is not None:
        weight = torch.where(weight < s["min_p"].double()[:, None].clamp(max=1.0), 0.0, weight)
    weight = torch.zeros_like(weight).scatter_(1, order.indices, weight)
    running = torch.cumsum(weight, dim=1)
    total = running[:, -1:]
    passed = (running > s["uniform"][:, None] * total) & (weight > 0)
    last = torch.where(weight > 0, place, -1).amax(dim=1)
    token = torch.where(passed.any(dim=1), passed.int().argmax(dim=1), last)
    share = weight.gather(1, token.clamp(min=0)[:, None]) / total
    return token, torch.log(share)[:, 0].float()


# -- the framework's calls ---------------------------------------------------------------------------------------


def _own_prefix(s):
    from continuous_depth_batching_amd import ops

    case, keep = s["case"], s["keep"]
    if not keep:
        plan = ops.prefix_decode_plan(s["group"], s["lengths"], num_heads=case["heads"], num_kv_heads=case["kv"])
        nbytes = ops.prefix_decode_workspace_bytes(plan, case["heads"], case["kv"], case["dim"], s["most"])
        keep.update(view=ops.KVPoolView(s["pool"], case["block"]), plan=plan.to(DEV),
                    workspace=torch.empty(nbytes, dtype=torch.uint8, device=DEV))
    out = torch.empty_like(s["q"], memory_format=torch.contiguous_format)
    ops.prefix_decode_attention_raw(s["q"], s["k"], s["v"], keep["view"], s["layer"], 0, s["table"], None,
                                    s["position"], s["cos"], s["sin"], case["rope"], s["q_bias"], s["k_bias"],
                                    keep["plan"], out, keep["workspace"], case["dim"] ** -0.5)
    return out, s["pool"]


def _own_sample(s):
    from continuous_depth_batching_amd import ops

    keep, (rows, vocab) = s["keep"], s["logits"].shape
    if not keep:
        keep["workspace"] = torch.empty(ops.sample_workspace_bytes(rows, vocab), dtype=torch.uint8, device=DEV)
    tokens = torch.empty(rows, dtype=torch.int64, device=DEV)
    logprobs = torch.empty(rows, dtype=torch.float32, device=DEV)
    ops.sample_raw(s["logits"], s["uniform"], s["temperature"], s["top_k"], s["top_p"], s["min_p"], tokens, logprobs,
                   keep["workspace"])
    return tokens, logprobs


def run(s):
    if s["case"]["kind"] == "prefix":
        return _own_prefix(s) if own else _plain_prefix(s)
    return _own_sample(s) if own else _plain_sample(s)


def work(case):
    e = 2 if case["dtype"] == "bf16" else 4
    if case["kind"] == "sample":
        given = 8 + 4 * {"mixed": 4, "filters": 4, "temperature": 1, "top_k": 1, "top_p": 2, "min_p": 2}[case["mix"]]
        return dict(bytes=case["rows"] * (case["vocab"] * e + given + 12), flops=0)
    h, g, d, rows = case["heads"], case["kv"], case["dim"], case["groups"] * case["rows"]
    prefix = int(_lengths(case["groups"], case["plo"], case["phi"]).sum())
    tokens = int(_lengths(rows, case["lo"], case["hi"]).sum())
    token = 2 * g * d * e + 4 / case["block"]  # keys, values and table entry of a cached token
    return dict(bytes=(prefix + tokens) * token + rows * (2 * h + 2 * g) * d * e,
                flops=4 * (prefix * case["rows"] + tokens) * h * d)


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


def _exact_prefix(case, seed):
    """Row by row over all of the row's tokens, as if nothing were shared."""
    s = prepare(case, seed)
    block, group = case["block"], case["heads"] // case["kv"]
    positions = s["position"].long()
    q = _exact_turn(s["q"], s["q_bias"], s, positions)
    k = _exact_turn(s["k"], s["k_bias"], s, positions)
    pool, out, layers = s["pool"].double(), [], s["layer"].tolist()
    for b, p in enumerate(positions.tolist()):
        slots = (s["table"][b, :p // block + 1].long()[:, None] * block + torch.arange(block, device=DEV)).flatten()
        slots = slots[:p + 1]
        # The cache holds the new token in its own type, and so does what the row attends over.
        pool[layers[b], 0, slots[-1]] = k[b]
        pool[layers[b], 1, slots[-1]] = s["v"][b].double()
        keys, values = pool[layers[b], 0, slots], pool[layers[b], 1, slots]
        keys[-1] = k[b].to(s["pool"].dtype).double()
        score = (keys.transpose(0, 1) @ q[b].view(case["kv"], group, -1).transpose(1, 2)) * case["dim"] ** -0.5
        share = torch.softmax(score, dim=1)  # [kv, tokens, group]
        out.append((share.transpose(1, 2) @ values.transpose(0, 1)).flatten(0, 1))
    return torch.stack(out), pool


def _exact_sample(case, seed):
    """Row by row on the host."""
    if case["rows"] * case["vocab"] > 40_000_000:
        return None
    s = prepare(case, seed)
    logits = s["logits"].double().cpu().numpy()
    given = {n: None if s[n] is None else s[n].cpu().numpy().astype(np.float64)
             for n in ("uniform", "temperature", "top_k", "top_p", "min_p")}
    tokens, shares = [], []
    for r, x in enumerate(logits):
        t, k, p, m = (1.0 if given[n] is None else float(given[n][r]) for n in ("temperature", "top_k", "top_p", "min_p"))
        kept = np.argsort(-x, kind="stable")
        kept = kept[x[kept] > -np.inf]
        if t <= 0:
            kept, t = kept[:1], 1.0
        if given["top_k"] is not None and k > 0:
            kept = kept[:int(k)]
        w = np.exp((x[kept] - x[kept[0]]) / t)
        if given["top_p"] is not None and p < 1:
            sums = np.cumsum(w)
            n = 1 + int(np.searchsorted(sums, p * sums[-1], side="left"))
            kept, w = kept[:n], w[:n]
        if given["min_p"] is not None:
            n = int((w >= min(m, 1.0)).sum())
            kept, w = kept[:n], w[:n]
        by_index = np.argsort(kept)
        kept, w = kept[by_index], w[by_index]
        sums = np.cumsum(w)
        n = min(int(np.searchsorted(sums, given["uniform"][r] * sums[-1], side="right")), len(kept) - 1)
        tokens.append(int(kept[n]))
        shares.append(math.log(w[n] / sums[-1]))
    return torch.tensor(tokens), torch.tensor(shares, dtype=torch.float64)


def exact(case, seed):
    return _exact_prefix(case, seed) if case["kind"] == "prefix" else _exact_sample(case, seed)
