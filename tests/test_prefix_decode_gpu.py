"""Decode attention of rows that share prefixes (cdb_prefix_decode_attention) against float64."""

from __future__ import annotations

from dataclasses import replace

import numpy as np
import pytest
import torch

import prefix_helpers as ph
from continuous_depth_batching_amd import ops
from oracle import sampling

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def run(*args, **kwargs):
    s = ph.make(*args, **kwargs)
    before = s.pool.clone()
    out = ph.call(s)
    ph.check(s, out, before)
    return s, out


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("dim", [64, 96, 128])
@pytest.mark.parametrize("heads,kv", [(4, 4), (8, 2), (7, 1), (5, 5)])
def test_shapes(heads, kv, dim, dtype):
    run([0, 1, 0, -1, 1, 0], [37, 64], [1, 2, 17, 5, 33, 40], heads=heads, kv=kv, dim=dim, dtype=dtype, rope=1,
        bias=True, seed=dim + heads)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("rope", [0, 1, 2])
@pytest.mark.parametrize("bias", [False, True])
def test_rotations_and_biases(rope, bias, dtype):
    run([0, 0, 1], [50, 16], [3, 20, 9], heads=6, kv=3, dim=96, dtype=dtype, rope=rope, bias=bias, seed=rope)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("length", [0, 1, 15, 16, 17, 31, 32, 33, 127, 129, 500, 1500])
def test_prefix_lengths(length, dtype):
    run([0, 0, 0], [length], [1, 16, 18], heads=2, kv=2, dtype=dtype, block=32, seed=length)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("own", [1, 2, 15, 16, 17, 32, 33, 65, 129, 1023, 1025, 1026, 2200])
def test_own_lengths(own, dtype):
    run([0, -1], [21], [own, own], heads=2, kv=1, dtype=dtype, seed=own)


@pytest.mark.parametrize("heads,kv", [(17, 1), (40, 1), (64, 2)])
@pytest.mark.parametrize("own", [5, 1200])
def test_many_heads_share_a_kv_head(heads, kv, own):
    run([0, 0, -1], [70], [own, 3, own], heads=heads, kv=kv, seed=heads)


@pytest.mark.parametrize("block", [16, 32, 64, 256])
def test_blocks_and_table_rows(block):
    run([1, 0, 1, -1, 0], [100, 333], [4, 90, 41, 300, 1], block=block, shuffle_rows=True, layers=3, layer0=1,
        seed=block)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("rows", [1, 3, 31, 40, 130])
@pytest.mark.parametrize("dim", [64, 96, 128])
def test_group_sizes(rows, dim, dtype):
    own = 1 + np.arange(rows) % 23
    run([0] * rows + [-1], [700], [*own, 30], heads=4, kv=2, dim=dim, dtype=dtype, seed=rows)


def test_many_groups_in_any_order():
    rng = np.random.default_rng(0)
    group = rng.integers(-1, 12, size=90)
    lengths = rng.integers(0, 900, size=12)
    run(group, lengths, rng.integers(1, 120, size=90), heads=4, kv=4, dim=128, layers=4, seed=7)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
def test_peaked_and_large_scores(dtype):
    # Scores up to some thousands: one key takes nearly all weight, in the prefix for some rows, among the own for others.
    run([0] * 20 + [-1], [333], [1 + 7 * i for i in range(21)], heads=4, kv=2, dim=64, dtype=dtype, scale_q=60.0,
        seed=3)


def test_padding_rows_get_zeros_and_leave_the_cache():
    s, out = run([0, 0, 1, -1], [40, 50], [3, 4, 5, 6], padding=[0, 3], seed=1)
    assert (out[[0, 3]] == 0).all()


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
def test_appends_what_paged_decode_attention_appends(dtype):
    """fp32: the same bits. In bf16 the other one rounds the sum with the bias, both products and their sum, as torch's
    operators do, each by 2^-8 of at most (|k| + |bias|)(|cos| + |sin|), and this one only the result."""

    s = ph.make([0, 0, -1], [64], [30, 5, 77], heads=4, kv=4, dim=128, dtype=dtype, rope=1, bias=True, dead=0.0)
    other = s.pool.clone()
    out = ph.call(s)
    ws = torch.empty(ops.decode_workspace_bytes(3, 4, 128, 4096, 16, 8) // 4, device="cuda")
    ref = torch.ops.cdb.paged_decode_attention(s.q, s.k, s.v, other, s.layer, s.layer0, s.table, None, s.seq, s.cos,
                                               s.sin, 1, s.q_bias, s.k_bias, ws, 16, ops.ADAPTIVE_SPLIT, s.scale)
    if dtype is F32:
        assert bool((s.pool == other).all())
        assert bool(((out - ref).abs() <= 2e-6 + 2e-5 * ref.abs()).all())
        return
    most = float((s.k.abs() + s.k_bias.abs()).max()) * 2
    assert bool(((s.pool.double() - other.double()).abs() <= 5 * 2.0 ** -8 * most).all())
    assert bool((s.pool[:, 1] == other[:, 1]).all())


def test_bad_rows_get_nan_and_no_append():
    group, lengths, own = [0, 0, 0, 1, 1, -1, -1], [48, 32], [9, 3, 5, 4, 6, 7, 8]
    s = ph.make(group, lengths, own, dead=0.0, layers=2)
    s.seq[1] = 20            # inside its prefix
    s.layer[4] = 0           # not its group's layer
    s.layer[5] = 7           # no such layer
    s.seq[6] = 1 << 20       # past its table
    before = s.pool.clone()
    out = ph.call(s)
    assert out[[1, 4, 5, 6]].isnan().all() and not out[[0, 2, 3]].isnan().any()
    good = ph.make(group, lengths, own, dead=0.0, layers=2)
    want = ph.call(good)
    assert torch.equal(out[[0, 2, 3]], want[[0, 2, 3]])
    s.seq[[1, 4, 5, 6]] = -1
    expected = before.clone()
    s.pool.copy_(before)
    ph.call(s)
    for b in (0, 2, 3):
        p = int(s.seq[b])
        slot = int(s.table[b, p // 16]) * 16 + p % 16
        expected[int(s.layer[b])][:, slot] = s.pool[int(s.layer[b])][:, slot]
    assert torch.equal(s.pool, expected)


def test_blocks_outside_the_pool_give_nan():
    s = ph.make([0, 0, -1, 1], [48, 48], [9, 30, 7, 5], dead=0.0)
    s.table[1, 3] = 1 << 30   # own block of row 1
    out = ph.call(s)
    assert out[1].isnan().all() and not out[[0, 2, 3]].isnan().any()
    s.table[1, 3] = -5
    s.table[0, 1] = -1        # of the prefix, read through row 0
    out = ph.call(s)
    assert out[[0, 1]].isnan().all() and not out[[2, 3]].isnan().any()


def test_malformed_plans_stay_in_bounds():
    s = ph.make([0, 0, 1], [200, 90], [4, 5, 6], dead=0.0)
    for name in ("listed", "items", "row_info"):
        for value in (-1, 1 << 20, -(1 << 31), (1 << 31) - 1):
            for column in range({"listed": 1, "items": 8, "row_info": 4}[name]):
                t = getattr(s.plan, name).clone()
                if name == "listed":
                    t[:] = value
                else:
                    t[:, column] = value
                ph.call(s, plan=replace(s.plan, **{name: t}))
                torch.cuda.synchronize()


def test_padded_items_are_none():
    s = ph.make([0, 0, 1], [200, 90], [4, 5, 6], dead=0.0)
    want = ph.call(s).clone()
    items = torch.cat([s.plan.items, torch.full((5, 8), -1, dtype=torch.int32, device="cuda")])
    plan = replace(s.plan, items=items)
    ws = torch.empty(ops.prefix_decode_workspace_bytes(plan, 8, 4, 64, 10), dtype=torch.uint8, device="cuda")
    assert torch.equal(ph.call(s, plan=plan, workspace=ws), want)


def test_longer_chunks_where_the_workspace_is_small():
    s = ph.make([0, -1], [100], [5000, 3100], heads=2, kv=1)
    before = s.pool.clone()
    small = torch.empty(ops.prefix_decode_workspace_bytes(s.host_plan, 2, 1, 64, 2000), dtype=torch.uint8, device="cuda")
    ph.check(s, ph.call(s, workspace=small), before)


def test_a_row_does_not_depend_on_others_own_tokens():
    s = ph.make([0, 0, -1, -1], [300], [40, 1500, 90, 2100], dead=0.0)
    want = ph.call(s).clone()
    s.seq[1] = -1
    s.seq[3] = -1
    got = ph.call(s)
    assert torch.equal(got[[0, 2]], want[[0, 2]])


def test_captured_calls_replay_and_share_a_workspace():
    a = ph.make([0, 0, -1], [300], [40, 1500, 2100], seed=1, dead=0.0)
    b = ph.make([0, 0, -1], [300], [1030, 60, 1700], seed=2, dead=0.0)
    want = [ph.call(s).clone() for s in (a, b)]
    ws = a.workspace if a.workspace.numel() >= b.workspace.numel() else b.workspace
    outs = [torch.empty_like(w) for w in want]
    graphs = []
    for s, out in zip((a, b), outs):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ph.call(s, out=out, workspace=ws)
        graphs.append(graph)
    for _ in range(3):
        for i, graph in enumerate(graphs):
            outs[i].zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(outs[i], want[i])
        assert torch.equal(ph.call(a, workspace=ws), want[0])


def test_on_another_stream():
    s = ph.make([0, 0, 1], [200, 90], [4, 50, 6], dead=0.0)
    want = ph.call(s).clone()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = ph.call(s)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(got, want)


def test_offsets_past_4_gib():
    s = ph.make([0, 0, -1], [200], [40, 70, 60], heads=4, kv=4, dim=128, dead=0.0, layers=1)
    small = s.pool
    rows = (9 << 30) // (2 * 4 * 128 * 2) // 16 * 16  # two planes of 4.5 GiB
    s.pool = torch.empty(1, 2, rows, 4, 128, dtype=BF16, device="cuda")
    shift = rows // 16 - small.shape[2] // 16
    s.pool[:, :, shift * 16:] = small
    s.table[s.table >= 0] += shift
    before = s.pool[:, :, shift * 16:].clone()
    out = ph.call(s)
    s.table[s.table >= 0] -= shift
    s.pool = s.pool[:, :, shift * 16:].clone()
    ph.check(s, out, before)


def test_the_registered_operator():
    s = ph.make([0, 0, 1], [200, 90], [4, 50, 6], dead=0.0)
    want, pool = ph.call(s).clone(), s.pool.clone()
    got = torch.ops.cdb.prefix_decode_attention(
        s.q, s.k, s.v, pool, s.layer, s.layer0, s.table, None, s.seq, s.cos, s.sin, s.rope, s.q_bias, s.k_bias,
        s.plan.listed, s.plan.items, s.plan.row_info, s.plan.few, s.workspace, s.block, s.scale)
    assert torch.equal(got, want) and torch.equal(pool, s.pool)


def test_answers_drawn_from_shared_prompts():
    """A few steps of a one-layer decoder: six answers each of two prompts, every step's attention against float64 and
    every token against the definition."""

    heads = kv = 4
    dim, vocab, answers, steps = 64, 512, 6, 5
    width = heads * dim
    group = np.repeat([0, 1], answers)
    s = ph.make(group, [45, 130], np.full(2 * answers, steps), heads=heads, kv=kv, dim=dim, layers=1, seed=5)
    gen = torch.Generator().manual_seed(11)
    embed = torch.randn(vocab, width, generator=gen).to(BF16).cuda()
    wqkv = (torch.randn(3 * width, width, generator=gen) * width ** -0.5).to(BF16).cuda()
    head = (torch.randn(vocab, width, generator=gen) * 4 * width ** -0.5).to(BF16).cuda()
    packed_qkv, packed_head = ops.maybe_pack_linear_weight(wqkv), ops.maybe_pack_linear_weight(head)
    # The rows start behind their prompts, with one token all of a group's answers share.
    first = s.seq - (steps - 1)
    tokens = torch.from_numpy(group * 7 + 3).cuda()
    temperature = torch.full((2 * answers,), 0.9, device="cuda")
    top_k = torch.full((2 * answers,), 60, dtype=torch.int32, device="cuda")
    top_p = torch.full((2 * answers,), 0.95, device="cuda")
    drawn = []
    for step in range(steps):
        qkv = torch.ops.cdb.linear(torch.ops.cdb.gather_rows(embed, tokens), wqkv, packed_qkv, False)
        s.q, s.k, s.v = (x.view(2 * answers, heads, dim) for x in qkv.split(width, dim=1))
        s.seq = first + step
        before = s.pool.clone()
        out = ph.call(s)
        ph.check(s, out, before)
        u = torch.rand(2 * answers, dtype=torch.float64, generator=gen).cuda()
        x = out.view(2 * answers, width)
        tokens, _ = ops.lm_head_sample(x, head, packed_head, u, temperature, top_k, top_p)
        logits = torch.ops.cdb.linear(x, head, packed_head, False).double().cpu().numpy()
        for r in range(2 * answers):
            assert int(tokens[r]) == sampling.draw(logits[r], float(u[r]), float(np.float32(0.9)), 60,
                                                   float(np.float32(0.95)))[0]
        drawn.append(tokens.tolist())
    assert len(set(map(tuple, zip(*drawn)))) > answers  # the answers differ
