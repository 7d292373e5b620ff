"""What a row's bits depend on in decode attention of rows that share prefixes: the parts that its prefix is cut into and
whether its group has few queries, both of which the plan says, and nothing else of the batch."""

from __future__ import annotations

from types import SimpleNamespace

import numpy as np
import pytest
import torch

import prefix_helpers as ph
from continuous_depth_batching_amd import ops

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def some(s, rows):
    """The scene with some of its rows, in that order, and a plan and workspace of their own."""

    at = torch.tensor(rows, device="cuda")
    heads, kv, dim = s.q.shape[1], s.k.shape[1], s.q.shape[2]
    plan = ops.prefix_decode_plan(s.group[rows], s.lengths, num_heads=heads, num_kv_heads=kv)
    nbytes = ops.prefix_decode_workspace_bytes(plan, heads, kv, dim, 2048)
    part = SimpleNamespace(**vars(s))
    part.q, part.k, part.v = s.q[at], s.k[at], s.v[at]
    part.seq, part.layer, part.table = s.seq[at], s.layer[at], s.table[at]
    part.pool, part.host_plan, part.plan = s.pool.clone(), plan, plan.to("cuda")
    part.workspace = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
    return part


def shape_of(plan, b):
    """(parts of row b's prefix, negative for few queries; their ends)"""

    _, _, item0, parts = plan.row_info[b]
    return int(parts), plan.items[item0:item0 + abs(parts), 6].tolist()


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("heads,kv", [(4, 4), (14, 2)])
def test_a_row_cut_alike_has_the_same_bits_in_any_batch(heads, kv, dtype):
    # Up to 32 queries a KV head, and more, in a group of each kind; prefixes short enough to be cut alike in all batches.
    group = np.array(([0] * 3 + [1] * 40) * 2 + [2, -1, -1])
    own = [1 + 37 * b % 113 for b in range(group.size - 2)] + [1500, 7]
    s = ph.make(group, [200, 120, 77], own, heads=heads, kv=kv, dim=64, dtype=dtype, seed=heads, dead=0.0)
    want = ph.call(some(s, list(range(group.size)))).clone()
    whole = some(s, list(range(group.size))).host_plan
    rng = np.random.default_rng(1)
    for size in (1, 4, 30, 70, group.size):
        rows = sorted(rng.choice(group.size, size=size, replace=False).tolist(), key=lambda _: rng.random())
        part = some(s, rows)
        got = ph.call(part)
        same = [i for i, b in enumerate(rows) if shape_of(part.host_plan, i) == shape_of(whole, b)]
        assert size < 70 or len(same) >= size // 2  # smaller ones leave few queries of the large group
        assert torch.equal(got[same], want[[rows[i] for i in same]])


def test_calls_on_two_streams_at_once():
    scenes = [ph.make([0] * 9 + [1] * 40 + [-1], [900, 333], [1 + 31 * b % 97 for b in range(49)] + [2900], heads=4, kv=4,
                      dim=128, seed=i, dead=0.0) for i in range(2)]
    want = [ph.call(s).clone() for s in scenes]
    streams = [torch.cuda.Stream() for _ in scenes]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(6):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(ph.call(scenes[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(out, want[i]) for out in got[i])


def test_no_rows():
    s = ph.make([0, -1], [40], [3, 4])
    plan = ops.prefix_decode_plan([], [40], num_heads=8, num_kv_heads=4).to("cuda")
    s.q, s.k, s.v, s.seq, s.layer = (t[:0] for t in (s.q, s.k, s.v, s.seq, s.layer))
    before = s.pool.clone()
    assert ph.call(s, plan=plan).shape == (0, 8, 64)
    assert torch.equal(s.pool.isnan(), before.isnan())
