"""What decode attention of rows that share prefixes writes: its workspace, its output and the new tokens' slots, with
plans as they are made and with plans that make no sense."""

from __future__ import annotations

from dataclasses import replace

import pytest
import torch

import prefix_helpers as ph
from continuous_depth_batching_amd import ops

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
GUARD, MARK = 1 << 20, 0xA5


def guarded(nbytes):
    """(the whole, a slice of it with marked bytes on both sides)"""

    whole = torch.full((nbytes + 2 * GUARD,), MARK, dtype=torch.uint8, device="cuda")
    return whole, whole[GUARD:GUARD + nbytes]


def untouched(whole, nbytes):
    return bool((whole[:GUARD] == MARK).all()) and bool((whole[GUARD + nbytes:] == MARK).all())


def scene(**kwargs):
    """Two groups of few queries, one of many, and a row alone."""

    s = ph.make([0] * 5 + [1] * 40 + [2] * 3 + [-1], [200, 300, 90], [1 + b % 21 for b in range(48)] + [1100], **kwargs)
    assert 0 < s.host_plan.few < s.host_plan.num_items
    return s


def new_slots(s, rows):
    """(cache layer, slot) of the rows' new tokens."""

    out = []
    for b in rows:
        p = int(s.seq[b])
        out.append((s.layer0 + int(s.layer[b]), int(s.table[b, p // s.block]) * s.block + p % s.block))
    return out


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("heads,kv,dim", [(8, 4, 64), (4, 4, 128), (20, 1, 96)])
def test_a_workspace_of_just_the_bytes(heads, kv, dim, dtype):
    s = ph.make([0] * 5 + [1] * 40 + [2] * 3 + [-1], [200, 300, 90], [1 + b % 21 for b in range(48)] + [1100],
                heads=heads, kv=kv, dim=dim, dtype=dtype, seed=dim)
    nbytes = ops.prefix_decode_workspace_bytes(s.host_plan, heads, kv, dim, 1100)
    whole, workspace = guarded(nbytes)
    out_bytes = s.q.numel() * s.q.element_size()
    out_whole, out = guarded(out_bytes)
    before = s.pool.clone()
    got = ph.call(s, out=out.view(dtype).view(s.q.shape), workspace=workspace)
    ph.check(s, got, before)
    assert untouched(whole, nbytes) and untouched(out_whole, out_bytes)


def spoiled():
    """(what is wrong, plan, rows that have to be NaN) of plans with a part set to something else."""

    s = scene(dead=0.0)
    rows = s.host_plan.num_rows
    grouped = list(range(rows - 1))
    for name in ("listed", "items", "row_info"):
        for value in (-1, 1 << 20, -(1 << 31), (1 << 31) - 1):
            for column in range({"listed": 1, "items": 8, "row_info": 4}[name]):
                t = getattr(s.plan, name).clone()
                if name == "listed":
                    t[:] = value
                else:
                    t[:, column] = value
                bad = []
                if name == "row_info":
                    # A first query, a prefix, a first item or parts that cannot be. Parts of -1 can: one part, an item of
                    # few queries, which the large group's are not.
                    bad = {0: grouped, 1: list(range(rows)), 2: grouped, 3: list(range(rows))}[column]
                    if column == 3 and value == -1:
                        bad = list(range(5, 45))
                yield (name, value, column), s, replace(s.plan, **{name: t}), bad
    t = s.plan.row_info.clone()
    t[:, 3] = -t[:, 3]
    yield ("row_info", "other kind", 3), s, replace(s.plan, row_info=t), grouped


def test_plans_that_make_no_sense_write_nothing_else():
    for what, s, plan, bad in spoiled():
        nbytes = ops.prefix_decode_workspace_bytes(s.host_plan, 8, 4, 64, 1100)
        whole, workspace = guarded(nbytes)
        out_bytes = s.q.numel() * s.q.element_size()
        out_whole, out = guarded(out_bytes)
        pool = s.pool.clone()
        got = ph.call(s, out=out.view(BF16).view(s.q.shape), plan=plan, workspace=workspace)
        torch.cuda.synchronize()
        assert untouched(whole, nbytes) and untouched(out_whole, out_bytes), what
        assert bool(got[bad].isnan().all()) if bad else True, what
        changed = s.pool != pool
        for layer, slot in new_slots(s, [b for b in range(s.host_plan.num_rows) if b not in bad]):
            changed[layer][:, slot] = False
        assert not bool(changed.any()), what
        s.pool.copy_(pool)
