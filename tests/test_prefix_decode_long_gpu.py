"""Long parts of a prefix, whose block ids a wave looks up 1024 tokens at a time, and prefixes of as many parts as there
can be, against float64."""

from __future__ import annotations

import pytest
import torch

import prefix_helpers as ph
from continuous_depth_batching_amd import _lib, ops

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def plan_for(s, num_cus):
    """The scene's plan and workspace as for a GPU of so many compute units: for one, a prefix with four KV heads is one
    part."""

    heads, kv, dim = s.q.shape[1], s.k.shape[1], s.q.shape[2]
    plan = ops.prefix_decode_plan(s.group, s.lengths, num_heads=heads, num_kv_heads=kv, num_cus=num_cus)
    own = int((s.seq.cpu() + 1 - torch.as_tensor(s.start)).max())
    nbytes = ops.prefix_decode_workspace_bytes(plan, heads, kv, dim, own)
    s.host_plan, s.plan = plan, plan.to("cuda")
    s.workspace = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
    return plan


def run(s):
    before = s.pool.clone()
    ph.check(s, ph.call(s), before)


# From below one look-up to a third one, ending in each place of a step of 32 tokens and in its second tile.
TAILS = [1008, 1023, 1024, 1025, 1039, 1041, 1055, 1056, 2047, 2049, 2057, 2064, 2065, 2117]


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("length", TAILS)
@pytest.mark.parametrize("rows", [3, 40], ids=["few", "many"])
def test_one_part_of_many_tokens(rows, length, dtype):
    s = ph.make([0] * rows, [length], [1 + b % 5 for b in range(rows)], heads=4, kv=4, dtype=dtype, seed=length)
    plan = plan_for(s, 1)
    assert (plan.items[:, 5] == 0).all() and (plan.items[:, 6] == length).all() and (plan.few == 0) == (rows == 40)
    run(s)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("dim", [64, 96, 128])
@pytest.mark.parametrize("block", [16, 64])
def test_long_parts_of_other_heads_and_blocks(block, dim, dtype):
    s = ph.make([0] * 20 + [1] * 35, [3109, 1333], [1 + b % 3 for b in range(55)], heads=6, kv=3, dim=dim, dtype=dtype,
                block=block, rope=2, seed=dim)
    assert (plan_for(s, 1).items[:, 6] > 1024).all()  # both of one part
    run(s)


@pytest.mark.parametrize("position", [0, 1023, 1024, 1100, 2047, 2048, 2116])
@pytest.mark.parametrize("rows", [3, 40], ids=["few", "many"])
def test_a_block_outside_the_pool_is_seen_in_every_look_up(rows, position):
    s = ph.make([0] * rows + [1, -1], [2117, 30], [1 + b % 5 for b in range(rows)] + [2, 9], heads=4, kv=4, dead=0.0,
                seed=rows)
    assert [0, 2117] in plan_for(s, 1).items[:, 5:7].tolist()
    want = ph.call(s).clone()
    s.table[0, position // 16] = 1 << 30
    got = ph.call(s)
    assert got[:rows].isnan().all() and torch.equal(got[rows:], want[rows:])


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("rows,heads", [(1, 1), (3, 5), (40, 1), (30, 5)])
@pytest.mark.parametrize("length", [8192, 8209, 9000])
def test_as_many_parts_as_there_can_be(length, rows, heads, dtype):
    s = ph.make([0] * rows, [length], [1 + 7 * (b % 9) for b in range(rows)], heads=heads, kv=1, dtype=dtype, seed=rows)
    parts = abs(int(s.host_plan.row_info[0, 3]))
    assert parts > 50 and (length != 8192 or parts == _lib.CDB_PREFIX_MAX_PARTS)
    run(s)
