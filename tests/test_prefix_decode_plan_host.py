"""A plan of rows that share prefixes is for one number of query heads a KV head, by which its queries are counted (CPU)."""

from __future__ import annotations

from dataclasses import replace

import pytest

import prefix_helpers as ph
from continuous_depth_batching_amd import ops


def test_plans_know_their_heads():
    plan = ops.prefix_decode_plan([0, 0, -1], [40], num_heads=12, num_kv_heads=4)
    assert plan.share == plan.to("cpu").share == 3


@pytest.mark.parametrize("heads,kv", [(4, 4), (16, 4), (8, 8)])
def test_a_plan_for_other_heads_is_refused(heads, kv):
    s = ph.make([0, 0, 1], [40, 20], [3, 4, 5], heads=8, kv=4, device="cpu")
    other = ops.prefix_decode_plan(s.group, s.lengths, num_heads=heads, num_kv_heads=kv).to("cpu")
    with pytest.raises(ValueError, match="query heads a KV head"):
        ph.call(s, plan=other)
    # The same number of them on other heads, or a number that is not known, is not refused for that.
    for plan in (ops.prefix_decode_plan(s.group, s.lengths, num_heads=2, num_kv_heads=1).to("cpu"),
                 replace(other, share=0)):
        with pytest.raises(RuntimeError):  # tensors of the CPU
            ph.call(s, plan=plan)
