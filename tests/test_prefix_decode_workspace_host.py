"""Workspace bytes of decode attention of rows that share prefixes (CPU)."""

from __future__ import annotations

import ctypes

from continuous_depth_batching_amd import _lib, ops


def test_bytes_of_items_of_few_queries():
    # 256 rows that share with nobody: 16 queries' room an item, not 128.
    plan = ops.prefix_decode_plan(range(256), [1000] * 256, num_heads=16, num_kv_heads=16)
    assert plan.few == plan.num_items
    nbytes = ops.prefix_decode_workspace_bytes(plan, 16, 16, 128, 1000)
    assert nbytes == (plan.few * 16 * 16 * 130 + 256 * 16 * 130) * 4 + 256 * 16 * 8
    assert nbytes * 7 < _lib.lib().cdb_prefix_decode_workspace_bytes(256, plan.num_items, 16, 16, 128, 1000)


def test_bytes_of_both_kinds():
    plan = ops.prefix_decode_plan([0] * 3 + [1] * 40 + [-1], [500, 700], num_heads=8, num_kv_heads=4)
    assert 0 < plan.few < plan.num_items
    room = (plan.few * 16 + (plan.num_items - plan.few) * 128) * 4 * 98
    for own, chunks in ((1, 1), (1024, 1), (1025, 2), (1 << 20, 64)):
        own_bytes = 44 * chunks * (8 * 98 * 4 + 4 * 8)
        assert ops.prefix_decode_workspace_bytes(plan, 8, 4, 96, own) == room * 4 + own_bytes


def test_queries():
    f, g = _lib.lib().cdb_prefix_decode_plan_workspace_bytes, _lib.lib().cdb_prefix_decode_workspace_bytes
    assert f(-1, 0, 0, 4, 4, 64, 1) == f(1, -1, 0, 4, 4, 64, 1) == f(1, 2, 1, 4, 4, 64, 1) == f(1, 0, 0, 4, 4, 64, 0) == -1
    for few in range(4):
        assert f(5, few, 3, 8, 2, 128, 3000) <= g(5, 3, 8, 2, 128, 3000)
    assert f(5, 0, 3, 8, 2, 128, 3000) == g(5, 3, 8, 2, 128, 3000)


def test_less_than_one_chunk_a_row_is_refused():
    fake = ctypes.c_void_p(0x1000)  # refused on the host: no kernel sees it
    for few in range(4):
        need = _lib.lib().cdb_prefix_decode_plan_workspace_bytes(4, few, 3, 4, 4, 64, 1)
        assert _lib.lib().cdb_prefix_decode_attention(
            fake, fake, fake, fake, fake, 64 * 16 * 256, 2, 64, None, 0, fake, None, 4, 8, fake, fake, fake, 1, 100,
            None, None, fake, 4, fake, 3, few, fake, fake, fake, need - 1, 4, 4, 4, 64, 16, 0.1, 0, 0,
            _lib.CDB_DTYPE_BF16, None) == _lib.CDB_ERR_CAPACITY
