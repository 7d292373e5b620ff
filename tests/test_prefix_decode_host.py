"""The plan of rows that share prefixes, and what cdb_prefix_decode_attention and its Python call refuse (CPU)."""

from __future__ import annotations

import ctypes
from dataclasses import replace

import numpy as np
import pytest
import torch

import prefix_helpers as ph
from continuous_depth_batching_amd import _lib, ops


def cover(plan, group, lengths, heads, kv):
    """Every query of every row meets each token of its prefix once, in consecutive parts."""

    share = heads // kv
    for b, n in enumerate(group):
        q0, length, item0, parts = plan.row_info[b]
        if n < 0 or lengths[n] == 0:
            assert not plan.row_info[b].any()
            continue
        size = ops.PREFIX_FEW if parts < 0 else ops.PREFIX_QUERIES
        assert (item0 < plan.few) == (parts < 0)
        parts = abs(parts)
        assert length == lengths[n] and 1 <= parts <= _lib.CDB_PREFIX_MAX_PARTS
        first, count, leader, tokens = plan.items[item0, :4]
        assert tokens == length and leader == plan.listed[first] and not plan.items[:, 7].any()
        assert b in plan.listed[first:first + count] and plan.listed[first + q0 // share] == b and q0 % share == 0
        for q in range(q0, q0 + share):
            run = item0 + q // size * parts
            of = plan.items[run:run + parts]
            assert (of[:, :4] == plan.items[item0, :4]).all()
            assert (of[:, 4] == q // size * size).all()
            assert of[0, 5] == 0 and of[-1, 6] == length and (of[1:, 5] == of[:-1, 6]).all()
            assert (of[:, 5] < of[:, 6]).all()


@pytest.mark.parametrize("heads,kv", [(1, 1), (16, 16), (32, 8), (28, 4), (7, 1), (64, 1)])
def test_plans_cover_every_query_and_token(heads, kv):
    rng = np.random.default_rng(heads)
    for rows, groups, longest in ((1, 1, 5), (9, 2, 300), (70, 5, 5000), (256, 1, 40000), (40, 40, 200), (5, 3, 0)):
        group = rng.integers(-1, groups, size=rows)
        lengths = rng.integers(0, longest + 1, size=groups)
        plan = ops.prefix_decode_plan(group, lengths, num_heads=heads, num_kv_heads=kv)
        assert plan.num_rows == rows and plan.items.dtype == plan.row_info.dtype == np.int32
        cover(plan, group, lengths, heads, kv)
        assert sorted(plan.listed.tolist()) == [b for b in range(rows) if group[b] >= 0 and lengths[group[b]]]


def test_plans_of_nothing():
    plan = ops.prefix_decode_plan([], [], num_heads=4, num_kv_heads=4)
    assert plan.num_rows == plan.num_items == 0
    plan = ops.prefix_decode_plan([-1, -1], [], num_heads=4, num_kv_heads=4)
    assert plan.num_rows == 2 and plan.num_items == 0 and not plan.row_info.any()
    device = plan.to("cpu")
    assert device.row_info.shape == (2, 4) and device.items.shape == (0, 8) and device.row_info.dtype is torch.int32


@pytest.mark.parametrize("group,lengths,heads,kv", [([0, 2], [5, 5], 4, 4), ([0], [-1], 4, 4), ([0], [1 << 31], 4, 4),
                                                    ([0], [5], 5, 2), ([0], [5], 0, 1)])
def test_plans_that_make_no_sense(group, lengths, heads, kv):
    with pytest.raises(ValueError):
        ops.prefix_decode_plan(group, lengths, num_heads=heads, num_kv_heads=kv)


def test_plans_for_no_compute_units():
    with pytest.raises(ValueError):
        ops.prefix_decode_plan([0, 0], [100], num_heads=4, num_kv_heads=4, num_cus=0)


def code(**over):
    fake = ctypes.c_void_p(0x1000)  # refused on the host: no kernel sees it
    a = dict(q=fake, k_new=fake, v_new=fake, k_pool=fake, v_pool=fake, layer_stride=64 * 16 * 256, layers=2,
             pool_blocks=64, cache_layer=None, cache_layer0=0, block_table=fake, table_row=None, table_rows=4,
             table_width=8, seqlens=fake, cos=fake, sin=fake, style=1, max_positions=100, q_bias=None, k_bias=None,
             listed=fake, num_listed=4, items=fake, num_items=1, num_few=1, row_info=fake, out=fake,
             workspace=fake, nbytes=1 << 24, rows=4, heads=4, kv=4, dim=64, block=16, scale=0.1, q_stride=0,
             kv_stride=0, dtype=_lib.CDB_DTYPE_BF16, stream=None)
    a.update(over)
    return _lib.lib().cdb_prefix_decode_attention(*a.values())


odd = ctypes.c_void_p(0x1004)


@pytest.mark.parametrize("over,expected", [
    (dict(style=3), _lib.CDB_ERR_UNSUPPORTED), (dict(dtype=9), _lib.CDB_ERR_UNSUPPORTED),
    (dict(dim=80), _lib.CDB_ERR_UNSUPPORTED), (dict(rows=-1), _lib.CDB_ERR_SHAPE),
    (dict(heads=0), _lib.CDB_ERR_SHAPE), (dict(kv=0), _lib.CDB_ERR_SHAPE), (dict(kv=3), _lib.CDB_ERR_SHAPE),
    (dict(table_rows=0), _lib.CDB_ERR_SHAPE), (dict(table_width=0), _lib.CDB_ERR_SHAPE),
    (dict(table_rows=3), _lib.CDB_ERR_SHAPE), (dict(table_width=1 << 27), _lib.CDB_ERR_SHAPE),
    (dict(layers=0), _lib.CDB_ERR_SHAPE), (dict(pool_blocks=0), _lib.CDB_ERR_SHAPE),
    (dict(pool_blocks=1 << 31), _lib.CDB_ERR_SHAPE), (dict(num_listed=-1), _lib.CDB_ERR_SHAPE),
    (dict(num_items=-1), _lib.CDB_ERR_SHAPE), (dict(num_few=2), _lib.CDB_ERR_SHAPE), (dict(num_few=-1), _lib.CDB_ERR_SHAPE), (dict(items=odd), _lib.CDB_ERR_SHAPE),
    (dict(block=8), _lib.CDB_ERR_SHAPE), (dict(block=48), _lib.CDB_ERR_SHAPE),
    (dict(layer_stride=64 * 16 * 256 - 8), _lib.CDB_ERR_SHAPE), (dict(scale=0.0), _lib.CDB_ERR_SHAPE),
    (dict(scale=float("inf")), _lib.CDB_ERR_SHAPE), (dict(scale=float("nan")), _lib.CDB_ERR_SHAPE),
    (dict(q_stride=255), _lib.CDB_ERR_SHAPE), (dict(kv_stride=255), _lib.CDB_ERR_SHAPE),
    (dict(workspace=odd), _lib.CDB_ERR_SHAPE), (dict(k_pool=odd), _lib.CDB_ERR_SHAPE),
    (dict(v_pool=odd), _lib.CDB_ERR_SHAPE), (dict(max_positions=0), _lib.CDB_ERR_SHAPE),
    (dict(kv=1 << 22, heads=1 << 22, layers=1), _lib.CDB_ERR_SHAPE),
    (dict(q=None), _lib.CDB_ERR_NULL), (dict(k_pool=None), _lib.CDB_ERR_NULL), (dict(out=None), _lib.CDB_ERR_NULL),
    (dict(row_info=None), _lib.CDB_ERR_NULL), (dict(listed=None), _lib.CDB_ERR_NULL),
    (dict(items=None), _lib.CDB_ERR_NULL),
    (dict(cos=None), _lib.CDB_ERR_NULL), (dict(workspace=None), _lib.CDB_ERR_NULL),
    (dict(nbytes=100), _lib.CDB_ERR_CAPACITY), (dict(nbytes=-1), _lib.CDB_ERR_CAPACITY),
    (dict(rows=0), _lib.CDB_OK),
])
def test_c_entry_refuses(over, expected):
    assert code(**over) == expected


def test_workspace_query():
    f = _lib.lib().cdb_prefix_decode_workspace_bytes
    assert f(-1, 0, 4, 4, 64, 1) == f(1, -1, 4, 4, 64, 1) == f(1, 0, 4, 3, 64, 1) == f(1, 0, 4, 4, 64, 0) == -1
    assert f(2, 0, 4, 4, 64, 100000) > f(2, 0, 4, 4, 64, 1) and f(2, 9, 4, 4, 64, 1) > f(2, 0, 4, 4, 64, 1)


def scene():
    return ph.make([0, 0, 1], [40, 20], [3, 4, 5], device="cpu")


@pytest.mark.parametrize("change,error", [
    (lambda s: setattr(s, "q", s.q[:, :, :32]), ValueError),
    (lambda s: setattr(s, "k", s.k[:2]), ValueError),
    (lambda s: setattr(s, "v", s.v.float()), TypeError),
    (lambda s: setattr(s, "pool", s.pool.float()), TypeError),
    (lambda s: setattr(s, "pool", s.pool[:, :, ::2]), ValueError),
    (lambda s: setattr(s, "block", 8), ValueError),
    (lambda s: setattr(s, "block", 48), ValueError),
    (lambda s: setattr(s, "q", s.q.repeat(1, 1, 1)[:, :7]), ValueError),
    (lambda s: setattr(s, "seq", s.seq.long()), TypeError),
    (lambda s: setattr(s, "seq", s.seq[:2]), ValueError),
    (lambda s: setattr(s, "table", s.table[:2]), ValueError),
    (lambda s: setattr(s, "layer", s.layer[:2]), ValueError),
    (lambda s: setattr(s, "rope", 3), ValueError),
    (lambda s: setattr(s, "cos", s.cos[:, :3]), ValueError),
    (lambda s: setattr(s, "q_bias", torch.zeros(8, 64)), ValueError),
    (lambda s: setattr(s, "plan", s.host_plan), TypeError),
    (lambda s: setattr(s, "plan", replace(s.plan, few=99)), ValueError),
    (lambda s: setattr(s, "plan", replace(s.plan, items=s.plan.items.long())), TypeError),
    (lambda s: setattr(s, "plan", replace(s.plan, row_info=s.plan.row_info[:2])), ValueError),
    (lambda s: setattr(s, "plan", replace(s.plan, items=s.plan.items[:, :3])), ValueError),
    (lambda s: setattr(s, "workspace", s.workspace[::2]), ValueError),
    (lambda s: None, RuntimeError),  # tensors of the CPU
])
def test_arguments_are_checked(change, error):
    s = scene()
    change(s)
    with pytest.raises(error):
        ph.call(s)


def test_operator_is_registered():
    from torch._subclasses.fake_tensor import FakeTensorMode

    op = torch.ops.cdb.prefix_decode_attention.default
    assert {a.name for a in op._schema.arguments if a.alias_info is not None and a.alias_info.is_write} == \
        {"kv_pool", "workspace"}
    with FakeTensorMode():
        def ints(*shape):
            return torch.empty(*shape, dtype=torch.int32, device="cuda")
        q, k = torch.empty(3, 8, 64, device="cuda"), torch.empty(3, 4, 64, device="cuda")
        out = torch.ops.cdb.prefix_decode_attention(q, k, k, torch.empty(1, 2, 64, 4, 64, device="cuda"), None, 0,
                                                    ints(3, 4), None, ints(3), None, None, 0, None, None, ints(3),
                                                    ints(1, 8), ints(3, 4), 1, ints(9), 16, 0.125)
        assert out.shape == q.shape
