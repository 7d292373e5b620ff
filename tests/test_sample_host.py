"""Refusals of cdb_sample and ops.sample_raw, and its float64 definition, on the CPU."""

from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
import torch

from continuous_depth_batching_amd import _lib, ops
from oracle import sampling


def code(**over):
    fake = ctypes.c_void_p(0x1000)  # refused on the host: no kernel sees it
    a = dict(logits=fake, row_stride=100, uniform=fake, temperature=None, top_k=None, top_p=None, min_p=None,
             tokens=fake, logprobs=fake, workspace=fake, workspace_bytes=1 << 20, rows=2, vocab=100,
             dtype=_lib.CDB_DTYPE_BF16, stream=None)
    a.update(over)
    return _lib.lib().cdb_sample(*a.values())


@pytest.mark.parametrize("over,expected", [
    (dict(dtype=7), _lib.CDB_ERR_UNSUPPORTED),
    (dict(rows=-1), _lib.CDB_ERR_SHAPE),
    (dict(vocab=0), _lib.CDB_ERR_SHAPE),
    (dict(vocab=_lib.CDB_SAMPLE_MAX_VOCAB + 1, row_stride=1 << 21), _lib.CDB_ERR_SHAPE),
    (dict(row_stride=99), _lib.CDB_ERR_SHAPE),
    (dict(logits=ctypes.c_void_p(0x1001)), _lib.CDB_ERR_SHAPE),
    (dict(logits=None), _lib.CDB_ERR_NULL),
    (dict(uniform=None), _lib.CDB_ERR_NULL),
    (dict(tokens=None), _lib.CDB_ERR_NULL),
    (dict(logprobs=None), _lib.CDB_ERR_NULL),
    (dict(workspace_bytes=-1), _lib.CDB_ERR_CAPACITY),
    (dict(rows=0), _lib.CDB_OK),
])
def test_c_entry_refuses(over, expected):
    assert code(**over) == expected


def test_workspace_query():
    assert _lib.lib().cdb_sample_workspace_bytes(-1, 5) == -1
    assert _lib.lib().cdb_sample_workspace_bytes(1, 0) == -1
    assert ops.sample_workspace_bytes(0, 5) >= 0
    with pytest.raises(ValueError):
        ops.sample_workspace_bytes(1, _lib.CDB_SAMPLE_MAX_VOCAB + 1)


def raw(**over):
    a = dict(logits=torch.zeros(2, 8), uniform=torch.zeros(2, dtype=torch.float64), temperature=None, top_k=None,
             top_p=None, min_p=None, tokens=torch.zeros(2, dtype=torch.int64), logprobs=torch.zeros(2),
             workspace=torch.zeros(64, dtype=torch.uint8))
    a.update(over)
    ops.sample_raw(**a)


@pytest.mark.parametrize("over,error", [
    (dict(logits=torch.zeros(8)), ValueError),
    (dict(logits=torch.zeros(2, 0)), ValueError),
    (dict(logits=torch.zeros(8, 2).t()), ValueError),
    (dict(logits=torch.zeros(1, 8).expand(2, 8)), ValueError),
    (dict(uniform=torch.zeros(2)), TypeError),
    (dict(uniform=torch.zeros(3, dtype=torch.float64)), ValueError),
    (dict(temperature=torch.zeros(2, dtype=torch.float64)), TypeError),
    (dict(top_k=torch.zeros(2, dtype=torch.int64)), TypeError),
    (dict(top_p=torch.zeros(1)), ValueError),
    (dict(min_p=torch.zeros(4)[::2]), ValueError),
    (dict(tokens=torch.zeros(2, dtype=torch.int32)), TypeError),
    (dict(logprobs=torch.zeros(2, 1)), ValueError),
    (dict(workspace=torch.zeros(64, 64).t()[:32]), ValueError),
    (dict(), RuntimeError),  # tensors of the CPU
])
def test_arguments_are_checked(over, error):
    with pytest.raises(error):
        raw(**over)


def test_definition():
    x = np.array([1.0, 3.0, 3.0, -np.inf, np.nan, 2.0])
    assert sampling.order(x).tolist() == [1, 2, 5, 0]
    assert sampling.draw(x, 0.9, temperature=0.0) == (1, 0.0)
    assert sampling.kept(x, top_k=2)[0].tolist() == [1, 2]
    assert sampling.kept(x, top_p=0.5)[0].tolist() == [1, 2]
    assert sampling.kept(x, top_p=0.3)[0].tolist() == [1]
    assert sampling.kept(x, min_p=0.3)[0].tolist() == [1, 2, 5]
    assert sampling.draw(x, 0.0)[0] == 0 and sampling.draw(x, 1.0)[0] == 5
    assert sampling.draw(np.full(3, -np.inf), 0.5) == (-1, -math.inf)
    assert sampling.draw(np.array([np.inf, 0.0, np.inf]), 0.6) == (2, math.log(0.5))


def test_operator_is_registered():
    from torch._subclasses.fake_tensor import FakeTensorMode

    op = torch.ops.cdb.sample.default
    assert not any(a.alias_info is not None and a.alias_info.is_write for a in op._schema.arguments)
    with FakeTensorMode():
        tok, lp = torch.ops.cdb.sample(torch.empty(3, 50, device="cuda"),
                                       torch.empty(3, dtype=torch.float64, device="cuda"), None, None, None, None)
        assert tok.shape == lp.shape == (3,) and tok.dtype is torch.int64 and lp.dtype is torch.float32
