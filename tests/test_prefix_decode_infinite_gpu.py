"""Infinite keys and values in decode attention of rows that share prefixes.

A column of the result is a sum of its own column of the values, so a value that is infinite there makes that element
infinite in every row that sees the token, and leaves the bits of all other elements as they are. A key that gives a
score of -infinity has no weight, as one whose score is finite and far below the others' has."""

from __future__ import annotations

import math

import pytest
import torch

import prefix_helpers as ph

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
INF = math.inf


def slot_of(s, row, position):
    trow = row if s.table_row is None else int(s.table_row[row])
    return int(s.table[trow, position // s.block]) * s.block + position % s.block


def scene(dtype, dim, rows, **kwargs):
    """Group 0 of `rows` rows after 70 tokens, group 1 of two rows after 33, and one row alone."""

    own = [1 + b % 37 for b in range(rows)] + [2, 40, 1500]
    return ph.make([0] * rows + [1, 1, -1], [70, 33], own, heads=4, kv=2, dim=dim, dtype=dtype, layers=2,
                   dead=float("nan"), seed=rows + dim, **kwargs)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("dim", [64, 96, 128])
@pytest.mark.parametrize("rows", [3, 40], ids=["few", "many"])
def test_infinite_values(rows, dim, dtype):
    s = scene(dtype, dim, rows)
    want = ph.call(s).clone()
    last = rows + 2
    expected = want.clone()

    def put(row, position, head, d, value, seen_by):
        s.pool[int(s.layer[row]), 1, slot_of(s, row, position), head, d] = value
        expected[seen_by, 2 * head:2 * head + 2, d] = value

    group = list(range(rows))
    put(0, 0, 0, 3, INF, group)          # the first token of a prefix
    put(0, 69, 1, dim - 1, -INF, group)  # the last one, in a tile that sticks out of the prefix
    put(0, 37, 1, 20, INF, group)
    put(rows, 32, 0, 8, INF, [rows, rows + 1])
    put(last, 0, 0, 1, -INF, [last])     # own tokens: the first, one of another chunk, the last that is cached
    put(last, 1100, 0, 7, INF, [last])
    put(last, 1498, 1, 33, INF, [last])
    put(rows + 1, 33, 1, 40, INF, [rows + 1])
    s.pool[int(s.layer[last]), 1, slot_of(s, last, 40), 1, 50] = INF  # both signs: no number
    s.pool[int(s.layer[last]), 1, slot_of(s, last, 1400), 1, 50] = -INF
    expected[last, 2:4, 50] = float("nan")
    s.k, s.v = s.k.clone(), s.v.clone()
    for row in (0, rows, last):          # the new token
        s.v[row, 1, 5] = -INF
        expected[row, 2:4, 5] = -INF
    got = ph.call(s)
    same = (got == expected) | (got.isnan() & expected.isnan())
    assert same.all(), (~same).nonzero()[:8].tolist()


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("rows", [3, 40], ids=["few", "many"])
def test_keys_of_minus_infinity_have_no_weight(rows, dtype):
    # Queries are positive at the key's element, one of them a bf16 number, so the score is -infinity.
    results = []
    for value in (-INF, -1e30):
        s = scene(dtype, 64, rows, rope=0)
        s.q, s.k, s.v = s.q.clone(), s.k.clone(), s.v.clone()
        s.q[:, :, 11] = s.q[:, :, 11].abs() + 0.5
        s.q[1, :, 11] = 8.0
        s.scale = 0.125 / math.log2(math.e)  # a query of 8 is about 1 scaled
        last = rows + 2
        for row, position in ((0, 5), (0, 69), (rows, 32), (last, 0), (last, 1200), (last, 1498)):
            s.pool[int(s.layer[row]), 0, slot_of(s, row, position), :, 11] = value
        s.k[2, :, 11] = value            # a new token's
        results.append(ph.call(s))
    assert torch.isfinite(results[0]).all() and torch.equal(*results)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
def test_a_value_that_only_one_row_sees_stays_with_it(dtype):
    s = scene(dtype, 128, 40)
    want = ph.call(s).clone()
    s.k, s.v = s.k.clone(), s.v.clone()
    s.v[7] = INF
    got = ph.call(s)
    others = [b for b in range(43) if b != 7]
    assert torch.equal(got[others], want[others]) and (got[7] == INF).all()
