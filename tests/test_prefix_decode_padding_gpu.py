"""Groups whose first rows are padding: an answer that has ended, whose table row and cache layer say nothing any more."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import prefix_helpers as ph

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def end(s, rows):
    """Makes padding of rows and takes away what their table rows and cache layers said."""

    s.seq[rows] = -1
    s.layer[rows] = 99
    s.table[rows if s.table_row is None else s.table_row[rows].long()] = -1


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("rows", [5, 40, 150], ids=["few", "many", "more_than_a_wave"])
@pytest.mark.parametrize("left", ["second", "last"])
@pytest.mark.parametrize("shuffle", [False, True])
def test_first_rows_that_are_padding(left, rows, shuffle, dtype):
    group, own = [0] * rows + [1, -1, 1], [1 + b % 19 for b in range(rows)] + [4, 50, 6]
    s = ph.make(group, [64, 96], own, dtype=dtype, shuffle_rows=shuffle, seed=rows)  # prefixes of whole blocks
    want = ph.call(s).clone()
    ended = [0, rows] if left == "second" else [*range(rows - 1), rows]
    end(s, torch.tensor(ended, device="cuda"))
    got = ph.call(s)
    others = [b for b in range(rows + 3) if b not in ended]
    assert (got[ended] == 0).all()
    assert torch.equal(got[others], want[others])


def test_a_group_that_is_all_padding():
    s = ph.make([0, 0, 1], [64, 32], [3, 4, 5], seed=1)
    want = ph.call(s).clone()
    end(s, torch.tensor([0, 1], device="cuda"))
    got = ph.call(s)
    assert (got[:2] == 0).all() and torch.equal(got[2], want[2])


def test_rows_that_end_between_a_graphs_replays():
    s = ph.make(np.repeat([0, 1], 20), [80, 48], np.arange(40) % 9 + 1, seed=2)
    want = ph.call(s).clone()
    out = torch.empty_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ph.call(s, out=out)
    for ended in (0, 1, 20, 19, 3):
        end(s, torch.tensor([ended], device="cuda"))
        want[ended] = 0
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
