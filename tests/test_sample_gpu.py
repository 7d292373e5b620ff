"""Sampled tokens (cdb_sample through torch.ops.cdb.sample and ops.sample_raw) against the float64 definition.

Tokens have to be equal: the kernel's weights are off by 2^-38 of themselves and, by rounding to whole units, by 2^-47 of
the largest (2^-43 at 2^20 tokens), so it could differ only where the given number, or p, falls within about 2^-38 of a
border between two tokens. The numbers are drawn from a fixed seed and fall on no such border, or exactly on one that both
sides compute exactly. A log-probability is the fp32 rounding, 2^-24 relative, of a value that is off by what the kept
weight is: 2^-38."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from continuous_depth_batching_amd import ops
from oracle import sampling

pytestmark = pytest.mark.gpu
DEV = "cuda"


def run(logits, u, temperature=None, top_k=None, top_p=None, min_p=None):
    rows = logits.shape[0]

    def dev(v, dtype):
        if v is None:
            return None
        return torch.as_tensor(np.broadcast_to(np.asarray(v), (rows,)).copy()).to(dtype).to(DEV)

    tok, lp = torch.ops.cdb.sample(logits.to(DEV), dev(u, torch.float64), dev(temperature, torch.float32),
                                   dev(top_k, torch.int32), dev(top_p, torch.float32), dev(min_p, torch.float32))
    return tok.cpu(), lp.cpu()


def check(logits, u, temperature=None, top_k=None, top_p=None, min_p=None):
    got, lp = run(logits, u, temperature, top_k, top_p, min_p)
    x = logits.double().cpu().numpy()
    rows = x.shape[0]

    def at(v, r, default, f32):
        if v is None:
            return default
        y = np.broadcast_to(np.asarray(v), (rows,))[r]
        return float(np.float32(y)) if f32 else y

    for r in range(rows):
        token, logprob = sampling.draw(x[r], float(at(u, r, 0.0, False)), at(temperature, r, 1.0, True),
                                       int(at(top_k, r, 0, False)), at(top_p, r, 1.0, True), at(min_p, r, 0.0, True))
        assert int(got[r]) == token, (r, int(got[r]), token)
        if math.isinf(logprob):
            assert float(lp[r]) == logprob
        else:
            assert abs(float(lp[r]) - logprob) <= 2.0 ** -24 * abs(logprob) + 2.0 ** -38, (r, float(lp[r]), logprob)


def logits_of(rows, vocab, dtype, seed, spread=2.5):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, vocab, generator=gen) * spread
    x[:, ::max(1, vocab // 9)] += 2 * spread
    return x.to(dtype)


FILTERS = {
    "none": {},
    "temperature": dict(temperature=[0.3, 0.7, 1.0, 2.0, 40.0]),
    "top_k": dict(top_k=[1, 2, 7, 100, 5000]),
    "top_p": dict(top_p=[0.05, 0.5, 0.9, 0.99, 0.9999]),
    "min_p": dict(min_p=[0.01, 0.1, 0.5, 0.999, 1.0]),
    "all": dict(temperature=[0.6, 0.8, 1.0, 1.3, 0.0], top_k=[5, 50, 0, 1000, 3], top_p=[0.9, 0.5, 0.95, 0.8, 0.3],
                min_p=[0.0, 0.02, 0.1, 0.05, 0.5]),
}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("vocab", [1, 2, 7, 63, 1025, 8191, 50001])
@pytest.mark.parametrize("name", sorted(FILTERS))
def test_matches_definition(name, vocab, dtype):
    u = np.random.default_rng(vocab).random(5)
    check(logits_of(5, vocab, dtype, seed=vocab), u, **FILTERS[name])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_equal_logits_go_by_index(dtype):
    # Every logit the same, more of them than a list holds: borders are whole numbers, computed exactly by both.
    vocab = 40000
    x = torch.zeros(4, vocab, dtype=dtype)
    check(x, [0.0, 0.5, 0.25, 0.999], top_k=[3, 30000, 0, 0], top_p=[1.0, 1.0, 0.5, 0.125])
    check(x[:1], [0.9999999], top_k=[1])
    got, _ = run(x, [0.5, 0.5, 0.5, 0.5], temperature=[0.0] * 4)
    assert got.tolist() == [0, 0, 0, 0]


def test_zeros_of_both_signs_are_equal():
    x = torch.tensor([[-0.0, 0.0, -0.0, 0.0, -1.0]], dtype=torch.float32)
    for u in (0.0, 0.3, 0.6, 0.99):
        check(x, [u], top_k=[2])
    check(x, [0.9], temperature=[0.0])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("name", sorted(FILTERS))
def test_masked_infinite_and_nan_logits(name, dtype):
    x = logits_of(5, 4099, dtype, seed=5)
    x[0, 1:] = -math.inf                      # one token left
    x[1] = -math.inf                          # nothing left
    x[2, 100:] = float("nan")                 # NaN is never drawn
    x[3, [7, 400, 4000]] = math.inf           # only these
    x[4, :] = torch.finfo(dtype).min          # the lowest value is a value
    x[4, 17] = -math.inf
    u = [0.7, 0.5, 0.3, 0.8, 0.9]
    check(x, u, **FILTERS[name])
    nan = torch.full((1, 33), float("nan"), dtype=dtype)
    got, lp = run(nan, [0.5])
    assert got.tolist() == [-1] and lp.tolist() == [-math.inf]


def test_extreme_temperatures_and_parameters():
    x = logits_of(6, 3001, torch.float32, seed=9)
    inf, nan = math.inf, float("nan")
    check(x, [0.2, 0.4, 0.6, 0.8, 0.1, 0.9], temperature=[1e-30, 1e30, 1e-3, 1e-38, 300.0, 1.0],
          top_k=[-3, 0, 3000, 3001, 2 ** 31 - 1, 4])
    got, _ = run(x, [0.5] * 6, temperature=[-1.0, nan, 0.0, inf, 1.0, 1.0], top_p=[1, 1, 1, 1, -1.0, 0.0],
                 min_p=[0, 0, 0, 0, -1.0, 7.0])
    best = x.argmax(dim=1)
    for r in (0, 1, 2, 4, 5):
        assert int(got[r]) == int(best[r])
    assert int(got[3]) == 1500  # an endless temperature makes all 3001 tokens equal
    big = torch.tensor([[3e38, -3e38, 2.9e38, 0.0]])
    check(big, [0.5], temperature=[1e38])
    check(big, [0.99], temperature=[1e38], top_p=[0.95])


def test_numbers_outside_the_unit_interval_are_the_nearest_inside():
    x = logits_of(4, 999, torch.float32, seed=2, spread=0.5)
    got, _ = run(x, [-3.0, float("nan"), 1.0, 8.0])
    assert got[:2].tolist() == [0, 0] and got[2:].tolist() == [998, 998]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("vocab", [8192, 8193, 70001])
def test_many_tokens_kept_by_several_filters(vocab, dtype):
    # More than a list holds by top-k, by top-p and by min-p, and together; low temperatures at which most tokens weigh
    # less than a unit, where the k-th of them is far behind the last that weighs anything.
    x = logits_of(10, vocab, dtype, seed=vocab)
    check(x, np.random.default_rng(vocab + 1).random(10),
          temperature=[0.3, 0.05, 0.3, 3.0, 3.0, 3.0, 9.0, 9.0, 1.0, 0.01],
          top_k=[1000, 1200, 1201, 5000, 5000, 0, 0, 7000, 2500, 900],
          top_p=[1.0, 0.9999, 0.9, 0.97, 1.0, 0.97, 1.0, 0.999, 0.9999999, 0.5],
          min_p=[0.0, 0.0, 1e-9, 0.0, 1e-3, 1e-3, 1e-2, 1e-4, 0.0, 0.0])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_top_p_and_min_p_end_near_each_other(dtype):
    # Many tokens kept; the largest weights lie close together, so min-p ends before, in and behind the bins in which
    # top-p does.
    vocab, shares = 20011, [0.2, 0.5, 0.8, 0.95, 0.999]
    for temperature in (3.0, 8.0, 40.0):
        x = logits_of(1, vocab, dtype, seed=31, spread=2.0).expand(40, vocab).contiguous()
        top = (x[0].double() / temperature).sort(descending=True).values
        w = (top - top[0]).exp()
        ends = [float(w[int((w.cumsum(0) < p * w.sum()).sum())]) for p in shares]  # what top-p's last token weighs
        top_p = [p for p in shares for _ in range(8)]
        min_p = [e * f for e in ends for f in (0.2, 0.9, 0.97, 0.999, 1.0, 1.001, 1.03, 1.1)]
        check(x, np.random.default_rng(int(temperature)).random(40), temperature=[temperature] * 40, top_p=top_p,
              min_p=[min(1.0, m) for m in min_p])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_largest_vocabulary(dtype):
    vocab = 1 << 20
    x = logits_of(6, vocab, dtype, seed=41, spread=1.0)
    check(x, [0.999999, 0.2, 0.5, 0.8, 0.4, 0.7], temperature=[1.0, 1.0, 2.0, 1.0, 0.7, 0.0],
          top_k=[0, 50, 0, 40000, 1100, 0], top_p=[1.0, 0.9, 0.97, 1.0, 0.9, 1.0],
          min_p=[0.0, 0.0, 0.0, 0.0, 0.0, 0.0])


def test_calls_on_two_streams_at_once():
    sets = [logits_of(40, 5003 + 31000 * i, torch.bfloat16, seed=50 + i).to(DEV) for i in range(2)]
    u = torch.rand(40, dtype=torch.float64, generator=torch.Generator().manual_seed(3)).to(DEV)
    p = torch.full((40,), 0.95, device=DEV)
    want = [torch.ops.cdb.sample(x, u, None, None, p, None) for x in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(8):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(torch.ops.cdb.sample(sets[i], u, None, None, p, None))
    torch.cuda.synchronize()
    for i in range(2):
        for tok, lp in got[i]:
            assert torch.equal(tok, want[i][0]) and torch.equal(lp, want[i][1])


def test_more_rows_than_compute_units_of_a_long_vocabulary():
    rows, vocab = 260, 9001
    x = logits_of(rows, vocab, torch.float32, seed=21)
    kinds = [dict(top_k=0, top_p=1.0, min_p=0.0), dict(top_k=40, top_p=0.9, min_p=0.0),
             dict(top_k=0, top_p=0.95, min_p=0.0), dict(top_k=3000, top_p=0.99, min_p=0.0),
             dict(top_k=0, top_p=1.0, min_p=0.01)]
    check(x, np.random.default_rng(22).random(rows), temperature=[(0.0, 0.5, 1.0, 2.5)[r % 4] for r in range(rows)],
          **{n: [kinds[r % 5][n] for r in range(rows)] for n in ("top_k", "top_p", "min_p")})


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_logits_crowded_around_the_border(dtype):
    # Almost all logits have two values next to each other, so a bin holds more than a list and is narrowed by index.
    vocab = 20011
    x = torch.full((6, vocab), 1.0, dtype=dtype)
    x[:, ::3] = 1.0078125
    x[:, 5] = 9.0
    x[4:, 6] = -30.0
    check(x, [0.1, 0.5, 0.77, 0.93, 0.31, 0.9], top_k=[0, 6000, 6671, 9000, 0, 1100],
          top_p=[0.7, 1.0, 0.9, 0.5, 0.9, 0.99], min_p=[0.0, 0.0, 0.0, 0.0, 1e-4, 0.0])


def test_far_apart_logits_and_high_temperatures():
    # Differences beyond the type's range, and none at all among the largest of the parts.
    x = torch.zeros(4, 4000)
    x[0, ::2], x[0, 1::2] = 3e38, -3e38
    x[1, 7], x[1, 9] = 3.4e38, -3.4e38
    x[2, 1::8] = 5.0
    x[3] = torch.linspace(-3e38, 3e38, 4000)
    check(x, [0.3, 0.6, 0.9, 0.999], temperature=[1e38, 3e38, 1.0, 2e38], top_k=[1100, 30, 400, 1000])
    check(x, [0.3, 0.6, 0.9, 0.999], temperature=[1e38, 3e38, 1.0, 2e38], top_p=[0.9, 0.5, 0.99, 0.3])
    check(x, [0.3, 0.6, 0.9, 0.999], temperature=[1e38, 3e38, 1.0, 2e38], min_p=[0.01, 0.5, 0.1, 0.05])


def test_frequencies_follow_the_weights():
    # 200000 evenly spread numbers: each token's count is its share to within one number.
    x = torch.tensor([[0.3, -math.inf, 1.7, -0.5, 1.7, 0.0]])
    n = 200000
    u = (np.arange(n) + 0.5) / n
    got, _ = run(x.expand(n, 6).contiguous(), u)
    counts = torch.bincount(got, minlength=6).double()
    assert (counts - torch.softmax(x[0].double(), 0) * n).abs().max() <= 1


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("offset", [0, 1, 3, 7])
def test_strided_and_unaligned_rows(dtype, offset):
    base = logits_of(3, 2100, dtype, seed=offset).to(DEV)
    view = base[:, offset:offset + 2050 - offset]
    u = np.random.default_rng(offset).random(3)
    check(view, u, top_k=[40, 0, 900], top_p=[0.9, 0.9, 1.0])


def test_rows_do_not_depend_on_the_batch_and_captured_calls_repeat():
    x = logits_of(40, 20000, torch.bfloat16, seed=4).to(DEV)
    u = torch.rand(40, dtype=torch.float64, generator=torch.Generator().manual_seed(1)).to(DEV)
    t = torch.full((40,), 0.8, device=DEV)
    p = torch.full((40,), 0.9, device=DEV)
    tok = torch.empty(40, dtype=torch.int64, device=DEV)
    lp = torch.empty(40, device=DEV)
    ws = torch.empty(ops.sample_workspace_bytes(40, 20000), dtype=torch.uint8, device=DEV)
    ops.sample_raw(x, u, t, None, p, None, tok, lp, ws)
    eager, eager_lp = tok.clone(), lp.clone()
    for r in (0, 17, 39):
        one, one_lp = torch.ops.cdb.sample(x[r:r + 1], u[r:r + 1], t[:1], None, p[:1], None)
        assert int(one) == int(eager[r]) and float(one_lp) == float(eager_lp[r])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.sample_raw(x, u, t, None, p, None, tok, lp, ws)
    for _ in range(3):
        tok.fill_(-7)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(tok, eager) and torch.equal(lp, eager_lp)
    u.copy_(u.flip(0))
    graph.replay()
    again, _ = torch.ops.cdb.sample(x, u, t, None, p, None)
    assert torch.equal(tok, again)


def test_lm_head_sample_draws_from_its_logits():
    gen = torch.Generator().manual_seed(3)
    w = (torch.randn(4096, 256, generator=gen) * 0.2).bfloat16().to(DEV)
    x = torch.randn(6, 256, generator=gen).bfloat16().to(DEV)
    u = torch.rand(6, dtype=torch.float64, generator=gen).to(DEV)
    packed = ops.maybe_pack_linear_weight(w)
    tok, lp = ops.lm_head_sample(x, w, packed, u, top_p=torch.full((6,), 0.8, device=DEV))
    logits = torch.ops.cdb.linear(x, w, packed, False)
    for r in range(6):
        token, logprob = sampling.draw(logits[r].double().cpu().numpy(), float(u[r]), top_p=float(np.float32(0.8)))
        assert int(tok[r]) == token and abs(float(lp[r]) - logprob) <= 2.0 ** -24 * abs(logprob) + 2.0 ** -38
    cold, _ = ops.lm_head_sample(x, w, packed, u, temperature=torch.zeros(6, device=DEV))
    assert torch.equal(cold, ops.lm_head_argmax(x, w, packed))


def test_no_rows():
    tok, lp = torch.ops.cdb.sample(torch.empty(0, 9, device=DEV), torch.empty(0, dtype=torch.float64, device=DEV),
                                   None, None, None, None)
    assert tok.shape == (0,) and lp.shape == (0,)
