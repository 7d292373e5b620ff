"""Log-probabilities of drawn tokens (cdb_sample) to what their weights are held in, 2^-38, where the largest logit is many
temperatures from zero."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from continuous_depth_batching_amd import ops  # noqa: F401  (registers torch.ops.cdb.*)
from oracle import sampling

pytestmark = pytest.mark.gpu
DEV = "cuda"


def far_logits(rows, vocab, dtype, temperatures):
    """Rows whose spread is a few temperatures and whose largest logit is some 2^19 of them in powers of two, as far as
    the type can tell them apart."""

    gen = torch.Generator().manual_seed(vocab)
    x = torch.randn(rows, vocab, generator=gen, dtype=torch.float64)
    return (x * 2 + torch.linspace(-3e5, 3e5, rows, dtype=torch.float64)[:, None] * math.log(2)).mul(
        torch.from_numpy(temperatures.astype(np.float64))[:, None]).to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("vocab", [3, 700, 20000])
def test_a_token_alone_is_certain(vocab, dtype):
    rows = 200
    t = np.float32(10.0) ** np.linspace(-6, 5, rows, dtype=np.float32)
    x = far_logits(rows, vocab, dtype, t)
    u = torch.from_numpy(np.random.default_rng(vocab).random(rows)).to(DEV)
    for filters in (dict(top_k=1), dict(top_p=0.0)):
        k = torch.full((rows,), filters["top_k"], dtype=torch.int32, device=DEV) if "top_k" in filters else None
        p = torch.full((rows,), filters["top_p"], device=DEV) if "top_p" in filters else None
        _, lp = torch.ops.cdb.sample(x.to(DEV), u, torch.from_numpy(t).to(DEV), k, p, None)
        assert (lp == 0).all(), lp[lp != 0][:5]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("vocab", [2, 40, 5000, 30011])
@pytest.mark.parametrize("top_k", [0, 2, 1500])
def test_far_from_zero(top_k, vocab, dtype):
    rows = 120
    t = np.float32(10.0) ** np.linspace(-6, 5, rows, dtype=np.float32)
    x = far_logits(rows, vocab, dtype, t)
    u = np.random.default_rng(vocab + 1).random(rows)
    k = torch.full((rows,), top_k, dtype=torch.int32, device=DEV)
    tok, lp = torch.ops.cdb.sample(x.to(DEV), torch.from_numpy(u).to(DEV), torch.from_numpy(t).to(DEV), k, None, None)
    assert (lp <= 0).all()
    xs = x.double().numpy()
    for r in range(rows):
        token, logprob = sampling.draw(xs[r], float(u[r]), float(t[r]), top_k)
        assert int(tok[r]) == token, r
        assert abs(float(lp[r]) - logprob) <= 2.0 ** -24 * abs(logprob) + 2.0 ** -38, (r, float(lp[r]), logprob)
