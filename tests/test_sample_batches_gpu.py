"""A row's token and log-probability, bit for bit, whatever batch it is drawn in: long rows are drawn by workgroups of 1024
threads up to 256 rows and of 512 beyond."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from continuous_depth_batching_amd import ops  # noqa: F401  (registers torch.ops.cdb.*)

pytestmark = pytest.mark.gpu
DEV = "cuda"


def batch(rows, vocab, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    rng = np.random.default_rng(seed)
    # Flat rows that keep thousands and rows in which a few stand out; some masked.
    x = torch.randn(rows, vocab, generator=gen) * torch.tensor([0.3, 1.0, 2.5])[torch.arange(rows) % 3, None]
    x[:, 5::997] += 6.0
    x[::7, ::2] = -math.inf
    x[3] = 1.0
    x[4] = -math.inf
    x[5, 100 % vocab] = math.inf

    def pick(values, dtype):
        return torch.from_numpy(rng.choice(np.asarray(values), size=rows)).to(dtype).to(DEV)

    return dict(logits=x.to(dtype).to(DEV), uniform=torch.rand(rows, dtype=torch.float64, generator=gen).to(DEV),
                temperature=pick([0.0, 0.3, 0.7, 1.0, 3.0, 40.0, 1e-6], torch.float32),
                top_k=pick([0, 0, 1, 40, 1000, 1201, 5000], torch.int32),
                top_p=pick([1.0, 0.3, 0.9, 0.97, 0.9999], torch.float32),
                min_p=pick([0.0, 0.0, 1e-6, 0.01, 0.3, 1.0], torch.float32))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("vocab", [8193, 20011, 49152])
def test_a_row_is_drawn_alike_in_any_batch(vocab, dtype):
    rows = 330
    b = batch(rows, vocab, dtype, vocab)
    tokens, logprobs = torch.ops.cdb.sample(*b.values())
    for size in (256, 41):
        for at in range(0, rows, size):
            part = {k: v[at:at + size] for k, v in b.items()}
            few, few_logprobs = torch.ops.cdb.sample(*part.values())
            assert torch.equal(few, tokens[at:at + size])
            assert torch.equal(few_logprobs, logprobs[at:at + size])
    for names in ((), ("temperature",), ("top_k",), ("top_p",), ("min_p",), ("top_p", "min_p")):
        only = {k: v if k in ("logits", "uniform") or k in names else None for k, v in b.items()}
        tokens, logprobs = torch.ops.cdb.sample(*only.values())
        head = {k: None if v is None else v[:256] for k, v in only.items()}
        few, few_logprobs = torch.ops.cdb.sample(*head.values())
        assert torch.equal(few, tokens[:256]) and torch.equal(few_logprobs, logprobs[:256]), names


def test_many_rows():
    b = batch(70001, 40, torch.float32, 5)
    tokens, logprobs = torch.ops.cdb.sample(*b.values())
    at = torch.arange(69900, 70001, device=DEV)
    few, few_logprobs = torch.ops.cdb.sample(*(v[at] for v in b.values()))
    assert torch.equal(few, tokens[at]) and torch.equal(few_logprobs, logprobs[at])
    assert int((tokens < 0).sum()) == int((~(b["logits"] > -math.inf).any(dim=1)).sum())
