"""Sums of exponentials over long rows, a warp a beam: the error of a beam's log-sum does not grow with the vocabulary.

In units of 2^-24, relative to the sum: a term is off by 4 (two units in the last place) and by what the rounding of its exponent does, at most 2.8 for logits up
to 3 below the largest (5.6 bits of exponent: half a unit of 2^-22, times ln 2) and less in proportion to its weight below; log2(e) rounded to fp32 by 0.7; a chain of four terms 3, the two
joins of a step 2, the compensated sum over the steps 2 - 14.5 in all, below 2^-20, an absolute 1e-6 in the logarithm.  The total is rounded to fp32 once more.
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def check(psb, x, vocab, batch, beams, t):
    """x: `beams` rows that every item has; the beams' totals of their best tokens lie 1e-5 apart, in an order of each item's own."""
    x = x.to(t)
    x64 = x.double()
    top, at = x64.max(1)
    log_sum = (x64 - top[:, None]).exp().sum(1).log()
    order = torch.stack([torch.randperm(beams, generator=torch.Generator().manual_seed(i)) for i in range(batch)]).cuda()
    scores = (log_sum[None] - 1e-5 * order).float()
    total = scores.double() - log_sum[None]
    best, parent = total.sort(1, descending=True)
    assert float((best[:, :-1] - best[:, 1:]).min()) > 4e-6
    logits = x.repeat(batch, 1)
    p, tokens = (torch.empty((batch, beams), dtype=torch.int32, device="cuda") for _ in range(2))
    v = torch.empty((batch, beams), device="cuda")
    psb.beam_select(logits, scores, batch, beams, vocab, beams, p, tokens, v)
    assert bool(((v.double() - best).abs() <= 1e-6 + best.abs() * 2.0**-23).all())
    assert torch.equal(p, parent.int()) and torch.equal(tokens, at[parent].int())


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("batch,beams,vocab", [(150, 16, 100_000), (150, 9, 200_000), (300, 3, 150_001), (1, 64, 262_144), (40, 33, 100_000)])
def test_rows_of_alike_logits(psb, t, batch, beams, vocab):
    """A beam's logits are all alike but for one; the beams differ a little."""
    x = -torch.linspace(0.2, 3.0, beams, device="cuda")[:, None].repeat(1, vocab)
    x[torch.arange(beams), torch.arange(beams) * 997 % vocab] = 0.0
    check(psb, x, vocab, batch, beams, t)


def test_the_longest_rows_a_warp_takes(psb):
    test_rows_of_alike_logits(psb, torch.float16, 150, 9, 1 << 22)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("batch,beams,vocab", [(150, 16, 100_000), (2, 12, 100_000)])
def test_rows_of_random_logits(psb, t, batch, beams, vocab):
    g = torch.Generator(device="cuda").manual_seed(vocab + beams)
    x = torch.rand((beams, vocab), generator=g, device="cuda") * torch.linspace(0.1, 8.0, beams, device="cuda")[:, None]
    x[:, 5] = 12.0
    check(psb, x, vocab, batch, beams, t)
