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


# Logits far from zero, where what fp32 holds of a logit times log2(e) leaves nothing of its exponent: the same totals and the same order as in 64 bits.
@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("batch,beams,vocab", [(1, 4, 3000), (2, 5, 50_000), (160, 3, 1500)])
@pytest.mark.parametrize("offset", [1e4, 1e6, 3.99e6, 4e6, -4e6, 1e7, -2e8, 1e9, 1.37e10, 1e11, -1e12, 1e20, -1e20, 1.37e37, 1e38, 3e38, -3e38])
def test_far_logits(psb, t, batch, beams, vocab, offset):
    from test_gpu_beams import check as check_all
    g = torch.Generator(device="cuda").manual_seed(vocab + beams)
    x = (torch.randn((batch * beams, vocab), generator=g, device="cuda") * 3 + offset).to(t)
    s = -5 * torch.rand((batch, beams), generator=g, device="cuda")
    check_all(psb, x, s, 7)
    x[:, ::2] = torch.randn(x[:, ::2].shape, generator=g, device="cuda").to(t)   # half of them near zero
    check_all(psb, x, s, 7)


@pytest.mark.parametrize("vocab", [2000, 60_000])
@pytest.mark.parametrize("batch", [1, 160])
def test_logits_that_rise_through_every_range(psb, batch, vocab):
    """From one way of holding the base to the next, up and down, within a share and between them."""
    from test_gpu_beams import check as check_all
    border = np.float32(4e6)
    around = torch.from_numpy(border + np.arange(-vocab // 2, vocab - vocab // 2, dtype=np.float32) * np.float32(0.25))
    rows = [around, -around, around.flip(0), -around.flip(0), torch.linspace(-5e6, 5e6, vocab), torch.logspace(0, 38, vocab), -torch.logspace(0, 38, vocab).flip(0),
            torch.full((vocab,), 1e38), torch.full((vocab,), float(np.nextafter(np.float32(1e38), np.float32(2e38))))]
    rows[-1][: vocab // 2] = 1e38
    x = torch.stack(rows).float().cuda().repeat(batch, 1)
    check_all(psb, x, -torch.arange(9.0, device="cuda").repeat(batch, 1) * 0.37, 12)


def check_totals(psb, x, vocab, batch, beams):
    """The same scores as in check(), where tokens and beams lie closer together than totals are exact: the totals, and each one's own."""
    x64 = x.double()
    log_sum = (x64 - x64.amax(1, keepdim=True)).exp().sum(1).log() + x64.amax(1)
    order = torch.stack([torch.randperm(beams, generator=torch.Generator().manual_seed(i)) for i in range(batch)]).cuda()
    scores = (log_sum[None] - x64.amax(1) - 1e-5 * order).float()
    p, tokens = (torch.empty((batch, beams), dtype=torch.int32, device="cuda") for _ in range(2))
    v = torch.empty((batch, beams), device="cuda")
    psb.beam_select(x.repeat(batch, 1), scores, batch, beams, vocab, beams, p, tokens, v)
    log_p = x64 - log_sum[:, None]
    for i in range(batch):
        total = scores[i].double()[:, None] + log_p
        best = total.flatten().topk(beams)[0]
        bound = 1e-6 + best.abs() * 2.0**-23
        assert bool(((v[i].double() - best).abs() <= bound).all())
        assert bool(((v[i].double() - total[p[i].long(), tokens[i].long()]).abs() <= bound).all())


def test_slowly_rising_rows(psb):
    """The base rises many times while what came before still makes up most of the sum."""
    vocab, batch, beams = 100_000, 150, 16
    x = torch.stack([torch.linspace(-d, 0, vocab, device="cuda") for d in torch.linspace(0.3, 20, beams).tolist()])
    check_totals(psb, x, vocab, batch, beams)
    y = torch.full((beams, vocab), -17.0, device="cuda")       # and a few logits that rise above many
    y[:, ::9973] = torch.linspace(-16, 0, y[:, ::9973].shape[1], device="cuda")
    y -= torch.linspace(0, 1, beams, device="cuda")[:, None]
    check_totals(psb, y, vocab, batch, beams)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("batch,vocab", [(150, 100_000), (1, 1 << 24)])
def test_sums_of_logits_far_below_the_largest(psb, t, batch, vocab):
    """One logit at the top, all others d below.  The exponent's rounding is then half a unit of up to 2^-19, times ln 2: 11 of the units above, and log2(e)'s for d up to
    17 3.8 - with the rest 4 + 11 + 3.8 + 7 = 25.8, 1.54e-6."""
    beams = 9
    x = -torch.linspace(9.0, 17.0, beams, device="cuda")[:, None].repeat(1, vocab).to(t)
    x[:, 7] = 0
    log_sum = torch.log(1 + (vocab - 1) * x[:, 0].double().exp())
    p, tokens = (torch.empty((batch, beams), dtype=torch.int32, device="cuda") for _ in range(2))
    v = torch.empty((batch, beams), device="cuda")
    scores = torch.zeros((batch, beams), device="cuda")
    psb.beam_select(x.repeat(batch, 1) if batch > 1 else x, scores, batch, beams, vocab, beams, p, tokens, v)
    assert (tokens == 7).all() and torch.equal(p.sort(1)[0], torch.arange(beams, device="cuda", dtype=torch.int32).repeat(batch, 1))
    want = -log_sum[p.long()]
    assert bool(((v.double() - want).abs() <= 1.54e-6 + want.abs() * 2.0**-23).all())
