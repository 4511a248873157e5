"""Beam selection and reordering of states against 64-bit arithmetic and indexing.

Parents and tokens have to be those of 64-bit totals, ties to the lowest (beam, token).  A total's error: a row's sum of exponentials has a
relative error below 2^-20 (terms of 2 units in the last place and their arguments' rounding, sums of some hundred terms in fp32), an absolute one of
1e-6 in its logarithm, and the total is rounded to fp32 once.
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def expected(logits, scores, k):
    """Totals in 64 bits, largest first, ties to the lowest index; -1, -1, -inf where nothing is left."""
    batch, beams = scores.shape
    x = logits.double().view(batch, beams, -1)
    vocab = x.shape[2]
    top = x.amax(2, keepdim=True)
    total = scores.double()[:, :, None] + ((x - top) - torch.exp(x - top).sum(2, keepdim=True).log())
    closed = ~torch.isfinite(top) | x.isnan().any(2, keepdim=True) | ~torch.isfinite(scores.double())[:, :, None]
    total = torch.where(closed, -torch.inf, total).view(batch, beams * vocab)
    if total.shape[1] < k:
        total = torch.cat([total, torch.full((batch, k - total.shape[1]), -torch.inf, dtype=torch.float64, device=total.device)], 1)
    total, at = torch.sort(total, dim=1, descending=True, stable=True)
    total, at = total[:, :k], at[:, :k]
    none = total == -torch.inf
    return torch.where(none, -1, at // vocab).int(), torch.where(none, -1, at % vocab).int(), total


def chosen(psb, logits, scores, k, row_stride=0, **kw):
    batch, beams = scores.shape
    parents = torch.full((batch + 1, k), 99, dtype=torch.int32, device="cuda")
    tokens, totals = parents.clone(), torch.full((batch + 1, k), 99.0, device="cuda")
    psb.beam_select(logits, scores, batch, beams, logits.shape[1], k, parents, tokens, totals, row_stride=row_stride, **kw)
    torch.cuda.synchronize()
    assert (parents[batch] == 99).all() and (tokens[batch] == 99).all() and (totals[batch] == 99).all()
    return parents[:batch], tokens[:batch], totals[:batch]


def check(psb, logits, scores, k, row_stride=0):
    p, t, v = chosen(psb, logits, scores, k, row_stride)
    wp, wt, wv = expected(logits, scores, k)
    assert torch.equal(p, wp) and torch.equal(t, wt)
    none = wv == -torch.inf
    assert torch.equal(v == -torch.inf, none)
    assert bool(((v.double() - wv).abs()[~none] <= 1e-6 + wv.abs()[~none] * 2.0**-23).all())


def make(batch, beams, vocab, t, seed, pad=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn((batch * beams, vocab + pad), generator=g, device="cuda") * 3).to(t)
    s = -5 * torch.rand((batch, beams), generator=g, device="cuda")
    return x[:, :vocab], s


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("batch,beams,vocab,k", [(1, 1, 1, 1), (1, 1, 5, 8), (2, 3, 2, 6), (1, 4, 255, 8), (3, 5, 257, 10), (2, 1, 1000, 1), (1, 64, 300, 64), (2, 16, 4099, 32),
                                                 (1, 4, 32000, 8), (7, 3, 50257, 6), (1, 1, 200000, 64), (40, 2, 8000, 4), (300, 1, 500, 5), (1, 64, 20000, 64), (150, 8, 3001, 16)])
def test_selection(psb, t, batch, beams, vocab, k):
    check(psb, *make(batch, beams, vocab, t, vocab + k), k)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("pad", [1, 8, 13])
def test_strides(psb, t, pad):
    x, s = make(3, 4, 1001, t, pad, pad)
    check(psb, x, s, 9, row_stride=1001 + pad)
    x, s = make(3, 4, 1008, t, pad, pad)
    check(psb, x, s, 9, row_stride=1008 + pad)


@pytest.mark.parametrize("t", TYPES)
def test_masks(psb, t):
    x, s = make(8, 4, 700, t, 3)
    low = torch.finfo(t).min
    x[0, :] = -torch.inf                    # a beam without a token
    x[4:8, 1:] = -torch.inf                 # one token a beam
    x[8:12, :] = -torch.inf                 # an item without any
    x[12, 5] = torch.nan
    x[13, 699] = torch.inf
    x[16:20, :] = low                       # the lowest value everywhere: all tokens alike
    x[20:24, 3:] = low
    x[24, :] = low
    x[24, 17] = -torch.inf
    s[5, 0] = -torch.inf
    s[6, :] = -torch.inf
    s[7, 1], s[7, 2] = torch.nan, torch.inf
    for k in (1, 7, 64):
        check(psb, x, s, k)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("vocab", [100, 3000, 40000])
def test_ties(psb, t, vocab):
    """All logits alike; few different values; the same row in every beam, at places of other alignment too."""
    s = torch.zeros((2, 3), device="cuda")
    check(psb, torch.zeros((6, vocab), device="cuda", dtype=t), s, 64)
    g = torch.Generator(device="cuda").manual_seed(vocab)
    check(psb, torch.randint(0, 3, (6, vocab), generator=g, device="cuda").to(t), s, 50)
    row = torch.randn(vocab, generator=g, device="cuda").to(t)
    for pad in (0, 1, 4):
        flat = torch.zeros(6 * (vocab + pad) + 8, dtype=t, device="cuda")
        x = flat[:6 * (vocab + pad)].view(6, vocab + pad)[:, :vocab]
        x[:] = row
        check(psb, x, s, 20, row_stride=vocab + pad)
        x[0::2] = torch.where(row == 0, -row, row)   # zeros of either sign are alike
        check(psb, x, s, 20, row_stride=vocab + pad)


@pytest.mark.parametrize("batch,beams,vocab", [(1, 4, 32000), (400, 3, 1000), (64, 8, 20000)])
def test_totals_in_place_of_the_scores(psb, batch, beams, vocab):
    logits, scores = make(batch, beams, vocab, torch.bfloat16, 91)
    parents, tokens, totals = chosen(psb, logits, scores, beams)
    p, t = torch.empty_like(parents), torch.empty_like(tokens)
    psb.beam_select(logits, scores, batch, beams, vocab, beams, p, t, scores)
    assert torch.equal(p, parents) and torch.equal(t, tokens) and torch.equal(scores, totals)


@pytest.mark.parametrize("vocab", [5000, 128000])
def test_sorted_and_concentrated_rows(psb, vocab):
    """The best tokens side by side, in one warp's share."""
    x = torch.linspace(-10, 10, vocab, device="cuda").repeat(4, 1)
    s = torch.tensor([[0.0, -0.1, -20.0, -0.3]], device="cuda")
    check(psb, x, s, 64)
    check(psb, x.flip(1).contiguous(), s, 64)
    y = torch.full((4, vocab), -50.0, device="cuda")
    y[:, 256:512] = torch.randn((4, 256), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    check(psb, y, s, 64)


def test_large_and_small_logits(psb):
    g = torch.Generator(device="cuda").manual_seed(9)
    x = torch.randn((4, 3000), generator=g, device="cuda")
    x[1] *= 1e4
    x[2] = x[2] * 1e-6 + 1e4
    x[3] -= 3e38
    check(psb, x, torch.zeros((1, 4), device="cuda"), 16)
    check(psb, x, torch.zeros((4, 1), device="cuda"), 16)


def test_streams_and_graph(psb):
    x, s = make(3, 4, 20000, torch.float32, 1)
    k = 8
    p, t, v = (torch.zeros((3, k), dtype=d, device="cuda") for d in (torch.int32, torch.int32, torch.float32))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    psb.beam_select(x, s, 3, 4, 20000, k, p, t, v, stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(t, expected(x, s, k)[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        psb.beam_select(x, s, 3, 4, 20000, k, p, t, v, stream=torch.cuda.current_stream().cuda_stream)
    x.copy_(make(3, 4, 20000, torch.float32, 2)[0])
    graph.replay()
    wp, wt, _ = expected(x, s, k)
    assert torch.equal(t, wt) and torch.equal(p, wp)


# ---- states ----

def reordered(states, parents, lengths, into):
    out = into.clone()
    for b in range(parents.shape[0]):
        n = states.shape[4] if lengths is None else min(max(int(lengths[b]), 0), states.shape[4])
        for j, p in enumerate(parents[b].tolist()):
            if 0 <= p < states.shape[2]:
                out[:, b, j, :, :n] = states[:, b, p, :, :n]
    return out


@pytest.mark.parametrize("layers,batch,beams,heads,tokens,bytes_", [(1, 1, 1, 1, 1, 1), (2, 3, 4, 2, 5, 32), (1, 2, 5, 3, 17, 6), (3, 1, 8, 8, 33, 128), (1, 2, 9, 2, 10, 20), (2, 2, 16, 1, 7, 256),
                                                                    (1, 1, 64, 2, 9, 48), (1, 3, 33, 1, 11, 7), (2, 5, 4, 8, 515, 128), (1, 1, 2, 1, 100000, 160), (300, 250, 2, 1, 2, 16)])
@pytest.mark.parametrize("place", [True, False])
@pytest.mark.parametrize("ragged", [True, False])
def test_reorder(psb, layers, batch, beams, heads, tokens, bytes_, place, ragged):
    rng = np.random.default_rng(tokens + beams)
    g = torch.Generator(device="cuda").manual_seed(beams)
    states = torch.randint(0, 256, (layers, batch, beams, heads, tokens, bytes_), generator=g, device="cuda", dtype=torch.uint8)
    parents = rng.integers(-1, beams + 1, (batch, beams)).astype(np.int32)   # some outside
    parents[0] = rng.permutation(beams)                                       # a permutation: cycles
    lengths = rng.integers(-1, tokens + 2, batch).astype(np.int32) if ragged else None
    d_parents, d_lengths = torch.from_numpy(parents).cuda(), torch.from_numpy(lengths).cuda() if ragged else None
    out = states.clone() if place else torch.randint(0, 256, states.shape, generator=g, device="cuda", dtype=torch.uint8)
    want = reordered(states, parents, lengths, out)
    before = states.clone()
    psb.beam_reorder(out if place else states, out, d_parents, layers, batch, beams, heads, tokens, bytes_, d_lengths=d_lengths)
    assert torch.equal(out, want)
    assert torch.equal(states, before)


def test_reorder_offset_buffers(psb):
    """States that begin at odd places."""
    flat = torch.arange(2 * 3 * 4 * 6 + 64, device="cuda").to(torch.uint8)
    for at in (1, 2, 4, 8, 16):
        a = flat.clone()
        s = a[at:at + 144].view(1, 2, 3, 1, 4, 6)
        parents = np.array([[2, 0, 1], [1, 1, 0]], np.int32)
        want = reordered(s.clone(), parents, None, s)
        psb.beam_reorder(s, s, torch.from_numpy(parents).cuda(), 1, 2, 3, 1, 4, 6)
        assert torch.equal(s, want) and torch.equal(a[:at], flat[:at]) and torch.equal(a[at + 144:], flat[at + 144:])


# ---- a generating model's step ----

@pytest.mark.parametrize("batch,beams", [(1, 4), (3, 5)])
def test_steps_of_a_beam_search(psb, batch, beams):
    """Norm, product with the vocabulary's rows, selection, reordering, in a captured graph, three steps: the same beams as the search in 64 bits on the same codes."""
    dim, vocab, steps, heads = 256, 1003, 3, 2
    rows = batch * beams
    g = torch.Generator(device="cuda").manual_seed(batch)
    table = torch.randn((vocab, dim), generator=g, device="cuda").bfloat16()
    w, ws = torch.empty((vocab, dim), dtype=torch.int8, device="cuda"), torch.empty(vocab, device="cuda")
    psb.i8_encode_rows(table, vocab, dim, w, ws)
    weight = (1 + 0.1 * torch.randn(dim, generator=g, device="cuda")).bfloat16()
    x = torch.randn((rows, dim), generator=g, device="cuda").bfloat16()
    stream = torch.randn((rows, dim), generator=g, device="cuda").bfloat16()
    codes, cs = torch.empty((rows, dim), dtype=torch.int8, device="cuda"), torch.empty(rows, device="cuda")
    logits = torch.empty((rows, vocab), device="cuda")
    scores = torch.zeros((batch, beams), device="cuda")
    parents, tokens = (torch.zeros((batch, beams), dtype=torch.int32, device="cuda") for _ in range(2))
    totals = torch.zeros((batch, beams), device="cuda")
    history = torch.full((1, batch, beams, heads, steps, 2), -1, dtype=torch.int16, device="cuda")

    def step(s):
        psb.i8_norm_rows(x, rows, dim, weight, 1e-5, codes, cs, d_residual=stream, d_sum=stream, stream=s)
        psb.i8_matmul(codes, cs, rows, w, ws, vocab, dim, logits, stream=s)
        psb.beam_select(logits, scores, batch, beams, vocab, beams, parents, tokens, totals, stream=s)
        psb.beam_reorder(history, history, parents, 1, batch, beams, heads, steps, 4, stream=s)
        psb.beam_reorder(stream, stream, parents, 1, batch, beams, 1, 1, dim * 2, stream=s)

    keep = stream.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(side.cuda_stream)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(torch.cuda.current_stream().cuda_stream)
    stream.copy_(keep)
    scores.zero_()
    scores[:, 1:] = -torch.inf               # the first step has one beam
    history.fill_(-1)
    ref_stream, ref_scores, ref_history = keep.clone(), scores.clone(), history.clone()
    for i in range(steps):
        graph.replay()
        # the same step in 64 bits, from the codes' definition
        h = x.double() + ref_stream.double()
        u = h * weight.double()
        top = u.abs().amax(1, keepdim=True)
        q = torch.round(127 * u / top) * (top / 127 / torch.sqrt((h * h).mean(1, keepdim=True) + 1e-5))
        table64 = torch.round(127 * table.double() / table.double().abs().amax(1, keepdim=True)) * (table.double().abs().amax(1, keepdim=True) / 127)
        wp, wt, wv = expected(q @ table64.T, ref_scores, beams)
        assert torch.equal(parents, wp) and torch.equal(tokens, wt)
        assert torch.allclose(totals.double(), wv, rtol=1e-5, atol=1e-5)
        at = torch.arange(batch, device="cuda")[:, None]
        ref_history = ref_history[:, at, wp.long()]
        assert torch.equal(history, ref_history)
        summed = (x.float() + ref_stream.float()).bfloat16().view(batch, beams, dim)
        ref_stream = summed[at, wp.long()].reshape(rows, dim)
        assert torch.equal(stream, ref_stream)
        for target in (history, ref_history):
            target[0, :, :, :, i, 0] = wt[:, :, None].to(torch.int16)
        scores.copy_(totals)
        ref_scores = totals.clone()
        x.copy_(table[tokens.flatten().long()])
