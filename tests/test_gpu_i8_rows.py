"""8-bit codes of rows, plain and behind the residual addition and the norm, against 64-bit arithmetic.

Codes have to be equal.  A scale comes from 64-bit values but for the mean of squares, a sum of at most 16 products a thread and ten
additions over threads in fp32: relative error below 26 * 2^-24 in the mean, half of it in the root, and one rounding to fp32: 1e-6.
The sum is the fp32 sum rounded to the type: equal to the same two steps of torch.
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def expected(x, residual=None, weight=None, eps=None):
    h = x.double()
    if residual is not None:
        h = h + residual.double()
    u = h if weight is None else h * weight.double()
    top = u.abs().amax(1)
    dead = ~torch.isfinite(top) | ~torch.isfinite(h).all(1)
    codes = torch.round(127 * u / torch.where(top > 0, top, 1.0)[:, None])
    codes = torch.where(dead[:, None], 0.0, codes).to(torch.int8)
    scale = top / 127 if eps is None else top / (127 * torch.sqrt((h * h).mean(1) + eps))
    return codes, torch.where(dead, torch.nan, torch.where(top > 0, scale, 0.0))


def check_scales(got, want):
    got, want = got.double().cpu().numpy(), want.cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(want))
    fine = ~np.isnan(want)
    assert np.allclose(got[fine], want[fine], rtol=1e-6, atol=2e-45)


def values(n, dim, t, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((n, dim), generator=g, device="cuda") * torch.exp(2 * torch.randn((n, 1), generator=g, device="cuda"))
    x[:, :: max(1, dim // 3)] *= 10
    if n > 3:
        x[n // 2] = 0
        x[n // 3] = torch.randint(-3, 4, (dim,), generator=g, device="cuda").float()   # few values: codes on ties
    return x.to(t)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("n,dim", [(1, 1), (1, 7), (5, 8), (3, 16), (1000, 96), (257, 100), (33, 127), (40, 128), (7, 129), (9, 512), (4, 513), (5, 1024), (3, 1030),
                                   (2, 2048), (3, 4095), (6, 4096), (2, 4104), (2, 8192), (3, 8200), (1, 16384), (2, 16385), (1, 32768), (2, 32776), (1, 131071)])
def test_encode(psb, t, n, dim):
    x = values(n, dim, t, n * 7 + dim)
    codes, scales = torch.full((n + 1, dim), 99, dtype=torch.int8, device="cuda"), torch.full((n + 1,), 7.0, device="cuda")
    psb.i8_encode_rows(x, n, dim, codes, scales)
    want, scale = expected(x)
    assert torch.equal(codes[:n], want)
    check_scales(scales[:n], scale)
    assert (codes[n] == 99).all() and scales[n] == 7   # behind the last row


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("n,dim", [(1, 1), (3, 8), (700, 64), (50, 100), (33, 127), (5, 1024), (3, 1031), (300, 4096), (2, 5003), (1, 8192), (5, 8192), (2, 16384), (1, 20001), (1, 40000), (3, 53248), (2, 131064), (1, 131071)])
@pytest.mark.parametrize("residual,weight", [(True, True), (False, True), (True, False)])
def test_norm(psb, t, n, dim, residual, weight):
    x = values(n, dim, t, n + dim)
    r = values(n, dim, t, n + dim + 1) if residual else None
    w = (1 + 0.2 * torch.randn(dim, device="cuda")).to(t) if weight else None
    codes, scales = torch.empty((n, dim), dtype=torch.int8, device="cuda"), torch.empty(n, device="cuda")
    total = torch.empty_like(x)
    psb.i8_norm_rows(x, n, dim, w, 1e-5, codes, scales, d_residual=r, d_sum=total)
    want, scale = expected(x, r, w, float(np.float32(1e-5)))
    assert torch.equal(codes, want)
    check_scales(scales, scale)
    assert torch.equal(total, (x.float() + (r.float() if residual else 0)).to(t))


# enough rows to fill the GPU, at both sides of every change in the threads a row and in the elements a thread, rows that begin at packs and that do not
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("n,dim", [(40000, 1), (40001, 17), (40000, 64), (40003, 65), (30000, 128), (30000, 129), (20001, 256), (20000, 263), (9001, 512), (9000, 519), (5000, 1024), (5003, 1031),
                                   (3000, 4096), (3001, 4101), (1300, 8192), (1301, 8193), (1200, 9216), (1203, 9221), (700, 16384), (701, 16391), (600, 32768)])
def test_many_rows(psb, t, n, dim):
    x, r, w = values(n, dim, t, n), values(n, dim, t, n + 1), (1 + 0.2 * torch.randn(dim, device="cuda")).to(t)
    codes, scales = torch.empty((n, dim), dtype=torch.int8, device="cuda"), torch.empty(n, device="cuda")
    psb.i8_encode_rows(x, n, dim, codes, scales)
    want, scale = expected(x)
    assert torch.equal(codes, want)
    check_scales(scales, scale)
    want, scale = expected(x, r, w, float(np.float32(1e-5)))
    total = (x.float() + r.float()).to(t)
    psb.i8_norm_rows(x, n, dim, w, 1e-5, codes, scales, d_residual=r, d_sum=r)
    assert torch.equal(codes, want) and torch.equal(r, total)
    check_scales(scales, scale)


# both sides of the lengths to which a thread of a warp has three quarters of its elements, and few rows of them
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("n,dim", [(40000, 48), (40001, 52), (20000, 72), (30000, 96), (3, 96), (30001, 104), (20000, 192), (20001, 200), (10000, 384), (1, 384), (9000, 392), (6000, 768), (6001, 776)])
def test_three_quarters(psb, t, n, dim):
    test_many_rows(psb, t, n, dim)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("dim,pads", [(96, (3, 5, 7, 9)), (96, (8, 16, 24, 32)), (1000, (0, 1, 0, 0)), (4096, (8, 8, 8, 16)), (50, (1, 1, 1, 1))])
@pytest.mark.parametrize("where", ["apart", "rows", "residual"])
def test_strides_and_sums_in_place(psb, t, dim, pads, where):
    n = 37
    wide = lambda pad, seed: values(n, dim + pad, t, seed)  # noqa: E731
    x, r, total = wide(pads[0], 1), wide(pads[1], 2), torch.full((n, dim + pads[2]), 3.0, device="cuda").to(t)
    w = (1 + 0.1 * torch.randn(dim, device="cuda")).to(t)
    codes, scales = torch.full((n, dim + pads[3]), 99, dtype=torch.int8, device="cuda"), torch.empty(n, device="cuda")
    x0, r0 = x.clone(), r.clone()
    into = dict(apart=total, rows=x, residual=r)[where]
    behind = into[:, dim:].clone()
    psb.i8_norm_rows(x, n, dim, w, 1e-6, codes, scales, d_residual=r, d_sum=into, row_stride=dim + pads[0], residual_stride=dim + pads[1],
                     sum_stride=into.stride(0), code_stride=dim + pads[3])
    want, scale = expected(x0[:, :dim], r0[:, :dim], w, float(np.float32(1e-6)))
    assert torch.equal(codes[:, :dim], want) and (codes[:, dim:] == 99).all()
    check_scales(scales, scale)
    assert torch.equal(into[:, :dim], (x0[:, :dim].float() + r0[:, :dim].float()).to(t)) and torch.equal(into[:, dim:], behind)


@pytest.mark.parametrize("dim", [24, 100, 3000, 9000])
def test_ranges(psb, dim):
    """Infinities, NaN, rows of the type's largest and smallest values, one large value among small ones, weights of zero."""
    g = torch.Generator(device="cuda").manual_seed(dim)
    x = torch.randn((12, dim), generator=g, device="cuda")
    x[0, 3] = float("inf")
    x[1, dim - 1] = float("nan")
    x[2] *= 1e38
    x[3] *= 1e-38
    x[4] *= 1e-44
    x[5, 7] = 3e38
    x[6] = 0
    x[7, 0] = float("-inf")
    x[7, 1] = float("inf")
    x[8] = 1e25
    x[9] = -1e-30
    r = torch.zeros_like(x)
    r[2] = x[2]                     # the sum leaves fp32's range
    codes, scales = torch.empty((12, dim), dtype=torch.int8, device="cuda"), torch.empty(12, device="cuda")
    psb.i8_encode_rows(x, 12, dim, codes, scales)
    want, scale = expected(x)
    assert torch.equal(codes, want)
    check_scales(scales, scale)
    w = torch.randn(dim, generator=g, device="cuda")
    w[5] = 0
    for eps in (0.0, 1e-5):
        for residual in (None, r):
            psb.i8_norm_rows(x, 12, dim, w, eps, codes, scales, d_residual=residual)
            want, scale = expected(x, residual, w, float(np.float32(eps)))
            assert torch.equal(codes, want)
            check_scales(scales, scale)
    w[:] = 0
    psb.i8_norm_rows(x, 12, dim, w, 1e-5, codes, scales)
    want, scale = expected(x, None, w, 1e-5)
    assert torch.equal(codes, want)
    check_scales(scales, scale)


def test_codes_next_to_ties(psb):
    """Values a few units in the last place to either side of every tie: codes of 64-bit arithmetic all the same."""
    top = np.float32(3.7)
    ties = (np.arange(0, 127) + 0.5) * np.float64(top) / 127
    x = []
    for t in ties:
        v = np.float32(t)
        near = [v]
        for _ in range(6):
            near.append(np.nextafter(near[-1], np.float32(10)))
        for _ in range(6):
            v = np.nextafter(v, np.float32(-10))
            near.append(v)
        x += near + [-n for n in near]
    x = torch.tensor(np.array([top] + x, np.float32), device="cuda")[None].repeat(3, 1)
    dim = x.shape[1]
    codes, scales = torch.empty((3, dim), dtype=torch.int8, device="cuda"), torch.empty(3, device="cuda")
    psb.i8_encode_rows(x, 3, dim, codes, scales)
    assert torch.equal(codes, expected(x)[0])
    w = torch.full((dim,), 1.7, device="cuda")
    psb.i8_norm_rows(x, 3, dim, w, 1e-5, codes, scales, d_residual=x * 1e-8)
    assert torch.equal(codes, expected(x, x * 1e-8, w, 1e-5)[0])


def test_no_rows(psb):
    x = torch.zeros((1, 8), device="cuda")
    codes, scales = torch.full((1, 8), 5, dtype=torch.int8, device="cuda"), torch.full((1,), 2.0, device="cuda")
    psb.i8_encode_rows(x, 0, 8, codes, scales)
    assert (codes == 5).all() and scales[0] == 2


def test_other_stream_and_graph(psb):
    x = values(300, 512, torch.bfloat16, 5)
    codes, scales = torch.zeros((300, 512), dtype=torch.int8, device="cuda"), torch.zeros(300, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    psb.i8_encode_rows(x, 300, 512, codes, scales, stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(codes, expected(x)[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        psb.i8_encode_rows(x, 300, 512, codes, scales, stream=torch.cuda.current_stream().cuda_stream)
    x.copy_(values(300, 512, torch.bfloat16, 6))
    codes.zero_()
    graph.replay()
    assert torch.equal(codes, expected(x)[0])
