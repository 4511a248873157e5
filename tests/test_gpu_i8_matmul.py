"""Products of 8-bit codes against 64-bit arithmetic.

The sums are exact; their conversion to fp32 and the two products with the scales round by 2^-24 each, the output's type by eps / 2 more.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def codes(n, k, seed, pad=0, full=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    pitch = (k + 15) // 16 * 16 + pad
    c = torch.randint(-128, 128, (n, pitch), generator=g, device="cuda", dtype=torch.int8)
    if full:
        c[:] = -128
    return c


def scales(n, seed, size):
    return torch.rand(n, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda") * size


def expected(x, xs, w, ws, k):
    return (x[:, :k].double() @ w[:, :k].double().T) * xs.double()[:, None] * ws.double()


def close(got, want, t):
    # fp16 below its normal range rounds by half its smallest step
    bound = want.abs() * (3.1 * 2.0**-24 + torch.finfo(t).eps / 2 * 1.001) + (2.0**-25 if t == torch.float16 else 1e-40)
    return bool(((got.double() - want).abs() <= bound).all())


def check(psb, m, n, k, t, x_pad=0, w_pad=0, out_pad=0, full=False, limited=None):
    x, w = codes(m, k, 1 + m, x_pad, full), codes(n, k, 2 + n, w_pad, full)
    xs, ws = scales(m, 3, 1.0), scales(n, 4, 1.0 / (64 * k))
    out = torch.full((m + 1, n + out_pad), 77.0, device="cuda").to(t)
    kw = dict(x_stride=x.stride(0), w_stride=w.stride(0), out_stride=n + out_pad)
    if limited is None:
        psb.i8_matmul(x, xs, m, w, ws, n, k, out, **kw)
    else:
        psb.i8_matmul_limited(x, xs, m, w, ws, n, k, out, tiles=limited, polls=2000, **kw)
    want = expected(x, xs, w, ws, k)
    assert close(out[:m, :n], want, t)
    assert (out[m] == 77).all() and (out[:, n:] == 77).all()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 128, 128), (1, 1000, 4096), (1, 3, 5000), (2, 1001, 1037), (3, 515, 2063), (4, 30, 8200), (4, 10000, 1024), (2, 129, 16), (16, 128, 100), (17, 127, 129), (31, 300, 31), (64, 64, 2048), (100, 513, 640),
                                   (128, 128, 128), (129, 257, 257), (255, 100, 33), (256, 256, 512), (257, 130, 1000), (300, 5000, 96), (513, 640, 300),
                                   (1000, 2000, 130), (3, 40000, 256), (70, 130, 20000), (2049, 70, 72)])
def test_products(psb, m, n, k, t):
    check(psb, m, n, k, t)


@pytest.mark.parametrize("m,n,k", [(1, 4096, 4096), (37, 4099, 4000), (256, 2048, 8192), (4096, 4096, 1024), (2500, 3001, 515), (600, 30000, 128),
                                   # pairs of blocks: odd sizes, one slab, last tiles of few channels and tokens
                                   (193, 40000, 100), (4097, 5001, 333), (5000, 2561, 129), (300, 20000, 2048), (10000, 1100, 16)])
def test_larger_products(psb, m, n, k):
    check(psb, m, n, k, torch.float32)
    check(psb, m, n, k, torch.bfloat16)


@pytest.mark.parametrize("m,n,k", [(5, 200, 131071), (1, 64, 131071), (300, 300, 131071)])
def test_longest_rows_do_not_overflow(psb, m, n, k):
    check(psb, m, n, k, torch.float32, full=True)   # every product is 16,384: the sum is 2^31 - 16,384
    check(psb, m, n, k, torch.float32)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m,n,k", [(5, 131, 100), (40, 700, 1500), (300, 200, 200), (1100, 900, 260)])
def test_strides(psb, m, n, k, t):
    check(psb, m, n, k, t, x_pad=16, w_pad=48, out_pad=5)
    check(psb, m, n, k, t, x_pad=0, w_pad=16, out_pad=8)


def test_codes_behind_a_row_do_not_count(psb):
    """k codes of longer rows: what lies behind them in the same 16 bytes belongs to nobody."""
    for k in (1, 5, 17, 120, 130):
        check(psb, 33, 65, k, torch.float32, x_pad=128, w_pad=128)


@pytest.mark.parametrize("m,n,k,tiles", [(1, 300, 512, 0), (1, 300, 512, 1), (40, 130, 4096, 0), (300, 500, 700, 3), (300, 500, 700, 0), (2000, 4000, 128, 200),
                                         (2000, 4000, 1100, 150), (520, 70, 5000, 0),
                                         (3000, 4000, 300, 0), (3000, 4000, 300, 130), (700, 20000, 1000, 80)])
def test_results_when_a_wait_gives_up(psb, m, n, k, tiles):
    for t in TYPES:
        check(psb, m, n, k, t, limited=tiles)


def test_nan_scales_reach_their_rows_and_columns_only(psb):
    m, n, k = 40, 300, 256
    x, w, xs, ws = codes(m, k, 1), codes(n, k, 2), scales(m, 3, 1.0), scales(n, 4, 1e-3)
    xs[7], ws[11], ws[12] = float("nan"), float("nan"), 0.0
    out = torch.empty((m, n), device="cuda")
    psb.i8_matmul(x, xs, m, w, ws, n, k, out)
    want = expected(x, xs, w, ws, k)
    assert torch.equal(out.isnan(), want.isnan())
    fine = ~want.isnan()
    assert close(out[fine], want[fine], torch.float32)


def test_nothing_to_do(psb):
    out = torch.full((2, 2), 5.0, device="cuda")
    one = torch.ones(2, device="cuda")
    psb.i8_matmul(codes(2, 16, 1), one, 0, codes(2, 16, 2), one, 2, 16, out)
    psb.i8_matmul(codes(2, 16, 1), one, 2, codes(2, 16, 2), one, 0, 16, out, out_stride=2)
    assert (out == 5).all()


@pytest.mark.parametrize("m,n,k", [(8, 1000, 2048), (700, 1000, 512)])
def test_two_streams_and_graphs(psb, m, n, k):
    sets = []
    for i in range(2):
        x, w, xs, ws = codes(m, k, 10 + i), codes(n, k, 20 + i), scales(m, 30 + i, 1.0), scales(n, 40 + i, 1e-4)
        sets.append((x, xs, w, ws, torch.zeros((m, n), device="cuda")))
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for _ in range(5):
        for s, (x, xs, w, ws, out) in zip(streams, sets):
            psb.i8_matmul(x, xs, m, w, ws, n, k, out, stream=s.cuda_stream)
    torch.cuda.synchronize()
    for x, xs, w, ws, out in sets:
        assert close(out, expected(x, xs, w, ws, k), torch.float32)
    graphs = []
    for x, xs, w, ws, out in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            psb.i8_matmul(x, xs, m, w, ws, n, k, out, stream=torch.cuda.current_stream().cuda_stream)
        out.zero_()
        x.copy_(x.flip(0))
        graphs.append(g)
    for _ in range(2):
        for g in graphs:
            g.replay()
    for x, xs, w, ws, out in sets:
        assert close(out, expected(x, xs, w, ws, k), torch.float32)


def test_many_streams_of_split_paired_and_single_products(psb):
    """Calls of every kernel under way together on eight streams, small rings and large: their blocks hold tensor memory while they wait for each other."""
    shapes = [(16, 300, 1100), (224, 30000, 256), (256, 9000, 128), (40, 700, 4096), (100, 513, 2048), (1, 4000, 4096), (200, 20000, 100), (30, 128, 9000)]
    calls = []
    for i, (m, n, k) in enumerate(shapes):
        x, w, xs, ws = codes(m, k, 50 + i), codes(n, k, 60 + i), scales(m, 70 + i, 1.0), scales(n, 80 + i, 1e-4)
        calls.append((torch.cuda.Stream(), x, xs, w, ws, torch.zeros((m, n), device="cuda"), m, n, k))
    torch.cuda.synchronize()
    for _ in range(20):
        for s, x, xs, w, ws, out, m, n, k in calls:
            psb.i8_matmul(x, xs, m, w, ws, n, k, out, x_stride=x.stride(0), w_stride=w.stride(0), stream=s.cuda_stream)
    torch.cuda.synchronize()
    for s, x, xs, w, ws, out, m, n, k in calls:
        assert close(out, expected(x, xs, w, ws, k), torch.float32)


# Single blocks that run through several tiles, the tile's tokens for one half of the epilogue (20, 32) and for both (33, 100, 250), and pairs with tiles left over: the
# warps that share a tile have to agree on how their wait ended.
@pytest.mark.parametrize("m,n,k,tiles", [(20, 40000, 128, 0), (20, 40000, 128, 100), (20, 40000, 128, 200), (20, 40000, 128, 312), (32, 30000, 700, 170), (33, 40000, 100, 150),
                                         (100, 40000, 128, 0), (100, 40000, 128, 100), (100, 40000, 128, 200), (100, 30011, 700, 149), (180, 20000, 260, 155),
                                         (2000, 4000, 128, 60), (2000, 4000, 1100, 80), (250, 40001, 300, 100)])
def test_results_when_a_wait_of_single_blocks_or_pairs_gives_up(psb, m, n, k, tiles):
    for t in TYPES:
        check(psb, m, n, k, t, limited=tiles)
