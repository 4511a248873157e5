"""Arrays of more than 2^31 elements or 2^32 bytes: what lies at their ends."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_rows(psb):
    n, dim = 70_001, 32_000                       # 2.24e9 elements
    x = torch.zeros((n, dim), dtype=torch.bfloat16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    some = [0, 1, n // 2, n - 2, n - 1]
    x[some] = torch.randn((len(some), dim), generator=g, device="cuda").bfloat16()
    codes, scales = torch.full((n, dim), 77, dtype=torch.int8, device="cuda"), torch.empty(n, device="cuda")
    psb.i8_encode_rows(x, n, dim, codes, scales)
    u = x[some].double()
    top = u.abs().amax(1, keepdim=True)
    want = torch.round(127 * u / top).to(torch.int8)
    assert torch.equal(codes[some], want)
    assert (codes[n // 2 + 1] == 0).all() and scales[n // 2 + 1] == 0
    w = torch.ones(dim, device="cuda").bfloat16()
    psb.i8_norm_rows(x, n, dim, w, 1e-5, codes, scales, d_residual=x, d_sum=x)   # in place
    assert torch.equal(codes[some], want)
    assert torch.equal(x[some].double(), 2 * u)


def test_products(psb):
    m, n, k = 301, 8_000_001, 32                  # 2.4e9 outputs
    g = torch.Generator(device="cuda").manual_seed(2)
    x, w = (torch.randint(-127, 128, (r, k), generator=g, device="cuda", dtype=torch.int8) for r in (m, n))
    xs, ws = torch.rand(m, generator=g, device="cuda"), torch.rand(n, generator=g, device="cuda") * 0.01
    out = torch.empty((m, n), dtype=torch.float16, device="cuda")
    psb.i8_matmul(x, xs, m, w, ws, n, k, out)
    cols = torch.cat([torch.arange(0, 300, device="cuda"), torch.arange(n - 300, n, device="cuda")])
    want = (x.double() @ w[cols].double().T) * xs.double()[:, None] * ws[cols].double()
    bound = want.abs() * (3.1 * 2.0**-24 + 2.0**-11 * 1.001) + 2.0**-25
    assert bool(((out[:, cols].double() - want).abs() <= bound).all())
    rows = [0, m - 1]
    one = torch.empty((1, n), dtype=torch.float16, device="cuda")
    for r in rows:                                # the other kernels' way to the same outputs
        psb.i8_matmul(x[r:r + 1], xs[r:r + 1], 1, w, ws, n, k, one)
        assert torch.equal(one[0], out[r])


def test_rows_of_codes_behind_4_gb(psb):
    n, k = 270_000, 16_000                        # 4.3e9 bytes of codes
    w = torch.zeros((n, k), dtype=torch.int8, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(3)
    w[-200:] = torch.randint(-127, 128, (200, k), generator=g, device="cuda", dtype=torch.int8)
    ws = torch.full((n,), 1e-4, device="cuda")
    for m in (1, 20):
        x = torch.randint(-127, 128, (m, k), generator=g, device="cuda", dtype=torch.int8)
        out = torch.empty((m, n), device="cuda")
        psb.i8_matmul(x, torch.ones(m, device="cuda"), m, w, ws, n, k, out)
        want = (x.double() @ w[-300:].double().T) * ws[-300:].double()
        assert bool(((out[:, -300:].double() - want).abs() <= want.abs() * 3.1 * 2.0**-24).all()) and (out[:, :1000] == 0).all()


def test_selection(psb):
    batch, beams, vocab, k = 71, 2, 1 << 24, 4    # 2.4e9 logits, the largest vocabulary
    x = torch.full((batch * beams, vocab), -20.0, dtype=torch.float16, device="cuda")
    x[:, vocab - 3], x[-1, vocab - 1], x[-1, 5], x[-2, 7] = 3.0, 9.0, 8.0, 1.0
    s = torch.zeros((batch, beams), device="cuda")
    p, t, v = torch.empty((batch, k), dtype=torch.int32, device="cuda"), torch.empty((batch, k), dtype=torch.int32, device="cuda"), torch.empty((batch, k), device="cuda")
    psb.beam_select(x, s, batch, beams, vocab, k, p, t, v)
    total = torch.log_softmax(x[-2:].double(), 1)
    top, at = torch.sort(total.flatten(), descending=True, stable=True)
    assert torch.equal(p[-1], (at[:k] // vocab).int()) and torch.equal(t[-1], (at[:k] % vocab).int())
    assert bool(((v[-1].double() - top[:k]).abs() <= 1e-6 + top[:k].abs() * 2.0**-23).all())
    assert (t[0, :2] == vocab - 3).all() and torch.equal(p[0, :2].cpu(), torch.tensor([0, 1], dtype=torch.int32))


@pytest.mark.parametrize("place", [True, False])
def test_states(psb, place):
    layers, batch, beams, heads, tokens, dim = 2, 9, 4, 8, 4097, 1024   # 4.8 GB of bf16
    s = torch.zeros((layers, batch, beams, heads, tokens, dim), dtype=torch.bfloat16, device="cuda")
    s[-1, -1, :, -1, -1] = torch.arange(beams, device="cuda", dtype=torch.bfloat16)[:, None] + 1
    s[0, 0, :, 0, 0] = torch.arange(beams, device="cuda", dtype=torch.bfloat16)[:, None] + 11
    out = s if place else torch.zeros_like(s)
    parents = torch.tensor([3, 0, 0, 2], dtype=torch.int32, device="cuda").repeat(batch, 1)
    psb.beam_reorder(s, out, parents, layers, batch, beams, heads, tokens, dim * 2)
    want = torch.tensor([4, 1, 1, 3], device="cuda", dtype=torch.bfloat16)
    assert torch.equal(out[-1, -1, :, -1, -1, 0], want) and torch.equal(out[0, 0, :, 0, 0, -1], want + 10)
    assert out[:, :, :, :, 1:-1].count_nonzero() == 0


@pytest.mark.parametrize("m,n", [((1 << 31) - 256, 1), (5, (1 << 31) - 256), (1, (1 << 31) - 256)])
def test_products_of_the_most_rows(psb, m, n):
    k = 16                                        # 34 GB of codes
    g = torch.Generator(device="cuda").manual_seed(4)

    def codes(rows):                              # zeros, but for rows at both ends and beside 2^30
        c = torch.zeros((rows, k), dtype=torch.int8, device="cuda")
        some = sorted({r for r in (0, 1, 200, 255, 256, 1 << 30, rows - 257, rows - 256, rows - 2, rows - 1) if 0 <= r < rows})
        c[some] = torch.randint(-127, 128, (len(some), k), generator=g, device="cuda", dtype=torch.int8)
        return c, some
    x, xr = codes(m)
    w, wr = codes(n)
    xs, ws = torch.full((m,), 0.5, device="cuda"), torch.full((n,), 0.25, device="cuda")
    out = torch.full((m, n), 7.0, dtype=torch.float16, device="cuda")
    psb.i8_matmul(x, xs, m, w, ws, n, k, out)
    want = (x[xr].double() @ w[wr].double().T) * 0.125     # halves of eighths: at most 17 bits
    assert torch.equal(out[xr][:, wr], want.half())
    assert int(out.count_nonzero()) == int(want.count_nonzero())   # and zeros everywhere else
