"""Products of 8-bit codes whose waits end after a few polls, with all products issued: any role of a block may give up, at any place.

What is under way then - products, copies - has to end before the block's memory is used for anything else, and the outputs are formed in another way: they
are the same, up to the roundings that tests/test_gpu_i8_matmul.py states.
"""
import pytest
import torch

from test_gpu_i8_matmul import close, codes, expected, scales

pytestmark = pytest.mark.gpu
POLLS = [1, 2, 3, 5, 8, 12, 20, 100]


def check(psb, m, n, k, polls):
    x, w, xs, ws = codes(m, k, 1 + m), codes(n, k, 2 + n), scales(m, 3, 1.0), scales(n, 4, 1.0 / (64 * k))
    out = torch.empty((m + 1, n), device="cuda")
    want = expected(x, xs, w, ws, k)
    for _ in range(3):
        out.fill_(77.0)
        psb.i8_matmul_limited(x, xs, m, w, ws, n, k, out, tiles=-1, polls=polls, x_stride=x.stride(0), w_stride=w.stride(0), out_stride=n)
        assert close(out[:m], want, torch.float32)
        assert (out[m] == 77).all()


# blocks of one tile, two and three, of one slab and of many; a tile's tokens for one half of the epilogue (20) and for both; tiles that blocks share
@pytest.mark.parametrize("polls", POLLS)
@pytest.mark.parametrize("m,n,k", [(20, 18000, 1000), (20, 37000, 128), (20, 50000, 300), (100, 18000, 4000), (100, 37000, 128), (180, 50000, 260), (40, 700, 4096), (130, 130, 9000)])
def test_single_and_split(psb, m, n, k, polls):
    check(psb, m, n, k, polls)


# pairs of blocks, whose two loading threads give up by themselves, so that one may have come further than the other
@pytest.mark.parametrize("polls", POLLS)
@pytest.mark.parametrize("m,n,k", [(200, 18000, 2000), (250, 30001, 300), (256, 18000, 128), (1000, 9000, 1100), (2000, 4000, 4096), (3000, 2561, 300)])
def test_pairs(psb, m, n, k, polls):
    check(psb, m, n, k, polls)
