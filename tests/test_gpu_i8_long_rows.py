"""Norms of long rows of alike values: the mean of squares is as exact as tests/test_gpu_i8_rows.py derives, however many squares a thread adds."""
import pytest
import torch

from test_gpu_i8_rows import check_scales, expected

pytestmark = pytest.mark.gpu


# values whose squares, added one after the other in fp32, are rounded to one side more often than not
@pytest.mark.parametrize("t", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim,pad", [(131071, 0), (131064, 0), (131064, 1), (65537, 0), (40000, 0), (3999, 1)])
@pytest.mark.parametrize("residual", [True, False])
def test_rows_of_alike_values(psb, t, dim, pad, residual):
    row = torch.cat([torch.linspace(0.5, 2, 301), torch.tensor([0.6914310297, 1.5468403560, 0.7874243885, 1.4476282883, 0.5508383757])]).cuda()
    n = len(row)
    x = row[:, None].repeat(1, dim).to(t)
    r = (x * 0.5).to(t) if residual else None
    if pad:                                   # the residual's rows begin at other places than the rows: element by element
        wide = torch.zeros((n, dim + pad), dtype=t, device="cuda")
        wide[:, :dim] = x
    codes, scales = torch.empty((n, dim), dtype=torch.int8, device="cuda"), torch.empty(n, device="cuda")
    psb.i8_norm_rows(wide if pad else x, n, dim, None, 1e-5, codes, scales, d_residual=r, row_stride=dim + pad)
    assert (codes == 127).all()
    check_scales(scales, expected(x[:, :8], None if r is None else r[:, :8], None, float(torch.tensor(1e-5)))[1])   # (a row's mean is its value's)
