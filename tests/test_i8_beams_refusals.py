"""Calls that the 8-bit row and beam operators refuse: before any device is looked for, so they run without one."""
import pytest
import torch

from paraselect_b200 import api, build


@pytest.fixture(scope="module", autouse=True)
def built():
    build.ensure_built()


def refused(status, call, *args, **kw):
    with pytest.raises(api.PsbError) as e:
        call(*args, **kw)
    assert e.value.status == status, e.value


def rows(n=4, dim=32, t=torch.float32):
    return torch.zeros((n, dim), dtype=t)


def codes(n=4, dim=32):
    return torch.zeros((n, dim), dtype=torch.int8)


def test_encode_refusals():
    x, c, s = rows(), codes(), torch.zeros(4)
    bad = lambda status, *a, **kw: refused(status, api.i8_encode_rows, *a, **kw)  # noqa: E731
    bad(1, x, -1, 32, c, s)
    bad(1, x, 4, 0, c, s)
    bad(1, x, 4, 32, c, s, row_stride=31)
    bad(1, x, 4, 32, c, s, code_stride=31)
    bad(1, x, 4, 32, None, s)
    bad(1, x, 4, 32, c, None)
    bad(1, rows(t=torch.float64), 4, 32, c, s)
    bad(1, x, 4, 32, x.view(torch.int8), s)                      # the codes lie over the rows
    bad(1, x, 4, 32, c, c.view(-1)[:16].view(torch.float32))      # the scales lie over the codes
    bad(2, x, 1, 131072, c, s)
    bad(2, x, 1 << 31, 32, c, s)


def test_norm_refusals():
    x, r, w, c, s = rows(), rows(), torch.zeros(32), codes(), torch.zeros(4)
    bad = lambda status, *a, **kw: refused(status, api.i8_norm_rows, *a, **kw)  # noqa: E731
    bad(1, x, 4, 32, w, -1e-5, c, s)
    bad(1, x, 4, 32, w, float("nan"), c, s)
    bad(1, x, 4, 32, w, float("inf"), c, s)
    bad(1, x, 4, 32, w.half(), 1e-5, c, s)
    bad(1, x, 4, 32, w, 1e-5, c, s, d_residual=r.bfloat16())
    bad(1, x, 4, 32, w, 1e-5, c, s, d_residual=r, residual_stride=16)
    bad(1, x, 4, 32, w, 1e-5, c, s, d_sum=r, sum_stride=16)
    flat = torch.zeros(4 * 32 + 8)
    bad(1, flat[:128].view(4, 32), 4, 32, w, 1e-5, c, s, d_sum=flat[4:132].view(4, 32))   # the sum lies over the rows, shifted
    wide = torch.zeros((4, 64))
    bad(1, wide, 4, 32, w, 1e-5, c, s, d_sum=wide, row_stride=64, sum_stride=32)
    bad(1, x, 4, 32, w, 1e-5, c, s, d_sum=w)
    bad(1, x, 4, 32, w, 1e-5, r.view(torch.int8), s, d_residual=r)


def test_matmul_refusals():
    x, w, out = codes(4, 32), codes(8, 32), torch.zeros((4, 8))
    xs, ws = torch.zeros(4), torch.zeros(8)
    bad = lambda status, *a, **kw: refused(status, api.i8_matmul, *a, **kw)  # noqa: E731
    bad(1, x, xs, -1, w, ws, 8, 32, out)
    bad(1, x, xs, 4, w, ws, -1, 32, out)
    bad(1, x, xs, 4, w, ws, 8, 0, out)
    bad(2, x, xs, 4, w, ws, 8, 131072, out, x_stride=131072, w_stride=131072)
    bad(1, x, xs, 4, w, ws, 8, 20, out)                                 # rows 20 bytes apart
    bad(1, x.view(-1)[1:], xs, 3, w, ws, 8, 32, out)                    # rows at odd places
    bad(1, x, xs, 4, w, ws, 8, 32, out, x_stride=16)
    bad(1, x, xs, 4, w, ws, 8, 32, out, out_stride=7)
    bad(1, x, xs, 4, w, ws, 8, 32, out.double())
    bad(1, x, xs, 4, w, ws, 8, 32, x.view(torch.float32).view(4, 8))   # the output lies over an input
    bad(1, x, xs, 4, w, ws, 8, 32, ws, out_stride=8)
    bad(1, None, xs, 4, w, ws, 8, 32, out)
    refused(1, api.i8_matmul_limited, x, xs, 4, w, ws, 8, 32, out, polls=0)


def test_select_refusals():
    logits, scores = torch.zeros((6, 10)), torch.zeros((2, 3))
    p, t, v = torch.zeros((2, 4), dtype=torch.int32), torch.zeros((2, 4), dtype=torch.int32), torch.zeros((2, 4))
    many = torch.zeros(9)
    bad = lambda status, *a, **kw: refused(status, api.beam_select, *a, **kw)  # noqa: E731
    bad(1, logits, scores, -1, 3, 10, 4, p, t, v)
    bad(1, logits, scores, 2, 0, 10, 4, p, t, v)
    bad(1, logits, scores, 2, 3, 0, 4, p, t, v)
    bad(1, logits, scores, 2, 3, 10, 0, p, t, v)
    bad(1, logits, scores, 2, 3, 10, 4, p, t, v, row_stride=9)
    bad(1, logits, None, 2, 3, 10, 4, p, t, v)
    bad(1, logits.long(), scores, 2, 3, 10, 4, p, t, v)
    for call in ((logits, scores, 2, 3, 10, 4, p, p, v),            # outputs over each other, over the logits, over the scores of other items
                 (logits, scores, 2, 3, 10, 4, p, t, t.view(torch.float32)), (logits, scores, 2, 3, 10, 4, p, t, logits),
                 (logits, scores, 2, 3, 10, 4, p, scores.view(torch.int32), v), (logits, scores, 2, 3, 10, 2, p, t, scores),
                 (logits, many, 2, 3, 10, 3, p, t, many[1:])):
        bad(1, *call)
    bad(2, logits, scores, 2, 65, 10, 4, p, t, v)
    bad(2, logits, scores, 2, 3, 10, 65, p, t, v)
    bad(2, logits, scores, 2, 3, (1 << 24) + 1, 4, p, t, v)


def test_reorder_refusals():
    a, b, p = torch.zeros(2 * 3 * 4 * 5 * 2), torch.zeros(2 * 3 * 4 * 5 * 2), torch.zeros((2, 3), dtype=torch.int32)
    bad = lambda status, *args, **kw: refused(status, api.beam_reorder, *args, **kw)  # noqa: E731
    bad(1, a, b, p, 1, 2, 0, 4, 5, 8)
    bad(1, a, b, p, 1, 2, 3, 0, 5, 8)
    bad(1, a, b, p, 1, 2, 3, 4, 5, 0)
    bad(1, a, b, p, -1, 2, 3, 4, 5, 8)
    bad(1, a, b, None, 1, 2, 3, 4, 5, 8)
    bad(1, a, a[2:], p, 1, 2, 3, 4, 5, 8)                 # the buffers overlap without being the same
    bad(1, a, b, b[6:].view(torch.int32), 1, 2, 3, 4, 5, 8)   # the parents, the lengths lie in the states
    bad(1, a, b, p, 1, 2, 3, 4, 5, 8, d_lengths=b[-2:].view(torch.int32))
    bad(2, a, b, p, 1, 2, 65, 4, 5, 8)
    bad(2, a, b, p, 70000, 2, 3, 4, 5, 8)
    bad(2, a, b, p, 1, 2, 3, 4, 2**31 - 1, 1 << 40)


def test_arrays_of_other_types():
    """Codes are int8, scales and totals fp32, parents and tokens int32: anything else is not read as if it were."""
    x, c, s, i = rows(), codes(), torch.zeros(4), torch.zeros((4, 4), dtype=torch.int32)
    refused(1, api.i8_encode_rows, x, 4, 32, c.to(torch.uint8), s)
    refused(1, api.i8_encode_rows, x, 4, 32, c, s.double())
    refused(1, api.i8_norm_rows, x, 4, 32, None, 1e-5, c.int(), s)
    refused(1, api.i8_norm_rows, x, 4, 32, None, 1e-5, c, s.half())
    refused(1, api.i8_matmul, c.short(), s, 4, codes(8), torch.zeros(8), 8, 32, torch.zeros((4, 8)))
    refused(1, api.i8_matmul, c, s.half(), 4, codes(8), torch.zeros(8), 8, 32, torch.zeros((4, 8)))
    refused(1, api.i8_matmul, c, s, 4, codes(8).short(), torch.zeros(8), 8, 32, torch.zeros((4, 8)))
    refused(1, api.i8_matmul, c, s, 4, codes(8), torch.zeros(8).double(), 8, 32, torch.zeros((4, 8)))
    for n, kind in ((0, torch.float64), (1, torch.int64), (2, torch.int64), (3, torch.bfloat16)):
        given = [torch.zeros((4, 4)), i, i.clone(), torch.zeros((4, 4))]
        given[n] = given[n].to(kind)
        refused(1, api.beam_select, torch.zeros((16, 10)), given[0], 4, 4, 10, 4, *given[1:])
    refused(1, api.beam_reorder, x, x.clone(), i.long(), 1, 4, 4, 1, 1, 8)
    refused(1, api.beam_reorder, x, x.clone(), i, 1, 4, 4, 1, 1, 8, d_lengths=i[0].long())


def test_without_a_device_there_is_no_fallback():
    if api.device_count() > 0:
        pytest.skip("a GPU is present")
    x, c, s = rows(), codes(), torch.zeros(4)
    refused(5, api.i8_encode_rows, x, 4, 32, c, s)
    refused(5, api.i8_matmul, c, s, 4, codes(8), torch.zeros(8), 8, 32, torch.zeros((4, 8)))


def test_sizes_beyond_32_bits():
    """They are refused, not cut to their lower half: 2^32 + 32 elements a row are not 32, 2^32 items are not none."""
    big = 1 << 32
    x, c, s, i = rows(), codes(), torch.zeros(4), torch.zeros((2, 3), dtype=torch.int32)
    refused(1, api.i8_encode_rows, x, 4, big + 32, c, s, row_stride=32, code_stride=32)
    refused(1, api.i8_norm_rows, x, 4, big + 32, None, 1e-5, c, s, row_stride=32, code_stride=32)
    refused(1, api.i8_matmul, c, s, 4, codes(8), torch.zeros(8), 8, big + 32, torch.zeros((4, 8)), x_stride=32, w_stride=32)
    refused(1, api.i8_matmul_limited, c, s, 4, codes(8), torch.zeros(8), 8, 32, torch.zeros((4, 8)), polls=big + 1)
    for sizes in ((big, 3, 10, 3), (2, big + 3, 10, 3), (2, 3, big + 10, 3), (2, 3, 10, big + 3), (2, 3, 10, (1 << 31) + 3), (2, -big + 3, 10, 3)):
        refused(1, api.beam_select, torch.zeros((6, 10)), torch.zeros((2, 3)), *sizes, i, i.clone(), torch.zeros((2, 3)), row_stride=10)
    a = torch.zeros(240)
    for n in range(5):
        sizes = [1, 2, 3, 4, 5]
        sizes[n] = big if n in (0, 1, 4) else big + sizes[n]
        refused(1, api.beam_reorder, a, a.clone(), i, *sizes, 8)
