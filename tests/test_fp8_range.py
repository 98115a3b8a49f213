"""The e4m3 products at the ends of the scale range.  A code times its scale enters the matrix unit as bf16: exact from scale byte 3 on
(2^-9 2^-124 = 2^-133 is bf16's smallest subnormal), rounded to a multiple of 2^-133 below, and 2^128, i.e. Inf, for a block maximum
above 248 * 2^120 (its code is 256)."""
import pytest
import torch

import row_ops_ref as R
from sipmask_amd import ops as P

pytestmark = pytest.mark.gpu
CODES = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()      # 0 .. 448


def _rows(byte):
    """127 rows, each with one code's value in column 0 and the block's maximum in column 1"""
    x = torch.zeros(127, 128, dtype=torch.float64)
    x[:, 0], x[:, 1] = CODES, 448.0 if byte < 247 else 240.0
    return x * 2.0 ** (byte - 127)


def _bf16(v):
    """f64 -> what bf16 holds of values with at most four digits: a multiple of 2^-133, half to even"""
    return torch.where(v.abs() < 2.0 ** -126, torch.round(v * 2.0 ** 133) * 2.0 ** -133, v)


@pytest.mark.parametrize("byte", [0, 1, 2, 3, 4, 9, 10, 246, 247])
def test_products_of_every_code(byte):
    x = _rows(byte)
    if byte == 247:
        x = x[CODES <= 240]                      # (the largest f32 are 255.99 * 2^120)
    q, s, v = R.fp8_quantize(x.float(), 1)
    assert bool((s == byte).all()) and torch.equal(v, x)
    t = 60 if byte < 127 else -60
    w = torch.zeros(40, 128)
    w[:, 0] = 2.0 ** t * torch.arange(1, 41)     # (five bits at most of them: up to 16 exact, the others rounded to e4m3 here as there)
    wv = R.fp8_quantize(w, 1)[2]
    want = _bf16(x[:, :1]) * wv[:, 0]
    if byte >= 3:
        assert torch.equal(want, x @ wv.t())
    assert torch.equal(want, want.float().double())
    xd, wd = x.float().cuda(), w.cuda()
    xq, wq = P.quantize_fp8(xd), P.quantize_fp8(wd)
    assert torch.equal(xq.code_matrix().view(torch.uint8).cpu(), q)
    for rows in (slice(0, 5), slice(0, 40), slice(0, None)):             # one product by registers, one by more of them, one by tiles
        r = P.quantize_fp8(xd[rows])
        assert torch.equal(P.matmul_fp8(r, wq, out_dtype=torch.float32).double().cpu(), want[rows])
        assert torch.equal(P.matmul_fp8(wq, r, out_dtype=torch.float32).double().cpu(), want[rows].t())
    w128 = torch.zeros(40, 128)
    w128[:, 0] = 2.0 ** t
    for m in (5, 100):                           # quantised on the way, and by a launch before
        y = P.linear_fp8(xd[:m], w128.cuda())
        assert torch.equal(y.double().cpu(), _bf16(x[:m, :1]) * 2.0 ** t * torch.ones(40, dtype=torch.float64))


@pytest.mark.parametrize("value", [248.5 * 2.0 ** 120, 3.4028234663852886e38])
@pytest.mark.parametrize("m", [3, 90])
def test_maxima_that_round_beyond_f32(value, m):
    x = torch.full((m, 128), value)
    q = P.quantize_fp8(x.cuda())
    assert bool((q.scale_matrix() == 247).all()) and bool((q.dequantize(torch.float64) == 2.0 ** 128).all())
    assert bool(torch.isinf(q.dequantize()).all())
    w = P.quantize_fp8(torch.full((24, 128), 2.0 ** -100).cuda())
    assert bool((P.matmul_fp8(q, w, out_dtype=torch.float32) == float("inf")).all())
    below = P.quantize_fp8(torch.full((m, 128), 247.5 * 2.0 ** 120).cuda())
    assert bool((P.matmul_fp8(below, w, out_dtype=torch.float32) == 128 * 240.0 * 2.0 ** 20).all())
