"""GroupNorm + activation, counter-based dropout and the e4m3 products on the device, against float64 (row_ops_ref.py has the bounds)."""
import ctypes as C
import math

import pytest
import torch

import row_ops_ref as R
from sipmask_amd import _lib
from sipmask_amd import hip_ops as H
from sipmask_amd import ops as P
from sipmask_amd import ops_rows as PR

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def rnd(*shape, seed=0, dtype=F32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


def within(got, want, bound, what=""):
    err = (got.double() - want).abs()
    bad = ~(err <= bound)
    assert not bad.any(), "%s: %d of %d out of bounds, worst %.3g times its bound" % (
        what, int(bad.sum()), bad.numel(), float((err / bound.clamp_min(1e-300)).max()))


def rows_of(y):
    """[N, C, *] -> [rows, C]"""
    return y.movedim(1, -1).reshape(-1, y.shape[1])


# ------------------------------------------------------------------------------------------------ GroupNorm + activation
GN_SHAPES = [  # batch, channels, groups, spatial
    (1, 256, 32, (7, 11)), (2, 64, 8, (13, 21)), (3, 60, 12, (5, 7)), (2, 24, 24, (9,)), (1, 8, 1, (1, 1)), (2, 30, 3, (2, 3, 4)),
    (1, 520, 5, (3, 5)), (2, 2056, 1, (6,)), (1, 512, 2, (40, 33)), (4, 16, 4, ()), (1, 1, 1, (300,)), (1, 72, 6, (130, 17))]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("shape", GN_SHAPES)
def test_group_norm_act_forward_backward(shape, dtype):
    n, c, g, sp = shape
    for k, act in enumerate(("none", "relu", "silu", "gelu")):
        x = (rnd(n, *sp, c, seed=k) * 1.5 + rnd(c, seed=9)).to(dtype).movedim(-1, 1).requires_grad_(True)
        ga, be = (1 + 0.3 * rnd(c, seed=5)).requires_grad_(True), (0.3 * rnd(c, seed=6)).requires_grad_(True)
        y = P.group_norm_act(x, ga, be, g, 1e-5, act)
        assert y.dtype == dtype and y.shape == x.shape and y.movedim(1, -1).is_contiguous()
        dy = rnd(n, *sp, c, seed=7 + k).to(dtype).movedim(-1, 1)
        dx, dga, dbe = torch.autograd.grad(y, [x, ga, be], dy)
        ref = R.GroupNormAct(rows_of(x.detach()), n, g, ga.detach(), be.detach(), 1e-5, act)
        ref.backward(rows_of(dy))
        within(rows_of(y.detach()), ref.y, ref.y_bound(dtype), "y %s" % act)
        bx, bg, bb = ref.bounds(dtype)
        within(rows_of(dx), ref.dx, bx, "dx %s" % act)
        within(dga, ref.dgamma, bg, "dgamma %s" % act)
        within(dbe, ref.dbeta, bb, "dbeta %s" % act)


def test_group_norm_act_without_parameters_and_other_parameter_types():
    x = rnd(2, 6, 5, 16, dtype=BF16).movedim(-1, 1)
    ref = R.GroupNormAct(rows_of(x), 2, 4, None, None, 1e-3, "silu")
    within(rows_of(P.group_norm_act(x, None, None, 4, 1e-3, "silu")), ref.y, ref.y_bound(BF16))
    w = (1 + 0.1 * rnd(16, seed=1)).to(BF16).requires_grad_(True)
    b = (0.1 * rnd(16, seed=2)).to(F16).requires_grad_(True)
    y = P.group_norm_act(x, w, b, 4, 1e-3, "relu")
    ref = R.GroupNormAct(rows_of(x), 2, 4, w.detach(), b.detach(), 1e-3, "relu")
    ref.backward(torch.ones_like(rows_of(x)))
    within(rows_of(y.detach()), ref.y, ref.y_bound(BF16))
    dw, db = torch.autograd.grad(y, [w, b], torch.ones_like(y))          # (x has no gradient: the element-wise pass is skipped)
    assert dw.dtype == BF16 and db.dtype == F16
    _, bg, bb = ref.bounds(BF16)
    within(dw, ref.dgamma, bg + R.half_step(BF16) * ref.dgamma.abs())
    within(db, ref.dbeta, bb + R.half_step(F16) * ref.dbeta.abs())


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_group_norm_act_layouts(dtype):
    """NCHW memory, a channel slice of a wider channels-last tensor, a slice that starts off a 16-byte boundary, gradients in another
    layout: the same numbers"""
    base = rnd(2, 9, 7, 40, dtype=dtype)
    w, b = 1 + 0.1 * rnd(16, seed=1), 0.1 * rnd(16, seed=2)
    dy = rnd(2, 9, 7, 16, seed=3, dtype=dtype)
    for off in (0, 8, 3):
        sl = base[..., off:off + 16].movedim(-1, 1)
        ref = R.GroupNormAct(rows_of(sl), 2, 4, w, b, 1e-5, "gelu")
        ref.backward(rows_of(dy.movedim(-1, 1)))
        bx = ref.bounds(dtype)[0]
        for x in (sl, sl.contiguous(), sl.contiguous(memory_format=torch.channels_last)):
            for d in (dy.movedim(-1, 1), dy.movedim(-1, 1).contiguous()):
                x = x.detach().requires_grad_(True)
                y = P.group_norm_act(x, w, b, 4, 1e-5, "gelu")
                within(rows_of(y.detach()), ref.y, ref.y_bound(dtype))
                within(rows_of(torch.autograd.grad(y, x, d)[0]), ref.dx, bx)
    x = base[..., :16].movedim(-1, 1).detach().requires_grad_(True)      # an expanded gradient (sum of the outputs)
    y = P.group_norm_act(x, w, b, 4, 1e-5, "none")
    ref = R.GroupNormAct(rows_of(x.detach()), 2, 4, w, b, 1e-5, "none")
    ref.backward(torch.ones_like(rows_of(x)))
    within(rows_of(torch.autograd.grad(y.sum(), x)[0]), ref.dx, ref.bounds(dtype)[0])


@pytest.mark.parametrize("ratio", [1e2, 1e4])
def test_group_norm_act_mean_far_from_zero(ratio):
    """|mean| = ratio standard deviations: the statistics and x - mean keep their digits (input rounding is the only loss)"""
    x = (rnd(2, 33, 31, 64) + ratio).movedim(-1, 1)
    ref = R.GroupNormAct(rows_of(x), 2, 8, None, None, 1e-5, "none")
    # E[x^2] - m^2 in f64: 2^-53 ratio^2 of the variance, far below the f32 roundings
    within(rows_of(P.group_norm_act(x, None, None, 8, 1e-5, "none")), ref.y, ref.y_bound(F32))


def test_group_norm_act_constant_group_and_single_value():
    x = torch.full((2, 8, 3, 3), 5.25, device=DEV).contiguous(memory_format=torch.channels_last)
    b = rnd(8, seed=1)
    y = P.group_norm_act(x, rnd(8, seed=2), b, 2, 1e-5, "none")
    assert torch.equal(y, b.view(1, 8, 1, 1).expand_as(y))
    x = rnd(3, 4, 1, 1)                                                   # groups of one value: xhat = 0
    assert torch.equal(P.group_norm_act(x, None, b[:4], 4, 1e-5, "none"), b[:4].view(1, 4, 1, 1).expand(3, 4, 1, 1))


def test_group_norm_act_relu_gate_at_the_border():
    """beta = -gamma * xhat for many elements: t is 0 up to rounding, and the gate is the one of the f64 definition"""
    c, hw = 64, 4096
    x = torch.where(torch.rand(hw, c, generator=torch.Generator().manual_seed(1)) < 0.5, 1.0, -1.0).to(DEV)
    x[:, 0] += 1e-3 * torch.arange(hw, device=DEV) / hw
    ref = R.GroupNormAct(x, 1, 8, None, None, 1e-5, "relu")
    beta = (-ref.xh[7]).float()                                           # off by up to 2^-25 |xh| from the border
    xl = x.view(1, hw, c).movedim(-1, 1).detach().requires_grad_(True)
    ref = R.GroupNormAct(x, 1, 8, None, beta, 1e-5, "relu")
    dy = rnd(hw, c, seed=4)
    ref.backward(dy)
    assert int((ref.t.abs() < 1e-6).sum()) > hw * c // 4
    y = P.group_norm_act(xl, None, beta, 8, 1e-5, "relu")
    dx, = torch.autograd.grad(y, xl, dy.view(1, hw, c).movedim(-1, 1))
    within(rows_of(dx), ref.dx, ref.bounds(F32)[0], "gate")


@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu"])
def test_group_norm_act_nan_and_inf_stay_in_their_group(act):
    x = rnd(2, 5, 5, 32, dtype=BF16)
    clean = P.group_norm_act(x.movedim(-1, 1), None, None, 4, 1e-5, act)
    for v in (float("nan"), float("inf"), -float("inf")):
        z = x.clone()
        z[1, 2, 3, 9] = v
        y = P.group_norm_act(z.movedim(-1, 1), None, None, 4, 1e-5, act)
        assert torch.isnan(y[1, 8:16]).all()
        mask = torch.ones_like(y, dtype=torch.bool)
        mask[1, 8:16] = False
        assert torch.equal(y[mask], clean[mask])


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("c,groups", [(256, 32), (20, 4), (48, 16)])
def test_gn_act_rows_pyramid_with_dropout(dtype, c, groups):
    lv = H.Levels(2, [(19, 23), (10, 12), (5, 6), (3, 3), (1, 1)])
    x = rnd(lv.rows, c, dtype=dtype).requires_grad_(True)
    ga, be = (1 + 0.2 * rnd(c, seed=1)).requires_grad_(True), (0.2 * rnd(c, seed=2)).requires_grad_(True)
    seed, offset, p = 0x1234567890ABCDEF, 77, 0.3
    y = PR.gn_act_rows(x, lv, ga, be, groups, 1e-5, "silu", dropout_p=p, seed=seed, offset=offset)
    dy = rnd(lv.rows, c, seed=3, dtype=dtype)
    dx, dga, dbe = torch.autograd.grad(y, [x, ga, be], dy)
    fac = R.keep_factor((lv.rows, c), p, seed, offset).to(DEV)
    dg, db, bgs, bbs = 0, 0, 0, 0
    for l, (h, w) in enumerate(lv.sizes):
        r = slice(lv.row0[l], lv.row0[l] + 2 * h * w)
        ref = R.GroupNormAct(x.detach()[r], 2, groups, ga.detach(), be.detach(), 1e-5, "silu", fac[r])
        ref.backward(dy[r])
        within(y.detach()[r], ref.y, ref.y_bound(dtype), "y level %d" % l)
        bx, bg, bb = ref.bounds(dtype)
        within(dx[r], ref.dx, bx, "dx level %d" % l)
        dg, db, bgs, bbs = dg + ref.dgamma, db + ref.dbeta, bgs + bg, bbs + bb
    within(dga, dg, bgs, "dgamma")
    within(dbe, db, bbs, "dbeta")
    assert bool((y.detach()[fac == 0] == 0).all())


def test_gn_act_rows_agrees_with_gn_rows():
    """the operator that was there before, on its own ground (bf16, groups of 8 channels, ReLU)"""
    lv = H.Levels(2, [(25, 42), (13, 21)])
    x = rnd(lv.rows, 256, dtype=BF16)
    ga, be = 1 + 0.2 * rnd(256, seed=1), 0.2 * rnd(256, seed=2)
    a, b = PR.gn_rows(x, lv, ga, be, 32, 1e-5, True), PR.gn_act_rows(x, lv, ga, be, 32, 1e-5, "relu")
    assert float((a.float() - b.float()).abs().max()) <= 2 ** -8 * float(b.float().abs().max())


def test_group_norm_act_empty_batches_and_levels():
    w = torch.ones(8, device=DEV, requires_grad=True)
    x = torch.zeros(0, 8, 4, 4, device=DEV, requires_grad=True)
    y = P.group_norm_act(x, w, None, 2)
    assert y.shape == (0, 8, 4, 4)
    dx, dw = torch.autograd.grad(y, [x, w], torch.zeros_like(y))
    assert dx.shape == x.shape and torch.equal(dw, torch.zeros(8, device=DEV))
    lv = H.Levels(2, [(3, 4), (0, 5), (2, 2), (0, 0)])
    x = rnd(lv.rows, 8).requires_grad_(True)
    y = PR.gn_act_rows(x, lv, w, None, 2, 1e-5, "none")
    dx, dw = torch.autograd.grad(y, [x, w], torch.ones_like(y))
    assert torch.isfinite(dx).all() and torch.isfinite(dw).all()
    for r, hw in ((slice(0, 24), 12), (slice(24, 32), 4)):
        ref = R.GroupNormAct(x.detach()[r], 2, 2, w.detach(), None, 1e-5, "none")
        within(y.detach()[r], ref.y, ref.y_bound(F32))


def test_group_norm_act_leaves_other_columns_alone():
    """a C call that writes a channel slice: what lies beside it stays"""
    lib = _lib.load()
    x, out = rnd(30, 16), torch.full((30, 40), 7.0, device=DEV)
    d = _lib.GnActDesc()
    d.nlev, d.batch, d.channels, d.groups, d.dtype, d.act, d.eps = 1, 2, 16, 4, 2, 0, 1e-5
    d.hw[0], d.x_stride, d.y_stride, d.dy_stride, d.dx_stride = 15, 16, 40, 16, 16
    ws = torch.empty(lib.sm_group_norm_act_workspace(C.byref(d), 0), dtype=torch.uint8, device=DEV)
    dst = out[:, 8:24]
    _lib.check(lib.sm_group_norm_act(C.byref(d), _lib.ptr(x), None, None, C.c_void_p(dst.data_ptr()), None, _lib.ptr(ws), ws.numel(),
                                     _lib.stream_ptr()), "sm_group_norm_act")
    ref = R.GroupNormAct(x, 2, 4, None, None, 1e-5, "none")
    within(dst, ref.y, ref.y_bound(F32))
    assert bool((out[:, :8] == 7).all()) and bool((out[:, 24:] == 7).all())


def test_group_norm_act_is_reproducible_and_follows_the_stream():
    x = rnd(4, 50, 84, 256, dtype=BF16).movedim(-1, 1).requires_grad_(True)
    w, b = rnd(256, seed=1).requires_grad_(True), rnd(256, seed=2).requires_grad_(True)
    dy = rnd(4, 50, 84, 256, seed=3, dtype=BF16).movedim(-1, 1)

    def step():
        y = P.group_norm_act(x, w, b, 32, 1e-5, "gelu", dropout_p=0.2, seed=3)
        return (y.detach(),) + torch.autograd.grad(y, [x, w, b], dy)
    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, second))


def test_group_norm_act_refusals():
    x = rnd(2, 8, 3, 3)
    for call, err in ((lambda: P.group_norm_act(x.double(), None, None, 2), TypeError),
                      (lambda: P.group_norm_act(x, None, None, 3), ValueError),
                      (lambda: P.group_norm_act(x, None, None, 0), ValueError),
                      (lambda: P.group_norm_act(x, None, None, 2, -1.0), ValueError),
                      (lambda: P.group_norm_act(x, None, None, 2, activation="tanh"), ValueError),
                      (lambda: P.group_norm_act(x, rnd(7), None, 2), ValueError),
                      (lambda: P.group_norm_act(x, None, torch.zeros(8), 2), NotImplementedError),
                      (lambda: P.group_norm_act(x, None, None, 2, dropout_p=1.5), ValueError),
                      (lambda: P.group_norm_act(x, None, None, 2, offset=torch.zeros(1, device=DEV)), ValueError),
                      (lambda: P.group_norm_act(rnd(8), None, None, 2), ValueError),
                      (lambda: PR.gn_act_rows(rnd(5, 8), H.Levels(1, [(2, 2)]), None, None, 2), ValueError),
                      (lambda: PR.gn_act_rows(rnd(6, 8), H.Levels(1, [(1, 1)] * 6), None, None, 2), ValueError)):
        with pytest.raises(err):
            call()


# ------------------------------------------------------------------------------------------------ dropout
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (9,), (33, 93), (5, 256), (3, 4, 8), (1000, 17), ()])
@pytest.mark.parametrize("residual", [False, True])
def test_dropout_forward_backward(shape, dtype, residual):
    seed, offset = 0xFEDCBA9876543210, (1 << 40) + 3
    for p in (0.0, 0.1, 0.5, 1.0):
        x = rnd(*shape, dtype=dtype).requires_grad_(True)
        r = rnd(*shape, seed=1, dtype=dtype).requires_grad_(True) if residual else None
        y = P.dropout(x, p, seed, offset, residual=r)
        fac = R.keep_factor(shape, p, seed, offset).to(DEV)
        rd = r.detach().double() if residual else torch.zeros((), dtype=torch.float64, device=DEV)
        xs = x.detach().double() * fac
        want = xs + rd
        # the factor, its product and the sum: 3 roundings
        within(y.detach(), want, R.half_step(dtype) * want.abs() + R.E * (2 * xs.abs() + want.abs()) + R.tiny(dtype))
        dy = rnd(*shape, seed=2, dtype=dtype)
        grads = torch.autograd.grad(y, [x] + ([r] if residual else []), dy)
        want = dy.double() * fac
        within(grads[0], want, (R.half_step(dtype) + 2 * R.E) * want.abs() + R.tiny(dtype))
        assert bool((grads[0][fac == 0] == 0).all())
        if residual:
            assert torch.equal(grads[1], dy)


def test_dropout_strides_do_not_change_the_mask():
    x = rnd(40, 64, dtype=BF16)
    want = P.dropout(x, 0.4, 11, 5)
    wide = torch.zeros(40, 80, dtype=BF16, device=DEV)
    for off in (0, 8, 3):
        wide[:, off:off + 64] = x
        assert torch.equal(P.dropout(wide[:, off:off + 64], 0.4, 11, 5), want)
        assert torch.equal(P.dropout(x, 0.4, 11, 5, residual=wide[:, off:off + 64]) != x, want != 0)
    assert torch.equal(P.dropout(x.t().contiguous().t(), 0.4, 11, 5), want)
    assert torch.equal(P.dropout(x.view(5, 8, 64), 0.4, 11, 5).view(40, 64), want)
    odd = torch.zeros(40 * 64 + 1, dtype=BF16, device=DEV)[1:].view(40, 64)
    odd.copy_(x)
    assert odd.data_ptr() % 16 != 0 and torch.equal(P.dropout(odd, 0.4, 11, 5), want)
    xg = x.clone().requires_grad_(True)                                    # an expanded gradient
    g, = torch.autograd.grad(P.dropout(xg, 0.4, 11, 5).sum(), xg)
    assert torch.equal(g != 0, P.dropout(torch.ones_like(x), 0.4, 11, 5) != 0)


def test_dropout_drops_nan_and_inf_and_keeps_the_mean():
    n = 1 << 20
    x = torch.full((n,), float("nan"), device=DEV)
    x[::2] = float("inf")
    y = P.dropout(x, 0.25, 5)
    keep = R.keep_factor((n,), 0.25, 5, 0).to(DEV) != 0
    assert bool((y[~keep] == 0).all()) and not torch.isfinite(y[keep]).any()
    # binomial: 6 standard deviations of n draws
    for p in (0.1, 0.5, 0.9):
        k = int((P.dropout(torch.ones(n, device=DEV), p, 123, 9) != 0).sum())
        assert abs(k - n * (1 - p)) < 6 * math.sqrt(n * p * (1 - p)) + n / 65536
    a, b = (P.dropout(torch.ones(n, device=DEV), 0.5, s, o) != 0 for s, o in ((1, 0), (1, 1)))
    assert abs(int((a == b).sum()) - n // 2) < 6 * math.sqrt(n) / 2        # neighbouring offsets are independent
    assert torch.equal(P.dropout(torch.ones(n, device=DEV), 0.5, 1, -1), P.dropout(torch.ones(n, device=DEV), 0.5, 1, (1 << 64) - 1))


def test_dropout_training_flag_and_refusals():
    x, r = rnd(4, 4), rnd(4, 4, seed=1)
    assert P.dropout(x, 0.5, 1, training=False) is x
    assert torch.equal(P.dropout(x, 0.5, 1, residual=r, training=False), x + r)
    assert P.dropout(torch.zeros(0, 4, device=DEV), 0.5, 1).shape == (0, 4)
    for call, err in ((lambda: P.dropout(x.double(), 0.5, 1), TypeError), (lambda: P.dropout(x, 2.0, 1), ValueError),
                      (lambda: P.dropout(x, 0.5, 1, residual=r[:2]), ValueError),
                      (lambda: P.dropout(x, 0.5, 1, residual=r.half()), ValueError),
                      (lambda: P.dropout(x, 0.5, 1, offset=torch.zeros(1, dtype=torch.int64)), ValueError),
                      (lambda: P.dropout(x.long(), 0.5, 1), TypeError)):
        with pytest.raises(err):
            call()


def test_dropout_element_numbers_pass_32_bits():
    n = (1 << 32) + 24
    x = torch.ones(n, dtype=BF16, device=DEV)
    y = P.dropout(x, 0.5, 99, 4)
    for first in (0, (1 << 31) - 13, (1 << 32) - 16, n - 40):
        want = torch.from_numpy(R.draws(first, 40 if first + 40 <= n else n - first, 99, 4).astype("int64") >= 32768)
        assert torch.equal(y[first:first + len(want)].cpu() != 0, want)


def test_dropout_device_offset_in_a_replayed_graph():
    x = rnd(333, 40, dtype=BF16)
    step = torch.zeros(1, dtype=torch.int64, device=DEV)
    P.dropout(x, 0.3, 21, step)                                            # warm-up outside the capture
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        with torch.cuda.graph(g, stream=s):
            y = P.dropout(x, 0.3, 21, step)
            z = P.group_norm_act(x.t().reshape(1, 40, 333), None, None, 4, 1e-5, "relu", dropout_p=0.3, seed=21, offset=step)
            step.add_(1)
    torch.cuda.current_stream().wait_stream(s)
    step.zero_()
    for i in range(4):
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, P.dropout(x, 0.3, 21, i))
        assert torch.equal(z, P.group_norm_act(x.t().reshape(1, 40, 333), None, None, 4, 1e-5, "relu", dropout_p=0.3, seed=21, offset=i))
    xg = x.clone().requires_grad_(True)
    out = P.dropout(xg, 0.3, 21, step)
    step.add_(1)
    with pytest.raises(RuntimeError):                                      # the offset changed before the backward ran
        torch.autograd.grad(out.sum(), xg)


# ------------------------------------------------------------------------------------------------ e4m3 blocks
def spread(rows, cols, seed=0, dtype=F32):
    """values of very unlike size between columns, some zeros"""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g) * torch.exp(2 * torch.randn(cols, generator=g))
    return torch.where(torch.rand(rows, cols, generator=g) < 0.2, torch.zeros(()), x).to(dtype).to(DEV)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 128), (3, 130), (128, 128), (129, 257), (300, 64), (77, 1000), (5, 8)])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("transpose", [False, True])
def test_quantize_fp8_codes_and_scales(rows, cols, block_rows, transpose, dtype):
    x = spread(rows, cols, seed=rows + cols, dtype=dtype)
    q = P.quantize_fp8(x, block_rows, transpose)
    src = x.t().contiguous() if transpose else x
    code, byte, val = R.fp8_quantize(src, block_rows)
    r, c = src.shape
    nkb = -(-c // 128)
    assert q.shape == (r, c) and q.codes.shape == (2 * nkb, r, 64) and q.scales.shape == (-(-nkb // 4), byte.shape[0], 4)
    got = q.code_matrix().view(torch.uint8)
    zero = (code & 0x7F) == 0                                              # (+0 and -0 stand for the same value)
    assert torch.equal(torch.where(zero, code & 0x7F, code), torch.where(zero, got & 0x7F, got))
    assert bool((q.codes.view(torch.uint8).transpose(0, 1).reshape(r, -1)[:, c:] & 0x7F == 0).all())
    assert torch.equal(q.scale_matrix().long(), byte)
    assert bool((q.scales.transpose(0, 1).reshape(byte.shape[0], -1)[:, nkb:] == 127).all())
    assert torch.equal(q.dequantize(torch.float64), val)


def test_quantize_fp8_every_code_and_every_exponent():
    codes = torch.arange(256, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn).float()
    x = torch.full((1, 256), 448.0, device=DEV)
    x[0, :127], x[0, 128:255] = codes[:127], codes[128:255]
    q = P.quantize_fp8(x)
    assert bool((q.scale_matrix() == 127).all()) and torch.equal(q.dequantize(), x)
    e = torch.arange(-149, 128, device=DEV)
    v = R.pow2(e).float().view(-1, 1).expand(-1, 128).contiguous()         # subnormals of f32 among them
    v[:, 1::2] *= 1.9375
    v = torch.where(torch.isfinite(v), v, torch.full_like(v, 3.4028234663852886e38))
    code, byte, val = R.fp8_quantize(v, 1)
    q = P.quantize_fp8(v)
    assert torch.equal(q.scale_matrix().long(), byte) and torch.equal(q.code_matrix().view(torch.uint8), code)


def test_quantize_fp8_nan_and_inf():
    x = spread(4, 256, seed=1)
    clean = P.quantize_fp8(x)
    z = x.clone()
    z[1, 3], z[2, 200], z[3, 5] = float("nan"), float("inf"), -float("inf")
    q = P.quantize_fp8(z)
    bad = torch.zeros(4, 256, dtype=torch.bool, device=DEV)
    bad[1, 3] = bad[2, 200] = bad[3, 5] = True
    v = q.dequantize()
    assert torch.isnan(v[bad]).all() and torch.isfinite(v[~bad]).all()
    code, byte, _ = R.fp8_quantize(z, 1)
    assert torch.equal(q.scale_matrix().long(), byte)
    assert torch.equal(v[0], clean.dequantize()[0])
    y = P.matmul_fp8(q, P.quantize_fp8(spread(8, 256, seed=2), 128), out_dtype=F32)
    assert torch.isfinite(y[0]).all() and torch.isnan(y[1:]).all()


def test_quantize_fp8_strided_rows():
    wide = spread(50, 300, seed=4, dtype=BF16)
    for off in (0, 8, 5):
        sl = wide[:, off:off + 200]
        for br, tr in ((1, False), (128, False), (1, True), (128, True)):
            a, b = P.quantize_fp8(sl, br, tr), P.quantize_fp8(sl.contiguous(), br, tr)
            assert torch.equal(a.codes.view(torch.uint8), b.codes.view(torch.uint8)) and torch.equal(a.scales, b.scales)


MM_SHAPES = [(1, 1, 1), (1, 8, 128), (7, 512, 2048), (16, 33, 130), (17, 64, 64), (33, 3, 2000), (64, 64, 1000), (128, 128, 128), (129, 257, 385),
             (300, 130, 16), (977, 333, 1131), (5, 1000, 4096), (2048, 256, 512), (700, 900, 640), (4100, 2050, 140),
             (500, 700, 44100), (8200, 2040, 2056)]


@pytest.mark.parametrize("m,n,k", MM_SHAPES)
def test_matmul_fp8(m, n, k):
    a, b = spread(m, k, seed=m), spread(n, k, seed=n + 1)
    bias = 10 * rnd(n, seed=3)
    for i, (bra, brb, dt) in enumerate(((1, 128, BF16), (1, 1, F32), (128, 128, F16), (128, 1, BF16))):
        qa, qb = P.quantize_fp8(a, bra), P.quantize_fp8(b * 2.0 ** -6, brb)
        av, bv = R.fp8_quantize(a, bra)[2], R.fp8_quantize(b * 2.0 ** -6, brb)[2]
        y = av @ bv.t()
        top = float(y.abs().max())
        if dt == F16 and top > 3e4:
            dt = F32
        within(P.matmul_fp8(qa, qb, out_dtype=dt), y, R.matmul_bound(av, bv, y, k, dt), "product %d" % i)
        res = rnd(m, n, seed=5).to(dt)
        full = y + bias.double() + res.double()
        got = P.matmul_fp8(qa, qb, bias, True, res, dt)
        within(got, full.clamp_min(0), R.matmul_bound(av, bv, full, k, dt, extra=2 * (bias.double().abs() + res.double().abs())), "epilogue %d" % i)


def test_matmul_fp8_wide_scales_and_exact_integers():
    g = torch.Generator().manual_seed(0)
    a = torch.randint(-7, 8, (200, 384), generator=g).float().to(DEV)
    b = torch.randint(-7, 8, (144, 384), generator=g).float().to(DEV)
    want = (a.double() @ b.double().t()).float()
    for sa, sb in ((0, 0), (60, -70), (-100, 90), (100, -100)):             # integers times powers of two: exact
        y = P.matmul_fp8(P.quantize_fp8(a * 2.0 ** sa), P.quantize_fp8(b * 2.0 ** sb, 128), out_dtype=F32)
        assert torch.equal(y, want * 2.0 ** (sa + sb))


def test_matmul_fp8_residual_strides_and_out_reuse():
    a, b = P.quantize_fp8(spread(70, 256, seed=1)), P.quantize_fp8(spread(24, 256, seed=2), 128)
    plain = P.matmul_fp8(a, b, out_dtype=F32)
    wide = rnd(70, 40)
    for off in (0, 4, 3):
        assert torch.equal(P.matmul_fp8(a, b, residual=wide[:, off:off + 24], out_dtype=F32), plain + wide[:, off:off + 24])
    assert torch.equal(P.matmul_fp8(a, b, residual=wide.t()[:24].t(), out_dtype=F32), plain + wide[:, :24])


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("m,n,k", [(1, 8, 16), (7, 40, 200), (130, 96, 256), (1013, 205, 331), (5000, 64, 128)])
def test_linear_fp8_forward_backward(m, n, k, dtype):
    x = spread(m, k, seed=1).clamp(-50, 50).to(dtype).requires_grad_(True)
    w = (rnd(n, k, seed=2) / math.sqrt(k)).requires_grad_(True)
    b = rnd(n, seed=3).requires_grad_(True)
    y = P.linear_fp8(x, w, b)
    dy = (0.01 * rnd(m, n, seed=4)).to(dtype)
    dx, dw, db = torch.autograd.grad(y, [x, w, b], dy)
    qv = lambda t, br: R.fp8_quantize(t, br)[2]
    xd, wd = x.detach(), w.detach()
    xq, wq, gq = qv(xd, 1), qv(wd, 128), qv(dy, 1)
    want = xq @ wq.t() + b.detach().double()
    within(y.detach(), want, R.matmul_bound(xq, wq, want, k, dtype, extra=2 * b.detach().double().abs()), "y")
    wt = wq.t().contiguous()
    want = gq @ wq
    within(dx, want, R.matmul_bound(gq, wt, want, n, dtype), "dx")
    gt, xt = qv(dy.t().contiguous(), 1), qv(xd.t().contiguous(), 1)
    want = gt @ xt.t()
    within(dw, want, R.matmul_bound(gt, xt, want, m, F32), "dw")
    want = dy.double().sum(0)
    within(db, want, R.E * (25 * dy.double().abs().sum(0) + 2 * want.abs()), "dbias")
    assert dw.dtype == w.dtype and db.dtype == b.dtype and dx.dtype == dtype


def test_linear_fp8_gradient_by_differences():
    """whole numbers small enough to be exact in e4m3: the layer is linear, and one step along an axis is the gradient itself"""
    g = torch.Generator().manual_seed(5)
    x = torch.randint(-3, 4, (20, 40), generator=g).float().to(DEV).requires_grad_(True)
    w = torch.randint(-3, 4, (12, 40), generator=g).float().to(DEV).requires_grad_(True)
    dy = torch.randint(-3, 4, (20, 12), generator=g).float().to(DEV)
    dx, dw = torch.autograd.grad(P.linear_fp8(x, w), [x, w], dy)
    f = lambda a, b: float((P.linear_fp8(a, b) * dy).double().sum())
    for i, j in ((0, 0), (19, 39), (7, 20), (3, 11)):
        e = torch.zeros_like(x)
        e[i, j] = 1
        assert (f(x.detach() + e, w.detach()) - f(x.detach() - e, w.detach())) / 2 == float(dx[i, j])
    for i, j in ((0, 0), (11, 39), (5, 2)):
        e = torch.zeros_like(w)
        e[i, j] = 1
        assert (f(x.detach(), w.detach() + e) - f(x.detach(), w.detach() - e)) / 2 == float(dw[i, j])


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("m", [1, 15, 16, 17, 64, 65, 200])
def test_linear_fp8_quantises_like_quantize_fp8(m, dtype):
    """the few-rows kernel quantises x itself, the others through a launch: the same codes"""
    for n, k in ((40, 130), (16, 2048), (300, 77)):
        wide, w = spread(m, k + 11, seed=m, dtype=dtype), P.quantize_fp8(spread(n, k, seed=2) * 2.0 ** -6, 128)
        for x in (wide[:, :k].contiguous(), wide[:, :k], wide[:, 3:3 + k]):
            want = P.matmul_fp8(P.quantize_fp8(x), w, out_dtype=dtype)
            assert torch.equal(P.linear_fp8(x, None, weight_q=w), want)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_linear_fp8_partial_gradients(dtype):
    """any subset of the gradients, with and without a ReLU, equals the whole set's"""
    x, w, b = spread(70, 96, seed=1).clamp(-50, 50).to(dtype), rnd(40, 96, seed=2) / 8, rnd(40, seed=3)
    dy = rnd(70, 40, seed=4, dtype=dtype)
    for relu in (False, True):
        leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
        full = torch.autograd.grad(P.linear_fp8(*leaves, relu=relu), leaves, dy)
        for pick in ((0,), (1,), (2,), (0, 1), (1, 2), (0, 2)):
            args = [t.clone().requires_grad_(i in pick) for i, t in enumerate((x, w, b))]
            got = torch.autograd.grad(P.linear_fp8(*args, relu=relu), [args[i] for i in pick], dy)
            assert all(torch.equal(g, full[i]) for g, i in zip(got, pick))
        wq = P.quantize_fp8(w, 128)
        args = [t.clone().requires_grad_(True) for t in (x, w)]
        got = torch.autograd.grad(P.linear_fp8(*args, b, relu=relu, weight_q=wq), args, dy)
        assert all(torch.equal(g, f) for g, f in zip(got, full))


def test_linear_fp8_serving_form_relu_and_shapes():
    x = spread(24, 96, seed=1, dtype=BF16)
    w, b = rnd(32, 96, seed=2) / 8, rnd(32, seed=3)
    wq = P.quantize_fp8(w, 128)
    y = P.linear_fp8(x, w, b, relu=True)
    assert torch.equal(y, P.linear_fp8(x, None, b, relu=True, weight_q=wq))
    assert torch.equal(y.view(2, 3, 4, 32), P.linear_fp8(x.view(2, 3, 4, 96), w.view(32, 96, 1, 1), b, relu=True))
    assert torch.equal(P.linear_fp8(x[5], w, b), P.linear_fp8(x, w, b)[5]) and bool((y >= 0).all())
    for i in range(0, 24, 5):                                              # a row's result does not depend on its batch
        assert torch.equal(P.linear_fp8(x[i:i + 1], w, b, relu=True), y[i:i + 1])
    xg = x.clone().requires_grad_(True)
    yg = P.linear_fp8(xg, w, b, relu=True)
    dy = rnd(24, 32, seed=4, dtype=BF16)
    dx, = torch.autograd.grad(yg, xg, dy)
    x2 = x.clone().requires_grad_(True)
    dx2, = torch.autograd.grad(P.linear_fp8(x2, w, b), x2, torch.where(yg.detach() > 0, dy, torch.zeros_like(dy)))
    assert torch.equal(dx, dx2)
    e = torch.zeros(0, 96, device=DEV, requires_grad=True)
    wg, bg = w.clone().requires_grad_(True), b.clone().requires_grad_(True)
    y0 = P.linear_fp8(e, wg, bg)
    assert y0.shape == (0, 32)
    gx, gw, gb = torch.autograd.grad(y0, [e, wg, bg], torch.zeros_like(y0))
    assert gx.shape == (0, 96) and torch.equal(gw, torch.zeros_like(w)) and torch.equal(gb, torch.zeros_like(b))


def test_fp8_refusals():
    x, w = rnd(4, 16), rnd(8, 16, seed=1)
    q, wq = P.quantize_fp8(x), P.quantize_fp8(w, 128)
    xg = x.clone().requires_grad_(True)
    for call, err in ((lambda: P.quantize_fp8(x.double()), TypeError), (lambda: P.quantize_fp8(x[0]), ValueError),
                      (lambda: P.quantize_fp8(x, 64), ValueError), (lambda: P.quantize_fp8(x[:0], transpose=True), ValueError),
                      (lambda: P.quantize_fp8(x[:, :0]), ValueError), (lambda: P.matmul_fp8(x, wq), TypeError),
                      (lambda: P.matmul_fp8(q, P.quantize_fp8(w[:, :8], 128)), ValueError),
                      (lambda: P.matmul_fp8(q, wq, out_dtype=torch.float64), TypeError),
                      (lambda: P.matmul_fp8(q, wq, bias=rnd(7)), ValueError),
                      (lambda: P.matmul_fp8(q, wq, residual=rnd(4, 8), out_dtype=BF16), ValueError),
                      (lambda: P.linear_fp8(x, None), ValueError), (lambda: P.linear_fp8(x, w[:, :8]), ValueError),
                      (lambda: P.linear_fp8(x, w, rnd(9)), ValueError), (lambda: P.linear_fp8(xg, None, weight_q=wq), ValueError),
                      (lambda: P.linear_fp8(x, w, weight_q=q), ValueError), (lambda: P.linear_fp8(x, w.double()), TypeError),
                      (lambda: P.linear_fp8(x, w.view(8, 4, 2, 2)), ValueError)):
        with pytest.raises(err):
            call()


def test_matmul_fp8_offsets_pass_32_bits():
    """4.3 GB of codes and an output of more than 2^31 bytes: the last rows are the first ones again"""
    m, k, n = (1 << 25) + 130, 128, 40
    base = spread(1024, k, seed=3, dtype=BF16)
    x = base.repeat(m // 1024 + 1, 1)[:m]
    w = spread(n, k, seed=4) * 2.0 ** -6
    y = P.linear_fp8(x, w)
    want = P.linear_fp8(base, w)
    for r0 in (0, 1 << 24, m - 1024 - m % 1024):
        assert torch.equal(y[r0:r0 + 1024], want)
    assert torch.equal(y[m - m % 1024:], want[:m % 1024])


def test_group_norm_act_rows_pass_32_bits():
    """more than 2^32 bytes of rows: every image equals the small one it repeats"""
    base = rnd(64, 64, 256, dtype=BF16)
    reps = 2100
    x = base.view(1, 4096, 256).repeat(reps, 1, 1).movedim(-1, 1)
    y = P.group_norm_act(x, None, None, 32, 1e-5, "silu")
    want = P.group_norm_act(base.view(1, 4096, 256).movedim(-1, 1), None, None, 32, 1e-5, "silu")
    for i in (0, 1023, 2047, 2048, reps - 1):
        assert torch.equal(y[i:i + 1], want)


# ------------------------------------------------------------------------------------------------ together
def test_residual_branch_forward_backward():
    """rows -> group_norm_act + dropout -> linear_fp8 -> dropout + residual, as a training step runs it, against the composition of the
    references on the intermediate values that the device produced"""
    lv = H.Levels(2, [(12, 17), (6, 9)])
    c = 96
    x = rnd(lv.rows, c, dtype=BF16).requires_grad_(True)
    ga, be = (1 + 0.2 * rnd(c, seed=1)).requires_grad_(True), (0.2 * rnd(c, seed=2)).requires_grad_(True)
    w, b = (rnd(c, c, seed=3) / math.sqrt(c)).requires_grad_(True), (0.1 * rnd(c, seed=4)).requires_grad_(True)
    h = PR.gn_act_rows(x, lv, ga, be, 12, 1e-5, "silu", dropout_p=0.1, seed=7, offset=0)
    v = P.linear_fp8(h, w, b)
    y = P.dropout(v, 0.2, 7, 1, residual=x)
    dy = rnd(lv.rows, c, seed=5, dtype=BF16)
    gx, gga, gbe, gw, gb, gh, gv = torch.autograd.grad(y, [x, ga, be, w, b, h, v], dy)
    f0, f1 = (R.keep_factor((lv.rows, c), p, 7, o).to(DEV) for p, o in ((0.1, 0), (0.2, 1)))
    qv = lambda t, br: R.fp8_quantize(t, br)[2]
    hd, vd, xd = h.detach(), v.detach(), x.detach()
    want = vd.double() * f1 + xd.double()
    within(y.detach(), want, R.half_step(BF16) * want.abs() + 3 * R.E * (want.abs() + (vd.double() * f1).abs()) + R.tiny(BF16), "y")
    want = dy.double() * f1
    within(gv, want, (R.half_step(BF16) + 2 * R.E) * want.abs() + R.tiny(BF16), "dv")
    hq, wq = qv(hd, 1), qv(w.detach(), 128)
    want = hq @ wq.t() + b.detach().double()
    within(vd, want, R.matmul_bound(hq, wq, want, c, BF16, extra=2 * b.detach().double().abs()), "v")
    gq = qv(gv, 1)
    want = gq @ wq
    within(gh, want, R.matmul_bound(gq, wq.t().contiguous(), want, c, BF16), "dh")
    gt, ht = qv(gv.t().contiguous(), 1), qv(hd.t().contiguous(), 1)
    want = gt @ ht.t()
    within(gw, want, R.matmul_bound(gt, ht, want, lv.rows, F32), "dw")
    want = gv.double().sum(0)
    within(gb, want, R.E * (25 * gv.double().abs().sum(0) + 2 * want.abs()), "dbias")
    dg, db, bgs, bbs = 0, 0, 0, 0
    for l, (hh, ww) in enumerate(lv.sizes):
        r = slice(lv.row0[l], lv.row0[l] + 2 * hh * ww)
        ref = R.GroupNormAct(xd[r], 2, 12, ga.detach(), be.detach(), 1e-5, "silu", f0[r])
        ref.backward(gh[r])
        within(hd[r], ref.y, ref.y_bound(BF16), "h")
        bx, bg, bb = ref.bounds(BF16)
        tot = ref.dx + dy.double()[r]                                      # autograd adds the branch (rounded) and the residual's gradient
        within(gx[r], tot, bx + R.half_step(BF16) * (tot.abs() + bx) + R.E * tot.abs(), "dx")
        dg, db, bgs, bbs = dg + ref.dgamma, db + ref.dbeta, bgs + bg, bbs + bb
    within(gga, dg, bgs, "dgamma")
    within(gbe, db, bbs, "dbeta")


def test_training_step_captured_and_replayed():
    """forward and backward of the branch in one graph: replays equal the eager step on the inputs of the moment"""
    c, lv = 64, H.Levels(1, [(10, 13)])
    w0 = rnd(c, c, seed=1) / 8
    ga0, be0 = 1 + 0.1 * rnd(c, seed=2), 0.1 * rnd(c, seed=3)
    dy = rnd(lv.rows, c, seed=4, dtype=BF16)

    def step(x, w, ga, be):
        x, w, ga, be = (t.detach().requires_grad_(True) for t in (x, w, ga, be))
        h = PR.gn_act_rows(x, lv, ga, be, 8, 1e-5, "gelu", dropout_p=0.25, seed=5, offset=3)
        y = P.dropout(P.linear_fp8(h, w), 0.1, 5, 4, residual=x)
        return (y.detach(),) + torch.autograd.grad(y, [x, w, ga, be], dy)
    xs = [rnd(lv.rows, c, seed=10 + i, dtype=BF16) for i in range(4)]
    buf = xs[0].clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(buf, w0, ga0, be0)
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = step(buf, w0, ga0, be0)
    for x in xs:
        buf.copy_(x)
        g.replay()
        torch.cuda.synchronize()
        want = step(x, w0, ga0, be0)
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_fp8_matrices_without_rows():
    q = P.quantize_fp8(torch.zeros(0, 40, device=DEV))
    assert q.shape == (0, 40) and q.dequantize().shape == (0, 40)
    w = P.quantize_fp8(rnd(8, 40), 128)
    assert P.matmul_fp8(q, w).shape == (0, 8)
    assert P.quantize_fp8(torch.zeros(0, 40, device=DEV), 128).scale_matrix().shape == (0, 1)


def test_fp8_operands_of_another_place_are_refused():
    x, w = rnd(4, 16), rnd(8, 16, seed=1)
    q, wq = P.quantize_fp8(x), P.quantize_fp8(w, 128)
    host = lambda t: P.Fp8Blocks(t.codes.cpu(), t.scales.cpu(), t.rows, t.cols, t.block_rows)
    half = P.Fp8Blocks(wq.codes, wq.scales.cpu(), 8, 16, 128)
    short = P.Fp8Blocks(wq.codes[:, :7], wq.scales, 8, 16, 128)
    with pytest.raises(NotImplementedError):
        P.matmul_fp8(q, host(wq))
    for bad in (host(wq), half, short):
        with pytest.raises(ValueError):
            P.linear_fp8(x, None, weight_q=bad)
    for bad in (half, short):
        with pytest.raises(ValueError):
            P.matmul_fp8(q, bad)
    with pytest.raises(TypeError):
        P.linear_fp8(x, w, weight_q=w)


@pytest.mark.parametrize("m", [3, 40, 700])
def test_linear_fp8_any_alignment(m):
    """rows, bias and gradient that start 2 or 4 bytes behind a 16-byte boundary"""
    k, n = 200, 56
    x, w, b, dy = rnd(m, k, seed=1, dtype=BF16), rnd(n, k, seed=2), rnd(n, seed=3), rnd(m, n, seed=4, dtype=BF16)

    def odd(t):
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=DEV)[1:].view(t.shape)
        return flat.copy_(t)
    got = []
    for f in (lambda t: t, odd):
        xl, wl, bl = (f(t).requires_grad_(True) for t in (x, w, b))
        y = P.linear_fp8(xl, wl, bl, relu=True)
        with torch.no_grad():
            serving = P.linear_fp8(xl, None, bl, relu=True, weight_q=P.quantize_fp8(wl, 128))
        got.append((y.detach(), serving) + torch.autograd.grad(y, [xl, wl, bl], f(dy)))
    for a, c in zip(*got):
        assert torch.equal(a, c)
    assert torch.equal(got[0][0], got[0][1])


def test_expanded_gradients_and_a_graph_walked_twice():
    lv = H.Levels(2, [(5, 7)])
    x, ga, be = rnd(lv.rows, 64, seed=1, dtype=BF16), 1 + 0.1 * rnd(64, seed=2), 0.1 * rnd(64, seed=3)
    w, b = rnd(48, 64, seed=4) / 8, rnd(48, seed=5)
    img = x.view(2, 5, 7, 64).permute(0, 3, 1, 2)
    calls = ((lambda x, g, h, w, b: PR.gn_act_rows(x, lv, g, h, 8, activation="gelu", dropout_p=0.2, seed=1)),
             (lambda x, g, h, w, b: P.group_norm_act(x.view(2, 5, 7, 64).permute(0, 3, 1, 2), g, h, 8, activation="silu")),
             (lambda x, g, h, w, b: P.dropout(x, 0.3, 2, residual=x)), (lambda x, g, h, w, b: P.linear_fp8(x, w, b, relu=True)))
    for call in calls:
        leaves = [t.clone().requires_grad_(True) for t in (x, ga, be, w, b)]
        y = call(*leaves)
        one = torch.ones((), dtype=y.dtype, device=DEV)
        first = torch.autograd.grad(y, leaves, one.expand(y.shape), retain_graph=True, allow_unused=True)
        dense = torch.autograd.grad(y, leaves, torch.ones_like(y), retain_graph=True, allow_unused=True)
        dy = rnd(*y.shape, seed=9, dtype=y.dtype)
        torch.autograd.grad(y, leaves, dy.transpose(-1, -2).contiguous().transpose(-1, -2), retain_graph=True, allow_unused=True)
        again = torch.autograd.grad(y, leaves, torch.ones_like(y), allow_unused=True)
        for a, c, d in zip(first, dense, again):
            assert (a is None) == (c is None) == (d is None)
            if a is not None:
                assert torch.equal(a, c) and torch.equal(a, d)
    assert img.shape == (2, 64, 5, 7)


def test_changed_tensors_are_noticed_by_the_backward():
    x, w = rnd(20, 64, seed=1, dtype=BF16).requires_grad_(True), (rnd(48, 64, seed=4) / 8).requires_grad_(True)
    y = P.linear_fp8(x, w, relu=True)
    y.detach().add_(1)                           # the ReLU's gate is the result itself
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()
    z = rnd(20, 64, seed=2, dtype=BF16)
    lv = H.Levels(1, [(4, 5)])
    h = PR.gn_act_rows(z, lv, (1 + 0 * rnd(64)).requires_grad_(True), rnd(64), 8)
    z.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        h.sum().backward()
    off = torch.zeros(1, dtype=torch.int64, device=DEV)
    d = P.dropout(x, 0.5, 1, off)
    off.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        d.sum().backward()


def test_calls_on_two_streams_at_once():
    """the same operators in two streams that run side by side: nothing is shared between the calls"""
    lv = H.Levels(2, [(40, 52), (20, 26)])
    ga, be, w = 1 + 0.1 * rnd(256, seed=2), 0.1 * rnd(256, seed=3), P.quantize_fp8(rnd(512, 256, seed=4) / 16, 128)
    xs = [rnd(lv.rows, 256, seed=i, dtype=BF16) for i in range(2)]

    def chain(x, seed):
        h = PR.gn_act_rows(x, lv, ga, be, 32, activation="silu", dropout_p=0.1, seed=seed)
        h = P.linear_fp8(h, None, relu=True, weight_q=w)
        return P.matmul_fp8(P.quantize_fp8(h, transpose=True), P.quantize_fp8(x, transpose=True), out_dtype=F32)
    want = [chain(x, i) for i, x in enumerate(xs)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(4):
        for i, (x, s) in enumerate(zip(xs, streams)):
            with torch.cuda.stream(s):
                got[i].append(chain(x, i))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


def test_two_captured_graphs_replayed_in_turn():
    """two graphs of one memory pool, one after the other and in the other order, with eager calls between: the workspaces are theirs"""
    c, lv = 128, H.Levels(1, [(30, 40), (15, 20)])
    ga, be, w = 1 + 0.1 * rnd(c, seed=2), 0.1 * rnd(c, seed=3), P.quantize_fp8(rnd(96, c, seed=4) / 8, 128)
    off = torch.zeros(1, dtype=torch.int64, device=DEV)

    def chain(x):
        h = PR.gn_act_rows(x, lv, ga, be, 16, activation="relu", dropout_p=0.1, seed=3, offset=off)
        return P.dropout(P.linear_fp8(h, None, weight_q=w), 0.2, 4, off)
    bufs = [rnd(lv.rows, c, seed=i, dtype=BF16) for i in range(2)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for b in bufs:
            chain(b)
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graphs, outs, pool = [], [], None
    for b in bufs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=pool):
            y = chain(b)
        pool = g.pool()
        graphs.append(g)
        outs.append(y)
    for turn, order in enumerate(((0, 1), (1, 0), (0, 1))):
        off.fill_(turn)
        for i in order:
            bufs[i].copy_(rnd(lv.rows, c, seed=10 * turn + i, dtype=BF16))
            want = chain(bufs[i])
            graphs[i].replay()
            torch.cuda.synchronize()
            assert torch.equal(outs[i], want)


def test_results_can_be_changed_in_place():
    """what a residual branch does to a result it owns; the gradient is that of the sum"""
    lv = H.Levels(2, [(5, 7)])
    for shape in ((2, 64, 5, 7), (2, 64, 35), (2, 64, 1, 5, 7), (70, 64)):
        for fmt in (0, 1):
            x = rnd(*shape, seed=1, dtype=BF16)
            x = (x.movedim(1, -1).contiguous().movedim(-1, 1) if fmt else x).requires_grad_(True)
            calls = [lambda x: P.group_norm_act(x, None, None, 8, activation="silu", dropout_p=0.1, seed=1), lambda x: P.dropout(x, 0.3, 2)]
            if x.dim() == 2:
                calls.append(lambda x: PR.gn_act_rows(x, lv, None, None, 8))
            else:
                w = rnd(48, shape[-1], seed=4) / 4
                calls += [lambda x: P.linear_fp8(x, w), lambda x: P.linear_fp8(x, w.clone().requires_grad_(True))]
            for call in calls:
                y = call(x)
                dy = rnd(*y.shape, seed=5, dtype=BF16)
                want, = torch.autograd.grad(y, [x], dy)
                z = call(x)
                z += 1
                got, = torch.autograd.grad(z, [x], dy)
                assert torch.equal(got, want) and torch.equal(z.detach(), y.detach() + 1)


@pytest.mark.parametrize("nkb", [1, 2, 3, 5, 7, 31, 63, 64, 65, 130])
def test_quantize_fp8_rows_of_any_number_of_blocks(nkb):
    """a workgroup's 64 blocks end inside a row, span many rows, or lie in one"""
    for rows in (1, 13, 70):
        for cols in (nkb * 128, nkb * 128 - 53):
            x = rnd(rows, cols, seed=nkb + rows, dtype=BF16)
            q = P.quantize_fp8(x)
            codes, byte, _ = R.fp8_quantize(x, 1)
            assert torch.equal(q.code_matrix().view(torch.uint8), codes.to(torch.uint8)) and torch.equal(q.scale_matrix().long(), byte)
            assert bool((q.codes.view(torch.uint8).transpose(0, 1).reshape(rows, -1)[:, cols:] == 0).all())
            assert bool((q.scales.transpose(0, 1).reshape(rows, -1)[:, nkb:] == 127).all())


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("cols", [1, 3, 8, 63, 64, 65, 100, 255, 513])
def test_dropout_rows_of_any_width_and_stride(cols, dtype):
    """strided x, residual and result through the C entry: the mask is that of the dense tensor, other columns stay as they were"""
    for rows in (1, 2, 41, 300):
        x, r = rnd(rows, cols, seed=1, dtype=dtype), rnd(rows, cols, seed=2, dtype=dtype)
        fac = R.keep_factor((rows, cols), 0.3, 7, 9).to(DEV)
        want = x.double() * fac
        bound = R.half_step(dtype) * want.abs() + 2 * R.E * want.abs() + R.tiny(dtype)
        both = want + r.double()
        bothb = R.half_step(dtype) * both.abs() + 2 * R.E * (want.abs() + both.abs()) + R.tiny(dtype)
        for ox, orr, oy, wide in ((0, 0, 0, cols), (1, 2, 3, cols + 5), (8, 0, 16, (cols + 23) // 8 * 8)):
            def place(t, o):
                buf = torch.full((rows, wide + o), 5.0, dtype=dtype, device=DEV)
                buf[:, o:o + cols] = t
                return buf
            bx, br, by = place(x, ox), place(r, orr), place(torch.zeros_like(x), oy)
            e = x.element_size()
            for res in (None, br):
                by[:, oy:oy + cols] = 0
                assert _lib.load().sm_dropout(H.DTYPE_CODES[dtype], bx.data_ptr() + ox * e, None if res is None else br.data_ptr() + orr * e,
                                              by.data_ptr() + oy * e, rows, cols, bx.stride(0), br.stride(0), by.stride(0),
                                              H.dropout_threshold(0.3), 7, 9, None, H._stream(x)) == 0
                within(by[:, oy:oy + cols], want if res is None else both, bound if res is None else bothb, "y")
                assert bool((by[:, :oy] == 5).all()) and bool((by[:, oy + cols:] == 5).all())


@pytest.mark.parametrize("c,groups,hw", [(256, 32, 900), (256, 32, 60), (60, 12, 300), (48, 4, 700)])
def test_group_norm_act_backward_over_its_own_gradient(c, groups, hw):
    """dx may be dy"""
    x, dy = rnd(2 * hw, c, seed=1, dtype=BF16), rnd(2 * hw, c, seed=2, dtype=BF16)
    ga, be = 1 + 0.1 * rnd(c, seed=3), 0.1 * rnd(c, seed=4)
    y = torch.empty_like(x)
    d, need, stats = H.group_norm_act(x, c, y, 2, (hw,), c, groups, 1e-5, H.ACTIVATIONS["silu"], H.dropout_threshold(0.2), 3, (4, None), ga, be,
                                      True)
    outs = []
    for dx in (torch.empty_like(x), dy):
        dg, db = torch.empty(c, device=DEV), torch.empty(c, device=DEV)
        H.group_norm_act_bwd(d, need, x, dy, c, dx, ga, be, stats, dg, db)
        outs.append((dx, dg, db))
    assert all(torch.equal(a, b) for a, b in zip(*outs))


@pytest.mark.parametrize("m,n,k", [(40, 70, 300), (500, 333, 1200), (300, 256, 9000), (3000, 512, 256)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_matmul_fp8_onto_its_residual(m, n, k, dtype):
    """residual may be y (with K split and without)"""
    a, b, r = P.quantize_fp8(rnd(m, k, seed=1)), P.quantize_fp8(rnd(n, k, seed=2), 128), rnd(m, n, seed=3, dtype=dtype)
    want = P.matmul_fp8(a, b, relu=True, residual=r, out_dtype=dtype)
    plan, need, _ = H._fp8_plan(m, n, k, 1, 128, H.DTYPE_CODES[dtype], 1)
    d = _lib.Fp8MatmulDesc.from_buffer_copy(plan)
    d.res_stride = n
    ws = torch.empty(max(need, 16), dtype=torch.uint8, device=DEV)
    assert _lib.load().sm_fp8_matmul(C.byref(d), a.codes.data_ptr(), a.scales.data_ptr(), b.codes.data_ptr(), b.scales.data_ptr(), None,
                                     r.data_ptr(), r.data_ptr(), ws.data_ptr(), need, H._stream(r)) == 0
    assert torch.equal(r, want)


@pytest.mark.parametrize("cols,stride", [(64, 64), (64, 80), (37, 41)])
def test_rows_written_over_their_input(cols, stride):
    """y may be x (dropout, GroupNorm) or the residual (dropout)"""
    for rows in (3, 500):
        def rows_like(seed):
            t = torch.zeros(rows, stride, dtype=F16, device=DEV)[:, :cols]
            return t.copy_(rnd(rows, cols, seed=seed, dtype=F16))
        x, r = rows_like(1), rows_like(2)
        thr, s = H.dropout_threshold(0.4), H._stream(x)
        want = P.dropout(x, 0.4, 5, 6, residual=r)
        for onto_x in (True, False):
            a, b = rows_like(1), rows_like(2)
            y = a if onto_x else b
            assert _lib.load().sm_dropout(1, a.data_ptr(), b.data_ptr(), y.data_ptr(), rows, cols, a.stride(0), b.stride(0), y.stride(0), thr, 5,
                                          6, None, s) == 0
            assert torch.equal(y, want)
        want = P.group_norm_act(x, None, None, 1, activation="gelu")
        plan, need, _ = H._gn_act_plan(rows, (1,), cols, 1, 1, 3, 1e-5, 0)
        d = _lib.GnActDesc.from_buffer_copy(plan)
        d.x_stride = d.y_stride = x.stride(0)
        ws = torch.empty(max(need, 16), dtype=torch.uint8, device=DEV)
        assert _lib.load().sm_group_norm_act(C.byref(d), x.data_ptr(), None, None, x.data_ptr(), None, ws.data_ptr(), need, s) == 0
        assert torch.equal(x, want)
