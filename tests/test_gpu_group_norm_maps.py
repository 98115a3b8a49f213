"""GroupNorm + activation on many small maps (a block takes several of them), against float64 (row_ops_ref.py has the bounds)."""
import pytest
import torch

import row_ops_ref as R
from sipmask_amd import hip_ops as H
from sipmask_amd import ops as P
from sipmask_amd import ops_rows as PR

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def rnd(*shape, seed=0, dtype=F32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def rows(t):
    return t.detach().movedim(1, -1).reshape(-1, t.shape[1])


def check(named):
    for name, got, want, bound in named:
        assert bool(((got.double() - want).abs() <= bound).all()), name


# images, channels, groups, map: one block a map, several maps a block, tiles with idle columns, groups of a whole tile of 32 columns
SHAPES = [(300, 64, 8, (7, 7)), (9001, 64, 8, (1, 1)), (70, 256, 32, (14, 14)), (1100, 256, 32, (2, 2)), (150, 72, 9, (5, 3)),
          (130, 512, 2, (3, 3)), (70, 1024, 4, (8, 7)), (200, 256, 2, (6, 6)), (400, 24, 1, (8, 8)), (66, 320, 10, (4, 4))]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("shape", SHAPES)
def test_many_small_maps(shape, dtype):
    n, c, g, (h, w) = shape
    x = (rnd(n, h, w, c, seed=1) * 1.5 + rnd(c, seed=9)).to(dtype).movedim(-1, 1).requires_grad_(True)
    ga, be = (1 + 0.3 * rnd(c, seed=5)).requires_grad_(True), (0.3 * rnd(c, seed=6)).requires_grad_(True)
    dy = rnd(n, h, w, c, seed=7, dtype=dtype).movedim(-1, 1)
    for act, p in (("relu", 0.0), ("gelu", 0.3)):
        y = P.group_norm_act(x, ga, be, g, 1e-5, act, p, 11, 3)
        fac = R.keep_factor((n * h * w, c), p, 11, 3).cuda() if p else None
        ref = R.GroupNormAct(rows(x), n, g, ga.detach(), be.detach(), 1e-5, act, fac)
        ref.backward(rows(dy))
        got = torch.autograd.grad(y, [x, ga, be], dy)
        bx, bg, bb = ref.bounds(dtype)
        check([("y", rows(y), ref.y, ref.y_bound(dtype)), ("dx", rows(got[0]), ref.dx, bx), ("dgamma", got[1], ref.dgamma, bg),
               ("dbeta", got[2], ref.dbeta, bb)])
        again = torch.autograd.grad(P.group_norm_act(x, ga, be, g, 1e-5, act, p, 11, 3), [x, ga, be], dy)
        assert all(torch.equal(u, v) for u, v in zip(got, again))


def test_many_small_maps_partial_gradients_and_layouts():
    n, c, h, w = 300, 64, 5, 5
    base = rnd(n, h, w, 80, seed=1, dtype=BF16)
    x = base[..., 8:72].movedim(-1, 1)
    ga, be = 1 + 0.3 * rnd(c, seed=5), 0.3 * rnd(c, seed=6)
    dy = rnd(n, h, w, c, seed=7, dtype=BF16).movedim(-1, 1)
    ref = R.GroupNormAct(rows(x), n, 8, ga, be, 1e-5, "silu")
    ref.backward(rows(dy))
    bx, bg, bb = ref.bounds(BF16)
    with torch.no_grad():
        check([("y", rows(P.group_norm_act(x, ga, be, 8, 1e-5, "silu")), ref.y, ref.y_bound(BF16))])
    for which in range(3):
        t = [x, ga, be]
        t[which] = t[which].detach().requires_grad_(True)
        got, = torch.autograd.grad(P.group_norm_act(*t, 8, 1e-5, "silu"), t[which], dy)
        check([(which, rows(got) if which == 0 else got, (ref.dx, ref.dgamma, ref.dbeta)[which], (bx, bg, bb)[which])])
    # neighbours of the slice stay as they were
    assert torch.equal(base, rnd(n, h, w, 80, seed=1, dtype=BF16))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_many_small_maps_of_a_pyramid(dtype):
    """levels of different sizes, an empty one among them, in one launch"""
    b, c = 90, 64
    lv = H.Levels(b, [(7, 9), (0, 4), (4, 5), (1, 1)])
    x = rnd(lv.rows, c, seed=2, dtype=dtype).requires_grad_(True)
    ga, be = (1 + 0.3 * rnd(c, seed=5)).requires_grad_(True), (0.3 * rnd(c, seed=6)).requires_grad_(True)
    dy = rnd(lv.rows, c, seed=7, dtype=dtype)
    y = PR.gn_act_rows(x, lv, ga, be, 8, 1e-5, "silu", 0.2, 5, 1)
    got = torch.autograd.grad(y, [x, ga, be], dy)
    fac = R.keep_factor((lv.rows, c), 0.2, 5, 1).cuda()
    dg, db, eg, eb = 0, 0, 0, 0
    for l, (h, w) in enumerate(lv.sizes):
        r = slice(lv.row0[l], lv.row0[l] + b * h * w)
        if h * w == 0:
            continue
        ref = R.GroupNormAct(x.detach()[r], b, 8, ga.detach(), be.detach(), 1e-5, "silu", fac[r])
        ref.backward(dy[r])
        bx, bg, bb = ref.bounds(dtype)
        check([("y", y.detach()[r], ref.y, ref.y_bound(dtype)), ("dx", got[0][r], ref.dx, bx)])
        dg, db, eg, eb = dg + ref.dgamma, db + ref.dbeta, eg + bg, eb + bb
    check([("dgamma", got[1], dg, eg), ("dbeta", got[2], db, eb)])


def test_many_small_maps_rows_written_over_their_input():
    n, c, h, w = 300, 64, 4, 4
    x = rnd(n, h, w, c, seed=1, dtype=BF16).movedim(-1, 1)
    want = P.group_norm_act(x, None, None, 8, 1e-5, "relu")
    y = x.clone(memory_format=torch.channels_last)
    H.group_norm_act(y, c, y, n, (h * w,), c, 8, 1e-5, 1, 0, 0, (0, None), None, None, False)
    assert torch.equal(y, want)
