"""Host side of the residual-block operators (GroupNorm + activation, dropout, e4m3 products): the float64 references themselves, the
C entry points' refusals (which return before anything is launched) and the Python entry points' refusals of CPU tensors."""
import ctypes as C

import pytest
import torch

import row_ops_ref as R
from sipmask_amd import _lib
from sipmask_amd import hip_ops as H
from sipmask_amd import ops as P
from sipmask_amd import ops_rows as PR


# ------------------------------------------------------------------------------------------------ references
@pytest.mark.parametrize("ctr,key,want", [
    ([0] * 4, [0] * 2, [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]),
    ([0xffffffff] * 4, [0xffffffff] * 2, [0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd]),
    ([0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344], [0xa4093822, 0x299f31d0], [0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1])])
def test_philox_known_answers(ctr, key, want):
    assert R.philox_block(ctr, key) == want


def test_draws_follow_the_blocks():
    seed, off = 0x0123456789abcdef, 0xfedcba9876543210
    for first in (0, 5, 8 * 3 + 7, (1 << 32) * 8 - 3):
        got = R.draws(first, 21, seed, off)
        for j, v in enumerate(got):
            i = first + j
            w = R.philox_block([(i // 8) & 0xffffffff, i // 8 >> 32, off & 0xffffffff, off >> 32], [seed & 0xffffffff, seed >> 32])
            assert int(v) == (w[i % 8 // 2] >> (16 * (i % 2))) & 0xffff


def test_fp8_reference_matches_every_code():
    """every finite e4m3 value is its own code, midpoints go to the even neighbour"""
    codes = torch.arange(256, dtype=torch.uint8)
    vals = codes.view(torch.float8_e4m3fn).double()
    fin = ~torch.isnan(vals)
    x = torch.full((1, 256 + 128), 448.0, dtype=torch.float64)      # a 448 in every block: scale 1
    x[0, :127], x[0, 128:255] = vals[:127], vals[128:255]
    c, s, v = R.fp8_quantize(x, 1)
    assert (s == 127).all()
    assert torch.equal(c[0, :127], codes[:127]) and torch.equal(c[0, 128:255], codes[128:255])
    pos = vals[:127]
    mid = (pos[1:] + pos[:-1]) / 2
    x = torch.full((1, 128), 448.0, dtype=torch.float64)
    x[0, :126] = mid
    c = R.fp8_quantize(x, 1)[0][0, :126].long()
    assert (c % 2 == 0).all() and ((c - torch.arange(126)).abs() <= 1).all()
    assert int(fin.sum()) == 254


@pytest.mark.parametrize("name", ["none", "relu", "silu", "gelu"])
def test_group_norm_reference_against_torch_and_differences(name):
    g = torch.Generator().manual_seed(3)
    b, hw, c, gr = 2, 11, 12, 3
    x = torch.randn(b * hw, c, generator=g, dtype=torch.float64)
    ga, be = (torch.randn(c, generator=g, dtype=torch.float64) for _ in range(2))
    dy = torch.randn(b * hw, c, generator=g, dtype=torch.float64)
    ref = R.GroupNormAct(x, b, gr, ga, be, 1e-5, name)
    n = torch.nn.functional.group_norm(x.view(b, hw, c).permute(0, 2, 1), gr, ga, be, 1e-5).permute(0, 2, 1).reshape(b * hw, c)
    want = {"none": n, "relu": n.relu(), "silu": torch.nn.functional.silu(n), "gelu": torch.nn.functional.gelu(n)}[name]
    torch.testing.assert_close(ref.y, want, rtol=1e-12, atol=1e-12)
    dx = ref.backward(dy)
    h = 1e-6
    f = lambda x_, ga_, be_: (R.GroupNormAct(x_, b, gr, ga_, be_, 1e-5, name).y * dy).sum()
    for v, grad, which in ((torch.randn(x.shape, generator=g, dtype=torch.float64), dx, 0),
                           (torch.randn(c, generator=g, dtype=torch.float64), ref.dgamma, 1),
                           (torch.randn(c, generator=g, dtype=torch.float64), ref.dbeta, 2)):
        args = [x, ga, be]
        hi, lo = list(args), list(args)
        hi[which], lo[which] = args[which] + h * v, args[which] - h * v
        num = (f(*hi) - f(*lo)) / (2 * h)
        assert abs(num - (grad * v).sum()) < 1e-6 * (1 + abs(num))


# ------------------------------------------------------------------------------------------------ C entry points
def _gn_desc(**kw):
    d = _lib.GnActDesc()
    d.nlev, d.batch, d.channels, d.groups, d.dtype, d.act, d.eps, d.drop_threshold = 1, 2, 64, 8, 0, 1, 1e-5, 0
    d.hw[0], d.row0[0] = 10, 0
    d.x_stride = d.y_stride = d.dy_stride = d.dx_stride = 64
    for k, v in kw.items():
        if k == "hw0":
            d.hw[0] = v
        elif k == "row00":
            d.row0[0] = v
        else:
            setattr(d, k, v)
    return d


def test_group_norm_workspace_is_host_arithmetic():
    lib = _lib.load()
    for back in (0, 1):
        assert lib.sm_group_norm_act_workspace(C.byref(_gn_desc(hw0=1000)), back) > 0
        assert lib.sm_group_norm_act_workspace(C.byref(_gn_desc(batch=0)), back) == 0
        assert lib.sm_group_norm_act_workspace(C.byref(_gn_desc(hw0=0)), back) >= 0


@pytest.mark.parametrize("bad", [dict(nlev=0), dict(nlev=6), dict(batch=-1), dict(channels=0), dict(groups=0), dict(groups=7), dict(dtype=3),
                                 dict(dtype=-1), dict(act=4), dict(eps=-1.0), dict(eps=float("nan")), dict(drop_threshold=-1),
                                 dict(drop_threshold=65537), dict(hw0=-1), dict(row00=-1), dict(x_stride=63), dict(y_stride=0),
                                 dict(dy_stride=63), dict(dx_stride=63), dict(batch=0x7fffffff)])
def test_group_norm_bad_descriptions(bad):
    lib = _lib.load()
    d = _gn_desc(**bad)
    one = C.c_void_p(16)
    assert lib.sm_group_norm_act_workspace(C.byref(d), 0) < 0
    assert lib.sm_group_norm_act(C.byref(d), one, None, None, one, None, one, 1 << 40, None) < 0
    assert lib.sm_group_norm_act_bwd(C.byref(d), one, one, None, None, one, one, one, one, one, 1 << 40, None) < 0


def test_group_norm_bad_pointers():
    lib = _lib.load()
    one, odd = C.c_void_p(16), C.c_void_p(24)
    d = _gn_desc(hw0=1000)                       # (a handful of rows needs no workspace)
    f = lambda x, y, st, ws, n: lib.sm_group_norm_act(C.byref(d), x, None, None, y, st, ws, n, None)
    assert f(None, one, None, one, 1 << 40) == -2 and f(one, None, None, one, 1 << 40) == -2 and f(one, one, None, None, 1 << 40) == -2
    assert f(one, one, odd, one, 1 << 40) == -2 and f(one, one, None, odd, 1 << 40) == -2
    assert f(one, one, None, one, 1) == -5
    assert lib.sm_group_norm_act_workspace(None, 0) == -2
    g = lambda x, dy, st, ws, n: lib.sm_group_norm_act_bwd(C.byref(d), x, dy, None, None, st, one, one, one, ws, n, None)
    assert g(None, one, one, one, 1 << 40) == -2 and g(one, None, one, one, 1 << 40) == -2 and g(one, one, None, one, 1 << 40) == -2
    assert g(one, one, one, one, 1) == -5
    # nothing to do: returns before it looks at a pointer
    d = _gn_desc(batch=0)
    assert lib.sm_group_norm_act(C.byref(d), None, None, None, None, None, None, 0, None) == 0


def test_dropout_bad_arguments():
    lib = _lib.load()
    one = C.c_void_p(16)

    def f(dt=0, x=one, res=None, y=one, rows=4, cols=8, lx=8, lr=8, ly=8, thr=100):
        return lib.sm_dropout(dt, x, res, y, rows, cols, lx, lr, ly, thr, 0, 0, None, None)
    assert f(dt=3) == -2 and f(dt=-1) == -2 and f(thr=-1) == -2 and f(thr=65537) == -2 and f(x=None) == -2 and f(y=None) == -2
    assert f(rows=-1) == -1 and f(cols=-1) == -1 and f(lx=7) == -1 and f(ly=7) == -1 and f(res=one, lr=7) == -1
    assert f(rows=1 << 60, cols=1 << 10, lx=1 << 10, ly=1 << 10) == -1
    assert f(rows=0, x=None, y=None) == 0 and f(cols=0, x=None, y=None) == 0


def test_fp8_bad_arguments():
    lib = _lib.load()
    one, odd = C.c_void_p(16), C.c_void_p(17)
    assert [lib.sm_fp8_codes_bytes(10, c) for c in (1, 128, 129)] == [1280, 1280, 2560] and lib.sm_fp8_codes_bytes(-1, 1) == -1
    assert [lib.sm_fp8_scales_bytes(200, c, br) for c, br in ((1, 1), (512, 1), (513, 1), (513, 128))] == [800, 800, 1600, 16]
    assert lib.sm_fp8_scales_bytes(1, 1, 2) == -2

    def q(dt=0, x=one, rows=4, cols=8, ld=8, br=1, gate=None, ldg=8, codes=one, sc=one, ct=None, st=None, cs=None, ws=None, n=0):
        return lib.sm_fp8_quantize(dt, x, rows, cols, ld, br, gate, ldg, codes, sc, ct, st, cs, ws, n, None)
    assert q(dt=5) == -2 and q(br=2) == -2 and q(x=None) == -2 and q(codes=None) == -2 and q(sc=None) == -2
    assert q(codes=odd) == -2 and q(sc=odd) == -2 and q(codes=None, sc=None) == -2 and q(ct=one) == -2 and q(ct=odd, st=one) == -2
    assert q(rows=-1) == -1 and q(cols=0) == -1 and q(ld=7) == -1 and q(rows=0, ct=one, st=one) == -1 and q(rows=0) == 0
    assert q(rows=1 << 33, ct=one, st=one) == -1 and q(gate=one, ldg=7) == -1
    assert q(cs=one) == -2 and q(cs=one, ws=one, n=31) == -5 and lib.sm_fp8_quantize_workspace(4, 8, 1) == 32
    assert lib.sm_fp8_quantize_workspace(-1, 8, 1) == -1 and lib.sm_fp8_quantize_workspace(1, 0, 0) == -1

    def mm(ws=1 << 40, res=None, a=one, y=one, wsp=one, **kw):
        d = _lib.Fp8MatmulDesc()
        d.m, d.n, d.k, d.a_block_rows, d.b_block_rows, d.out_dtype, d.relu, d.y_stride, d.res_stride = 4, 8, 128, 1, 128, 0, 0, 8, 8
        for k, v in kw.items():
            setattr(d, k, v)
        return lib.sm_fp8_matmul(C.byref(d), a, one, one, one, None, res, y, wsp, ws, None)
    for bad in (dict(m=-1), dict(n=0), dict(k=0), dict(y_stride=7), dict(res=one, res_stride=7)):
        assert mm(**bad) == -1, bad
    for bad in (dict(a_block_rows=2), dict(b_block_rows=0), dict(out_dtype=3), dict(a=None), dict(a=odd), dict(y=None)):
        assert mm(**bad) == -2, bad
    assert mm(m=0, a=None, y=None) == 0
    d = _lib.Fp8MatmulDesc()
    d.m, d.n, d.k, d.a_block_rows, d.b_block_rows, d.y_stride = 100, 512, 1 << 16, 1, 1, 512
    need = lib.sm_fp8_matmul_workspace(C.byref(d))
    assert need > 16                             # few tiles, long sum: split
    assert lib.sm_fp8_matmul(C.byref(d), one, one, one, one, None, None, one, one, need - 1, None) == -5
    assert lib.sm_fp8_matmul(C.byref(d), one, one, one, one, None, None, one, None, need, None) == -2
    d.m = 1000
    need = lib.sm_fp8_linear_workspace(C.byref(d))

    def lin(dt=0, x=one, ld=1 << 16, y=one, ws=one, n=need):
        return lib.sm_fp8_linear(C.byref(d), dt, x, ld, one, one, None, None, y, ws, n, None)
    assert lin(dt=3) == -2 and lin(x=None) == -2 and lin(y=None) == -2 and lin(ws=None) == -2 and lin(ld=10) == -1 and lin(n=need - 1) == -5
    d.a_block_rows = 128
    assert lin() == -2


def test_fp8_launch_limits():
    """more blocks than a launch holds: refused, not truncated"""
    lib = _lib.load()
    one = C.c_void_p(16)
    d = _lib.Fp8MatmulDesc()
    d.m, d.n, d.k, d.a_block_rows, d.b_block_rows, d.y_stride = 1, 1 << 30, 128, 1, 128, 1 << 30
    assert lib.sm_fp8_matmul_workspace(C.byref(d)) == lib.sm_fp8_linear_workspace(C.byref(d)) != 0
    assert lib.sm_fp8_linear_workspace(C.byref(d)) < 0
    assert lib.sm_fp8_matmul(C.byref(d), one, one, one, one, None, None, one, one, 1 << 40, None) < 0
    cols = 1 << 30
    assert lib.sm_fp8_quantize(0, one, 1, cols, cols, 1, None, 0, one, one, None, None, one, one, 1 << 40, None) < 0


def test_fp8_layer_bad_arguments():
    lib = _lib.load()
    one, odd = C.c_void_p(16), C.c_void_p(17)
    out = [C.c_int64() for _ in range(3)]

    def desc(**kw):
        d = _lib.Fp8LayerDesc()
        d.m, d.n, d.k, d.need_dx, d.need_dw, d.need_db, d.x_stride, d.dy_stride = 200, 96, 300, 1, 1, 1, 300, 96
        for k, v in kw.items():
            setattr(d, k, v)
        return d

    def size(**kw):
        st = lib.sm_fp8_layer_bytes(C.byref(desc(**kw)), *map(C.byref, out))
        return st or tuple(v.value for v in out)
    full = size()
    # codes of x^T (300 x 200) and w^T (300 x 96) with their scales, 256 bytes apart
    assert full[0] == 300 * 256 + 1280 + 300 * 128 + 256
    assert size(need_dx=0, need_dw=0)[0] == 0 and size(need_dx=0)[0] == 300 * 256 + 1280
    assert size(have_wq=1)[1] < full[1] and size(need_dw=0, need_db=0)[2] < full[2]
    for bad in (dict(m=0), dict(n=0), dict(k=0), dict(x_stride=299), dict(dy_stride=95), dict(m=1 << 31)):
        assert size(**bad) == -1, bad
    for bad in (dict(dtype=3), dict(w_dtype=-1)):
        assert size(**bad) == -2, bad
    assert lib.sm_fp8_layer_bytes(C.byref(desc()), None, C.byref(out[1]), C.byref(out[2])) == -2
    assert lib.sm_fp8_layer_bytes(None, *map(C.byref, out)) == -2

    def fwd(x=one, w=one, ld=300, wc=None, ws=None, y=one, saved=one, wsp=one, n=full[1], **kw):
        return lib.sm_fp8_layer_fwd(C.byref(desc(**kw)), x, w, ld, wc, ws, None, y, saved, wsp, n, None)
    for bad in (dict(x=None), dict(y=None), dict(saved=None), dict(saved=odd), dict(wsp=None), dict(w=None), dict(ld=299), dict(have_wq=1),
                dict(have_wq=1, wc=one)):
        assert fwd(**bad) == -2, bad
    assert fwd(n=full[1] - 1) == -5

    def bwd(dy=one, y=None, saved=one, dx=one, dw=one, db=one, wsp=one, n=full[2], **kw):
        return lib.sm_fp8_layer_bwd(C.byref(desc(**kw)), dy, y, saved, dx, dw, db, wsp, n, None)
    for bad in (dict(dy=None), dict(saved=None), dict(saved=odd), dict(dx=None), dict(dw=None), dict(db=None), dict(wsp=odd), dict(relu=1)):
        assert bwd(**bad) == -2, bad
    assert bwd(n=full[2] - 1) == -5
    assert bwd(need_dx=0, need_dw=0, need_db=0, dx=None, dw=None, db=None, saved=None, wsp=None, n=0) == 0



# ------------------------------------------------------------------------------------------------ Python entry points
def test_cpu_tensors_are_refused():
    x, w = torch.randn(4, 8), torch.randn(8)
    for call in (lambda: P.group_norm_act(x, w, w, 2), lambda: PR.gn_act_rows(x, H.Levels(1, [(2, 2)]), w, w, 2),
                 lambda: P.dropout(x, 0.5, 1), lambda: P.quantize_fp8(x), lambda: P.linear_fp8(x, torch.randn(3, 8))):
        with pytest.raises(NotImplementedError):
            call()


def test_dropout_probability_and_offset_checks():
    assert H.dropout_threshold(0) == 0 and H.dropout_threshold(1) == 65536 and H.dropout_threshold(0.1) == 6554
    for p in (-0.1, 1.1, float("nan")):
        with pytest.raises(ValueError):
            H.dropout_threshold(p)
    dev = torch.device("cpu")
    assert H.dropout_offset(-1, dev) == ((1 << 64) - 1, None)
    t = torch.zeros(1, dtype=torch.int64)
    assert H.dropout_offset(t, dev) == (0, t)
    for bad in (torch.zeros(2, dtype=torch.int64), torch.zeros(1, dtype=torch.int32)):
        with pytest.raises(ValueError):
            H.dropout_offset(bad, dev)


def test_dense_rows_views_and_copies():
    t = torch.arange(4 * 6 * 8.0).view(4, 6, 8)
    assert H.dense_rows(t, 8).data_ptr() == t.data_ptr() and H.dense_rows(t, 8).shape == (24, 8)
    v = H.dense_rows(t[..., 2:5], 3)
    assert v.data_ptr() == t[..., 2:5].data_ptr() and H.row_stride(v) == 8 and torch.equal(v, t[..., 2:5].reshape(24, 3))
    for odd in (t.transpose(1, 2), t[:, ::2, ::2], t[:1, :1].expand(5, 6, 8), t[..., :1].expand(4, 6, 3)):
        c = odd.shape[-1]
        r = H.dense_rows(odd, c)
        assert torch.equal(r, odd.reshape(-1, c)) and r.stride(1) == 1 and (r.shape[0] == 1 or r.stride(0) >= c)
    one = H.dense_rows(t[0, :1, 1:4], 3)
    assert H.row_stride(one) == 3
    assert H.dense_rows(t[:0], 8).shape == (0, 8)
    col = H.dense_rows(torch.zeros(1).expand(5, 1), 1)
    assert col.stride(0) >= 1
