"""How the residual-block operators are called by autograd and the tracer: forward mode, torch.jit.trace, saved-tensor hooks, activation
checkpointing.  On the CPU the C entry points are replaced by stand-ins that note what they are given (and fill the result with something
that depends on x), on the device they are the real ones."""
import contextlib
import ctypes as C

import numpy as np
import pytest
import torch
import torch.utils.checkpoint
from torch.autograd import forward_ad

import row_ops_ref as R
from sipmask_amd import _lib
from sipmask_amd import hip_ops as H
from sipmask_amd import ops as P
from sipmask_amd import ops_rows as PR
from sipmask_amd import sipmask_head  # noqa: F401
from sipmask_amd.registry import build_head

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def floats(address, rows, cols, stride):
    """f32 rows at an address as a numpy view"""
    flat = np.ctypeslib.as_array((C.c_float * ((rows - 1) * stride + cols)).from_address(address))
    return np.lib.stride_tricks.as_strided(flat, (rows, cols), (4 * stride, 4))


class StandIn:
    """the library with its launches on f32 rows replaced: y = 2 x (products: y[i][j] = x[i][0])"""

    def __init__(self, lib):
        self.lib, self.calls = lib, []

    def __getattr__(self, name):
        return getattr(self.lib, name)

    @staticmethod
    def struct(d, cls):
        return cls.from_buffer_copy(d if isinstance(d, (bytes, cls)) else d._obj)

    def sm_group_norm_act(self, d, x, gamma, beta, y, stats, ws, need, stream):
        d = self.struct(d, _lib.GnActDesc)
        rows = d.batch * sum(d.hw[l] for l in range(d.nlev))
        floats(y, rows, d.channels, d.y_stride)[...] = 2 * floats(x, rows, d.channels, d.x_stride)
        self.calls.append(("gn", d, x))
        return 0

    def sm_group_norm_act_bwd(self, d, x, dy, gamma, beta, stats, dx, dgamma, dbeta, ws, need, stream):
        self.calls.append(("gn_bwd", self.struct(d, _lib.GnActDesc), x))
        return 0

    def sm_dropout(self, dtype, x, res, y, rows, cols, ldx, ldr, ldy, *rest):
        floats(y, rows, cols, ldy)[...] = 2 * floats(x, rows, cols, ldx)
        self.calls.append(("dropout", rows, cols))
        return 0

    def _product(self, m, n, x, stride, y):
        floats(y, m, n, n)[...] = floats(x, m, 1, stride)
        return 0

    def sm_fp8_quantize(self, *args):
        return 0

    def sm_fp8_linear(self, d, dtype, x, stride, *rest):
        d = self.struct(d, _lib.Fp8MatmulDesc)
        return self._product(d.m, d.n, x, stride, rest[4])

    def sm_fp8_layer_fwd(self, d, x, w, ldw, wc, ws, bias, y, *rest):
        d = self.struct(d, _lib.Fp8LayerDesc)
        return self._product(d.m, d.n, x, d.x_stride, y)


@pytest.fixture
def standin(monkeypatch):
    s = StandIn(_lib.load())
    monkeypatch.setattr(_lib, "load", lambda: s)
    monkeypatch.setattr(_lib, "require_cuda", lambda *t: None)
    monkeypatch.setattr(_lib, "on_device", lambda t: contextlib.nullcontext())
    monkeypatch.setattr(_lib, "here", lambda t: True)
    monkeypatch.setattr(H, "_stream", lambda t: 0)
    return s


def _cl(*shape, seed=0, dtype=F32, device="cpu"):
    t = torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(device)
    return t.movedim(-1, 1) if t.dim() == 4 else t


LV = H.Levels(1, [(2, 3), (1, 2)])


def _operators(device="cpu"):
    """name -> (function of one tensor, shape of that tensor (channels last))"""
    c = 16
    w, b = 1 + 0.1 * _cl(c, seed=1, device=device), 0.1 * _cl(c, seed=2, device=device)
    lw, lb = 0.3 * _cl(24, c, seed=3, device=device), 0.1 * _cl(24, seed=4, device=device)
    return {
        "group_norm_act": (lambda x: P.group_norm_act(x, w, b, 4, 1e-5, "silu", 0.25, 3, 5), (2, 3, 4, c)),
        "gn_act_rows": (lambda x: PR.gn_act_rows(x, LV, w, b, 4, 1e-5, "gelu"), (LV.rows, c)),
        "dropout": (lambda x: P.dropout(x, 0.5, 7, 1), (5, c)),
        "dropout_residual": (lambda x: P.dropout(x, 0.5, 7, 1, residual=x), (5, c)),
        "linear_fp8": (lambda x: P.linear_fp8(x, lw, lb, relu=True), (6, c)),
        "linear_fp8_3d": (lambda x: P.linear_fp8(x, lw, lb), (2, 3, c)),
    }


NAMES = sorted(_operators())


def _trace(f, x):
    with torch.no_grad():
        return torch.jit.trace(f, (x,), check_trace=False)


# ------------------------------------------------------------------------------------------------ forward mode and the tracer
@pytest.mark.parametrize("name", NAMES)
def test_forward_mode_is_refused(standin, name):
    f, shape = _operators()[name]
    x = _cl(*shape)
    with forward_ad.dual_level():
        d = forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(RuntimeError, match="forward mode|jvp"):
            f(d)
        f(x)                                     # (a tensor without a tangent is none of its business)
    assert torch.equal(f(x), f(x))


@pytest.mark.parametrize("name", NAMES)
def test_function_transforms_are_refused(standin, name):
    """torch.func: no rule of these operators, so an error and no result"""
    f, shape = _operators()[name]
    x = _cl(*shape)
    for call in (lambda: torch.func.jvp(f, (x,), (torch.ones_like(x),)), lambda: torch.func.jacfwd(f)(x), lambda: torch.func.vmap(f)(x[None])):
        with pytest.raises(RuntimeError):
            call()
    assert not standin.calls


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
@pytest.mark.parametrize("name", NAMES)
def test_a_traced_call_follows_its_input(standin, name):
    f, shape = _operators()[name]
    t = _trace(f, _cl(*shape, seed=10))
    for seed in (11, 12):
        x = _cl(*shape, seed=seed)
        y = t(x)
        assert y.shape == f(x).shape and torch.equal(y, f(x)) and float(y.abs().max()) > 0


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
def test_operators_on_codes_are_not_traced(standin):
    """their results are filled behind the tracer's back and are no inputs of an autograd function"""
    w = _cl(24, 16, seed=3)
    wq = P.quantize_fp8(w, 128)
    for f in (lambda x: P.matmul_fp8(P.quantize_fp8(x), wq), lambda x: P.quantize_fp8(x).dequantize(), lambda x: P.matmul_fp8(wq, wq) + x[0, 0]):
        with pytest.raises(RuntimeError, match="torch.jit.trace"):
            _trace(f, _cl(6, 16))
    t = _trace(lambda x: P.linear_fp8(x, None, weight_q=wq), _cl(6, 16))
    x = _cl(6, 16, seed=1)
    assert torch.equal(t(x), P.linear_fp8(x, None, weight_q=wq))


@pytest.mark.gpu
@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
@pytest.mark.parametrize("name", NAMES)
def test_forward_mode_and_trace_on_the_device(name):
    f, shape = _operators("cuda")[name]
    x = _cl(*shape, seed=10, device="cuda")
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="forward mode|jvp"):
            f(forward_ad.make_dual(x, torch.ones_like(x)))
    t = _trace(f, x)
    for seed in (11, 12):
        x = _cl(*shape, seed=seed, device="cuda")
        assert torch.equal(t(x), f(x))


# ------------------------------------------------------------------------------------------------ saved tensors that come back as others
def _dense_copy(t):
    return torch.empty(t.shape, dtype=t.dtype, device=t.device).copy_(t)


@pytest.mark.parametrize("pyramid", [False, True])
def test_backward_takes_strides_and_offset_from_the_saved_tensors(standin, pyramid):
    """hooks that hand back dense copies: the backward steps x by the copy's stride and reads the copy of the offset, not the address that
    the forward's (long freed) one had; the descriptor that the graph keeps stays the forward's"""
    if pyramid:
        x = _cl(LV.rows, 40)[:, 8:24].requires_grad_(True)
        call = lambda off: PR.gn_act_rows(x, LV, None, None, 4, 1e-5, "relu", 0.5, 3, off)
    else:
        x = _cl(2, 3, 4, 40)[:, 8:24].requires_grad_(True)
        call = lambda off: P.group_norm_act(x, None, None, 4, 1e-5, "relu", 0.5, 3, off)
    copies = []

    def unpack(t):
        copies.append(_dense_copy(t))
        return copies[-1]
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
        y = call(torch.tensor([7]) * 2 + 1)
    (_, fwd, _), = standin.calls
    assert fwd.x_stride == 40 and fwd.drop_offset_dev
    for turn in range(2):
        del standin.calls[:], copies[:]
        torch.autograd.grad(y, x, torch.ones_like(y), retain_graph=True)
        (_, bwd, address), = standin.calls
        off, = [t for t in copies if t.dtype == torch.int64]
        dense, = [t for t in copies if t.shape == x.shape]
        assert bwd.x_stride == 16 and bwd.drop_offset_dev == off.data_ptr() and int(off) == 15
        if pyramid:
            assert address == dense.data_ptr()
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t):
        y = call(0)                              # nothing changed hands: as the forward had it, no offset
    del standin.calls[:]
    torch.autograd.grad(y, x, torch.ones_like(y))
    (_, bwd, address), = standin.calls
    assert bwd.x_stride == 40 and not bwd.drop_offset_dev and address == x.data_ptr()


def _gn_case(layout, dev):
    """(x, function of x and an offset) of a slice of channels"""
    w, b = (1 + 0.1 * _cl(16, seed=1, device=dev)).requires_grad_(True), (0.1 * _cl(16, seed=2, device=dev)).requires_grad_(True)
    if layout == "rows":
        lv = H.Levels(2, [(9, 13), (5, 7)])
        x = _cl(lv.rows, 40, dtype=BF16, device=dev)[:, 8:24]
        return x, w, b, lambda x, off: PR.gn_act_rows(x, lv, w, b, 4, 1e-5, "silu", 0.3, 5, off)
    x = _cl(2, 33, 31, 40, dtype=BF16, device=dev)[:, 8:24]
    return x, w, b, lambda x, off: P.group_norm_act(x, w, b, 4, 1e-5, "silu", 0.3, 5, off)


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["rows", "nchw"])
@pytest.mark.parametrize("how", ["cpu", "pinned", "checkpoint", "checkpoint_reentrant"])
def test_group_norm_act_through_hooks_and_checkpoints(layout, how):
    """saved tensors that were on the host in between, and an activation that is computed again, with an offset that lives only inside the
    region: the gradients of the plain call, bit for bit (no atomics)"""
    x, w, b, f = _gn_case(layout, "cuda")
    base = torch.tensor([20], device="cuda")
    layer = lambda x: f(x, base * 2 + 1)
    plain = x.detach().requires_grad_(True)
    y0 = layer(plain)
    dy = torch.randn(y0.shape, generator=torch.Generator().manual_seed(3)).to(BF16).cuda()
    want = torch.autograd.grad(y0, [plain, w, b], dy)
    x = x.detach().requires_grad_(True)
    assert x.stride() == plain.stride()
    if how in ("cpu", "pinned"):
        with torch.autograd.graph.save_on_cpu(pin_memory=how == "pinned"):
            y = layer(x)
    else:
        y = torch.utils.checkpoint.checkpoint(layer, x, use_reentrant=how == "checkpoint_reentrant")
    junk = [torch.full((1,), 999, device="cuda") for _ in range(64)]     # (where the forward's offset was)
    assert torch.equal(y, y0)
    if how == "checkpoint_reentrant":
        for t in (w, b):
            t.grad = None
        y.backward(dy)
        got = (x.grad, w.grad, b.grad)
    else:
        got = torch.autograd.grad(y, [x, w, b], dy)
    for u, v in zip(got, want):
        assert torch.equal(u, v)
    del junk


@pytest.mark.parametrize("reentrant", [False, True])
def test_tower_dropout_is_not_computed_again(reentrant):
    """the counter has moved on when a checkpoint calls the forward a second time: refused, not another mask"""
    h = build_head(dict(type="SipMaskHead", num_classes=5, in_channels=64, feat_channels=64, stacked_convs=2, tower_dropout=0.25)).train()

    def layer(x):
        d = h._tower_drop()
        return x.square() * R.keep_factor(x.shape, d["dropout_p"], d["seed"], d["offset"])
    x = torch.randn(4, 8, dtype=torch.float64, requires_grad=True)
    y = torch.utils.checkpoint.checkpoint(layer, x, use_reentrant=reentrant)
    assert h.tower_dropout_calls == 1
    with pytest.raises(RuntimeError, match="checkpoint computes again"):
        y.sum().backward()
    assert h.tower_dropout_calls == 1
    layer(x).sum().backward()                    # without one, and behind that: as ever
    assert h.tower_dropout_calls == 2 and torch.equal(x.grad, 2 * x.detach() * R.keep_factor(x.shape, 0.25, 0, 2))


def test_tower_dropout_is_not_traced():
    """the tracer would bake the counter in: every call of the traced function would repeat one mask"""
    h = build_head(dict(type="SipMaskHead", num_classes=5, in_channels=64, feat_channels=64, stacked_convs=2, tower_dropout=0.25)).train()
    with pytest.raises(RuntimeError, match="repeat its masks"):
        _trace(lambda x: x * h._tower_drop()["offset"], torch.randn(4))
    assert h.tower_dropout_calls == 0
    assert torch.equal(_trace(lambda x: x * len(h.eval()._tower_drop()), torch.randn(4))(torch.ones(4)), torch.zeros(4))


@pytest.mark.gpu
@pytest.mark.parametrize("how", ["cpu", "checkpoint"])
def test_dropout_and_linear_through_hooks_and_checkpoints(how):
    w, b = (0.3 * _cl(24, 40, seed=3, device="cuda")).requires_grad_(True), (0.1 * _cl(24, seed=4, device="cuda")).requires_grad_(True)
    x = _cl(70, 56, device="cuda")[:, 8:48].requires_grad_(True)
    base = torch.tensor([20], device="cuda")
    layer = lambda x: P.dropout(P.linear_fp8(x, w, b, relu=True), 0.3, 5, base * 2 + 1)
    y0 = layer(x)
    dy = _cl(70, 24, seed=6, device="cuda")
    want = torch.autograd.grad(y0, [x, w, b], dy)
    if how == "cpu":
        with torch.autograd.graph.save_on_cpu():
            y = layer(x)
    else:
        y = torch.utils.checkpoint.checkpoint(layer, x, use_reentrant=False)
    junk = [torch.full((1,), 999, device="cuda") for _ in range(64)]
    assert torch.equal(y, y0)
    for u, v in zip(torch.autograd.grad(y, [x, w, b], dy), want):
        assert torch.equal(u, v)
    del junk


# ------------------------------------------------------------------------------------------------ sizes
def test_sizes_beyond_the_descriptors_fields_are_refused():
    """2^32 + 2 images are not 2: the descriptors hold 32 bits"""
    big = (1 << 32) + 2
    for call in (lambda: H._gn_act_plan(big, (1,), 8, 2, 0, 1, 1e-5, 0), lambda: H._gn_act_plan(1, (1,), big, 2, 0, 1, 1e-5, 0),
                 lambda: H._fp8_plan(4, big, 16, 1, 128, 0, 0), lambda: H._fp8_plan(4, 8, big, 1, 128, 0, 0),
                 lambda: H._fp8_layer_plan(4, big, 16, 0, 0, 0, 1, 1, 1, 0), lambda: H._fp8_layer_plan(4, 8, big, 0, 0, 0, 1, 1, 1, 0)):
        with pytest.raises(ValueError, match="at most"):
            call()
    assert H._fp8_plan(4, 8, 16, 1, 128, 0, 0)[1:] == (0, 0)
    with pytest.raises(RuntimeError):            # (rows are 64 bits wide; a layer's gradients sum over them)
        H._fp8_layer_plan(big, 8, 16, 0, 0, 0, 1, 1, 1, 0)


# ------------------------------------------------------------------------------------------------ groups and column tiles of every relation
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("shape", [(1, 256, 256, 130, 127),      # one channel a group, more row blocks than the partials alone would allow
                                   (1, 768, 256, 40, 33),        # groups of three channels that lie in two tiles
                                   (2, 264, 88, 50, 31),         # ... in tiles of 17 vectors
                                   (1, 1024, 2, 41, 37),         # a group of two whole tiles
                                   (1, 640, 2, 60, 23),          # ... of one and a half
                                   (1, 130, 26, 97, 30),         # five channels, any alignment
                                   (3, 96, 96, 70, 61)])
def test_group_norm_act_groups_and_tiles(shape, dtype):
    n, c, g, h, w = shape
    x = (_cl(n, h, w, c, seed=1, device="cuda") * 1.5 + torch.linspace(-1, 1, c, device="cuda").view(1, c, 1, 1)).to(dtype)
    x = x.contiguous(memory_format=torch.channels_last).requires_grad_(True)
    ga, be = (1 + 0.3 * _cl(c, seed=5, device="cuda")).requires_grad_(True), (0.3 * _cl(c, seed=6, device="cuda")).requires_grad_(True)
    dy = _cl(n, h, w, c, seed=7, dtype=dtype, device="cuda")
    y = P.group_norm_act(x, ga, be, g, 1e-5, "silu")
    got = torch.autograd.grad(y, [x, ga, be], dy)
    rows = lambda t: t.detach().movedim(1, -1).reshape(-1, c)
    ref = R.GroupNormAct(rows(x), n, g, ga.detach(), be.detach(), 1e-5, "silu")
    ref.backward(rows(dy))
    # a block of at most h w / 4 rows has 512 / 64 threads or more to a column: their rows, then the tree over the threads
    bounds = ref.bounds(dtype, run=h * w // 32 + 10)
    for name, u, want, bound in [("y", rows(y), ref.y, ref.y_bound(dtype)), ("dx", rows(got[0]), ref.dx, bounds[0]),
                                 ("dgamma", got[1], ref.dgamma, bounds[1]), ("dbeta", got[2], ref.dbeta, bounds[2])]:
        assert bool(((u.double() - want).abs() <= bound).all()), name
    again = torch.autograd.grad(P.group_norm_act(x, ga, be, g, 1e-5, "silu"), [x, ga, be], dy)
    assert all(torch.equal(u, v) for u, v in zip(got, again))
