"""SipMaskHead(tower_dropout=..., mask_lat_fp8=...): arguments, counter and masks on the host; the layers against float64 on the
device."""
import pytest
import torch

import row_ops_ref as R
from sipmask_amd import hip_ops as H
from sipmask_amd import ops_rows as PR
from sipmask_amd import sipmask_head  # noqa: F401
from sipmask_amd.registry import build_head

SMALL = dict(type="SipMaskHead", num_classes=5, in_channels=64, feat_channels=64, stacked_convs=2)
BF16 = torch.bfloat16


def head(**kw):
    torch.manual_seed(3)
    return build_head(dict(SMALL, **kw))


def test_probability_is_checked():
    for p in (-0.1, 1.0, float("nan")):
        with pytest.raises(ValueError):
            head(tower_dropout=p)


def test_off_by_default_and_not_part_of_the_state():
    a, b = head(), head(tower_dropout=0.3)
    assert a._tower_drop() == {} and a.tower_dropout_calls == 0
    assert list(a.state_dict()) == list(b.state_dict())
    assert all(torch.equal(u, v) for u, v in zip(a.state_dict().values(), b.state_dict().values()))


def test_a_mask_of_its_own_for_every_call():
    h = head(tower_dropout=0.25, tower_dropout_seed=7).train()
    got = [h._tower_drop() for _ in range(4)]
    assert [d["offset"] for d in got] == [1, 2, 3, 4] and all(d["seed"] == 7 and d["dropout_p"] == 0.25 for d in got)
    h.eval()
    assert h._tower_drop() == {} and h.tower_dropout_calls == 4


def test_ranks_draw_different_masks(monkeypatch):
    h = head(tower_dropout=0.25).train()
    monkeypatch.setattr(torch.distributed, "is_initialized", lambda: True)
    monkeypatch.setattr(torch.distributed, "get_rank", lambda: 3)
    assert h._tower_drop()["offset"] == (3 << 48) + 1


def _bf(*shape, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(BF16).cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("norm", [True, False])
def test_tower_layer_on_rows(norm):
    """the tower's layer = the convolution's own output, then GroupNorm + ReLU (or ReLU) and the mask, in float64"""
    p, seed = 0.3, 11
    kw = {} if norm else dict(norm_cfg=None)
    h = head(tower_dropout=p, tower_dropout_seed=seed, **kw).cuda().train()
    h.tower_dropout_calls = 40
    lv = H.Levels(2, [(9, 13), (5, 7)])
    x = _bf(lv.rows, 64, seed=1).requires_grad_(True)
    dy = _bf(lv.rows, 64, seed=2)
    m = h.cls_convs[0]
    y = h._tower_rows(x, lv, h.cls_convs)
    assert h.tower_dropout_calls == 41
    gx, = torch.autograd.grad(y, [x], dy)
    x2 = x.detach().requires_grad_(True)
    fac = R.keep_factor((lv.rows, 64), p, seed, 41).cuda()
    if not norm:
        v, _ = PR.conv_rows(x2, lv, m.conv.weight, m.conv.bias, 1, 1, relu=True)
        want = v.detach().double() * fac
        err = (y.detach().double() - want).abs()
        assert bool((err <= R.half_step(BF16) * want.abs() + 2 * R.E * want.abs() + R.tiny(BF16)).all())
        assert bool((y[fac == 0] == 0).all())
        g2, = torch.autograd.grad(v, [x2], (dy.double() * fac).to(BF16))
    else:
        v, _ = PR.conv_rows(x2, lv, m.conv.weight, None, 1, 1)
        dv = torch.empty_like(v)
        for l, (a, b) in enumerate(lv.sizes):
            r = slice(lv.row0[l], lv.row0[l] + 2 * a * b)
            ref = R.GroupNormAct(v.detach()[r], 2, 32, m.norm.weight.detach(), m.norm.bias.detach(), 1e-5, "relu", fac[r])
            assert bool(((y.detach()[r].double() - ref.y).abs() <= ref.y_bound(BF16)).all())
            dv[r] = ref.backward(dy[r]).to(BF16)
        g2, = torch.autograd.grad(v, [x2], dv)
    # dx: the layer's gradient went through one more rounding to bf16 on each side; 2^-8 twice, relative in norm (9 * 64 terms add
    # rounding errors that are independent)
    assert float((gx.float() - g2.float()).norm() / g2.float().norm()) < 2 * 2.0 ** -8


@pytest.mark.gpu
def test_the_counter_fixes_the_masks():
    wide = dict(in_channels=256, feat_channels=256)      # (gn_rows, the path without dropout, wants 8 channels per group)
    h = head(tower_dropout=0.5, **wide).cuda().train()
    lv = H.Levels(1, [(8, 8)])
    x = _bf(lv.rows, 256, seed=3)
    with torch.no_grad():
        a, b = h._tower_rows(x, lv, h.reg_convs), h._tower_rows(x, lv, h.reg_convs)
        h.tower_dropout_calls = 0
        c = h._tower_rows(x, lv, h.reg_convs)
        assert not torch.equal(a, b) and torch.equal(a, c)
        plain = head(**wide).cuda().train()
        u, v = plain._tower_rows(x, lv, plain.reg_convs), h.eval()._tower_rows(x, lv, h.reg_convs)
        assert h.tower_dropout_calls == 2 and torch.allclose(u.float(), v.float(), rtol=2.0 ** -7, atol=1e-3)


@pytest.mark.gpu
@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("rows", ["1", "0"])
def test_training_step_reaches_every_parameter(monkeypatch, norm, rows):
    """both training graphs; the NCHW one draws per level, the row one per layer"""
    monkeypatch.setenv("SIPMASK_TRAIN_ROWS", rows)
    kw = {} if norm else dict(norm_cfg=None, ssd_flag=True)
    h = build_head(dict(type="SipMaskHead", num_classes=81, in_channels=256, stacked_convs=2, tower_dropout=0.1, **kw)).cuda().train()
    g = torch.Generator().manual_seed(3)
    sizes = [(16, 20), (8, 10), (4, 5), (2, 3), (1, 2)]
    feats = [torch.randn(2, 256, a, b, generator=g).cuda() for a, b in sizes]
    out = h(feats)
    assert h.tower_dropout_calls == (3 if rows == "1" else 15)
    tot = sum(t.float().square().mean() for lev in out[:4] for t in lev) + out[4].float().square().mean()
    tot.backward()
    for name, p in h.named_parameters():
        if name.startswith("feat_align.norm") and not norm:
            continue
        assert p.grad is not None and bool(torch.isfinite(p.grad).all()), name


@pytest.mark.gpu
def test_capture_is_refused():
    h = head(tower_dropout=0.5).cuda().train()
    lv = H.Levels(1, [(8, 8)])
    x = _bf(lv.rows, 64, seed=3)
    with torch.no_grad():
        h._tower_rows(x, lv, h.cls_convs)
    torch.cuda.synchronize()
    s = torch.zeros(4, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.add_(1)
        with pytest.raises(RuntimeError, match="counter from the host"):
            h._tower_drop()
    graph.replay()
    torch.cuda.synchronize()
    assert float(s[0]) == 1 and h.tower_dropout_calls == 1


@pytest.mark.gpu
@pytest.mark.parametrize("rows", ["1", "0"])
def test_mask_branch_with_e4m3_operands(monkeypatch, rows):
    """the mask branch's 1x1 convolution as one e4m3 layer: what it was given and returned, against float64 of the quantised operands;
    the other outputs do not change, and every parameter of the branch gets its gradient"""
    monkeypatch.setenv("SIPMASK_TRAIN_ROWS", rows)
    from sipmask_amd import ops as P
    h = build_head(dict(type="SipMaskHead", num_classes=81, in_channels=256, stacked_convs=2, mask_lat_fp8=True)).cuda().train()
    with torch.no_grad():
        h.sip_mask_lat0.bias.copy_(0.1 * torch.randn(512, generator=torch.Generator().manual_seed(5)))
    g = torch.Generator().manual_seed(4)
    feats = [torch.randn(1, 256, a, b, generator=g).cuda() for a, b in [(16, 20), (8, 10), (4, 5), (2, 3), (1, 2)]]
    seen = []
    call = P.linear_fp8
    monkeypatch.setattr(P, "linear_fp8", lambda x, w, b, relu: seen.append((x, w, b, call(x, w, b, relu=relu))) or seen[-1][3])
    out = h(feats)
    (x, w, b, y), = seen
    assert x.shape[-1] == 768 and y.shape == x.shape[:-1] + (512,) and out[4].shape == (1, 32, 64, 80)
    xq = R.fp8_quantize(x.detach().reshape(-1, 768), 1)[2]
    wq = R.fp8_quantize(w.detach(), 128)[2]
    pre = xq @ wq.t() + b.detach().double()
    bound = R.matmul_bound(xq, wq, pre, 768, y.dtype, extra=2 * b.detach().double().abs())
    assert bool(((y.detach().reshape(-1, 512).double() - pre.clamp_min(0)).abs() <= bound).all())
    out[4].float().square().mean().backward()
    for p in (h.sip_mask_lat0.weight, h.sip_mask_lat0.bias, h.sip_mask_lat.weight, h.reg_convs[0].conv.weight):
        assert p.grad is not None and bool(torch.isfinite(p.grad).all()) and float(p.grad.abs().max()) > 0


@pytest.mark.gpu
def test_gradients_in_allreduce_buckets_match_plain_training():
    """both options on: gradients that live in all-reduce buckets (a census step through autograd's add, then written directly) equal those
    of a plain step with the same masks.  5e-3 relative, not bits: the deformable convolution's and the split-K convolutions' gradients are
    added with float atomics; a lost or doubled contribution would be of the gradient's own size."""
    from test_gpu_api import _synthetic_gt
    from sipmask_amd.dist_train import GradBucketer, HipSGD, head_train_step
    torch.manual_seed(9)
    h = build_head(dict(type="SipMaskHead", num_classes=81, in_channels=256, stacked_convs=3, center_sampling=True,
                        strides=[8, 16, 32, 64, 128], tower_dropout=0.1, tower_dropout_seed=5, mask_lat_fp8=True)).cuda()
    g = torch.Generator().manual_seed(5)
    feats = [torch.randn(2, 256, a, b, generator=g).cuda() for a, b in [(16, 20), (8, 10), (4, 5), (2, 3), (1, 2)]]
    gtb, gtl, gtm = _synthetic_gt(g, 2, 128, 160, 4)
    gtb, gtl = [b.cuda() for b in gtb], [l.cuda() for l in gtl]
    metas = [dict(img_shape=(128, 160, 3), pad_shape=(128, 160, 3), scale_factor=1.0) for _ in range(2)]
    opt = HipSGD(h.named_parameters(), lr=0.0, momentum=0.0, weight_decay=0.0)

    def step(**kw):
        h.tower_dropout_calls = 100
        return head_train_step(h, feats, gtb, gtl, gtm, metas, opt, **kw)
    plain_loss = step()
    plain = {n: (None if p.grad is None else p.grad.detach().clone()) for n, p in h.named_parameters()}
    opt.zero_grad()
    bucket = GradBucketer([p for p in h.parameters() if p.requires_grad], bucket_bytes=4 << 20)
    try:
        for turn in range(3):
            loss = step(bucketer=bucket)
            if turn:
                norm = h.cls_convs[0].norm
                assert not H.GRAD_SINK.census and {norm.weight.data_ptr(), norm.bias.data_ptr()} <= H.GRAD_SINK.written
            for k in plain_loss:
                assert abs(loss[k] - plain_loss[k]) <= 1e-4 * max(1.0, abs(plain_loss[k])), (turn, k)
            for n, p in h.named_parameters():
                if plain[n] is None:
                    assert float(p.grad.abs().max()) == 0.0, n
                else:
                    assert float((p.grad - plain[n]).norm() / (plain[n].norm() + 1e-20)) <= 5e-3, (turn, n)
    finally:
        bucket.remove()
