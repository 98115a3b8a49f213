"""Measured cases of the normalisation, dropout and 8-bit product operators.

group_norm_act   GroupNorm + activation (+ dropout) on channels-last tensors and on pyramid rows, forward and backward
dropout          inverted dropout whose mask is a function of (seed, offset, element), never stored; optional residual
linear_fp8       rows x weight^T in e4m3 with one power-of-two scale per block of 128, forward and backward
matmul_fp8       the product alone, on operands that are quantised already

Three computations of the same values: `run` with `own` false is the plain form in elementary torch operations, `run` with
`own` true calls the framework, `exact` follows the definitions in 64 bits.

Definitions
  group norm   per (image, level, group): m = mean x, v = mean (x - m)^2, t = (x - m) / sqrt(v + eps) * gamma_c + beta_c,
               y = act(t) * keep / (1 - p);   act in {none, relu, silu = t sigmoid(t), gelu = t Phi(t)}
  dropout      element i (row-major; channels fastest for channels-last tensors) takes 16-bit lane i % 8 of the block
               Philox-4x32-10(counter = (i / 8, offset), key = seed), lane j = bits 16 (j % 2) .. of word j / 2;
               keep = lane >= round(65536 p), kept values are multiplied by 65536 / (65536 - round(65536 p))
  fp8 block    scale = the smallest power of two (not below 2^-127) with max |x| / scale <= 448 over the block, 1 for a block
               of zeros; code = x / scale rounded to e4m3 (nearest, ties to even).  Activations and gradients: 1 x 128 blocks
               along the summed axis; weights: 128 x 128
  linear_fp8   y = q(x) q(w)^T + bias;  dx = q(dy) q(w);  dw = q(dy^T) q(x^T)^T;  dbias = column sums of dy
"""
import math

import numpy as np
import torch

own = False

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}
PYRAMID = ((100, 168), (50, 84), (25, 42), (13, 21), (7, 11))      # the head's five levels of an 800 x 1344 canvas


# ---------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # the coarsest head level of one image: a launch-bound call
        dict(name="gn_p7_one_image", op="gn", dtype="f16", batch=1, channels=256, groups=32, h=7, w=11, pyramid=False,
             act="silu", p=0.0, train=False),
        # the training towers of the head: five levels of four 800 x 1344 images, ReLU, with dropout
        dict(name="gn_tower_train", op="gn", dtype="bf16", batch=4, channels=256, groups=32, h=0, w=0, pyramid=True,
             act="relu", p=0.1, train=True),
        # a map whose channel count is no multiple of a vector, float32
        dict(name="gn_odd_train", op="gn", dtype="f32", batch=2, channels=60, groups=12, h=33, w=47, pyramid=False,
             act="gelu", p=0.0, train=True),
        # stride-4 maps of a batch of 544 x 544 images
        dict(name="gn_stride4_batch16", op="gn", dtype="bf16", batch=16, channels=256, groups=32, h=136, w=136,
             pyramid=False, act="silu", p=0.0, train=False),
        # one image's coarsest level through a residual branch
        dict(name="dropout_small_residual", op="dropout", dtype="f16", rows=77, cols=256, p=0.1, residual=True, train=False),
        # an odd row width, forward and backward, float32
        dict(name="dropout_odd_train", op="dropout", dtype="f32", rows=4099, cols=93, p=0.25, residual=True, train=True),
        # the stride-4 rows of four 800 x 1344 images, forward and backward
        dict(name="dropout_stride4_train", op="dropout", dtype="bf16", rows=268800, cols=256, p=0.5, residual=False,
             train=True),
        # a handful of detections through a wide layer: the weight is what has to be read
        dict(name="linear_few_rows", op="linear", dtype="bf16", m=7, k=2048, n=512, bias=True, relu=False, train=False),
        # layer3's 1x1 conv of four 800 x 1344 images, bias and ReLU fused
        dict(name="linear_layer3_conv1", op="linear", dtype="bf16", m=16800, k=1024, n=256, bias=True, relu=True,
             train=False),
        # the mask branch's 1x1 conv, forward and backward
        dict(name="linear_lat0_train", op="linear", dtype="bf16", m=67200, k=768, n=512, bias=True, relu=False, train=True),
        # odd sizes everywhere, float32 result
        dict(name="matmul_odd", op="matmul", dtype="f32", m=977, k=1131, n=333),
        # a large product
        dict(name="matmul_large", op="matmul", dtype="bf16", m=8192, k=4096, n=4096),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["gn", "gn", "dropout", "linear", "linear", "matmul"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "gn":
        cpg = rng.choice([1, 2, 3, 4, 5, 7, 8, 8, 8, 16, 16, 24, 32, 64])
        groups = rng.choice([1, 2, 3, 8, 16, 32, 32, 32])
        train = rng.random() < 0.5
        pyramid = rng.random() < 0.25
        batch = _log(rng, 1, 16)
        if pyramid:
            h = w = 0
            batch = 1 + batch % 4
        else:
            top = 40_000_000 if not train else 20_000_000
            hw = _log(rng, 1, max(1, min(136 * 136, top // (batch * cpg * groups))))
            h = _log(rng, 1, hw)
            w = max(1, hw // h)
        return dict(op="gn", dtype=dtype, batch=batch, channels=cpg * groups, groups=groups, h=h, w=w, pyramid=pyramid,
                    act=rng.choice(["none", "relu", "silu", "gelu"]), p=rng.choice([0.0, 0.0, 0.1, 0.5]), train=train)
    if op == "dropout":
        cols = _log(rng, 1, 2048)
        return dict(op="dropout", dtype=dtype, rows=_log(rng, 1, max(1, 30_000_000 // cols)), cols=cols,
                    p=rng.choice([0.05, 0.1, 0.25, 0.5, 0.9]), residual=rng.random() < 0.5, train=rng.random() < 0.5)
    if op == "linear":
        k, n = _log(rng, 16, 2304), _log(rng, 8, 2048)
        return dict(op="linear", dtype=dtype, m=_log(rng, 1, min(67200, 26_000_000_000 // (k * n), 50_000_000 // max(k, n))),
                    k=k, n=n, bias=rng.random() < 0.7, relu=False, train=rng.random() < 0.5)
    m, n, k = _log(rng, 1, 8192), _log(rng, 1, 4096), _log(rng, 1, 4096)
    return dict(op="matmul", dtype=dtype, m=m, k=k, n=n)


def _sizes(case):
    return PYRAMID if case["pyramid"] else ((case["h"], case["w"]),)


def work(case):
    e = BYTES[case["dtype"]]
    if case["op"] == "gn":
        n = case["batch"] * case["channels"] * sum(h * w for h, w in _sizes(case))
        par = 4 * case["channels"]
        if case["train"]:       # x, dy in; y, dx out; the two parameters in, their gradients out
            return {"bytes": 4 * n * e + 4 * par, "flops": 24 * n}
        return {"bytes": 2 * n * e + 2 * par, "flops": 8 * n}
    if case["op"] == "dropout":
        n = case["rows"] * case["cols"]
        tensors = (3 if case["residual"] else 2) + (2 if case["train"] else 0)
        return {"bytes": tensors * n * e, "flops": 2 * n * (2 if case["train"] else 1)}
    m, k, n = case["m"], case["k"], case["n"]
    if case["op"] == "matmul":
        kb = -(-k // 128)
        return {"bytes": m * k + n * k + m * kb + -(-n // 128) * kb + m * n * e, "flops": 2 * m * n * k}
    if case["train"]:           # x, dy in; y, dx out; the weight in, its gradient out
        return {"bytes": 2 * m * k * e + 2 * m * n * e + 8 * n * k, "flops": 6 * m * n * k}
    return {"bytes": m * k * e + m * n * e + n * k, "flops": 2 * m * n * k}


# --------------------------------------------------------------------------------------------------------------- inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _rand(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _inputs(case, seed):
    """the tensors of a case, from the seed alone"""
    g, dt = _gen(seed), DT[case["dtype"]]
    if case["op"] == "gn":
        c = case["channels"]
        rows = case["batch"] * sum(h * w for h, w in _sizes(case))
        # a conv's output: a scale and an offset of its own in every channel
        amp, off = 0.5 + _rand(g, c).abs(), 0.7 * _rand(g, c)
        x = (_rand(g, rows, c) * amp + off).to(dt)
        s = dict(x=x, gamma=1.0 + 0.2 * _rand(g, c), beta=0.2 * _rand(g, c))
        if case["train"]:
            s["dy"] = (1e-2 * _rand(g, rows, c)).to(dt)
        return s
    if case["op"] == "dropout":
        r, c = case["rows"], case["cols"]
        s = dict(x=_rand(g, r, c).to(dt), residual=_rand(g, r, c).to(dt) if case["residual"] else None)
        if case["train"]:
            s["dy"] = (1e-2 * _rand(g, r, c)).to(dt)
        return s
    m, k, n = case["m"], case["k"], case["n"]
    # activations behind a ReLU with channels of unlike size; weights of a trained layer
    x = (torch.relu(_rand(g, m, k)) * torch.exp(0.8 * _rand(g, k)))
    w = _rand(g, n, k) * (1.0 / math.sqrt(k)) * torch.exp(0.3 * _rand(g, n, 1))
    if case["op"] == "matmul":
        return dict(x=x.to(torch.bfloat16), w=w)
    s = dict(x=x.to(dt), w=w, bias=0.1 * _rand(g, n) if case["bias"] else None)
    if case["train"]:
        s["dy"] = (1e-3 * _rand(g, m, n) * torch.exp(0.5 * _rand(g, m, 1))).to(dt)
    return s


def _rng_of(seed):
    """(seed, offset) of a case's dropout"""
    return (0x9E3779B97F4A7C15 * (seed + 1)) & 0x7FFFFFFFFFFFFFFF, (seed * 2654435761 + 12345) & 0xFFFFFFFF


def prepare(case, seed):
    s = dict(case=case, seed=seed, **_inputs(case, seed))
    if case["op"] == "gn":
        if case["pyramid"]:
            if own:
                from sipmask_amd.hip_ops import Levels
                s["lv"] = Levels(case["batch"], PYRAMID)
        else:
            shape = (case["batch"], case["h"], case["w"], case["channels"])
            s["x"] = s["x"].view(shape).permute(0, 3, 1, 2)
            if case["train"]:
                s["dy"] = s["dy"].view(shape).permute(0, 3, 1, 2)
        leaves = ("x", "gamma", "beta")
    elif case["op"] == "dropout":
        leaves = ("x", "residual")
    elif case["op"] == "linear":
        leaves = ("x", "w", "bias")
        if not case["train"]:                 # a serving program lays its weight out once
            if own:
                from sipmask_amd import ops
                s["wq"] = ops.quantize_fp8(s["w"], block_rows=128)
            else:
                s["wq"] = _plain_quantize(s["w"], 128)
    else:
        if own:
            from sipmask_amd import ops
            s["a"], s["b"] = ops.quantize_fp8(s["x"]), ops.quantize_fp8(s["w"], block_rows=128)
        else:
            s["a"], s["b"] = _plain_quantize(s["x"], 1), _plain_quantize(s["w"], 128)
        del s["x"], s["w"]
        leaves = ()
    if own and case.get("train"):
        for k in leaves:
            if s[k] is not None:
                s[k].requires_grad_(True)
    return s


# ----------------------------------------------------------------------------------------------------------- plain form
def _plain_philox(n, seed, offset, device):
    """16-bit draws of elements 0 .. n-1: [n] int64"""
    i = torch.arange((n + 7) // 8, dtype=torch.int64, device=device)
    mask = 0xFFFFFFFF
    c = [i & mask, i >> 32, torch.full_like(i, offset & mask), torch.full_like(i, (offset >> 32) & mask)]
    k0, k1 = seed & mask, (seed >> 32) & mask
    for _ in range(10):
        p0, p1 = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57       # the low 64 bits are right whatever the sign
        c = [((p1 >> 32) & mask) ^ c[1] ^ k0, p1 & mask, ((p0 >> 32) & mask) ^ c[3] ^ k1, p0 & mask]
        k0, k1 = (k0 + 0x9E3779B9) & mask, (k1 + 0xBB67AE85) & mask
    lanes = torch.stack([w for v in c for w in (v & 0xFFFF, v >> 16)], 1)
    return lanes.reshape(-1)[:n]


def _plain_keep(n, p, seed, offset, device):
    """(keep mask [n], factor of the kept elements)"""
    thr = int(round(p * 65536))
    keep = _plain_philox(n, seed, offset, device) >= thr
    return keep, (65536.0 / (65536 - thr) if thr < 65536 else 0.0)


def _plain_act(t, act):
    if act == "relu":
        return torch.where(t < 0, torch.zeros_like(t), t)
    if act == "silu":
        return t / (1 + torch.exp(-t))
    if act == "gelu":
        return t * 0.5 * (1 + torch.erf(t * math.sqrt(0.5)))
    return t


def _plain_act_grad(t, t64, act):
    if act == "relu":                                # the border decides a whole gradient: it is found in 64 bits
        return (t64 > 0).to(t.dtype)
    if act == "silu":
        s = 1 / (1 + torch.exp(-t))
        return s * (1 + t * (1 - s))
    if act == "gelu":
        return 0.5 * (1 + torch.erf(t * math.sqrt(0.5))) + t * torch.exp(-0.5 * t * t) * (1 / math.sqrt(2 * math.pi))
    return torch.ones_like(t)


def _plain_gn(s):
    case = s["case"]
    nchw = not case["pyramid"]
    flat = lambda t: t.permute(0, 2, 3, 1).reshape(-1, case["channels"]) if nchw else t
    x, dy = flat(s["x"]), flat(s["dy"]) if case["train"] else None
    b, c, gr, eps = case["batch"], case["channels"], case["groups"], 1e-5
    keep = None
    if case["p"] > 0:
        keep, fac = _plain_keep(x.numel(), case["p"], *_rng_of(s["seed"]), x.device)
        keep = keep.view(x.shape).float() * fac
    ys, dxs, dgamma, dbeta, r0 = [], [], 0, 0, 0
    for h, w in _sizes(case):
        r1 = r0 + b * h * w
        blk = x[r0:r1].float().view(b, h * w, gr, c // gr)
        cnt = h * w * (c // gr)
        mean = blk.sum((1, 3), keepdim=True, dtype=torch.float64) / cnt
        dev = blk.double() - mean
        var = (dev * dev).sum((1, 3), keepdim=True) / cnt
        rstd = 1 / torch.sqrt(var + eps)
        xh64 = dev * rstd
        xh = xh64.float()
        g4, b4 = s["gamma"].view(gr, c // gr), s["beta"].view(gr, c // gr)
        t = xh * g4 + b4
        y = _plain_act(t, case["act"])
        k4 = None if keep is None else keep[r0:r1].view(blk.shape)
        if k4 is not None:
            y = y * k4
        ys.append(y.reshape(-1, c).to(x.dtype))
        if case["train"]:
            d = dy[r0:r1].float().view(blk.shape)
            if k4 is not None:
                d = d * k4
            t64 = xh64 * g4 + b4 if case["act"] == "relu" else None
            d = d * _plain_act_grad(t, t64, case["act"])
            dgamma = dgamma + (d * xh).sum((0, 1)).reshape(-1)
            dbeta = dbeta + d.sum((0, 1)).reshape(-1)
            dg = d * g4
            m1 = dg.sum((1, 3), keepdim=True) / cnt
            m2 = (dg * xh).sum((1, 3), keepdim=True) / cnt
            dxs.append((rstd.float() * (dg - m1 - xh * m2)).reshape(-1, c).to(x.dtype))
        r0 = r1
    back = lambda ts: (torch.cat(ts) if not nchw else
                       ts[0].view(b, case["h"], case["w"], c).permute(0, 3, 1, 2))
    if not case["train"]:
        return back(ys)
    return back(ys), back(dxs), dgamma, dbeta


def _plain_dropout(s):
    case, x = s["case"], s["x"]
    keep, fac = _plain_keep(x.numel(), case["p"], *_rng_of(s["seed"]), x.device)
    keep = keep.view(x.shape)
    zero = torch.zeros((), device=x.device)
    y = torch.where(keep, x.float() * fac, zero)
    if case["residual"]:
        y = y + s["residual"].float()
    y = y.to(x.dtype)
    if not case["train"]:
        return y
    dx = torch.where(keep, s["dy"].float() * fac, zero).to(x.dtype)
    return (y, dx, s["dy"]) if case["residual"] else (y, dx)


def _pow2(e):
    """2^e in float64, exactly (torch's ldexp multiplies by a pow() that may be off by an ulp), e a whole number"""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _plain_quantize(x, block_rows):
    """(e4m3 codes of x / scale, scale spread over the elements): codes float8 [rows, cols], scale f32 [row blocks, blocks]"""
    r, c = x.shape
    nr, nc = -(-r // block_rows), -(-c // 128)
    pad = torch.zeros(nr * block_rows, nc * 128, device=x.device)
    pad[:r, :c] = x.float()
    blk = pad.view(nr, block_rows, nc, 128)
    amax = blk.abs().amax((1, 3))
    m, e = torch.frexp(amax)                                # amax = m 2^e, 0.5 <= m < 1; 448 = 0.875 * 2^9
    e = torch.where(m > 0.875, e - 8, e - 9).clamp(-127, 127)
    e = torch.where(amax == 0, torch.zeros_like(e), e)
    scale = _pow2(e.double()).float()
    q = (blk / scale[:, None, :, None]).reshape(nr * block_rows, nc * 128)[:r, :c].to(torch.float8_e4m3fn)
    return q, scale, block_rows


def _plain_values(qs):
    q, scale, block_rows = qs
    r, c = q.shape
    full = scale.repeat_interleave(block_rows, 0)[:r].repeat_interleave(128, 1)[:, :c]
    return q.float() * full


def _plain_linear(s):
    case, x = s["case"], s["x"]
    wv = _plain_values(_plain_quantize(s["w"], 128) if case["train"] else s["wq"])
    y = _plain_values(_plain_quantize(x, 1)) @ wv.t()
    if case["bias"]:
        y = y + s["bias"]
    if case["relu"]:
        y = torch.where(y < 0, torch.zeros_like(y), y)
    y = y.to(x.dtype)
    if not case["train"]:
        return y
    dy = s["dy"]
    dx = (_plain_values(_plain_quantize(dy, 1)) @ wv).to(x.dtype)
    dw = _plain_values(_plain_quantize(dy.t(), 1)) @ _plain_values(_plain_quantize(x.t(), 1)).t()
    if not case["bias"]:
        return y, dx, dw
    return y, dx, dw, dy.sum(0, dtype=torch.float64).float()


def _plain_matmul(s):
    return (_plain_values(s["a"]) @ _plain_values(s["b"]).t()).to(DT[s["case"]["dtype"]])


# ------------------------------------------------------------------------------------------------------ the framework's
def _own(s):
    from sipmask_amd import ops, ops_rows
    case = s["case"]
    if case["op"] == "gn":
        seed, offset = _rng_of(s["seed"])
        if case["pyramid"]:
            y = ops_rows.gn_act_rows(s["x"], s["lv"], s["gamma"], s["beta"], case["groups"], 1e-5, case["act"],
                                     dropout_p=case["p"], seed=seed, offset=offset)
        else:
            y = ops.group_norm_act(s["x"], s["gamma"], s["beta"], case["groups"], 1e-5, case["act"],
                                   dropout_p=case["p"], seed=seed, offset=offset)
        if not case["train"]:
            return y
        return (y.detach(),) + torch.autograd.grad(y, [s["x"], s["gamma"], s["beta"]], s["dy"])
    if case["op"] == "dropout":
        seed, offset = _rng_of(s["seed"])
        y = ops.dropout(s["x"], case["p"], seed, offset, residual=s["residual"])
        if not case["train"]:
            return y
        return (y.detach(),) + torch.autograd.grad(y, [s["x"]] + ([s["residual"]] if case["residual"] else []), s["dy"])
    if case["op"] == "linear":
        if not case["train"]:
            return ops.linear_fp8(s["x"], None, s["bias"], relu=case["relu"], weight_q=s["wq"])
        y = ops.linear_fp8(s["x"], s["w"], s["bias"], relu=case["relu"])
        return (y.detach(),) + torch.autograd.grad(y, [s["x"], s["w"]] + ([s["bias"]] if case["bias"] else []), s["dy"])
    return ops.matmul_fp8(s["a"], s["b"], out_dtype=DT[case["dtype"]])


def run(state):
    if own:
        return _own(state)
    return {"gn": _plain_gn, "dropout": _plain_dropout, "linear": _plain_linear, "matmul": _plain_matmul}[
        state["case"]["op"]](state)


# ---------------------------------------------------------------------------------------- the definitions in 64 bits
def _exact_keep(shape, p, seed, offset):
    """float64 factors 0 or 1 / (1 - p') of a dropout, on the host in blocks"""
    n = int(np.prod(shape))
    thr = int(round(p * 65536))
    u = np.uint64
    lo = u(0xFFFFFFFF)
    out = np.empty(n, dtype=np.uint16)
    step = 1 << 22
    for b0 in range(0, -(-n // 8), step):
        ctr = np.arange(b0, min(b0 + step, -(-n // 8)), dtype=np.uint64)
        x0, x1 = ctr & lo, ctr >> u(32)
        x2, x3 = np.full_like(ctr, offset & 0xFFFFFFFF), np.full_like(ctr, offset >> 32)
        ka, kb = seed & 0xFFFFFFFF, seed >> 32
        for _ in range(10):
            pa, pb = x0 * u(0xD2511F53), x2 * u(0xCD9E8D57)
            x0, x1, x2, x3 = (pb >> u(32)) ^ x1 ^ u(ka), pb & lo, (pa >> u(32)) ^ x3 ^ u(kb), pa & lo
            ka, kb = (ka + 0x9E3779B9) % 2 ** 32, (kb + 0xBB67AE85) % 2 ** 32
        words = np.stack([x0, x1, x2, x3], 1).astype("<u4")
        part = words.view("<u2").reshape(-1)
        out[8 * b0:8 * b0 + part.size] = part[:n - 8 * b0]
    keep = torch.from_numpy((out >= thr) if thr < 65536 else np.zeros(n, bool)).cuda().view(shape)
    return keep.double() * (65536.0 / max(65536 - thr, 1))


def _exact_fp8(x, block_rows):
    """the values that the codes of x stand for, float64"""
    v = x.double()
    r, c = v.shape
    out = torch.empty_like(v)
    # one scale per block, from the block's largest magnitude
    a = v.abs()
    a = torch.nn.functional.pad(a, (0, -c % 128, 0, -r % block_rows))
    top = a.view(a.shape[0] // block_rows, block_rows, a.shape[1] // 128, 128).amax(3).amax(1)
    ex = torch.ceil(torch.log2(torch.where(top > 0, top, torch.full_like(top, 448.0)) / 448.0))
    sc = (ex.long() + 1023).bitwise_left_shift(52).view(torch.float64)                          # 2^ex from its bits
    sc = torch.where(top / sc > 448, sc * 2, torch.where(top / (sc / 2) <= 448, sc / 2, sc))    # log2's own rounding
    sc = torch.where(top > 0, sc, torch.ones_like(sc)).clamp_min(2.0 ** -127)
    del a
    for i in range(sc.shape[0] if block_rows > 1 else 1):
        rows = slice(i * block_rows, min((i + 1) * block_rows, r)) if block_rows > 1 else slice(0, r)
        srow = (sc[i:i + 1] if block_rows > 1 else sc).repeat_interleave(128, 1)[:, :c]
        z = v[rows] / srow
        _, e = torch.frexp(z)
        quantum = ((e - 1).clamp_min(-6).long() + (1023 - 3)).bitwise_left_shift(52).view(torch.float64)    # 3 bits behind the first
        out[rows] = torch.round(z / quantum) * quantum * srow
    return out


def _exact_gn(case, s, seed):
    x = s["x"].double()
    gamma, beta = s["gamma"].double(), s["beta"].double()
    b, c, gr = case["batch"], case["channels"], case["groups"]
    fac = _exact_keep(tuple(x.shape), case["p"], *_rng_of(seed)) if case["p"] > 0 else torch.ones((), device=x.device,
                                                                                                  dtype=torch.float64)
    y, dx = torch.empty_like(x), torch.empty_like(x)
    ga, be = torch.zeros_like(gamma), torch.zeros_like(beta)
    r = 0
    for h, w in _sizes(case):
        for _ in range(b):
            rows = slice(r, r + h * w)
            r += h * w
            z = x[rows].reshape(h * w, gr, c // gr)
            mu = z.mean((0, 2), keepdim=True)
            sd = ((z - mu).square().mean((0, 2), keepdim=True) + 1e-5).sqrt()
            n = ((z - mu) / sd).reshape(h * w, c)
            t = n * gamma + beta
            f = fac if fac.dim() == 0 else fac[rows]
            if case["act"] == "relu":
                a, da = t.clamp_min(0), (t > 0).double()
            elif case["act"] == "silu":
                sg = torch.sigmoid(t)
                a, da = t * sg, sg + t * sg * (1 - sg)
            elif case["act"] == "gelu":
                cdf = 0.5 * torch.erfc(-t / math.sqrt(2.0))
                a, da = t * cdf, cdf + t * torch.exp(-t * t / 2) / math.sqrt(2 * math.pi)
            else:
                a, da = t, torch.ones_like(t)
            y[rows] = a * f
            if case["train"]:
                d = s["dy"][rows].double() * f * da
                ga += (d * n).sum(0)
                be += d.sum(0)
                u = (d * gamma).reshape(h * w, gr, c // gr)
                nn = n.reshape(h * w, gr, c // gr)
                dx[rows] = ((u - u.mean((0, 2), keepdim=True) - nn * (u * nn).mean((0, 2), keepdim=True)) / sd).reshape(h * w, c)
    shape = (lambda t: t) if case["pyramid"] else (lambda t: t.view(b, case["h"], case["w"], c).permute(0, 3, 1, 2))
    return (shape(y), shape(dx), ga, be) if case["train"] else shape(y)


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "gn":
        return _exact_gn(case, s, seed)
    if case["op"] == "dropout":
        f = _exact_keep(tuple(s["x"].shape), case["p"], *_rng_of(seed))
        y = s["x"].double() * f
        if case["residual"]:
            y = y + s["residual"].double()
        if not case["train"]:
            return y
        return (y, s["dy"].double() * f) + ((s["dy"].double(),) if case["residual"] else ())
    w = _exact_fp8(s["w"], 128)
    y = torch.matmul(_exact_fp8(s["x"], 1), w.t().contiguous())
    if case["op"] == "matmul":
        return y
    if case["bias"]:
        y = y + s["bias"].double()
    if case["relu"]:
        y = y.clamp_min(0)
    if not case["train"]:
        return y
    dy = s["dy"]
    out = (y, torch.matmul(_exact_fp8(dy, 1), w),
           torch.matmul(_exact_fp8(dy.t().contiguous(), 1), _exact_fp8(s["x"].t().contiguous(), 1).t().contiguous()))
    return out + ((dy.double().sum(0),) if case["bias"] else ())
