"""Float64 restatement of the residual-block operators (GroupNorm + activation, counter-based dropout, e4m3 blocks), on the CPU or
the GPU, and the error bounds their f32 kernels are held to.  u = half a step of the output type; every bound is u |value| plus
2^-24 times the number of f32 roundings on the path, weighted with the magnitudes that were rounded."""
import math

import numpy as np
import torch

E = 2.0 ** -24                                   # half a step of f32


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """half of the smallest subnormal: what a value near 0 may lose"""
    return {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -149}[dtype]


# ------------------------------------------------------------------------------------------------ dropout
def philox_block(counter, key):
    """Philox-4x32-10 on Python ints: counter = 4 words, key = 2 words"""
    c, k = list(counter), list(key)
    for _ in range(10):
        a, b = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [(b >> 32) ^ c[1] ^ k[0], b & 0xFFFFFFFF, (a >> 32) ^ c[3] ^ k[1], a & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def draws(first, n, seed, offset):
    """16-bit draws of elements first .. first + n - 1 (numpy)"""
    seed, offset = seed & (2 ** 64 - 1), offset & (2 ** 64 - 1)
    b0, b1 = first // 8, (first + n + 7) // 8
    ctr = np.arange(b1 - b0, dtype=np.uint64) + np.uint64(b0)
    lo = np.uint64(0xFFFFFFFF)
    s32 = np.uint64(32)
    x = [ctr & lo, ctr >> s32, np.full_like(ctr, offset & 0xFFFFFFFF), np.full_like(ctr, offset >> 32)]
    k0, k1 = seed & 0xFFFFFFFF, seed >> 32
    for _ in range(10):
        a, b = x[0] * np.uint64(0xD2511F53), x[2] * np.uint64(0xCD9E8D57)
        x = [(b >> s32) ^ x[1] ^ np.uint64(k0), b & lo, (a >> s32) ^ x[3] ^ np.uint64(k1), a & lo]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    w = np.stack(x, 1).astype("<u4").view("<u2").reshape(-1)
    return w[first - 8 * b0:][:n]


def keep_factor(shape, p, seed, offset, first=0):
    """float64 tensor of 0 or 1 / (1 - p')"""
    thr = int(round(p * 65536))
    n = int(np.prod(shape))
    k = draws(first, n, seed, offset).astype(np.int64) >= thr
    return torch.from_numpy(k.astype(np.float64)).reshape(shape) * (65536.0 / max(65536 - thr, 1))


# ------------------------------------------------------------------------------------------------ GroupNorm + activation
def act(t, name):
    if name == "relu":
        return torch.where(t < 0, torch.zeros_like(t), t)
    if name == "silu":
        return t * torch.sigmoid(t)
    if name == "gelu":
        return 0.5 * t * torch.erfc(-t / math.sqrt(2.0))
    return t


def act_grad(t, name):
    if name == "relu":
        return torch.where(t <= 0, torch.zeros_like(t), torch.ones_like(t))
    if name == "silu":
        s = torch.sigmoid(t)
        return s * (1 + t * (1 - s))
    if name == "gelu":
        return 0.5 * torch.erfc(-t / math.sqrt(2.0)) + t * torch.exp(-0.5 * t * t) / math.sqrt(2 * math.pi)
    return torch.ones_like(t)


class GroupNormAct:
    """rows [batch * hw, C] of one level, everything in float64"""

    def __init__(self, x, batch, groups, gamma, beta, eps, name, fac=None):
        rows, c = x.shape
        self.x, self.batch, self.groups, self.name = x.double(), batch, groups, name
        self.gamma = torch.ones(c, dtype=torch.float64, device=x.device) if gamma is None else gamma.double()
        self.beta = torch.zeros(c, dtype=torch.float64, device=x.device) if beta is None else beta.double()
        self.fac = torch.ones((), dtype=torch.float64, device=x.device) if fac is None else fac.to(x.device)
        z = self._g(self.x)
        mu = z.mean((1, 3), keepdim=True)
        self.rstd = 1 / torch.sqrt((z - mu).square().mean((1, 3), keepdim=True) + eps)
        self.xh = self._r((z - mu) * self.rstd)
        self.t = self.xh * self.gamma + self.beta
        self.y = act(self.t, name) * self.fac

    def _g(self, t):
        return t.reshape(self.batch, -1, self.groups, t.shape[1] // self.groups)

    def _r(self, t):
        return t.reshape(self.x.shape)

    def y_bound(self, dtype):
        """x - m: the difference against the mean's high part, the low part, the product with rstd * gamma (itself rounded) and the
        sum with beta: 4 roundings of |xh gamma|, 1 of |t|; the activations add at most 6 roundings of their result and have slopes
        of at most 1.13; dropout one more"""
        a = (self.xh * self.gamma).abs()
        return half_step(dtype) * self.y.abs() + E * (8 * self.y.abs() + 1.13 * self.fac * (5 * a + 2 * self.t.abs() + self.beta.abs())) + \
            tiny(dtype)

    def backward(self, dy):
        self.dy = dy.double()
        self.da = act_grad(self.t, self.name)
        d = self.dy * self.fac * self.da
        self.d = d
        self.dgamma, self.dbeta = (d * self.xh).sum(0), d.sum(0)
        u = self._g(d * self.gamma)
        xh = self._g(self.xh)
        self.m1, self.m2 = u.mean((1, 3), keepdim=True), (u * xh).mean((1, 3), keepdim=True)
        self.dx = self._r(self.rstd * (u - self.m1 - xh * self.m2))
        return self.dx

    def _d_err(self):
        """error of d in units of 2^-24: t is off by 6 roundings (see y_bound), |act''| <= 1.2; act' itself by 10 roundings of terms of
        at most 1.3; two products.  The ReLU's gate is exact (taken in f64 at the border)."""
        if self.name in ("relu", "none", None):
            return 2 * self.d.abs()
        terr = 6 * ((self.xh * self.gamma).abs() + self.beta.abs())
        return self.dy.abs() * self.fac * (1.2 * terr + 13 + 2 * self.da.abs())

    def bounds(self, dtype, run=256):
        """(dx, dgamma, dbeta).  `run`: f32 additions in a row before the sums go on in f64 (rows of a thread + the tree)"""
        de = self._d_err()
        xe = 4 * self.xh.abs()
        g = self.gamma.abs()
        s1 = self._g((de + run * self.d.abs()) * g).mean((1, 3), keepdim=True)
        s2 = self._g((de + (run + 5) * self.d.abs()) * g * self.xh.abs()).mean((1, 3), keepdim=True)
        one = lambda t: self._r(t.expand(self._g(self.x).shape))
        m1, m2, rs = one(self.m1.abs()), one(self.m2.abs()), one(self.rstd)
        dx = half_step(dtype) * self.dx.abs() + tiny(dtype) + E * rs * (
            (de + 3 * self.d.abs()) * g + one(s1) + 3 * m1 + one(s2) * self.xh.abs() + (xe + 4 * self.xh.abs()) * m2 + 2 * (
                (self.d * self.gamma).abs() + m1 + self.xh.abs() * m2))
        dg = E * ((de * self.xh.abs() + (run + 6) * (self.d * self.xh).abs()).sum(0) + 2 * self.dgamma.abs())
        db = E * ((de + run * self.d.abs()).sum(0) + 2 * self.dbeta.abs())
        return dx, dg, db


# ------------------------------------------------------------------------------------------------ e4m3 blocks
def fp8_quantize(x, block_rows):
    """-> (codes uint8 [rows, cols], scale bytes int64 [row blocks, col blocks], values float64 [rows, cols]); NaN / Inf -> 0x7f"""
    v = x.double()
    r, c = v.shape
    fin = torch.isfinite(v)
    a = torch.where(fin, v.abs(), torch.zeros_like(v))
    a = torch.nn.functional.pad(a, (0, -c % 128, 0, -r % block_rows))
    top = a.view(a.shape[0] // block_rows, block_rows, a.shape[1] // 128, 128).amax(3).amax(1)
    m, e = torch.frexp(top)                      # top = m 2^e, 1/2 <= m < 1, and 448 = 7/8 2^9
    e = torch.where(m > 0.875, e - 8, e - 9).clamp_min(-127)
    e = torch.where(top == 0, torch.zeros_like(e), e).long()
    byte = e + 127
    sc = pow2(e).repeat_interleave(block_rows, 0)[:r].repeat_interleave(128, 1)[:, :c]
    z = torch.where(fin, v, torch.zeros_like(v)) / sc
    _, ze = torch.frexp(z)
    step = pow2((ze - 1).clamp_min(-6).long() - 3)
    n = torch.round(z / step)                    # half to even
    q = n * step
    qa = q.abs()
    _, qe = torch.frexp(qa)
    exp = (qe - 1).clamp_min(-6).long()
    mant = (qa / pow2(exp - 3)).long()           # 0 .. 15; < 8 only for subnormals
    code = torch.where(mant >= 8, ((exp + 7) << 3) | (mant - 8), mant)
    code = torch.where((v < 0) | ((v == 0) & (torch.signbit(v))), code + 128, code)
    code = torch.where(fin, code, torch.full_like(code, 0x7F))
    return code.to(torch.uint8), byte, torch.where(fin, q * sc, torch.full_like(q, math.nan))


def pow2(e):
    return ((e + 1023) << 52).view(torch.float64)


def matmul_bound(av, bv, y, k, dtype, splits=64, extra=0.0):
    """f32 accumulation of k products: exact products, a product passes at most 16 additions inside an instruction, k / 16 between them and
    one per K split; 2^-23 each (the matrix unit's own additions may truncate)"""
    mag = av.abs() @ bv.abs().t()
    return half_step(dtype) * y.abs() + tiny(dtype) + 2 * E * ((k / 16 + 18 + splits) * mag + extra)
