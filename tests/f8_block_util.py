"""Plain forms in 64 bits of the operators around the 8-bit products, and their error
bounds from counts of float32 roundings (U = 2^-24 each, relative)."""
import math

import numpy as np
import torch

from f8_util import F32, F64, rounding

U = 2.0 ** -24
ACTS = (None, "relu", "relu2", "silu", "gelu", "gelu_tanh")
# A row's sum of D <= 2^15 terms in float32: at most 32 of a thread one after the other, four steps over
# a DPP row, two over a wave, 15 over the waves, 53 in all; the division by D and a few products beside it.
SUM = 64


# ---- Philox4x32-10 on Python's integers.

def philox(counter, key):
    """Four 32-bit words of a counter of four and a key of two."""
    x, k = list(counter), list(key)
    for _ in range(10):
        a, b = 0xD2511F53 * x[0], 0xCD9E8D57 * x[2]
        x = [(b >> 32) ^ x[1] ^ k[0], b & 0xFFFFFFFF, (a >> 32) ^ x[3] ^ k[1], a & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return x


def kept(seed, offset, drop, M, D):
    """Which elements of an M x D matrix stay, by numpy's unsigned integers."""
    u = np.uint64
    low, half = u(0xFFFFFFFF), u(32)
    seed, offset = seed % 2 ** 64, offset % 2 ** 64
    c = np.arange(M * -(-D // 8), dtype=u)
    x = [c & low, c >> half, u(offset) & low, u(offset) >> half]
    k = [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(10):
        a, b = u(0xD2511F53) * x[0], u(0xCD9E8D57) * x[2]
        x = [(b >> half) ^ x[1] ^ u(k[0]), b & low, (a >> half) ^ x[3] ^ u(k[1]), a & low]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    bits = np.stack([w >> s & u(0xFFFF) for w in x for s in (u(0), u(16))], -1)
    return torch.from_numpy(bits.reshape(M, -1)[:, :D].astype(np.int32)) >= drop


def factors(seed, offset, p, M, D):
    """What drop() multiplies by, in 64 bits."""
    drop = round(p * 65536)
    if drop == 0:
        return torch.ones(M, D, dtype=F64)
    return kept(seed, offset, drop, M, D).to(F64) * (65536 / (65536 - drop))


# ---- Activations: value, slope, and bounds of their float32 errors.

def _phi(h):
    return torch.exp(-0.5 * h * h) / math.sqrt(2 * math.pi)


def _cdf(h):
    return 0.5 * torch.special.erfc(-h * math.sqrt(0.5))


def _tanh_arg(h):
    c = 2 * math.sqrt(2 / math.pi)
    return c * (h + 0.044715 * h ** 3), c * (1 + 3 * 0.044715 * h * h)


def act(h, name):
    if name in ("relu", "relu2"):
        return h.clamp_min(0) ** (1 if name == "relu" else 2)
    if name == "silu":
        return h * torch.sigmoid(h)
    if name == "gelu":
        return h * _cdf(h)
    return h * torch.sigmoid(_tanh_arg(h)[0]) if name else h


def slope(h, name):
    if name in ("relu", "relu2"):
        return (h > 0).to(h.dtype) * (1 if name == "relu" else 2 * h)
    if name == "silu":
        s = torch.sigmoid(h)
        return s * (1 + h * (1 - s))
    if name == "gelu":
        return _cdf(h) + h * _phi(h)
    if name == "gelu_tanh":
        u, du = _tanh_arg(h)
        s = torch.sigmoid(u)
        return s + h * s * (1 - s) * du
    return torch.ones_like(h)


def _far(u):
    """Roundings of sigmoid(u) from |u| log2 e = 126 on, where e^-u is 2^t with t rounded: half a last place of
    t in 64 .. 128 is 2^-18, the part of log2 e past float32 adds 1.93e-8 |u| = 1.7e-6 < 2^-19 (up to 88.8, past which
    the result is 0 or 1); together below 5.6e-6, times ln 2 below 66 U relative."""
    return 72 * (u.abs() > 87.3).to(u.dtype)


# A sigmoid or e^(-h^2 / 2) below 2^-126 comes as zero (the hardware's reciprocal and 2^x): off by that, and what it is a factor of by
# that times the other factors.
LEAST = 2.0 ** -126


def act_error(h, name):
    """Of act(h) in float32.  sigmoid(u): e^-u within 4 U of itself and u's own error, a reciprocal: 8 U + |u's
    error| of itself, and for 16-bit values 1.25 U |u| more, u log2 e being rounded once (and log2 e, by 0.22 U).  u of gelu_tanh: three products and a sum, with two rounded constants, 6 U of
    itself.  Phi(-x) by a fit: 8 U, a reciprocal, a product and e^(-x^2 / 2), whose
    argument's roundings are 2.3 U of x^2 / 2, below 4 U x phi / Phi; the other side is 1 less that."""
    a = h.abs()
    if name == "silu":
        return (12 + 1.25 * a + _far(h)) * U * (h * torch.sigmoid(h)).abs() + a * LEAST
    if name == "gelu":
        return U * a * (40 * _cdf(h) + 4 * a * _phi(h)) + a * LEAST
    if name == "gelu_tanh":
        u = _tanh_arg(h)[0]
        return U * (h * torch.sigmoid(u)).abs() * (12 + 7.25 * u.abs() + _far(u)) + a * LEAST
    return 2 * U * act(h, name).abs()


def slope_error(h, name):
    a = h.abs()
    if name == "silu":
        s = torch.sigmoid(h)
        return (24 + 2.5 * a + _far(h)) * U * s * (1 + a) + (1 + a) * LEAST
    if name == "gelu":
        # (exp of -h^2 / 2, which has two roundings of itself)
        return U * (40 * _cdf(h) + 4 * a * _phi(h) + a * _phi(h) * (8 + 2 * h * h)) + (1 + a) * LEAST
    if name == "gelu_tanh":
        u, du = _tanh_arg(h)
        s = torch.sigmoid(u)
        # (1 - s is within U of 1 absolutely where s nears it, so s (1 - s) is within s U)
        return U * (s * (12 + 7.25 * u.abs() + _far(u)) + a * du * s * (4 + (1 - s) * (24 + 14.5 * u.abs() + _far(u)))) + (1 + a * du) * LEAST
    return 2 * U * slope(h, name).abs()


# ---- Norms.

def inverse_rms(v, eps):
    return (v.square().mean(-1, keepdim=True) + eps).rsqrt()


def norm(r, w, y=None, post=None, gate=None, scale=1.0, drop=None, eps=1e-6):
    """(r', x, i(r'), i(y)) and bounds of the float32 errors of r' and x; all in 64 bits."""
    one = torch.ones((), dtype=F64, device=r.device)
    if y is None:
        v, iy, verr = r, None, torch.zeros_like(r)
    else:
        iy = inverse_rms(y, eps) if post is not None else one
        k = one if drop is None else drop
        branch = (gate if gate is not None else one) * k * (y * iy * post if post is not None else y)
        v = scale * r + branch
        # scale r one rounding, the sum one; the branch five products, and i(y): half its sum's errors and four more.
        verr = U * (2 * (scale * r).abs() + (6 + SUM / 2 + 4) * branch.abs())
    iv = inverse_rms(v, eps)
    x = v * iv * w
    off = verr.square().sum(-1, keepdim=True).sqrt() / v.square().sum(-1, keepdim=True).sqrt().clamp_min(1e-300)
    xerr = (w * iv).abs() * verr + x.abs() * (U * (SUM / 2 + 6) + off)
    return v, x, iv, iy, verr, xerr


def norm_grad(dx, dr, r, w, iv, y=None, iy=None, post=None, gate=None, scale=1.0, drop=None):
    """{"dr", "dy", "dw", "dpost", "dgate" (a row's)}: (value, bound of its float32 error)."""
    M, D = r.shape
    one = torch.ones((), dtype=F64, device=r.device)
    mean = lambda t: t.mean(-1, keepdim=True)  # noqa: E731
    vh, gw = r * iv, dx * w
    e, abse = dr + iv * gw, dr.abs() + (iv * gw).abs()
    c1, absc1 = mean(gw * vh), mean((gw * vh).abs())
    t, abst = e - iv * vh * c1, abse + (iv * vh).abs() * absc1
    N = SUM + 8                                  # roundings of any one term of a sum over a row, and after it
    out = {"dr": (scale * t, U * N * (scale * abst).abs()), "dw": ((dx * vh).sum(0), U * (M + 8) * (dx * vh).abs().sum(0))}
    if y is None:
        return out
    k = one if drop is None else drop
    f = (gate if gate is not None else one) * k
    z = y * (iy * post if post is not None else one)
    dz, absdz = t * f, abst * f.abs()
    if post is None:
        out["dy"] = dz, U * (N + 2) * absdz
    else:
        yh = y * iy
        c2 = mean(dz * post * yh)
        u = (f * post * yh).abs()
        absc2 = mean(u * abse) + absc1 * mean(u * (iv * vh).abs())
        out["dy"] = (iy * (dz * post - yh * c2),
                     U * (N + 8) * iy * ((absdz * post).abs() + yh.abs() * absc2))
        out["dpost"] = (dz * yh).sum(0), U * (M + N + 4) * (absdz * yh.abs()).sum(0)
    dg, absdg = t * k * z, abst * (k * z).abs()
    out["dgate"] = dg, U * (N + 6) * absdg
    out["dgate sum"] = dg.sum(0), U * (M + N + 6) * absdg.sum(0)
    return out


def close(got, want, err, dtype=None):
    """got within err and one rounding to its type of want; an infinity of want's sign where want
    lies past the type's largest value, rounded, (65504 of float16: from half a step of 32 past it on)."""
    r, a = rounding(dtype or got.dtype)
    bound = err * (1 + r) + want.abs() * r + a
    off = (got.to(F64) - want).abs()
    past = want.abs() + err >= torch.finfo(got.dtype).max * (1 + torch.finfo(got.dtype).eps / 4)
    infinite = torch.isinf(got) & (got > 0).eq(want > 0)
    fine = (off <= bound) & torch.isfinite(got) | past & infinite
    assert fine.all(), ((off / bound)[~fine].max().item(), (~fine).sum().item(), tuple(got.shape))


def close_codes(q, s, want, err):
    """Codes and scales by rows of what is within err of want: a scale is a block's largest
    magnitude over 448, a value within half a code's step."""
    K = want.shape[-1]
    j = torch.arange(K, device=want.device) // 128
    pad = torch.nn.functional.pad
    top = pad(want.abs(), (0, -K % 128)).unflatten(-1, (-1, 128)).amax(-1).clamp_min(2.0 ** -110)
    slack = pad(err, (0, -K % 128)).unflatten(-1, (-1, 128)).amax(-1)
    assert ((s.to(F64) - top / 448).abs() <= slack / 448 + top / 448 * 4 * U).all()
    wide = s.to(F64)[..., j]
    off = (q.to(F64) * wide - want).abs()
    bound = (want.abs() * 2.0 ** -4).maximum(wide * 2.0 ** -10) * (1 + 2.0 ** -10) + err * 1.07 + want.abs() * 8 * U
    assert (off <= bound).all(), ((off / bound).max().item(), (off > bound).sum().item())


def randn(*shape, seed=0, dtype=F32, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def rng(seed, offset=0, device="cuda"):
    return torch.tensor([seed, offset], device=device)
