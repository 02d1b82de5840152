"""GPU tier: operands in 8-bit floating point with scales by blocks of 128
(fp64_emu/f8.py).  Codes and scales equal the definition's float32 steps bit for
bit; products, the gated activation and its gradient stay within bounds
derived from the formats' roundings (f8_util.py), against float64."""
import math

import pytest
import torch

import fp64_emu
from f8_util import (BLOCK, E4M3, E5M2, F64, operand, product_bound, quantised, rounding,
                     same_codes, values)

pytestmark = pytest.mark.gpu

BF16, FP16, F32 = torch.bfloat16, torch.float16, torch.float32


def _say(*what):
    print("case", *what, flush=True)


def _randn(shape, seed, dtype=BF16):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * torch.exp2(torch.randint(-4, 5, shape[-1:], generator=g).float())
    return x.to(dtype)


def _check_quant(x, fmt, dev, **kw):
    got = fp64_emu.quant_f8(x.to(dev) if not x.is_cuda else x, rows=True, cols=True, fmt=fmt)
    q, s = quantised(x, fmt)
    qt, st = quantised(x.transpose(-1, -2), fmt)
    for g, w in zip(got, (q, s, qt, st)):
        assert g.shape == w.shape
    assert same_codes(got[0], q) and torch.equal(got[1].cpu().nan_to_num(-1.0), s.nan_to_num(-1.0))
    assert same_codes(got[2], qt) and torch.equal(got[3].cpu().nan_to_num(-1.0), st.nan_to_num(-1.0))
    return got


SHAPES = [(1, 1), (1, 128), (1, 8192), (2, 5), (3, 129), (17, 333), (127, 255), (128, 128), (130, 1),
          (129, 640), (300, 777), (257, 1024), (3, 40, 200), (5, 128, 131)]


@pytest.mark.parametrize("fmt", [E4M3, E5M2])
@pytest.mark.parametrize("dtype", [BF16, FP16, F32])
@pytest.mark.parametrize("shape", SHAPES)
def test_quant_rows_and_cols(dev, shape, dtype, fmt):
    _say("quant", shape, dtype, fmt)
    x = _randn(shape, sum(shape), dtype)
    both = _check_quant(x, fmt, dev)
    only = fp64_emu.quant_f8(x.to(dev), fmt=fmt)
    turned = fp64_emu.quant_f8(x.to(dev), rows=False, cols=True, fmt=fmt)
    for a, b in zip(both, only + turned):
        assert torch.equal(a.float(), b.float())


@pytest.mark.parametrize("fmt", [E4M3, E5M2])
@pytest.mark.parametrize("shape", SHAPES)
def test_quant_tiles(dev, shape, fmt):
    _say("tiles", shape, fmt)
    for dtype in (BF16, F32):
        x = _randn(shape, 7 + sum(shape), dtype)
        q, s, qt, st = fp64_emu.quant_f8_tiles(x.to(dev), transposed=True, fmt=fmt)
        wq, ws = quantised(x, fmt, BLOCK)
        assert same_codes(q, wq) and torch.equal(s.cpu(), ws)
        assert same_codes(qt, wq.transpose(-1, -2)) and torch.equal(st.cpu(), ws.transpose(-1, -2))
        q1, s1 = fp64_emu.quant_f8_tiles(x.to(dev), fmt=fmt)
        assert same_codes(q1, wq) and torch.equal(s1.cpu(), ws)


def test_quant_every_bfloat16(dev):
    """All 65536 bit patterns, blocks of the finite ones apart from those with NaN or infinity."""
    bits = torch.arange(65536, dtype=torch.int32)
    x = bits.to(torch.int16).view(BF16)
    finite = x[torch.isfinite(x.float())]
    rest = x[~torch.isfinite(x.float())]
    for name, part in (("finite", finite), ("not finite", rest), ("mixed", x)):
        _say("every bfloat16", name)
        n = part.numel() // 256 * 256
        for fmt in (E4M3, E5M2):
            _check_quant(part[:n].reshape(-1, 256), fmt, dev)


@pytest.mark.parametrize("fmt", [E4M3, E5M2])
def test_quant_values(dev, fmt):
    """Zeros, the floor of the block's magnitude, the ends of float32's range, one odd element
    in a block: and whole blocks of NaN where one element is not finite."""
    x = _randn((140, 400), 3, F32)
    x[0] = 0.0
    x[1, :130] = 1e-41
    x[2] = 3.3e38
    x[3, 5] = 3.4e38
    x[4] = -1e-33
    x[5, 200] = 1e30
    x[6, 130] = math.inf
    x[7, 0] = math.nan
    x[8, 399] = -math.inf
    _say("values", fmt)
    q, s, _, _ = _check_quant(x, fmt, dev)
    v = values(q, s).cpu()
    assert torch.isnan(v[6, 128:256]).all() and torch.isfinite(v[6, :128]).all()
    assert torch.isnan(v[7, :128]).all() and torch.isnan(v[8, 384:]).all()
    assert (v[0] == 0).all()
    # Half a step of the code: 2^-4 (e4m3) or 2^-3 (e5m2) relative, or half of the
    # least code's value, and three float32 roundings on the way.
    top, half, least = {E4M3: (448.0, 2.0 ** -4, 2.0 ** -10), E5M2: (57344.0, 2.0 ** -3, 2.0 ** -17)}[fmt]
    ok = torch.isfinite(v)
    a = s.double().cpu().repeat_interleave(BLOCK, 1)[:, :400]
    bound = torch.maximum(x.double().abs() * half, a * least) * (1 + 2.0 ** -21)
    assert ((v - x.double()).abs() <= bound)[ok].all()


@pytest.mark.parametrize("what", ["rows apart", "odd start", "odd rows", "transposed", "members apart"])
def test_quant_strides(dev, what):
    _say("quant strides", what)
    big = _randn((3, 200, 520), 11).to(dev)
    x = {"rows apart": big[0, ::2, :384], "odd start": big[0, :, 3:390], "odd rows": big[0].reshape(-1)[:200 * 519].view(200, 519),
         "transposed": big[0].t(), "members apart": big[::2, 10:90, 8:200]}[what]
    _check_quant(x, E4M3, dev)


# ---- products ----

def _product(shape, out_dtype, fa=E4M3, fb=E4M3, tiles=True, accumulate=False, seed=0, dev="cuda"):
    *batch, M, N, K = shape
    qa, sa = operand((*batch, M, K), seed + 1, fa, device=dev)
    qb, sb = operand((*batch, N, K), seed + 2, fb, tiles, device=dev)
    A, B = values(qa, sa), values(qb, sb)
    want = A @ B.transpose(-1, -2).contiguous()
    fn = fp64_emu.bmm_f8 if batch else fp64_emu.mm_f8
    out = None
    if accumulate:
        out = torch.randn(want.shape, device=dev, generator=torch.Generator(dev).manual_seed(seed)).to(out_dtype)
        want = want + out.to(F64)
    bound = product_bound(A, B, want, out_dtype, out_dtype == F32)
    got = fn(qa, sa, qb, sb, out_dtype=out_dtype, out=out, accumulate=accumulate)
    assert got.dtype == out_dtype and got.shape == want.shape
    err = (got.to(F64) - want).abs()
    assert (err <= bound).all(), ((err / bound).max().item(), (err > bound).sum().item())
    return got, (qa, sa, qb, sb)


MM = [(1, 1, 1), (1, 7, 128), (1, 512, 4096), (1, 8192, 333), (5, 130, 1000), (16, 256, 129), (17, 100, 640),
      (33, 257, 777), (64, 64, 64), (64, 512, 16384), (65, 65, 65), (128, 128, 128), (129, 1, 300),
      (200, 333, 127), (256, 256, 256), (300, 500, 4100), (257, 513, 1025), (512, 4096, 384),
      (4100, 4200, 128), (4097, 4111, 300), (1000, 3, 5000), (2048, 2048, 2048)]


@pytest.mark.parametrize("tiles", [True, False])
@pytest.mark.parametrize("out_dtype", [BF16, F32])
@pytest.mark.parametrize("shape", MM)
def test_mm(dev, shape, out_dtype, tiles):
    _say("mm", shape, out_dtype, "tiles" if tiles else "rows")
    _product(shape, out_dtype, tiles=tiles, seed=sum(shape))


@pytest.mark.parametrize("fa,fb", [(E4M3, E5M2), (E5M2, E4M3), (E5M2, E5M2)])
@pytest.mark.parametrize("shape", [(3, 200, 500), (20, 96, 384), (50, 300, 1000), (300, 200, 700), (4096, 4096, 256)])
def test_mm_formats(dev, shape, fa, fb):
    for out_dtype in (F32, FP16, BF16):
        _say("mm formats", shape, fa, fb, out_dtype)
        _product(shape, out_dtype, fa, fb, tiles=shape[0] % 2 == 0, seed=3)


@pytest.mark.parametrize("out_dtype", [F32, BF16, FP16])
@pytest.mark.parametrize("shape", [(1, 100, 300), (40, 130, 20000), (300, 257, 640), (64, 128, 0), (4096, 4352, 130)])
def test_mm_accumulates(dev, shape, out_dtype):
    _say("mm accumulate", shape, out_dtype)
    _product(shape, out_dtype, accumulate=True, seed=9)


@pytest.mark.parametrize("shape", [(3, 1, 40, 300), (5, 70, 90, 200), (64, 128, 128, 128), (2, 300, 513, 385),
                                   (70, 256, 256, 130), (300, 16, 16, 16)])
def test_bmm(dev, shape):
    for out_dtype, tiles in ((BF16, True), (F32, False)):
        _say("bmm", shape, out_dtype, tiles)
        _product(shape, out_dtype, tiles=tiles, seed=5)


@pytest.mark.parametrize("shape", [(3, 50, 300), (200, 300, 777), (4096, 4096, 300)])
def test_mm_layouts(dev, shape):
    """Operands whose rows start anywhere, scales in either order, out rows apart: the same bits."""
    M, N, K = shape
    for out_dtype in (BF16, F32):
        _say("mm layouts", shape, out_dtype)
        got, (qa, sa, qb, sb) = _product(shape, out_dtype, seed=21)

        def shifted(q, ld, start):
            room = torch.full((q.shape[0] * ld + start + 64,), 0x7f, dtype=torch.uint8, device=dev)
            v = room.view(q.dtype).as_strided(q.shape, (ld, 1), start)
            v.copy_(q)
            return v

        for ld, start in ((K + 1, 1), (K, 0), (-(-K // 16) * 16, 0), (-(-K // 16) * 16 + 48, 32), (K + 5, 3)):
            a, b = shifted(qa, ld, start), shifted(qb, ld, start)
            s1 = sa.t().contiguous().t()
            s2 = sb.contiguous()
            out = torch.full((M, N + 5), -7.0, dtype=out_dtype, device=dev)[:, 2:N + 2]
            fp64_emu.mm_f8(a, s1, b, s2, out=out)
            assert torch.equal(out, got), (ld, start)
            assert (out.as_strided((M, 2), (N + 5, 1), 0) == -7).all()


def test_expanded_and_transposed_inputs(dev):
    """Rows that lie on each other (an expanded tensor's) and columns that lie apart: as their copies."""
    _say("expanded")
    x = _randn((1, 400), 31).to(dev).expand(140, 400)
    for a, b in zip(fp64_emu.quant_f8(x, cols=True), fp64_emu.quant_f8(x.contiguous(), cols=True)):
        assert torch.equal(a.float(), b.float())
    for y, w in ((x, x.contiguous()), (_randn((400, 140), 32).to(dev).t(), None)):
        w = y.contiguous() if w is None else w
        for a, b in zip(fp64_emu.swiglu_f8(y), fp64_emu.swiglu_f8(w)):
            assert torch.equal(a.float(), b.float())
    _, hq, hs = fp64_emu.swiglu_f8(x)
    dy = torch.ones(1, 200, device=dev).expand(140, 200)
    assert torch.equal(fp64_emu.swiglu_f8_backward(dy, hq[:1].expand(140, 400), hs[:1].expand(140, 4)),
                       fp64_emu.swiglu_f8_backward(dy.contiguous(), hq, hs))
    qa, sa = operand((1, 300), 33, device=dev)
    qb, sb = operand((200, 300), 34, device=dev)
    want = fp64_emu.mm_f8(qa, sa, qb, sb).expand(150, 200)
    turned = qb.view(torch.uint8).t().contiguous().t().view(E4M3)
    assert not turned.is_contiguous()
    for b in (qb, turned):
        got = fp64_emu.mm_f8(qa.expand(150, 300), sa.expand(150, 3), b, sb)
        assert (got.double() - want.double()).abs().max() <= want.abs().max() * 2.0 ** -7
    x = _randn((60, 256), 35).to(dev).requires_grad_()
    w = _randn((128, 256), 36, F32).to(dev).requires_grad_()
    (dx,) = torch.autograd.grad(fp64_emu.linear_f8(x, w).sum(), x)       # an expanded gradient
    (want,) = torch.autograd.grad(fp64_emu.linear_f8(x, w), x, torch.ones(60, 128, device=dev, dtype=BF16))
    assert torch.equal(dx, want)


def test_mm_nothing_to_do(dev):
    _say("mm empty")
    def e(r, k, fmt=E4M3):
        return (torch.empty(r, k, dtype=fmt, device=dev), torch.empty(r, -(-k // 128), device=dev))
    assert fp64_emu.mm_f8(*e(0, 128), *e(5, 128)).shape == (0, 5)
    assert fp64_emu.mm_f8(*e(5, 128), *e(0, 128)).shape == (5, 0)
    out = torch.full((5, 7), 3.0, device=dev)
    assert (fp64_emu.mm_f8(*e(5, 0), *e(7, 0), out=out, accumulate=True) == 3).all()
    assert (fp64_emu.mm_f8(*e(5, 0), *e(7, 0), out=out) == 0).all()
    x = torch.empty(0, 256, device=dev, dtype=BF16, requires_grad=True)
    w = torch.ones(128, 256, device=dev, requires_grad=True)
    y = fp64_emu.linear_f8(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), torch.empty_like(y))
    assert y.shape == (0, 128) and dx.shape == x.shape and (dw == 0).all()
    assert [t.shape for t in fp64_emu.quant_f8(torch.empty(0, 300, device=dev), cols=True)] == [
        (0, 300), (0, 3), (300, 0), (300, 0)]
    assert fp64_emu.swiglu_f8(torch.empty(0, 8, device=dev))[0].shape == (0, 4)


def test_mm_not_finite(dev):
    """A NaN scale or code reaches its row's or column's outputs and no others."""
    for shape in ((3, 50, 300), (300, 260, 700), (4096, 4096, 128)):
        for out_dtype in (BF16, F32):
            _say("mm NaN", shape, out_dtype)
            M, N, K = shape
            qa, sa = operand((M, K), 1, device=dev)
            qb, sb = operand((N, K), 2, device=dev)
            clean = fp64_emu.mm_f8(qa, sa, qb, sb, out_dtype=out_dtype)
            sa[1, 0] = math.nan
            qb.view(torch.uint8)[7, K - 1] = 0x7f
            got = fp64_emu.mm_f8(qa, sa, qb, sb, out_dtype=out_dtype)
            hit = torch.zeros(M, N, dtype=torch.bool, device=dev)
            hit[1] = True
            hit[:, 7] = True
            assert torch.isnan(got[hit]).all() and torch.equal(got[~hit], clean[~hit])


def test_mm_same_bits_again(dev):
    for shape in ((1, 300, 30000), (100, 100, 20000), (600, 500, 3000)):
        _say("mm again", shape)
        qa, sa = operand((shape[0], shape[2]), 1, device=dev)
        qb, sb = operand((shape[1], shape[2]), 2, device=dev)
        first = fp64_emu.mm_f8(qa, sa, qb, sb, out_dtype=F32)
        for _ in range(3):
            assert torch.equal(fp64_emu.mm_f8(qa, sa, qb, sb, out_dtype=F32), first)


def test_far_offsets(dev):
    """Codes past 2^32 bytes and outputs past 2^31 elements: sampled rows."""
    N, K = 70000, 65536
    _say("far quant", N, K)
    w = torch.empty(N, K, dtype=BF16, device=dev)
    for i in range(0, N, 10000):
        w[i:i + 10000] = torch.randn(10000, K, device=dev, generator=torch.Generator(dev).manual_seed(i))
    q, s, qt, st = fp64_emu.quant_f8_tiles(w, transposed=True)
    wq, ws = quantised(w[-112:], E4M3, BLOCK)              # 70000 = 546 128 + 112
    assert same_codes(q[-112:], wq) and torch.equal(s[-1:].cpu(), ws)
    assert same_codes(qt[:, -112:], wq.t()) and torch.equal(st[:, -1:].cpu(), ws.t())
    del w, qt, st
    qa, sa = operand((300, K), 4, device=dev)
    for M in (2, 300):
        _say("far mm", M, N, K)
        got = fp64_emu.mm_f8(qa[:M], sa[:M], q, s, out_dtype=F32)
        A, B = values(qa[:M], sa[:M]), values(q[-200:], s[torch.arange(N - 200, N, device=dev) // BLOCK])
        want = A @ B.t().contiguous()
        assert ((got[:, -200:].to(F64) - want).abs() <= product_bound(A, B, want, F32, True)).all()
    del q, s
    M, N, K = 33000, 66000, 128
    _say("far out", M, N, K)
    qa, sa = operand((M, K), 5, device=dev)
    qb, sb = operand((N, K), 6, device=dev)
    got = fp64_emu.mm_f8(qa, sa, qb, sb)
    A, B = values(qa[-100:], sa[-100:]), values(qb, sb)
    want = A @ B.t().contiguous()
    assert ((got[-100:].to(F64) - want).abs() <= product_bound(A, B, want, BF16, False)).all()


# ---- the gated activation ----

def _silu(g):
    return g / (1 + torch.exp(-g))


def _close(got, want, dtype, ops):
    """`ops` float32 operations (each within 2^-22 relative: the exponential's and the
    division's are not correctly rounded) and one rounding."""
    r, a = rounding(dtype)
    return ((got.to(F64) - want).abs() <= want.abs() * (r + ops * 2.0 ** -22) + a + 2.0 ** -140).all()


def _check_codes(q, s, x, rel):
    """Codes and scales of float32 values within `rel` of x: scales within that, codes
    within half a step of x (a value next to a tie may go either way)."""
    x = x.to(q.device)
    K = x.shape[-1]
    pad = torch.nn.functional.pad(x, (0, -K % BLOCK)).reshape(*x.shape[:-1], -1, BLOCK)
    a = pad.abs().amax(-1).clamp_min(2.0 ** -110)
    assert ((s.to(F64) * 448 - a).abs() <= a * (rel + 2.0 ** -23)).all()
    spread = s.to(F64).repeat_interleave(BLOCK, -1)[..., :K]
    # half a step (2^-4 of the value, or half of the least code) and rel on top of it
    bound = torch.maximum(x.abs() * 2.0 ** -4, spread * 2.0 ** -10) * (1 + 2 * rel + 2.0 ** -20) + x.abs() * 2 * rel
    assert ((q.to(F64) * spread - x).abs() <= bound).all()


SWIGLU = [(1, 1), (1, 4096), (3, 130), (127, 128), (130, 257), (300, 776), (257, 640)]


@pytest.mark.parametrize("dtype", [BF16, FP16, F32])
@pytest.mark.parametrize("M,F", SWIGLU)
def test_swiglu(dev, M, F, dtype):
    _say("swiglu", M, F, dtype)
    h = (_randn((M, 2 * F), M + F, F32) * 0.7).to(dtype)
    g, u = h.to(F64)[:, :F], h.to(F64)[:, F:]
    want = (_silu(g) * u).to(dev)
    y, hq, hs = fp64_emu.swiglu_f8(h.to(dev))
    assert y.dtype == dtype and _close(y, want, dtype, 8)
    for half, x in ((0, g), (1, u)):
        q, s = quantised(x.to(F32), E4M3)
        blocks = -(-F // BLOCK)
        assert same_codes(hq[:, half * F:(half + 1) * F], q)
        assert torch.equal(hs[:, half * blocks:(half + 1) * blocks].cpu(), s)
    q, s, qt, st, hq2, hs2 = fp64_emu.swiglu_f8(h.to(dev), quant="both")
    assert same_codes(hq2, hq.cpu()) and torch.equal(hs2, hs)
    _check_codes(q, s, want, 8 * 2.0 ** -22)
    _check_codes(qt, st, want.t().contiguous(), 8 * 2.0 ** -22)
    q3, s3 = fp64_emu.swiglu_f8(h.to(dev), quant="rows", keep=False)
    assert same_codes(q3, q.cpu()) and torch.equal(s3, s)


def test_swiglu_values(dev):
    """Far out on both sides, where e^-g leaves float32, and not finite."""
    g = torch.tensor([0.0, -0.0, 90.0, -85.0, -87.0, -100.0, -1e4, 1e30, 1e-40, math.inf, math.nan, 20.0])
    h = torch.cat((g, torch.full((12,), 0.5))).repeat(3, 1)
    _say("swiglu values")
    (y,) = fp64_emu.swiglu_f8(h.to(dev), keep=False)
    want = _silu(g.to(F64)) * 0.5
    got = y[0].cpu().to(F64)
    ok = torch.isfinite(want)
    assert torch.isnan(got[10]) and got[9] == math.inf
    # below e^-87 the quotient is a denormal or zero
    assert ((got - want).abs() <= want.abs() * 2.0 ** -19 + 1e-36)[ok].all()


def _kept(M, F, seed, dev):
    h = _randn((M, 2 * F), seed, F32) * 0.7
    _, hq, hs = fp64_emu.swiglu_f8(h.to(dev))
    blocks = -(-F // BLOCK)
    g, u = values(hq[:, :F], hs[:, :blocks]), values(hq[:, F:], hs[:, blocks:])
    return hq, hs, g, u


def _grad(dy, g, u):
    s = 1 / (1 + torch.exp(-g))
    return torch.cat((dy * u * s * (1 + g * (1 - s)), dy * g * s), 1)


@pytest.mark.parametrize("dtype", [BF16, FP16, F32])
@pytest.mark.parametrize("M,F", SWIGLU)
def test_swiglu_backward(dev, M, F, dtype):
    _say("swiglu backward", M, F, dtype)
    hq, hs, g, u = _kept(M, F, M + F, dev)
    dy = _randn((M, F), 2 * M + F, dtype).to(dev)
    want = _grad(dy.to(F64), g, u)
    dh = fp64_emu.swiglu_f8_backward(dy, hq, hs)
    # 1 + g (1 - s) loses up to |g| + 1 roundings where it is near zero: an absolute term.
    slack = dy.to(F64).abs() * u.abs() * (1 + g.abs()) * 12 * 2.0 ** -22
    slack = torch.cat((slack, slack * 0), 1)
    r, a = rounding(dtype)
    assert dh.dtype == dtype
    assert ((dh.to(F64) - want).abs() <= want.abs() * (r + 12 * 2.0 ** -22) * (1 + r) + slack * (1 + r) + a + 2.0 ** -140).all()
    got = fp64_emu.swiglu_f8_backward(dy, hq, hs, quant="both")
    rows = fp64_emu.swiglu_f8_backward(dy, hq, hs, quant="rows")
    full = fp64_emu.swiglu_f8_backward(dy.to(F32), hq, hs)     # the same float32 values, unrounded
    q, s = quantised(full, E4M3)
    qt, st = quantised(full.t(), E4M3)
    assert same_codes(got[0], q) and torch.equal(got[1].cpu(), s)
    assert same_codes(got[2], qt) and torch.equal(got[3].cpu(), st)
    assert same_codes(rows[0], q) and torch.equal(rows[1].cpu(), s)


def test_swiglu_backward_differences(dev):
    """Against central differences of the activation, in float64, at the kept values: third
    derivatives of silu are below 1, so a step of 1e-4 errs by 1e-8."""
    _say("swiglu differences")
    M, F, e = 40, 200, 1e-4
    hq, hs, g, u = _kept(M, F, 5, dev)
    dh = fp64_emu.swiglu_f8_backward(torch.ones(M, F, device=dev), hq, hs).to(F64)
    dg = (_silu(g + e) - _silu(g - e)) / (2 * e) * u
    du = _silu(g) * ((u + e) - (u - e)) / (2 * e)
    scale = 1 + g.abs() + u.abs()
    assert ((dh[:, :F] - dg).abs() <= (1e-8 * u.abs() + 12 * 2.0 ** -22 * (1 + g.abs()) * u.abs() + 1e-9 * scale)).all()
    assert ((dh[:, F:] - du).abs() <= 12 * 2.0 ** -22 * g.abs() + 1e-9 * scale).all()


# ---- the layer ----

@pytest.mark.parametrize("shape,N", [((1, 300), 200), ((5, 17, 256), 130), ((200, 777), 501), ((2, 150, 128), 1)])
def test_linear_and_gradients(dev, shape, N):
    _say("linear", shape, N)
    K = shape[-1]
    x = _randn(shape, 1).to(dev).requires_grad_()
    w = (_randn((N, K), 2, F32) * 0.05).to(dev).requires_grad_()
    y = fp64_emu.linear_f8(x, w)
    dy = _randn(y.shape, 3).to(dev)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    assert y.shape == (*shape[:-1], N) and y.dtype == BF16 and dx.shape == x.shape and dw.dtype == F32
    rows, grads = x.detach().reshape(-1, K), dy.reshape(-1, N)

    def v(t, tall=1):
        q, s = quantised(t, E4M3, tall)
        return values(q, s).to(dev)

    for got, A, B in ((y.reshape(-1, N), v(rows), v(w, BLOCK)), (dx.reshape(-1, K), v(grads), v(w, BLOCK).t()),
                      (dw, v(grads.t()), v(rows.t()))):
        want = A @ B.t().contiguous()
        bound = product_bound(A, B, want, got.dtype, got.dtype == F32)
        assert ((got.to(F64) - want).abs() <= bound).all()
    # A weight quantised earlier gives the same; without its transposed half only where x needs no gradient.
    wq = fp64_emu.quant_f8_tiles(w.detach(), transposed=True)
    assert torch.equal(fp64_emu.linear_f8(x, w, wq), y)
    assert torch.equal(fp64_emu.linear_f8(x.detach(), w, wq[:2]), y)
    with pytest.raises(ValueError, match="transposed half"):
        fp64_emu.linear_f8(x, w, wq[:2])


def test_linear_gradient_differences(dev):
    """<dy, y(x + d) - y(x)> = <dx, d> for a linear map, up to the quantisation of x, w and dy: steps of
    2^-4 of a block's elements average out over 256 x 384 terms to well below 3%."""
    _say("linear differences")
    x = _randn((256, 384), 1, F32).to(dev).requires_grad_()
    w = (_randn((320, 384), 2, F32) * 0.05).to(dev).requires_grad_()
    dy = torch.randn(256, 320, device=dev, generator=torch.Generator(dev).manual_seed(4))
    y = fp64_emu.linear_f8(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    dy64 = dy.to(F64)
    with torch.no_grad():
        d = dx / dx.norm() * x.norm()              # along the gradient: the change does not cancel
        far = fp64_emu.linear_f8(x + d, w)
        assert abs(((far - y).to(F64) * dy64).sum() / (dx.to(F64) * d.to(F64)).sum() - 1) < 0.03
        e = dw / dw.norm() * w.norm()
        far = fp64_emu.linear_f8(x, w + e)
        assert abs(((far - y).to(F64) * dy64).sum() / (dw.to(F64) * e.to(F64)).sum() - 1) < 0.03


def test_linear_keeps_one_byte(dev):
    """What waits for the backward pass: x's codes and scales and the weight's, nothing in 16 bits."""
    x = _randn((512, 1024), 1).to(dev).requires_grad_()
    w = _randn((256, 1024), 2, F32).to(dev).requires_grad_()
    kept = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t) or t, lambda t: t):
        fp64_emu.linear_f8(x, w)
        fp64_emu.swiglu_ckpt_f8(x)
    codes = sum(t.numel() for t in kept if t.element_size() == 1)
    rest = sum(t.numel() * t.element_size() for t in kept if t.element_size() > 1)
    assert codes == 512 * 1024 + 256 * 1024 + 512 * 1024 and rest <= codes // 16


def test_swiglu_ckpt(dev):
    _say("swiglu checkpoint")
    h = _randn((6, 50, 600), 1).to(dev).requires_grad_()
    y = fp64_emu.swiglu_ckpt_f8(h)
    dy = _randn(y.shape, 2).to(dev)
    (dh,) = torch.autograd.grad(y, h, dy)
    want = fp64_emu.swiglu_f8_backward(dy.reshape(-1, 300), *fp64_emu.swiglu_f8(h.detach().reshape(-1, 600))[1:])
    assert torch.equal(dh.reshape(-1, 600), want) and y.shape == (6, 50, 300)


# ---- streams, graphs, tracing, refusals ----

def test_other_stream(dev):
    _say("other stream")
    x = _randn((300, 700), 1).to(dev)
    w = _randn((400, 700), 2).to(dev)
    want = fp64_emu.linear_f8(x, w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = fp64_emu.linear_f8(x, w)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_graph_replays(dev):
    """A captured layer (partial sums and a relaid operand among its kernels) replays to the eager bits,
    with eager work between the replays."""
    _say("graph")
    x = _randn((70, 9001), 1).to(dev)
    w = _randn((130, 9001), 2).to(dev)

    def layer():
        q, s = fp64_emu.quant_f8(x)
        wq, ws = fp64_emu.quant_f8_tiles(w)
        packed = q.contiguous()                    # rows of 9001 bytes
        h = fp64_emu.mm_f8(packed, s, wq, ws)
        return fp64_emu.swiglu_f8(h, quant="both")

    want = layer()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = layer()
    for r in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a.float(), b.float()), r
        layer()
        torch.cuda.synchronize()


def test_refusals(dev):
    x = torch.zeros(4, 256, device=dev)
    q, s = fp64_emu.quant_f8(x)
    w, ws = fp64_emu.quant_f8_tiles(torch.zeros(300, 256, device=dev))
    for call, msg in [
            (lambda: fp64_emu.quant_f8(x.double()), "expect float32"),
            (lambda: fp64_emu.mm_f8(q, s, w[:, :128], ws[:, :1]), "expect B as"),
            (lambda: fp64_emu.mm_f8(q, s, w, ws[:2]), "scales by rows or by tiles"),
            (lambda: fp64_emu.mm_f8(q, s[:, :1], w, ws), "one scale per 128"),
            (lambda: fp64_emu.mm_f8(w, ws, q, s), "A's scales are by rows"),
            (lambda: fp64_emu.mm_f8(x, s, w, ws), "codes are float8"),
            (lambda: fp64_emu.mm_f8(q, s.double(), w, ws), "scales are float32"),
            (lambda: fp64_emu.mm_f8(q.cpu(), s, w, ws), "one GPU|CPU"),
            (lambda: fp64_emu.mm_f8(q, s, w, ws, out=torch.empty(4, 299, device=dev)), "out"),
            (lambda: fp64_emu.mm_f8(q, s, w, ws, out=torch.empty(1, 300, device=dev).expand(4, 300)), "overlap|memory"),
            (lambda: fp64_emu.mm_f8(q, s, w, ws, out_dtype=torch.float64), "expect float32"),
            (lambda: fp64_emu.swiglu_f8_backward(x, q, s), "hq"),
            (lambda: fp64_emu.swiglu_f8_backward(x[:, :128], q, s[:, :1]), "hs")]:
        with pytest.raises(RuntimeError, match=msg):
            call()
