"""GPU tier: products with an epilogue, the gradient of an activation and its bias, and dropout
against float64 and against the generator's definition; the layer with all of it through
autograd; other streams, captured graphs, refusals."""
import pytest
import torch

import fp64_emu
from fp64_emu import capi
from f8_block_util import (ACTS, F64, U, act, act_error, close, close_codes, factors, kept, randn, rng, slope, slope_error)
from f8_util import E4M3, E5M2, operand, product_bound, quantised, same_codes, values

pytestmark = pytest.mark.gpu

BF16, FP16, F32 = torch.bfloat16, torch.float16, torch.float32
CODE = {F32: 0, BF16: 1, FP16: 2}


# ---- Products with an epilogue.

# Members, M, N, K and the form they are there for: (tile_m, tile_n, splits or not).
MM = [((16, 16, False), 1, 5, 130, 1000), ((16, 16, True), 1, 16, 64, 65536), ((32, 32, False), 1, 20, 97, 1023),
      ((64, 32, True), 1, 257, 513, 1025), ((128, 128, False), 1, 1000, 1101, 300), ((128, 128, True), 1, 1000, 1001, 8000),
      ((128, 128, False), 5, 513, 700, 600)]
MM16 = MM + [((256, 256, False), 1, 3001, 3010, 2900), ((256, 256, False), 1, 4096, 4096, 1024),
             ((256, 256, True), 1, 2000, 2101, 8200), ((256, 256, False), 64, 512, 512, 512)]
MM32 = MM + [((128, 256, False), 1, 2000, 2101, 8200), ((128, 256, False), 2, 1500, 1501, 6000)]


def _product(case, dtype, name, parts, dev, tiles=True, fa=E4M3, fb=E4M3, seed=0):
    form, batch, M, N, K = case
    plan = capi.mm_f8_plan(M, N, K, CODE[dtype], batch)
    if form:
        assert (plan.tile_m, plan.tile_n, plan.splits > 1) == form
    lead = (batch,) if batch > 1 else ()
    qa, sa = operand((*lead, M, K), seed + 1, fa, device=dev)
    qb, sb = operand((*lead, N, K), seed + 2, fb, tiles, device=dev)
    if "small" in parts or name in ("silu", "gelu", "gelu_tanh"):       # (where the activation is curved)
        sb = sb / (8 * K ** 0.5)
    kw = {"act": name, "keep": "keep" in parts, "out_dtype": dtype}
    if "bias" in parts:
        kw["bias"] = randn(*(lead if "biases" in parts else ()), N, seed=seed + 3).to(dev)
    if "residual" in parts:
        kw["residual"] = randn(*lead, M, N, seed=seed + 4, dtype=dtype, scale=2.0).to(dev)
    fn = fp64_emu.bmm_f8 if lead else fp64_emu.mm_f8
    got = fn(qa, sa, qb, sb, **kw)
    got, kept_h = got if kw["keep"] else (got, None)
    A, B = values(qa, sa), values(qb, sb)
    h = A @ B.transpose(-1, -2).contiguous()
    herr = product_bound(A, B, h, F32, bool(plan.exact))
    if "bias" in kw:
        h = h + kw["bias"].to(F64).unsqueeze(-2)
        herr = herr + U * h.abs()
    if kept_h is not None:
        assert kept_h.dtype == dtype
        close(kept_h, h, herr)
    # The activation of h moved by herr: by its slope (at most 1.13 but for relu2's) and curvature (below 2).
    steep = 2 * (h.abs() + herr) if name == "relu2" else torch.full_like(h, 1.13)
    y, err = act(h, name), steep * herr + 2 * herr * herr + act_error(h, name)
    if "residual" in kw:
        y = y + kw["residual"].to(F64)
        err = err + U * y.abs()
    assert got.shape == h.shape and got.dtype == dtype
    close(got, y, err)
    return got


@pytest.mark.parametrize("name", ACTS)
@pytest.mark.parametrize("case", MM16)
def test_epilogue(dev, case, name):
    dtype = (BF16, FP16)[(case[2] + ACTS.index(name)) % 2]
    print("case epilogue", case, name, dtype, flush=True)
    parts = ("bias residual keep", "bias biases keep", "bias residual", "residual")[(case[3] + ACTS.index(name)) % 4]
    _product(case, dtype, name, parts, dev, tiles=bool(case[4] % 3))


@pytest.mark.parametrize("name", ACTS)
@pytest.mark.parametrize("case", MM32)
def test_epilogue_float32(dev, case, name):
    print("case epilogue float32", case, name, flush=True)
    parts = ("bias residual keep", "bias biases keep", "bias residual", "residual")[(case[2] + ACTS.index(name)) % 4]
    _product(case, F32, name, parts, dev, tiles=not case[4] % 3)


@pytest.mark.parametrize("parts", ["bias", "residual", "keep", "bias keep", "bias residual keep"])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("M,N,K", [(1, 3, 200), (30, 70, 300), (300, 515, 257), (1100, 1031, 129)])
def test_epilogue_parts(dev, M, N, K, dtype, parts):
    """Any of the parts alone, at odd sizes."""
    print("case epilogue parts", M, N, K, dtype, parts, flush=True)
    _product((None, 1, M, N, K), dtype, None, parts, dev, tiles=False)


@pytest.mark.parametrize("fa,fb", [(E5M2, E4M3), (E4M3, E5M2), (E5M2, E5M2)])
@pytest.mark.parametrize("M,N,K", [(5, 130, 300), (1000, 1101, 300)])
def test_epilogue_formats(dev, M, N, K, fa, fb):
    print("case epilogue formats", M, N, K, fa, fb, flush=True)
    for dtype in (BF16, F32):
        _product((None, 1, M, N, K), dtype, "relu", "bias residual keep small", dev, fa=fa, fb=fb)


def test_epilogue_depth_of_none(dev):
    """An empty sum: act(bias) + residual."""
    print("case epilogue depth 0", flush=True)
    q, s = torch.empty(7, 0, device=dev, dtype=E4M3), torch.empty(7, 0, device=dev)
    bias, res = randn(7, seed=1).to(dev), randn(7, 7, seed=2).to(dev)
    y, h = fp64_emu.mm_f8(q, s, q, s, torch.float32, bias=bias, act="relu", residual=res, keep=True)
    assert torch.equal(h, bias.expand(7, 7)) and torch.equal(y, bias.clamp_min(0) + res)


@pytest.mark.parametrize("M,N,K", [(20, 50, 300), (1000, 1101, 300)])
def test_epilogue_layouts(dev, M, N, K):
    """Residuals with rows apart, at odd places, transposed and expanded; a bias of stride 2 and of each type."""
    print("case epilogue layouts", M, N, K, flush=True)
    qa, sa = operand((M, K), 1, device=dev)
    qb, sb = operand((N, K), 2, tiles=True, device=dev)
    bias, res = randn(N, seed=3, dtype=BF16).to(dev), randn(M, N, seed=4, dtype=BF16).to(dev)
    call = lambda b, r: fp64_emu.mm_f8(qa, sa, qb, sb, bias=b, residual=r)  # noqa: E731
    want = call(bias, res)
    assert torch.equal(call(torch.stack([bias, bias], 1)[:, 1], res.t().contiguous().t()), want)
    assert torch.equal(call(bias.float(), torch.nn.functional.pad(res, (3, 4))[:, 3:3 + N]), want)
    row = res[:1]
    assert torch.equal(call(bias, row.expand(M, N)), call(bias, row.expand(M, N).contiguous()))


def test_epilogue_writes_nothing_beside(dev):
    """Rows past a product's last and columns past its width stay as they were (the C entry point)."""
    print("case epilogue beside", flush=True)
    import ctypes
    L = capi.lib()
    for M, N, K in ((5, 37, 300), (300, 301, 640), (1000, 1101, 300)):
        qa, sa = operand((M, K), 1, device=dev)
        qb, sb = operand((N, K), 2, device=dev)
        room = torch.full((2, M + 3, N + 5), 7.0, dtype=BF16, device=dev)
        bias = randn(N, seed=3).to(dev)
        f8 = lambda q, s: capi.F8(q.data_ptr(), s.data_ptr(), K, 0, s.stride(0), s.stride(1), 0, 0, 0)  # noqa: E731
        p = capi.MmF8(room[0].data_ptr(), N + 5, 0, 1, 0, f8(qa, sa), f8(qb, sb), 1, M, N, K)
        e = capi.Epilogue(bias.data_ptr(), None, room[1].data_ptr(), 0, 0, 0, N + 5, 0, 0, 3)
        need = L.fp64emu_mm_f8_epilogue_workspace(ctypes.byref(p), ctypes.byref(e))
        ws = torch.empty(max(need, 1), dtype=torch.uint8, device=dev)
        st = L.fp64emu_mm_f8_epilogue(ctypes.byref(p), ctypes.byref(e), ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream)
        assert st == 0, L.fp64emu_last_error()
        y, h = fp64_emu.mm_f8(qa, sa, qb, sb, bias=bias, act="silu", keep=True)
        for i, t in enumerate((y, h)):
            assert torch.equal(room[i, :M, :N], t) and (room[i, M:] == 7).all() and (room[i, :, N:] == 7).all()


def test_epilogue_residual_in_place(dev):
    """The residual may be the output itself (the C entry point)."""
    print("case epilogue in place", flush=True)
    import ctypes
    L = capi.lib()
    for M, N, K in ((5, 40, 300), (16, 64, 65536), (1000, 1104, 300)):
        qa, sa = operand((M, K), 1, device=dev)
        qb, sb = operand((N, K), 2, device=dev)
        res = randn(M, N, seed=3, dtype=BF16).to(dev)
        want, out = fp64_emu.mm_f8(qa, sa, qb, sb, residual=res), res.clone()
        f8 = lambda q, s: capi.F8(q.data_ptr(), s.data_ptr(), K, 0, s.stride(0), s.stride(1), 0, 0, 0)  # noqa: E731
        p = capi.MmF8(out.data_ptr(), N, 0, 1, 0, f8(qa, sa), f8(qb, sb), 1, M, N, K)
        e = capi.Epilogue(None, out.data_ptr(), None, 0, N, 0, 0, 0, 0, 0)
        need = L.fp64emu_mm_f8_epilogue_workspace(ctypes.byref(p), ctypes.byref(e))
        ws = torch.empty(max(need, 1), dtype=torch.uint8, device=dev)
        assert L.fp64emu_mm_f8_epilogue(ctypes.byref(p), ctypes.byref(e), ws.data_ptr(), need,
                                        torch.cuda.current_stream().cuda_stream) == 0
        assert torch.equal(out, want)


# ---- Activations at their ends, by products of one code each: 1 x h.

@pytest.mark.parametrize("name", ACTS[1:])
def test_activation_values(dev, name):
    """From far below zero to far above, zeros, infinities and NaN."""
    print("case activation values", name, flush=True)
    h = torch.cat([torch.linspace(-30, 30, 1201), torch.tensor([0.0, -0.0, 1e-30, -1e-30, 88.0, -88.0, 1e4, -1e4, 1e18, -1e18])]).to(dev)
    n = h.numel()
    q, s = torch.zeros(3, 16, device=dev, dtype=E4M3), torch.ones(3, 1, device=dev)
    w, t = torch.zeros(n, 16, device=dev, dtype=E4M3), torch.ones(n, 1, device=dev)
    y, kept_h = fp64_emu.mm_f8(q, s, w, t, torch.float32, bias=h, act=name, keep=True)
    assert torch.equal(kept_h[1], h)
    wide = h.to(F64)
    close(y[2], act(wide, name), act_error(wide, name) + 2.0 ** -126)
    d, = fp64_emu.act_f8_backward(torch.ones(3, n, device=dev), h.expand(3, n), name)
    close(d[1], slope(wide, name), slope_error(wide, name) + 2.0 ** -126)
    ends = torch.tensor([float("inf"), float("nan")], device=dev)
    y = fp64_emu.mm_f8(q, s, w[:2], t[:2], torch.float32, bias=ends, act=name)
    assert y[0, 0] == float("inf") and torch.isnan(y[0, 1])


@pytest.mark.parametrize("name", ["silu", "gelu_tanh"])
def test_slopes_near_one(dev, name):
    """Where sigmoid(u) nears 1 what is left of 1 keeps its own accuracy.  In roundings U of 2^-24: u of gelu_tanh is off by 6 of
    itself, e^-u by 4 and u's, sigmoid by 3 and (1 - s) of e^-u's, s (1 - s) by 8 and e^-u's, gelu_tanh's derivative of u by 4, products and
    sums by one each; up to u = 2, where it is taken from 1, 1 - s by what s is.  So taken everywhere, slopes were off by 31 U
    (gelu_tanh) and 8.5 U (silu) past h = 4."""
    print("case slopes near one", name, flush=True)
    h = torch.linspace(-8, 8, 2 ** 20 + 1).to(dev)[None]
    got, = fp64_emu.act_f8_backward(torch.ones_like(h), h, name)
    x = h.to(F64)
    want = slope(x, name)
    if name == "silu":
        s = torch.sigmoid(x)
        err = 6 * want.abs() + s * (1 - s) * (8 * x.abs() + 4) + (x <= 2) * x.abs() * s * s * (3 + 4 * (1 - s))
    else:
        c = 2 * (2 / torch.pi) ** 0.5
        u, du = c * (x + 0.044715 * x ** 3), c * (1 + 3 * 0.044715 * x * x)
        s, rest = torch.sigmoid(u), torch.sigmoid(-u)
        err = 2 * want.abs() + 3 * s + s * rest * ((6 * u.abs() + 4) + x.abs() * du * (6 * u.abs() + 17))
        err += (u <= 2) * x.abs() * du * s * s * (3 + rest * (6 * u.abs() + 4))
    assert ((got.to(F64) - want).abs() <= U * err).all()


@pytest.mark.parametrize("name", ["silu", "gelu", "gelu_tanh"])
def test_slopes_far_out(dev, name):
    """From far out on slopes are 1 and 0, however large h (an e^-u that is not quite 0 would be multiplied by it)."""
    print("case slopes far out", name, flush=True)
    h = torch.tensor([2.0 ** i for i in range(7, 128)]).to(dev)[None]
    for sign, want in ((1, 1.0), (-1, 0.0)):
        got, = fp64_emu.act_f8_backward(torch.ones_like(h), sign * h, name)
        assert torch.equal(got, torch.full_like(got, want))


# ---- The gradient of an activation and its bias.

GRAD = [(1, 1), (1, 300), (5, 17), (16, 128), (17, 129), (333, 777), (130, 1000), (300, 256), (2100, 264)]


@pytest.mark.parametrize("name", ACTS)
@pytest.mark.parametrize("M,N", GRAD)
def test_act_gradient(dev, M, N, name):
    dtype = (BF16, FP16, F32)[(M + ACTS.index(name)) % 3]
    print("case act gradient", M, N, name, dtype, flush=True)
    dy, h = randn(M, N, seed=1, dtype=dtype).to(dev), randn(M, N, seed=2, dtype=dtype, scale=3.0).to(dev)
    if M > 4:
        h[2:4] = 0
    wide, at = dy.to(F64), h.to(F64)
    want = wide * slope(at, name)
    err = wide.abs() * slope_error(at, name) + U * want.abs()
    sums, sum_err = want.sum(0), err.sum(0) + U * M * (want.abs() + err).sum(0)
    plain, db = fp64_emu.act_f8_backward(dy, h, name, bias=True)
    close(plain, want, err)
    close(db, sums, sum_err)
    q, s, db = fp64_emu.act_f8_backward(dy, h, name, "rows", bias=True)
    close_codes(q, s, want, err)
    close(db, sums, sum_err)
    q, s, qt, st, db = fp64_emu.act_f8_backward(dy, h, name, "both", bias=True)
    close_codes(q, s, want, err)
    close_codes(qt, st, want.t().contiguous(), err.t().contiguous())
    close(db, sums, sum_err)
    alone = fp64_emu.act_f8_backward(dy, h, name, "both")
    assert len(alone) == 4 and all(torch.equal(a.float(), b.float()) for a, b in zip(alone, (q, s, qt, st)))
    if name is None:
        assert torch.equal(plain, dy) and same_codes(q, quantised(dy, E4M3)[0])
        assert torch.equal(fp64_emu.act_f8_backward(dy, bias=True)[1], fp64_emu.act_f8_backward(dy, h, bias=True)[1])


@pytest.mark.parametrize("name", ACTS[1:])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_act_gradient_in_float32(dev, dtype, name):
    """16-bit operands are float32 values: codes, scales and dbias have the bits that the same values in float32 give,
    the plain gradient theirs rounded."""
    print("case act gradient in float32", dtype, name, flush=True)
    for M, N in ((5, 300), (700, 520)):
        dy, h = randn(M, N, seed=1, dtype=dtype).to(dev), randn(M, N, seed=2, dtype=dtype, scale=3.0).to(dev)
        for quant in ("rows", "both", None):
            got = fp64_emu.act_f8_backward(dy, h, name, quant, bias=True)
            want = fp64_emu.act_f8_backward(dy.float(), h.float(), name, quant, bias=True)
            if quant is None:
                want = (want[0].to(dtype), want[1])
            assert _same(got, want), (M, N, quant)


@pytest.mark.parametrize("M,N,K,ld", [(3, 264, 300, 2 ** 30 + 8), (1000, 1101, 300, 2 ** 22 + 8)])
def test_far_offsets(dev, M, N, K, ld):
    """Rows whose elements lie past 2^31 elements (and 2^32 bytes) from the first."""
    print("case far offsets", M, N, K, ld, flush=True)
    buf = torch.zeros((M - 1) * ld + N, dtype=BF16, device=dev)
    far = buf.as_strided((M, N), (ld, 1))
    near, h = (randn(M, N, seed=i, dtype=BF16).to(dev) for i in (96, 97))
    far.copy_(near)
    qa, sa = operand((M, K), 1, device=dev)
    qb, sb = operand((N, K), 2, device=dev)
    assert torch.equal(*(fp64_emu.mm_f8(qa, sa, qb, sb, act="relu", residual=t) for t in (far, near)))
    state = rng(5, 6, dev)
    for quant in (None, "rows", "both"):
        for call in (lambda t: fp64_emu.act_f8_backward(t, h, "silu", quant, bias=True),
                     lambda t: fp64_emu.act_f8_backward(h, t, "silu", quant, bias=True),
                     lambda t: fp64_emu.dropout_f8(t, 0.3, state, quant)):
            assert all(torch.equal(u.float(), v.float()) for u, v in zip(call(far), call(near)))


def test_act_gradient_layouts(dev):
    print("case act gradient layouts", flush=True)
    M, N = 150, 200
    dy, h = randn(M, N, seed=1, dtype=BF16).to(dev), randn(M, N, seed=2, dtype=BF16).to(dev)
    for quant in (None, "rows", "both"):
        want = fp64_emu.act_f8_backward(dy, h, "silu", quant, bias=True)
        for a, b in ((torch.nn.functional.pad(dy, (3, 8))[:, 3:203], torch.nn.functional.pad(h, (1, 2))[:, 1:201]),
                     (dy.t().contiguous().t(), h.t().contiguous().t())):
            got = fp64_emu.act_f8_backward(a, b, "silu", quant, bias=True)
            assert all(torch.equal(u.float(), v.float()) for u, v in zip(got, want))
    one = dy[:1].expand(M, N)
    for u, v in zip(fp64_emu.act_f8_backward(one, h, "silu", bias=True), fp64_emu.act_f8_backward(one.contiguous(), h, "silu", bias=True)):
        assert torch.equal(u, v)


def test_act_gradient_empty(dev):
    none = torch.empty(0, 40, device=dev)
    out = fp64_emu.act_f8_backward(none, none, "silu", "both", bias=True)
    assert [tuple(t.shape) for t in out] == [(0, 40), (0, 1), (40, 0), (40, 0), (40,)] and not out[-1].any()
    none = torch.empty(5, 0, device=dev)
    assert [tuple(t.shape) for t in fp64_emu.act_f8_backward(none, none, "silu", bias=True)] == [(5, 0), (0,)]


# ---- Dropout.

@pytest.mark.parametrize("p", [0.0, 2.0 ** -16, 0.1, 0.5, 1 - 2.0 ** -16])
@pytest.mark.parametrize("M,K", [(1, 1), (3, 7), (16, 128), (5, 300), (150, 257), (129, 1000)])
def test_dropout(dev, M, K, p):
    """The generator's mask, and the kept values rounded once; what is quantised is the float32 values."""
    print("case dropout", M, K, p, flush=True)
    seed, offset = 2 ** 62 + M, -3 + K
    state, drop = rng(seed, offset, dev), round(p * 65536)
    mask = kept(seed, offset, drop, M, K).to(dev)
    for dtype in (BF16, FP16, F32):
        x = randn(M, K, seed=K, dtype=dtype).to(dev)
        want = torch.where(mask, x.float() * torch.tensor(65536 / (65536 - drop), device=dev), 0.0)
        y, = fp64_emu.dropout_f8(x, p, state)
        assert y.dtype == dtype and torch.equal(y, want.to(dtype))
        q, s = fp64_emu.dropout_f8(x, p, state, "rows")
        qr, sr, qt, st = fp64_emu.dropout_f8(x, p, state, "both")
        for t, a, b in ((want, q, s), (want, qr, sr), (want.t(), qt, st)):
            wq, ws = quantised(t, E4M3)
            assert same_codes(a, wq) and torch.equal(b.cpu(), ws)


def test_dropout_share(dev):
    """Of 2^24 elements the share that is dropped is within five deviations of p, for each of the
    eight places of a chunk, and so is that of neighbours dropped together; another offset, another mask."""
    print("case dropout share", flush=True)
    x = torch.ones(4096, 4096, device=dev, dtype=BF16)
    state = rng(123, 0, dev)
    for p in (0.1, 0.5):
        gone = fp64_emu.dropout_f8(x, p, state)[0] == 0
        n = gone.numel()
        assert abs(gone.double().mean().item() - p) < 5 * (p * (1 - p) / n) ** 0.5 + 2.0 ** -17
        for j in range(8):
            assert abs(gone[:, j::8].double().mean().item() - p) < 5 * (p * (1 - p) * 8 / n) ** 0.5 + 2.0 ** -17
        both = (gone[:, 1:] & gone[:, :-1]).double().mean().item()
        assert abs(both - p * p) < 5 * (2 * p * p / n) ** 0.5 + 2.0 ** -15
        state += torch.tensor([0, 1], device=dev)
        other = fp64_emu.dropout_f8(x, p, state)[0] == 0
        assert abs((gone & other).double().mean().item() - p * p) < 5 * (2 * p * p / n) ** 0.5 + 2.0 ** -15


def test_dropout_layouts_and_values(dev):
    print("case dropout layouts", flush=True)
    x, state = randn(50, 200, seed=1).to(dev), rng(1, 2, dev)
    y, = fp64_emu.dropout_f8(x, 0.5, state)
    for t in (x.t().contiguous().t(), torch.nn.functional.pad(x, (3, 2))[:, 3:203]):
        assert torch.equal(fp64_emu.dropout_f8(t, 0.5, state)[0], y)
    z = torch.where(y == 0, float("nan"), x)
    assert torch.equal(fp64_emu.dropout_f8(z, 0.5, state)[0], y)
    assert fp64_emu.dropout_f8(x[:0], 0.5, state, "both")[2].shape == (200, 0)
    assert torch.equal(fp64_emu.dropout_f8(x, 0.0, None)[0], x)


def test_seeded_dropout(dev):
    """The gradient has the call's own mask, though rng goes on in place."""
    print("case seeded dropout", flush=True)
    x, state = randn(3, 5, 40, seed=1).to(dev).requires_grad_(), rng(7, 0, dev)
    y = fp64_emu.seeded_dropout_f8(x, 0.25, state)
    state += 1
    dy = randn(3, 5, 40, seed=2).to(dev)
    g, = torch.autograd.grad(y, x, dy, create_graph=True)
    k = factors(7, 0, 0.25, 15, 40).view(3, 5, 40).float().to(dev)
    assert torch.equal(g, dy * k) and torch.equal(y, x.detach() * k)
    with torch.no_grad():
        assert fp64_emu.seeded_dropout_f8(x, 0.25, state).grad_fn is None


# ---- The layer.

@pytest.mark.parametrize("name", ACTS)
@pytest.mark.parametrize("shape,N", [((1, 300), 200), ((5, 17, 256), 130), ((200, 777), 501)])
def test_linear_epilogue(dev, shape, N, name):
    """Output and gradients, given the operands' codes: the 8-bit forms are the quantiser's own, so what is left is
    the products' errors and what the quantised dh is off by, 2^-4 of an element at most."""
    print("case linear epilogue", shape, N, name, flush=True)
    K = shape[-1]
    x = randn(*shape, seed=1).to(dev).requires_grad_()
    w = randn(N, K, seed=2, scale=K ** -0.5).to(dev).requires_grad_()
    b = randn(N, seed=3, scale=0.5).to(dev).requires_grad_()
    r = randn(*shape[:-1], N, seed=4).to(dev).requires_grad_()
    y = fp64_emu.linear_f8(x, w, bias=b, act=name, residual=r)
    dy = randn(*y.shape, seed=5).to(dev)
    got = torch.autograd.grad(y, (x, w, b, r), dy)
    with torch.no_grad():
        rows = x.reshape(-1, K)
        q, s, qt, st = fp64_emu.quant_f8(rows, cols=True)
        wq = fp64_emu.quant_f8_tiles(w, transposed=True)
        out, h = fp64_emu.mm_f8(q, s, *wq[:2], F32, bias=b, act=name, residual=r.reshape(-1, N), keep=True)
        assert torch.equal(out.view(y.shape), y)
        dq, ds, dqt, dst, db = fp64_emu.act_f8_backward(dy.reshape(-1, N), h, name, "both", bias=True)
        assert torch.equal(got[0].reshape(-1, K), fp64_emu.mm_f8(dq, ds, *wq[2:], F32))
        assert torch.equal(got[1], fp64_emu.mm_f8(dqt, dst, qt, st, F32))
        assert torch.equal(got[2], db) and torch.equal(got[3], dy)
    # Beside float64: each operand off by about 2.6% in norm, a product by 3.7%, dh's argument by 3.7% of h: 12%.
    wide = [t.detach().double().requires_grad_() for t in (x, w, b, r)]
    full = act(wide[0] @ wide[1].t() + wide[2], name) + wide[3]
    want = torch.autograd.grad(full, wide, dy.double())
    # relu's slope jumps: h off by 3.7% of its deviation changes sign with a probability of E|error| times the density
    # at 0, 0.037 0.8 0.4 = 1.2%, and of the half that is on that is sqrt(0.012 / 0.5) = 15.4% in norm: with 12% 20%.
    for u, v in zip((y, *got), (full, *want)):
        assert (u.double() - v).norm() <= (0.20 if name == "relu" else 0.12) * v.norm()


@pytest.mark.parametrize("needs", ["x", "w", "b", "r", "xb", "wb", ""])
def test_linear_epilogue_needs(dev, needs):
    """Any of the leaves alone has the gradient that all of them have (the bias's in another order of its 30
    terms of at most 1.2 |dy|, where dh is not asked for both ways)."""
    print("case linear needs", needs, flush=True)
    t = {n: randn(*s, seed=i).to(dev) for i, (n, s) in enumerate({"x": (30, 200), "w": (70, 200), "b": (70,), "r": (30, 70)}.items())}
    full = {n: v.clone().requires_grad_() for n, v in t.items()}
    some = {n: v.clone().requires_grad_(n in needs) for n, v in t.items()}
    call = lambda t: fp64_emu.linear_f8(t["x"], t["w"], bias=t["b"], act="gelu", residual=t["r"])  # noqa: E731
    dy = randn(30, 70, seed=9).to(dev)
    want = dict(zip(full, torch.autograd.grad(call(full), list(full.values()), dy)))
    y = call(some)
    assert y.requires_grad == bool(needs)
    if needs:
        for n, g in zip(needs, torch.autograd.grad(y, [some[n] for n in needs], dy)):
            room = 2 * 30 * U * 1.2 * dy.abs().sum(0) if n == "b" else torch.zeros((), device=dev)
            assert ((g - want[n]).abs() <= room).all()
    b = t["b"].to(BF16).requires_grad_()
    g, = torch.autograd.grad(fp64_emu.linear_f8(t["x"], t["w"], bias=b), b, dy)
    assert g.dtype == BF16
    close(g, dy.to(F64).sum(0), 30 * U * dy.to(F64).abs().sum(0))


def test_together(dev):
    """Two blocks as a model runs them: norm, layer, activation, layer, and the next block's norm with the
    first's output, dropped; through autograd against float64 with the same masks."""
    print("case together", flush=True)
    M, D, F = 70, 256, 384
    g = lambda *s, seed, scale=1.0: randn(*s, seed=seed, scale=scale).to(dev).requires_grad_()  # noqa: E731
    r, w0, w1, po, ga = (g(M, D, seed=1), *(g(D, seed=i) for i in (2, 3, 4, 5)))
    u, bu, d, bd = g(F, D, seed=6, scale=D ** -0.5), g(F, seed=7, scale=0.1), g(D, F, seed=8, scale=F ** -0.5), g(D, seed=9, scale=0.1)
    leaves = (r, w0, w1, po, ga, u, bu, d, bd)
    state = rng(31, 0, dev)
    x = fp64_emu.residual_norm_f8(r, w0)
    h = fp64_emu.seeded_dropout_f8(fp64_emu.linear_f8(x, u, bias=bu, act="gelu_tanh"), 0.125, state)
    y = fp64_emu.linear_f8(h, d, bias=bd)
    new, out = fp64_emu.residual_norm_f8(r, w1, y, po, ga, p=0.25, rng=state)
    a, b = randn(M, D, seed=10).to(dev), randn(M, D, seed=11).to(dev)
    got = torch.autograd.grad((new, out), leaves, (a, b))
    r2, w02, w12, po2, ga2, u2, bu2, d2, bd2 = wide = [t.detach().double().requires_grad_() for t in leaves]
    k1, k2 = factors(31, 0, 0.125, M, F).to(dev), factors(31, 0, 0.25, M, D).to(dev)
    rms = lambda v: (v.square().mean(-1, keepdim=True) + 1e-6).rsqrt()  # noqa: E731
    h2 = act(r2 * rms(r2) * w02 @ u2.t() + bu2, "gelu_tanh") * k1
    y2 = h2 @ d2.t() + bd2
    new2 = r2 + ga2 * k2 * (y2 * rms(y2) * po2)
    out2 = new2 * rms(new2) * w12
    want = torch.autograd.grad((new2, out2), wide, (a.double(), b.double()))
    for s, t in zip((new, out, *got), (new2, out2, *want)):
        # two products one after the other and back: four of 3.7% and the slopes between them
        assert (s.double() - t).norm() <= 0.15 * t.norm(), (s.double() - t).norm() / t.norm()


# ---- Streams, graphs, refusals.

def _everything(t):
    """Every operator once."""
    got = list(fp64_emu.norm_f8(t["r"], t["w"], t["y"], t["w"], t["w"], 0.5, 0.25, t["rng"], "both", keep=True))
    got += fp64_emu.norm_f8(t["r"], t["w"], t["y"], t["w"], t["w"], 0.5, 0.25, t["rng"])
    got += [v for v in fp64_emu.norm_f8_backward(t["y"], t["r"], got[0], t["w"], got[5], t["y"], t["w"], t["w"], 0.5, 0.25, t["rng"])]
    got += fp64_emu.mm_f8(*got[1:3], t["q"], t["s"], bias=t["b"], act="silu", residual=t["res"], keep=True)
    got += fp64_emu.act_f8_backward(got[-2], got[-1], "silu", "both", bias=True)
    got += fp64_emu.dropout_f8(t["y"], 0.5, t["rng"], "both")
    return got


def _state(dev, M=700, D=520, seed=0):
    q, s = operand((300, D), seed + 9, tiles=True, device=dev)
    return {"r": randn(M, D, seed=seed + 1, dtype=BF16).to(dev), "y": randn(M, D, seed=seed + 2, dtype=BF16).to(dev),
            "w": randn(D, seed=seed + 3).to(dev), "b": randn(300, seed=seed + 4).to(dev), "q": q, "s": s,
            "res": randn(M, 300, seed=seed + 5, dtype=BF16).to(dev), "rng": rng(3, 5 + seed, dev)}


def _same(a, b):
    return len(a) == len(b) and all(torch.equal(u.float(), v.float()) for u, v in zip(a, b))


def test_block_other_stream(dev):
    print("case block stream", flush=True)
    t = _state(dev)
    want = _everything(t)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = _everything(t)
    side.synchronize()
    assert _same(got, want)


def test_block_graph_replays(dev):
    """Two captured graphs, replayed in turn with other inputs, masks that go on in place, and eager work
    between them: every replay gives the eager results."""
    print("case block graphs", flush=True)
    states = [_state(dev), _state(dev, M=130, D=1500, seed=50)]
    for t in states:
        _everything(t)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for t in states:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(_everything(t))
        graphs.append(graph)
    for turn in range(3):
        for t in states:
            t["y"].mul_(0.5)
            t["rng"] += 1
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for t, out in zip(states, outs):
            assert _same(out, _everything(t)), turn
        torch.cuda.synchronize()


def test_block_refusals(dev):
    x, w = torch.zeros(4, 64, device=dev), torch.zeros(64, device=dev)
    q, s = operand((4, 64), 1, device=dev)
    for call in (lambda: fp64_emu.mm_f8(q, s, q, s, bias=w), lambda: fp64_emu.mm_f8(q, s, q, s, bias=w[:4].cpu()),
                 lambda: fp64_emu.mm_f8(q, s, q, s, bias=w[:4].double()), lambda: fp64_emu.mm_f8(q, s, q, s, residual=x),
                 lambda: fp64_emu.mm_f8(q, s, q, s, residual=x[:, :4]), lambda: fp64_emu.mm_f8(q, s, q, s, bias=x[:, :4]),
                 lambda: fp64_emu.mm_f8(q, s, q, s, residual=torch.zeros(4, 4, dtype=BF16)),
                 lambda: fp64_emu.bmm_f8(q[None], s[None], q[None], s[None], bias=x[:2, :4]),
                 lambda: fp64_emu.act_f8_backward(x, x.half(), "silu"), lambda: fp64_emu.act_f8_backward(x, x.cpu(), "silu"),
                 lambda: fp64_emu.act_f8_backward(x.double(), x.double(), "silu"), lambda: fp64_emu.dropout_f8(x.double(), 0.0, None),
                 lambda: fp64_emu.dropout_f8(x, 0.5, torch.zeros(2, dtype=torch.int64)),
                 lambda: fp64_emu.dropout_f8(x, 0.5, torch.zeros(2, dtype=torch.int32, device=dev)),
                 lambda: fp64_emu.dropout_f8(x, 0.5, torch.zeros(4, dtype=torch.int64, device=dev)[::2])):
        with pytest.raises(RuntimeError):
            call()
    leaf = x.clone().requires_grad_()
    for call in (lambda: fp64_emu.act_f8_backward(leaf, x, "silu")[0], lambda: fp64_emu.dropout_f8(leaf, 0.0, None)[0],
                 lambda: fp64_emu.mm_f8(q, s, q, s, F32, bias=leaf[0, :4])):
        with pytest.raises(RuntimeError):
            call().sum().backward()


@pytest.mark.parametrize("shape,N", [((0, 256), 70), ((5, 0), 70), ((2, 0, 128), 40), ((3, 128), 0)])
def test_linear_epilogue_of_nothing(dev, shape, N):
    """No rows, no depth, no columns: an empty sum's epilogue and gradients of zeros."""
    print("case linear of nothing", shape, N, flush=True)
    K = shape[-1]
    x, w, b = (torch.ones(s, device=dev).requires_grad_() for s in (shape, (N, K), (N,)))
    r = torch.ones(*shape[:-1], N, device=dev).requires_grad_()
    y = fp64_emu.linear_f8(x, w, bias=b, act="relu", residual=r)
    assert y.shape == r.shape and (K != 0 or torch.equal(y, torch.full_like(y, 2.0)))
    grads = torch.autograd.grad(y, (x, w, b, r), torch.ones_like(y))
    assert [g.shape for g in grads] == [t.shape for t in (x, w, b, r)]
    assert torch.equal(grads[2], torch.full_like(b, float(y.numel() // max(N, 1)))) and not grads[1].any()


@pytest.mark.parametrize("lead", [(6,), (2, 3), ()])
def test_results_in_place(dev, lead):
    """Results written in place before the backward pass: values and gradients of the same step out of place."""
    print("case results in place", lead, flush=True)
    x, w, v = randn(*lead, 256, seed=1).to(dev).requires_grad_(), randn(256, seed=2).to(dev), randn(64, 256, seed=3).to(dev).requires_grad_()
    state = rng(3, 4, dev)
    for call in (lambda: fp64_emu.seeded_dropout_f8(x, 0.5, state), lambda: fp64_emu.linear_f8(x, v, act="silu"),
                 lambda: fp64_emu.swiglu_ckpt_f8(x), lambda: fp64_emu.residual_norm_f8(x, w), lambda: fp64_emu.residual_norm_f8(x, w, x)[1]):
        a, b = call().mul(2.0), call().mul_(2.0)
        dy = randn(*a.shape, seed=5).to(dev)
        assert torch.equal(a, b) and torch.equal(*(torch.autograd.grad(t, x, dy)[0] for t in (a, b)))
    new, out = fp64_emu.residual_norm_f8(x, w, x)
    new.add_(1.0)                           # (kept, and therefore said)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(out, x, torch.ones_like(out))


@pytest.mark.parametrize("name", [None, "silu"])
def test_linear_bias_alone(dev, name):
    """Where the bias alone wants a gradient dh is not written; its sum is act_f8_backward's, of plain dh's order."""
    print("case linear bias alone", name, flush=True)
    x, w, b = randn(70, 200, seed=1).to(dev), randn(130, 200, seed=2).to(dev), randn(130, seed=3).to(dev).requires_grad_()
    y, dy = fp64_emu.linear_f8(x, w, bias=b, act=name), randn(70, 130, seed=4).to(dev)
    q, s = fp64_emu.quant_f8(x)
    _, h = fp64_emu.mm_f8(q, s, *fp64_emu.quant_f8_tiles(w), F32, bias=b.detach(), act=name, keep=True)
    assert torch.equal(torch.autograd.grad(y, b, dy)[0], fp64_emu.act_f8_backward(dy, h, name, bias=True)[1])


def test_expanded_operands_of_nothing(dev):
    """No rows, spread from a scalar, as the gradient of a sum over them comes."""
    print("case expanded operands of nothing", flush=True)
    x = torch.ones((), device=dev).expand(0, 256)
    w = torch.ones(256, device=dev)
    assert x.stride() == (0, 0)
    assert [t.shape for t in fp64_emu.quant_f8(x, cols=True)] == [(0, 256), (0, 2), (256, 0), (256, 0)]
    assert fp64_emu.dropout_f8(x, 0.5, rng(1, 2, dev))[0].shape == (0, 256)
    assert not fp64_emu.act_f8_backward(x, x, "silu", bias=True)[1].any()
    assert fp64_emu.norm_f8(x, w, x, gate=x)[1].shape == (0, 256)
    leaf = torch.ones(0, 256, device=dev).requires_grad_()
    for call in (lambda: fp64_emu.residual_norm_f8(leaf, w), lambda: fp64_emu.seeded_dropout_f8(leaf, 0.5, rng(1, 2, dev)),
                 lambda: fp64_emu.linear_f8(leaf, torch.ones(8, 256, device=dev), act="silu"), lambda: fp64_emu.swiglu_ckpt_f8(leaf)):
        g, = torch.autograd.grad(call().sum(), leaf)
        assert g.shape == leaf.shape
