"""CPU tier: the operators around the 8-bit products, without a GPU: the C entry points' refusals and
workspaces, the Python functions' refusals, fake tensors, and the tests' own plain forms."""
import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import fp64_emu
from fp64_emu import capi
from f8_block_util import ACTS, F64, act, factors, kept, norm, norm_grad, philox, slope
from f8_util import E4M3

EINVAL, EWORKSPACE = 1, 2
F32, BF16, F16 = 0, 1, 2
P = 0x1000            # a pointer that no call below gets as far as using
R = ctypes.byref


def _f8(rows, depth, fmt=0, tiles=0, q=P, s=P, ld=None):
    return capi.F8(q, s, depth if ld is None else ld, 0, 1, rows, 0, fmt, tiles)


def _says(status, part):
    text = capi.lib().fp64emu_last_error().decode()
    assert status in (EINVAL, EWORKSPACE) and part in text, (status, text, part)


def test_epilogue_refusals():
    L = capi.lib()

    def call(accumulate=0, fmt=0, M=256, ws=None, n=0, **kw):
        p = capi.MmF8(P, 256, 0, BF16, accumulate, _f8(M, 256, fmt), _f8(256, 256), 1, M, 256, 256)
        e = capi.Epilogue(kw.get("bias"), kw.get("residual"), kw.get("keep"), 0, kw.get("ldr", 256), 0,
                          kw.get("ldk", 256), 0, kw.get("bias_dtype", 0), kw.get("act", 0))
        return L.fp64emu_mm_f8_epilogue(R(p), R(e), ws, n, None), L.fp64emu_mm_f8_epilogue_workspace(R(p), R(e))

    _says(call(act=6)[0], "FP64EMU_ACT")
    _says(call(act=-1)[0], "FP64EMU_ACT")
    _says(call(bias_dtype=3)[0], "dtype must be")
    _says(call(accumulate=1)[0], "does not accumulate")
    _says(call(residual=P, ldr=255)[0], "shorter than N")
    _says(call(keep=P, ldk=255)[0], "shorter than N")
    # e5m2 operands on tiles pass their sums through the workspace.
    st, need = call(fmt=1, bias=P)
    assert st == EWORKSPACE and need == 4 * 256 * 256 and call(bias=P, M=0) == (0, 0)


def test_pointwise_refusals():
    L = capi.lib()

    def grad(dy=P, h=P, dtype=BF16, a=3, M=4, N=256, ld=256, ldh=256, dh=P, ldd=256, rows=None, cols=None, db=None, ws=None, n=0):
        return L.fp64emu_act_f8_backward(dy, h, dtype, a, M, N, ld, ldh, dh, ldd, rows and R(rows), cols and R(cols), db, ws, n, None)

    for kw, text in ((dict(M=-1), "non-negative"), (dict(N=1 << 31), "2^31"), (dict(dtype=5), "dtype must"),
                     (dict(a=9), "FP64EMU_ACT"), (dict(dh=None), "no output"), (dict(dy=None), "null"), (dict(h=None), "null"),
                     (dict(ld=255), "shorter"), (dict(ldh=255), "shorter"), (dict(ldd=255), "shorter"),
                     (dict(cols=_f8(256, 4)), "plain form"), (dict(dh=None, rows=_f8(4, 256, fmt=1)), "e4m3"),
                     (dict(dh=None, rows=_f8(4, 256, tiles=1)), "e4m3"), (dict(dh=None, rows=_f8(4, 256, ld=128)), "shorter"),
                     (dict(dh=None, rows=_f8(4, 256, q=None)), "null 8-bit"), (dict(M=1 << 40), "too large"),
                     (dict(M=400, db=P), "workspace too small"), (dict(M=400, db=P, ws=0x1002, n=1 << 20), "aligned")):
        _says(grad(**kw), text)
    assert grad(N=0) == 0 and grad(M=0) == 0
    assert L.fp64emu_act_f8_backward_workspace(16, 256, 0) == 0 and L.fp64emu_act_f8_backward_workspace(0, 256, 0) == 0
    assert L.fp64emu_act_f8_backward_workspace(300, 100, 1) == 4 * 3 * 100

    def drop(x=P, dtype=BF16, M=4, K=256, ld=256, d=100, rng=P, y=P, ldy=256, rows=None, cols=None):
        return L.fp64emu_dropout_f8(x, dtype, M, K, ld, d, rng, y, ldy, rows and R(rows), cols and R(cols), None)

    for kw, text in ((dict(M=-1), "non-negative"), (dict(dtype=5), "dtype must"), (dict(d=65536), "0 .. 65535"), (dict(d=-1), "0 .. 65535"),
                     (dict(rng=None), "needs rng"), (dict(y=None), "no output"), (dict(x=None), "null"), (dict(ld=255), "shorter"),
                     (dict(ldy=255), "shorter"), (dict(cols=_f8(256, 4)), "plain form"), (dict(rows=_f8(4, 256, fmt=1)), "e4m3"),
                     (dict(M=1 << 40), "too large")):
        _says(drop(**kw), text)
    assert drop(M=0) == 0 and drop(K=0, rng=None, d=0) == 0


def _norm(M=4, D=256, **kw):
    p = {"r": P, "y": P, "w": P, "post": P, "gate": P, "rng": P, "M": M, "D": D, "ld_r": D, "ld_y": D, "ld_gate": 0, "r_dtype": BF16,
         "y_dtype": BF16, "w_dtype": F32, "post_dtype": F32, "gate_dtype": F32, "drop": 0, "scale": 1.0, "eps": 1e-6, **kw}
    return capi.Norm(*(p[n] for n, _ in capi.Norm._fields_))


NORM_REFUSALS = [
    (dict(M=-1), "non-negative"), (dict(D=0), "no norm"), (dict(D=1 << 27), "2^27"), (dict(M=1 << 40), "2^40"), (dict(r_dtype=4), "dtype must"),
    (dict(w_dtype=4), "dtype must"), (dict(post_dtype=-1), "dtype must"), (dict(gate_dtype=3), "dtype must"),
    (dict(r_dtype=BF16, y_dtype=F32), "y's dtype"), (dict(r_dtype=F16, y_dtype=BF16), "y's dtype"), (dict(eps=0.0), "eps"), (dict(eps=1e-40), "eps"),
    (dict(eps=float("nan")), "eps"), (dict(drop=65536), "0 .. 65535"), (dict(drop=-1), "0 .. 65535"), (dict(y=None), "need y"),
    (dict(y=None, post=None, gate=None, drop=7), "need y"), (dict(drop=7, rng=None), "needs rng"), (dict(r=None), "null"),
    (dict(w=None), "null"), (dict(ld_r=255), "shorter than D"), (dict(ld_y=255), "shorter than D"),
    (dict(ld_gate=255), "rows of gate"), (dict(ld_gate=256), "y's dtype")]


def test_norm_refusals():
    L = capi.lib()

    def call(out=P, ldo=256, x=P, ldx=256, stats=P, rows=None, cols=None, **kw):
        return L.fp64emu_norm_f8(R(_norm(**kw)), out, ldo, x, ldx, stats, rows and R(rows), cols and R(cols), None)

    for kw, text in NORM_REFUSALS:
        _says(call(**kw), text)
    plain = dict(y=None, post=None, gate=None)
    for kw, text in ((dict(out=None, x=None, stats=None), "no output"), (dict(**plain), "needs y"), (dict(ldo=255), "shorter"),
                     (dict(ldx=255), "shorter"), (dict(cols=_f8(256, 4)), "plain form"),
                     (dict(x=None, stats=None, cols=_f8(256, 4)), "need stats"),
                     (dict(x=None, cols=_f8(256, 4)), "elsewhere"), (dict(rows=_f8(4, 256, fmt=1)), "e4m3"),
                     (dict(rows=_f8(4, 256, tiles=1)), "e4m3"), (dict(rows=_f8(4, 256, s=None)), "null 8-bit")):
        _says(call(**kw), text)
    assert call(M=0) == 0 and L.fp64emu_norm_f8(None, P, 1, P, 1, P, None, None, None) == EINVAL


def test_norm_grad_refusals():
    L = capi.lib()

    def call(stats=P, ws=None, n=0, grad={}, **kw):
        g = {**dict.fromkeys(("dx", "dr", "dr_out", "dy", "dw", "dpost", "dgate"), P), "dgates": None,
             **dict.fromkeys(("ld_dx", "ld_dr", "ld_dr_out", "ld_dy", "ld_dgates"), 256), **grad}
        return L.fp64emu_norm_f8_backward(R(_norm(**kw)), stats, R(capi.NormGrad(*(g[n] for n, _ in capi.NormGrad._fields_))), ws, n, None)

    for kw, text in NORM_REFUSALS:
        if kw.get("y", P) is not None:
            _says(call(ws=P, n=1 << 40, **kw), text)
    for kw, text in ((dict(stats=None), "null"), (dict(grad={"dx": None}), "null"), (dict(grad={"ld_dx": 255}), "shorter"),
                     (dict(grad={"ld_dr": 255}), "shorter"), (dict(grad={"ld_dr_out": 255}), "shorter"), (dict(grad={"ld_dy": 255}), "shorter"),
                     (dict(post=None), "absent"), (dict(gate=None), "absent"), (dict(grad={"dgates": P}), "a row or a matrix"),
                     (dict(grad={"dgates": P, "dgate": None}), "y's dtype"), (dict(y=None, post=None, gate=None), "absent"),
                     (dict(ld_gate=256, gate_dtype=BF16), "of one gate"),
                     (dict(gate_dtype=BF16, grad={"dgates": P, "dgate": None}), "of one gate"), (dict(M=300), "workspace too small"), (dict(M=300, ws=0x1002, n=1 << 30), "aligned")):
        _says(call(**kw), text)
    assert L.fp64emu_norm_f8_backward(R(_norm()), P, None, None, 0, None) == EINVAL
    assert L.fp64emu_norm_f8_backward_workspace(R(_norm(M=0))) == 0
    assert L.fp64emu_norm_f8_backward_workspace(R(_norm(M=1))) == 0               # one group writes the sums itself
    assert L.fp64emu_norm_f8_backward_workspace(R(_norm(M=10 ** 6, D=8192))) <= 4 * 3 * 1024 * 8192


def test_python_refusals():
    x, w = torch.zeros(4, 256), torch.zeros(256)
    rng = torch.zeros(2, dtype=torch.int64)
    e = fp64_emu
    for call in (lambda: e.mm_f8(x, x, x, x, act="tanh"), lambda: e.mm_f8(x, x, x, x, bias=w, out=x),
                 lambda: e.mm_f8(x, x, x, x, keep=True, accumulate=True), lambda: e.bmm_f8(x, x, x, x, bias=w),
                 lambda: e.act_f8_backward(x, x, "tanh"), lambda: e.act_f8_backward(x, None, "silu"),
                 lambda: e.act_f8_backward(x, x[:2], "silu"), lambda: e.act_f8_backward(x[0], x[0], "silu"),
                 lambda: e.act_f8_backward(x, x, "silu", "cols"), lambda: e.dropout_f8(x, -0.1, rng),
                 lambda: e.dropout_f8(x, 1.0, rng), lambda: e.dropout_f8(x, float("nan"), rng), lambda: e.dropout_f8(x, 0.5, None),
                 lambda: e.dropout_f8(x[0], 0.5, rng), lambda: e.dropout_f8(x, 0.5, rng, "cols"), lambda: e.norm_f8(x[0], w),
                 lambda: e.norm_f8(x, w[:3]), lambda: e.norm_f8(x, w, post=w), lambda: e.norm_f8(x, w, gate=w),
                 lambda: e.norm_f8(x, w, x[:2]), lambda: e.norm_f8(x, w, x, post=x), lambda: e.norm_f8(x, w, x, gate=w[:5]),
                 lambda: e.norm_f8(x, w, eps=0.0), lambda: e.norm_f8(x[:, :0], w[:0]), lambda: e.norm_f8(x, w, scale=2.0), lambda: e.norm_f8(x, w, p=0.5, rng=rng),
                 lambda: e.norm_f8(x, w, x, p=0.5), lambda: e.norm_f8(x, w, quant="cols"),
                 lambda: e.norm_f8_backward(x[:2], None, x, w, x), lambda: e.norm_f8_backward(x, x[:2], x, w, x),
                 lambda: e.norm_f8_backward(x, None, x, w, x, post=w), lambda: e.norm_f8_backward(x, None, x, w, x, scale=0.5),
                 lambda: e.linear_f8(x, x, act="tanh"), lambda: e.linear_f8(x, x, bias=w), lambda: e.linear_f8(x, x, residual=x),
                 lambda: e.linear_f8(x, torch.zeros(8, 256), residual=torch.zeros(4, 8).half()),
                 lambda: e.residual_norm_f8(w[0], w), lambda: e.residual_norm_f8(x, x), lambda: e.residual_norm_f8(x, w, x[:2]),
                 lambda: e.seeded_dropout_f8(w[0], 0.5, rng)):
        with pytest.raises(ValueError):
            call()


def test_host_tensors_are_refused():
    x, w = torch.zeros(4, 256), torch.zeros(256)
    for call in (lambda: fp64_emu.norm_f8(x, w), lambda: fp64_emu.norm_f8_backward(x, None, x, w, x[:1, :4]),
                 lambda: fp64_emu.act_f8_backward(x, x, "silu"), lambda: fp64_emu.dropout_f8(x, 0.0, None),
                 lambda: fp64_emu.residual_norm_f8(x, w), lambda: fp64_emu.seeded_dropout_f8(x, 0.0, None)):
        with pytest.raises((RuntimeError, NotImplementedError)):
            call()


def test_fake_tensors():
    e = fp64_emu
    shapes = lambda out: [tuple(t.shape) if t is not None else None for t in out]  # noqa: E731
    with FakeTensorMode():
        x = torch.empty(40, 300, dtype=torch.bfloat16, device="cuda")
        w = torch.empty(300, device="cuda")
        rng = torch.empty(2, dtype=torch.int64, device="cuda")
        q, s = e.quant_f8(x)
        assert shapes(e.mm_f8(q, s, q, s, bias=w[:40], act="gelu", keep=True)) == [(40, 40), (40, 40)]
        assert e.mm_f8(q, s, q, s, act="relu", out_dtype=torch.float32).dtype == torch.float32
        assert shapes(e.act_f8_backward(x, x, "silu", "both", bias=True)) == [(40, 300), (40, 3), (300, 40), (300, 1), (300,)]
        assert shapes(e.dropout_f8(x, 0.5, rng, "rows")) == [(40, 300), (40, 3)]
        out = e.norm_f8(x.float(), w, x, w, w, 0.5, 0.1, rng, "both", keep=True)
        assert shapes(out) == [(40, 300), (40, 300), (40, 3), (300, 40), (300, 1), (2, 40)]
        assert out[0].dtype == torch.float32 and out[1].dtype == E4M3
        r, y = e.norm_f8(x.float(), w, x)
        assert r.dtype == torch.float32 and y.dtype == torch.bfloat16
        assert shapes(e.norm_f8(x, w, keep=True)) == [(40, 300), (1, 40)]
        assert shapes(e.norm_f8_backward(x, None, x, w, torch.empty(2, 40, device="cuda"), x, w, x)) == [
            (40, 300), (40, 300), (300,), (300,), (40, 300)]
        assert shapes(e.norm_f8_backward(x, x, x, w, torch.empty(1, 40, device="cuda"))) == [(40, 300), None, (300,), None, None]
        assert e.linear_f8(x, torch.empty(70, 300, device="cuda"), bias=torch.empty(70, device="cuda"), act="silu").shape == (40, 70)


def test_philox_known_answers():
    """The generator's published answers for a counter and key of zeros, of ones, and of the digits of pi."""
    ones = 0xFFFFFFFF
    assert philox((0,) * 4, (0,) * 2) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert philox((ones,) * 4, (ones,) * 2) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    assert philox((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0)) == [
        0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]


@pytest.mark.parametrize("seed,offset", [(0, 0), (2 ** 63 - 1, 2 ** 40 + 3), (-5, -1)])
def test_plain_mask(seed, offset):
    """The mask by numpy against the generator on Python's integers, element by element."""
    M, D, drop = 3, 21, 20000
    got, halves = kept(seed, offset, drop, M, D), lambda v: (v & 0xFFFFFFFF, v >> 32 & 0xFFFFFFFF)
    for m in range(M):
        for d in range(D):
            words = philox((m * 3 + d // 8, 0, *halves(offset)), halves(seed))
            assert got[m, d].item() == (words[d % 8 // 2] >> 16 * (d % 2) & 0xFFFF >= drop)


@pytest.mark.parametrize("name", ACTS)
def test_plain_slopes(name):
    """The tests' slopes against torch's derivatives of the tests' activations."""
    h = torch.linspace(-6, 6, 97, dtype=F64).add(1e-3).requires_grad_()
    d, = torch.autograd.grad(act(h, name).sum() + 0.0 * h.sum(), h)
    assert torch.allclose(d, slope(h.detach(), name), rtol=1e-12, atol=1e-13)


@pytest.mark.parametrize("post,gates,p", [(True, False, 0.3), (False, True, 0.0), (True, True, 0.5)])
def test_plain_norm_gradient(post, gates, p):
    """The tests' gradient against torch's derivative of the tests' norm."""
    g = torch.Generator().manual_seed(3)
    M, D = 5, 24
    new = lambda *s: torch.randn(s, generator=g, dtype=F64).requires_grad_()  # noqa: E731
    r, w, y, po, ga = new(M, D), new(D), new(M, D), new(D) if post else None, new(*((M, D) if gates else (D,)))
    drop = factors(99, 3, p, M, D)
    v, x, iv, iy, *_ = norm(r, w, y, po, ga, 0.7, drop)
    dv, dx = torch.randn(M, D, generator=g, dtype=F64), torch.randn(M, D, generator=g, dtype=F64)
    leaves = [t for t in (r, y, w, po, ga) if t is not None]
    want = torch.autograd.grad((v, x), leaves, (dv, dx))
    with torch.no_grad():
        got = norm_grad(dx, dv, v, w, iv, y, iy, po, ga, 0.7, drop)
    names = ["dr", "dy", "dw"] + (["dpost"] if post else []) + ["dgate" if gates else "dgate sum"]
    for n, t in zip(names, want):
        assert torch.allclose(got[n][0], t, rtol=1e-9, atol=1e-11), n


def test_no_derivative_is_said():
    """Results of the ops for tensors that require a gradient raise in the backward pass; under no_grad, or
    where nothing requires one, they have no history."""
    e = fp64_emu
    with FakeTensorMode():
        x = torch.empty(8, 256, device="cuda")
        w, h = torch.empty(256, device="cuda"), torch.empty(8, 256, device="cuda", requires_grad=True)
        q, s = e.quant_f8(x)
        rng, stats = torch.empty(2, dtype=torch.int64, device="cuda"), torch.empty(1, 8, device="cuda")
        calls = (lambda t: e.norm_f8(t, w), lambda t: e.norm_f8(x, w, t), lambda t: e.norm_f8_backward(t, x, x, w, stats)[:1],
                 lambda t: e.act_f8_backward(t, x, "silu"), lambda t: e.dropout_f8(t, 0.5, rng),
                 lambda t: [e.mm_f8(q, s, q, s, torch.float32, bias=t[0, :8], act="relu")])
        for call in calls:
            for out in call(h):
                assert out.requires_grad and out.grad_fn.name().endswith("NotImplemented")
            assert not any(t.requires_grad for t in call(x))
            with torch.no_grad():
                assert not any(t.requires_grad for t in call(h))


@pytest.mark.parametrize("p", [0.0, 1e-6, 2.0 ** -17])
def test_shares_that_round_to_none_need_no_rng(p):
    """A share of at most 2^-17 drops nothing: rng may be absent, with gradients and without."""
    with FakeTensorMode():
        r = torch.empty(4, 256, device="cuda", requires_grad=True)
        w = torch.empty(256, device="cuda")
        new, x = fp64_emu.residual_norm_f8(r, w, r, p=p)
        assert new.requires_grad and x.shape == r.shape
        assert fp64_emu.seeded_dropout_f8(r, p, None).requires_grad
        with torch.no_grad():
            assert fp64_emu.residual_norm_f8(r, w, r, p=p)[1].shape == r.shape


def test_norm_places():
    """Outputs on their operands: the same rows at the same distance without columns, or rows side by side in one buffer."""
    L, M, D = capi.lib(), 4, 256
    r, y, g, o, x = (0x100000 * (i + 1) for i in range(5))

    def call(out=o, ldo=D, x=x, ldx=D, cols=None, **kw):
        kw = {"r": r, "y": y, "gate": g, "ld_gate": D, "gate_dtype": BF16, **kw}
        return L.fp64emu_norm_f8(R(_norm(M, D, **kw)), out, ldo, x, ldx, P, None, cols and R(cols), None)

    cols = _f8(D, M)
    for at in (r, y, g):
        _says(call(out=at, x=None, cols=cols), "elsewhere")
        _says(call(out=at + 2 * D, x=None, cols=cols), "elsewhere")
        for kw in (dict(out=at, ldo=D + 8), dict(out=at + 2), dict(out=at + 2 * D), dict(out=at - 2 * D), dict(x=at, ldx=D + 8),
                   dict(x=at + 2 * (M * D - 1))):
            _says(call(**kw), "operand itself")
    _says(call(out=r, r_dtype=F32, y=r, ld_y=2 * D), "operand itself")          # the same start and pitch, half the width
    _says(call(out=o, x=o), "outputs overlap")
    _says(call(out=o, x=o + 2 * D), "outputs overlap")
    # Side by side: half a row's distance away, an element into the neighbour's.
    _says(call(ld_r=2 * D, out=r + 2 * D - 2, ldo=2 * D), "operand itself")
    _says(call(ld_r=2 * D, out=r + 2 * D + 2, ldo=2 * D), "operand itself")


@pytest.mark.parametrize("lead", [(6,), (2, 3), ()])
def test_results_may_be_written_in_place(lead):
    """Results of the differentiable functions are tensors of their own, as a plain operator's; the new stream, which is
    kept, is so for a program that has no gradients."""
    e = fp64_emu
    with FakeTensorMode():
        x = torch.empty(*lead, 256, device="cuda", requires_grad=True)
        w, v = torch.empty(256, device="cuda"), torch.empty(64, 256, device="cuda", requires_grad=True)
        state = torch.empty(2, dtype=torch.int64, device="cuda")
        for call in (lambda: e.seeded_dropout_f8(x, 0.5, state), lambda: e.linear_f8(x, v, act="relu"), lambda: e.linear_f8(x, v),
                     lambda: e.swiglu_ckpt_f8(x), lambda: e.residual_norm_f8(x, w), lambda: e.residual_norm_f8(x, w, x)[1]):
            out = call()
            assert out.requires_grad and out.mul_(2.0).shape[:-1] == x.shape[:-1]
        with torch.no_grad():
            e.residual_norm_f8(x, w, x)[0].mul_(2.0)


def test_norm_grad_wide_refusals():
    """The entry point with a gate's gradient in float32 refuses as the other does."""
    L = capi.lib()
    call = lambda p, d, stats=P: L.fp64emu_norm_f8_backward_wide(R(p), stats, d and R(d), P, 1 << 40, None)  # noqa: E731
    lds = dict.fromkeys(("ld_dx", "ld_dr", "ld_dr_out", "ld_dy", "ld_dgates"), 256)
    _says(call(_norm(), None), "NULL")
    _says(call(_norm(), capi.NormGrad(dx=P, dgates=P, **lds)), "y's dtype")
    _says(call(_norm(gate_dtype=BF16), capi.NormGrad(dx=P, dgates=P, **lds)), "of one gate")
    _says(call(_norm(gate_dtype=BF16, ld_gate=256), capi.NormGrad(dx=P, dgates=P, dgate=P, **lds)), "a row or a matrix")
    _says(call(_norm(gate_dtype=BF16, ld_gate=256), capi.NormGrad(dx=P, dgates=P, **{**lds, "ld_dgates": 255})), "shorter")
    _says(call(_norm(gate_dtype=BF16, ld_gate=256), capi.NormGrad(dx=P, dgates=P, **lds), None), "null")
