"""CPU tier: the 8-bit operators' checks, which run before any device work: the
C entry points' status codes and messages, the workspace rule, the Python
functions' refusals, host tensors refused, and tracing with fake tensors."""
import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import fp64_emu
from fp64_emu import capi
from f8_util import E4M3, E5M2, quantised, values

EINVAL, EWORKSPACE = 1, 2
F32, BF16 = 0, 1
P = 0x1000            # a pointer that no call below gets as far as using


def _f8(rows, depth, fmt=0, tiles=0, q=P, s=P, ld=None):
    return capi.F8(q, s, depth if ld is None else ld, 0, 1, rows, 0, fmt, tiles)


def _mm(M=256, N=256, K=256, batch=1, dtype=BF16, out=P, ws=None, ws_bytes=0, **kw):
    p = capi.MmF8(out, kw.pop("ldo", N), 0, dtype, 0, kw.pop("A", _f8(M, K)), kw.pop("B", _f8(N, K)),
                  batch, M, N, K)
    assert not kw
    return p, capi.lib().fp64emu_mm_f8(ctypes.byref(p), ws, ws_bytes, None), capi.lib().fp64emu_last_error().decode()


def test_mm_refusals():
    for kw, msg in [(dict(M=-1), "non-negative"), (dict(M=1 << 31), "below 2^31"), (dict(dtype=7), "dtype must be"),
                    (dict(A=_f8(256, 256, fmt=3)), "fmt must be"), (dict(A=_f8(256, 256, tiles=1)), "by rows"),
                    (dict(out=None), "null operand"), (dict(B=_f8(256, 256, q=None)), "null 8-bit"),
                    (dict(B=_f8(256, 256, s=None)), "null 8-bit"), (dict(ldo=255), "shorter than N"),
                    (dict(A=_f8(256, 256, ld=200)), "shorter than their depth")]:
        _, st, text = _mm(**kw)
        assert st == EINVAL and msg in text, (kw, st, text)
    assert capi.lib().fp64emu_mm_f8(None, None, 0, None) == EINVAL
    for kw in (dict(M=0), dict(N=0), dict(batch=0)):
        assert _mm(**kw)[1] == 0                  # nothing to do, no device touched


def test_mm_workspace():
    """Deep products of few tiles and operands whose rows cannot be copied ask for room; the call refuses less."""
    L = capi.lib()
    p, st, text = _mm(M=16, N=64, K=65536)
    need = L.fp64emu_mm_f8_workspace(ctypes.byref(p))
    assert need >= 2 * 4 * 16 * 64 and st == EWORKSPACE and "fp64emu_mm_f8_workspace" in text
    p, st, _ = _mm(M=300, N=300, K=256, A=_f8(300, 256, ld=257))
    assert L.fp64emu_mm_f8_workspace(ctypes.byref(p)) >= 300 * 256 and st == EWORKSPACE
    p, st, _ = _mm(M=300, N=300, K=256, A=_f8(300, 256, ld=257), ws=0x1008, ws_bytes=1 << 30)
    assert st == EINVAL
    big = capi.MmF8(P, 8192, 0, BF16, 0, _f8(8192, 8192), _f8(8192, 8192), 1, 8192, 8192, 8192)
    assert L.fp64emu_mm_f8_workspace(ctypes.byref(big)) == 0
    # A rule of the shapes: partial sums never exceed 32 times the output.
    for M in (1, 20, 64, 65, 300, 2000):
        for N in (1, 100, 5000):
            for K in (1, 1000, 10 ** 6):
                p = capi.MmF8(P, N, 0, F32, 0, _f8(M, K, ld=-(-K // 16) * 16), _f8(N, K, ld=-(-K // 16) * 16), 1, M, N, K)
                assert L.fp64emu_mm_f8_workspace(ctypes.byref(p)) <= 32 * 4 * M * N + 256


def test_quant_refusals():
    L = capi.lib()

    def call(rows, cols, x=P, dtype=BF16, batch=1, M=4, K=256, ld=256):
        r = ctypes.byref(rows) if rows else None
        c = ctypes.byref(cols) if cols else None
        return L.fp64emu_quant_f8(x, dtype, batch, M, K, ld, 0, r, c, None), L.fp64emu_last_error().decode()

    ok = _f8(4, 256)
    for args, kw, msg in [((ok, None), dict(dtype=9), "dtype must be"), ((None, None), {}, "no output"),
                          ((ok, _f8(256, 4, tiles=1)), {}, "agree"), ((ok, _f8(256, 4, fmt=1)), {}, "agree"),
                          ((ok, None), dict(x=None), "null operand"), ((ok, None), dict(ld=255), "shorter than K"),
                          ((_f8(4, 256, q=None), None), {}, "null 8-bit"), ((_f8(4, 256, ld=128), None), {}, "shorter"),
                          ((_f8(4, 256, fmt=5), None), {}, "fmt must be"), ((ok, None), dict(M=-1), "non-negative"),
                          ((ok, None), dict(M=1 << 40, K=256), "too large")]:
        st, text = call(*args, **kw)
        assert st == EINVAL and msg in text, (kw, st, text)
    assert call(ok, None, M=0)[0] == 0


def test_swiglu_refusals():
    L = capi.lib()
    r = ctypes.byref
    keep, rows = _f8(4, 512), _f8(4, 256)
    fw = lambda **k: L.fp64emu_swiglu_f8(k.get("h", P), k.get("dtype", BF16), 4, k.get("F", 256), k.get("ldh", 512),  # noqa: E731
                                         k.get("y"), k.get("ldy", 256), k.get("keep"), k.get("rows"), None, None)
    assert fw() == EINVAL and fw(y=P, ldh=511) == EINVAL and fw(y=P, ldy=255) == EINVAL and fw(y=P, h=None) == EINVAL
    assert fw(rows=r(_f8(4, 256, fmt=1))) == EINVAL and fw(rows=r(_f8(4, 256, tiles=1))) == EINVAL
    assert fw(keep=r(_f8(4, 512, ld=256))) == EINVAL and fw(y=P, F=0) == 0
    bw = lambda **k: L.fp64emu_swiglu_f8_backward(k.get("dy", P), BF16, 4, k.get("F", 256), k.get("ldy", 256),  # noqa: E731
                                                  k.get("keep", r(keep)), k.get("dh"), k.get("out", BF16), 512,
                                                  k.get("rows"), None, None)
    assert bw() == EINVAL and bw(dh=P, keep=None) == EINVAL and bw(dh=P, out=2) == EINVAL and bw(dh=P, dy=None) == EINVAL
    assert bw(rows=r(rows)) == EINVAL             # rows of 2 F codes do not fit 256
    assert bw(rows=r(_f8(4, 400)), F=200) == EINVAL and "multiple of 128" in L.fp64emu_last_error().decode()


def test_python_refusals():
    x = torch.zeros(4, 256)
    for call in (lambda: fp64_emu.quant_f8(x[0]), lambda: fp64_emu.quant_f8(x, rows=False),
                 lambda: fp64_emu.quant_f8(x, fmt=torch.int8), lambda: fp64_emu.quant_f8_tiles(x[0]),
                 lambda: fp64_emu.mm_f8(x[None], x, x, x), lambda: fp64_emu.bmm_f8(x, x, x, x),
                 lambda: fp64_emu.mm_f8(x, x, x, x, accumulate=True), lambda: fp64_emu.swiglu_f8(x[:, :3]),
                 lambda: fp64_emu.swiglu_f8(x, quant="cols"), lambda: fp64_emu.swiglu_f8_backward(x, x, x, quant="cols"),
                 lambda: fp64_emu.swiglu_f8_backward(x[0], x, x), lambda: fp64_emu.linear_f8(x, x[:, :5]),
                 lambda: fp64_emu.linear_f8(x, x, (x,)), lambda: fp64_emu.linear_f8(x, x, (x[:2], x)),
                 lambda: fp64_emu.swiglu_ckpt_f8(x[:, :3])):
        with pytest.raises(ValueError):
            call()


def test_host_tensors_are_refused():
    x = torch.zeros(4, 256)
    q, s = quantised(x, E4M3)
    for call in (lambda: fp64_emu.quant_f8(x), lambda: fp64_emu.quant_f8_tiles(x), lambda: fp64_emu.mm_f8(q, s, q, s),
                 lambda: fp64_emu.swiglu_f8(x), lambda: fp64_emu.swiglu_f8_backward(x, q, s),
                 lambda: fp64_emu.linear_f8(x, x)):
        with pytest.raises((RuntimeError, NotImplementedError)):
            call()


def test_fake_tensors():
    with FakeTensorMode():
        x = torch.empty(40, 300, dtype=torch.bfloat16, device="cuda")
        w = torch.empty(200, 300, device="cuda")
        q, s, qt, st = fp64_emu.quant_f8(x, cols=True)
        assert (q.shape, s.shape, qt.shape, st.shape) == ((40, 300), (40, 3), (300, 40), (300, 1))
        assert q.dtype == E4M3 and fp64_emu.quant_f8(x, fmt=E5M2)[0].dtype == E5M2
        wq, ws, wqt, wst = fp64_emu.quant_f8_tiles(w, transposed=True)
        assert (ws.shape, wqt.shape, wst.shape) == ((2, 3), (300, 200), (3, 2))
        assert fp64_emu.mm_f8(q, s, wq, ws).shape == (40, 200)
        assert [tuple(t.shape) for t in fp64_emu.swiglu_f8(x, quant="both")] == [
            (40, 150), (40, 2), (150, 40), (150, 1), (40, 300), (40, 4)]
        assert fp64_emu.linear_f8(x, w).shape == (40, 200)


def test_rows_start_at_sixteen_bytes():
    """Codes come in rows of a multiple of 16 bytes, scales block by block."""
    with FakeTensorMode():
        q, s = fp64_emu.quant_f8(torch.empty(5, 777, device="cuda"))
        assert q.stride() == (784, 1) and s.stride() == (1, 5)


def test_plain_form():
    """The tests' own plain form: the nearest code (against every code's value), the scales, tiles."""
    x = torch.randn(130, 260, generator=torch.Generator().manual_seed(1))
    codes = torch.arange(256, dtype=torch.uint8).view(E4M3).double()
    codes = codes[torch.isfinite(codes)]
    q, s = quantised(x, E4M3)
    scaled = x.double() / s.double().repeat_interleave(128, 1)[:, :260]
    nearest = (scaled[..., None] - codes).abs().amin(-1)
    assert torch.allclose((q.double() - scaled).abs(), nearest, atol=1e-4, rtol=0)
    qt, st = quantised(x, E4M3, 128)
    assert st.shape == (2, 3) and (values(qt, st) - x.double()).abs().max() < x.abs().max() / 16
