"""Fake-tensor registrations so the ops trace under torch.compile
(torch-ext/fp64_emu/_meta.py:1-22): the mutating ops return nothing and only
write their `out` (and `times`) arguments, so the fake is a no-op; the 8-bit
ops' fakes return empty tensors of their outputs' shapes and layouts."""
import torch

from ._ops import ops


def _noop(*args, **kwargs):
    return None


for _name in ("fp64_emu_mm", "fp64_emu_bmm", "fp64_emu_mm_nt", "fp64_emu_bmm_nt",
              "fp64_emu_mm_timed", "fp64_emu_mm_f8_out"):
    _packet = getattr(ops, _name, None)
    _qual = getattr(_packet, "_qualified_op_name", None) if _packet is not None else None
    if _qual is None:
        continue
    try:
        torch.library.register_fake(_qual)(_noop)
    except (AttributeError, RuntimeError):
        pass


def _blocks(n):
    return -(-n // 128)


def _f8(like, batch, rows, depth, scale_rows, blocks, fmt):
    q = like.new_empty((*batch, rows, -(-depth // 16) * 16), dtype=fmt)
    s = like.new_empty((*batch, blocks, scale_rows), dtype=torch.float32).transpose(-1, -2)
    return [q[..., :depth], s]


def _quant(x, rows, cols, tiles, fmt):
    *batch, M, K = x.shape
    out = []
    if rows:
        out += _f8(x, batch, M, K, _blocks(M) if tiles else M, _blocks(K), fmt)
    if cols:
        out += _f8(x, batch, K, M, _blocks(K) if tiles else K, _blocks(M), fmt)
    return out


def _mm(A, sA, B, sB, dtype):
    return A.new_empty((*A.shape[:-1], B.shape[-2]), dtype=dtype)


def _swiglu(h, quant, keep):
    M, F, e4m3 = h.shape[0], h.shape[1] // 2, torch.float8_e4m3fn
    out = [h.new_empty((M, F))] if quant == 0 else _f8(h, (), M, F, M, _blocks(F), e4m3)
    if quant == 2:
        out += _f8(h, (), F, M, F, _blocks(M), e4m3)
    if keep:
        out += _f8(h, (), M, 2 * F, M, 2 * _blocks(F), e4m3)
    return out


def _swiglu_backward(dy, hq, hs, quant):
    M, F, e4m3 = dy.shape[0], dy.shape[1], torch.float8_e4m3fn
    if quant == 0:
        return [dy.new_empty((M, 2 * F))]
    out = _f8(dy, (), M, 2 * F, M, _blocks(2 * F), e4m3)
    if quant == 2:
        out += _f8(dy, (), 2 * F, M, 2 * F, _blocks(M), e4m3)
    return out


def _asked(like, M, D, quant):
    e4m3 = torch.float8_e4m3fn
    if quant in (0, 3):
        return [like.new_empty((M, D))] if quant == 0 else []
    return _f8(like, (), M, D, M, _blocks(D), e4m3) + (_f8(like, (), D, M, D, _blocks(M), e4m3) if quant == 2 else [])


def _mm_epilogue(A, sA, B, sB, dtype, bias, act, residual, keep):
    return [_mm(A, sA, B, sB, dtype) for _ in range(2 if keep else 1)]


def _act_backward(dy, h, act, quant, bias):
    M, N = dy.shape
    return _asked(dy, M, N, quant) + ([dy.new_empty((N,), dtype=torch.float32)] if bias else [])


def _dropout(x, drop, rng, quant):
    return _asked(x, *x.shape, quant)


def _norm(r, w, y, post, gate, scale, drop, rng, quant, keep, eps):
    M, D = r.shape
    out = [] if y is None else [r.new_empty((M, D))]
    out += _asked(r if y is None else y, M, D, quant)
    return out + ([r.new_empty((1 if post is None else 2, M), dtype=torch.float32)] if keep else [])


def _norm_backward(dx, dr, r, w, stats, y, post, gate, scale, drop, rng, wide=False):
    M, D = r.shape
    out = [r.new_empty((M, D))] + ([] if y is None else [y.new_empty((M, D))])
    out += [r.new_empty((D,), dtype=torch.float32) for _ in range(1 if post is None else 2)]
    if gate is not None:
        shape = (D,) if gate.dim() == 1 else (M, D)
        out.append(gate.new_empty(shape, dtype=torch.float32 if wide or gate.dim() == 1 else gate.dtype))
    return out


for _name, _fake in (("mm_f8_epilogue", _mm_epilogue), ("act_f8_backward", _act_backward), ("dropout_f8", _dropout),
                     ("norm_f8", _norm), ("norm_f8_backward", _norm_backward)):
    torch.library.register_fake("fp64_emu::fp64_emu_" + _name)(_fake)

for _name, _fake in (("quant_f8", _quant), ("mm_f8", _mm), ("swiglu_f8", _swiglu),
                     ("swiglu_f8_backward", _swiglu_backward)):
    torch.library.register_fake("fp64_emu::fp64_emu_" + _name)(_fake)
