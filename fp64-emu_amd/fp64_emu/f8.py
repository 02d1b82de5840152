"""Matrices in 8-bit floating point with one float32 scale per block of 128:
the quantiser, products of such matrices, and the gated activation whose
checkpoint is held so.

A quantised matrix is a pair (q, s) with x ~ q s: q holds float8_e4m3fn or
float8_e5m2 codes, s one float32 scale for a block.  Blocks lie along K, 128
elements of one row ("rows", s [M, ceil(K / 128)]) or 128 x 128 elements
("tiles", s [ceil(M / 128), ceil(K / 128)]); the last ones may be shorter.
With a = max(largest magnitude of the block, 2^-110) and F the format's largest
value (448, 57344), s = a / F and q = x ((1 / a) F) rounded to the nearest code,
each step one float32 operation.  A block that holds an infinity or a NaN
stands for NaN throughout.

A product sums a block of K by matrix instructions, scales that by both blocks'
scales and adds it to a running float32 sum.  With a float32 output a block's sum
is a float32 one, too.  With a 16-bit output of more than a few rows it comes from
the 8-bit instruction, which keeps a product to about 13 bits below the largest
beside it: typically 2e-5 to 4e-5 of a block's sum (a float16 result rounds by 2e-4, a bfloat16
one by 2e-3), at most 2^-10 of the sum of magnitudes, and relative to the blocks where
they cancel.  A caller who needs more takes out_dtype=torch.float32 and rounds.
Products take their operands' rows along K, so a gradient needs its operands
quantised along another dimension; the quantiser's "cols" form gives blocks
along M with the codes laid transposed, in the same pass over x.

Differentiable are linear_f8 and swiglu_ckpt_f8, once.  The other functions have no
derivative: given tensors that require a gradient, their results raise in a
backward pass, and a product into `out` raises at once.

No reference counterpart: the reference's products are float64 ones.  The
work runs in hand-written gfx950 kernels; host tensors are refused.
"""
import math

import torch
from torch.autograd.function import once_differentiable

from ._ops import ops

E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2
BLOCK = 128
_FORMS = {None: 0, "rows": 1, "both": 2}

# The overloads themselves: resolving a packet's overload costs a microsecond a call.
_quant = ops.fp64_emu_quant_f8.default
_mm = ops.fp64_emu_mm_f8.default
_mm_out = ops.fp64_emu_mm_f8_out.default
_swiglu = ops.fp64_emu_swiglu_f8.default
_swiglu_backward = ops.fp64_emu_swiglu_f8_backward.default


def _check_x(x, fmt):
    if x.dim() not in (2, 3):
        raise ValueError(f"expect x as [M, K] or [batch, M, K], got {tuple(x.shape)}")
    if fmt is not E4M3 and fmt is not E5M2:
        raise ValueError(f"fmt must be float8_e4m3fn or float8_e5m2, got {fmt}")


def _form(quant):
    if quant not in _FORMS:
        raise ValueError(f"quant must be one of {tuple(_FORMS)}, got {quant!r}")
    return _FORMS[quant]


def quant_f8(x: torch.Tensor, rows: bool = True, cols: bool = False, fmt: torch.dtype = E4M3):
    """x [M, K] or [batch, M, K] (float32, bfloat16, float16) by blocks of 128.

    rows: (q, s) with blocks along K, q [.., M, K]; cols: (qt, st) with blocks
    along M and the codes laid transposed, qt [.., K, M]; with both
    (q, s, qt, st), from one pass over x.  Codes come in rows of a multiple of
    16 bytes, scales stored block by block."""
    _check_x(x, fmt)
    if not (rows or cols):
        raise ValueError("neither rows nor cols are asked for")
    return tuple(_quant(x, rows, cols, False, fmt))


def quant_f8_tiles(x: torch.Tensor, transposed: bool = False, fmt: torch.dtype = E4M3):
    """x [M, K] or [batch, M, K] by tiles of 128 x 128: (q, s), and with
    `transposed` (q, s, qt, st), the same values laid out as x^T.  The form of
    a weight, whose forward product and input gradient read it both ways."""
    _check_x(x, fmt)
    return tuple(_quant(x, True, transposed, True, fmt))


def _product(dim, A, sA, B, sB, out_dtype, out, accumulate):
    if A.dim() != dim or B.dim() != dim:
        raise ValueError(f"expect {dim}-D operands, got {A.dim()}-D and {B.dim()}-D")
    if out is None:
        if accumulate:
            raise ValueError("accumulate needs out")
        return _mm(A, sA, B, sB, out_dtype)
    _mm_out(out, A, sA, B, sB, accumulate)
    return out


def mm_f8(A: torch.Tensor, sA: torch.Tensor, B: torch.Tensor, sB: torch.Tensor,
          out_dtype: torch.dtype = torch.bfloat16, out: torch.Tensor = None,
          accumulate: bool = False) -> torch.Tensor:
    """C = A @ B^T of quantised A [M, K] and B [N, K], A's scales by rows, B's by
    rows or tiles.  out: where to (float32, bfloat16 or float16, rows any
    distance apart; out_dtype is then out's); accumulate: C is added to it, the
    sum rounded once.  16-bit outputs of more than a few rows take less exact sums of a
    block than float32 ones (the module's notes say how much)."""
    return _product(2, A, sA, B, sB, out_dtype, out, accumulate)


def bmm_f8(A: torch.Tensor, sA: torch.Tensor, B: torch.Tensor, sB: torch.Tensor,
           out_dtype: torch.dtype = torch.bfloat16, out: torch.Tensor = None,
           accumulate: bool = False) -> torch.Tensor:
    """C[b] = A[b] @ B[b]^T, as mm_f8 for each member."""
    return _product(3, A, sA, B, sB, out_dtype, out, accumulate)


def swiglu_f8(h: torch.Tensor, quant: str = None, keep: bool = True):
    """y = silu(g) u for h = [g | u], [M, 2 F].

    quant None: (y,) in h's type; "rows": (q, s), the next product's operand;
    "both": (q, s, qt, st), with the columns its weight's gradient reads, y
    quantised from its float32 values.  keep: then also (hq, hs), h by blocks of
    128 along each half in e4m3 (scales [M, 2 ceil(F / 128)]): the checkpoint
    swiglu_f8_backward takes, a byte for each element of h."""
    form = _form(quant)
    if h.dim() != 2 or h.size(1) % 2:
        raise ValueError(f"expect h as [M, 2 F], got {tuple(h.shape)}")
    return tuple(_swiglu(h, form, keep))


def swiglu_f8_backward(dy: torch.Tensor, hq: torch.Tensor, hs: torch.Tensor, quant: str = None):
    """The gradient of swiglu_f8 for dy [M, F], taken at the values its checkpoint
    (hq, hs) stands for.  quant None: dh [M, 2 F] in dy's type; "rows": (q, s);
    "both": (q, s, qt, st), quantised from the float32 values."""
    form = _form(quant)
    if dy.dim() != 2:
        raise ValueError(f"expect dy as [M, F], got {tuple(dy.shape)}")
    got = _swiglu_backward(dy, hq, hs, form)
    return got[0] if form == 0 else tuple(got)


def _as_rows(t):
    """t [.., K] as [rows, K]; the count is written out, since with K = 0 it cannot be inferred."""
    return t.reshape(math.prod(t.shape[:-1]), t.size(-1))


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, wq, ws, wqt, wst, grad):
        rows = _as_rows(x)
        # (needs_input_grad does not heed no_grad, and in here gradients are always off.)
        wants_x, wants_w = (grad and n for n in ctx.needs_input_grad[:2])
        q, s, *kept = quant_f8(rows, cols=wants_w)
        if wq is None:
            wq, ws, *across = quant_f8_tiles(w.detach(), transposed=wants_x)
            wqt, wst = across if wants_x else (None, None)
        elif wants_x and wqt is None:
            raise ValueError("wq lacks the transposed half that x's gradient reads")
        ctx.save_for_backward(*(kept if wants_w else (None, None)),
                              *((wqt, wst) if wants_x else (None, None)))
        ctx.shape, ctx.w_dtype, ctx.x_dtype = x.shape, w.dtype, x.dtype
        return mm_f8(q, s, wq, ws, out_dtype=x.dtype).view(*x.shape[:-1], w.size(0))

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        xqt, xst, wqt, wst = ctx.saved_tensors
        rows = _as_rows(dy)
        dx = dw = None
        got = quant_f8(rows, rows=wqt is not None, cols=xqt is not None)
        if wqt is not None:
            dx = mm_f8(got[0], got[1], wqt, wst, out_dtype=ctx.x_dtype).view(ctx.shape)
        if xqt is not None:
            dw = mm_f8(got[-2], got[-1], xqt, xst, out_dtype=ctx.w_dtype)
        return dx, dw, None, None, None, None, None


def linear_f8(x: torch.Tensor, w: torch.Tensor, wq: tuple = None) -> torch.Tensor:
    """y = x @ w^T for x [.., K] and w [N, K], in x's type, by 8-bit products:
    x by rows, w by tiles.  Differentiable once, in x and w; what is kept for w's
    gradient is x in 8 bits (blocks along its rows' direction), not x.  Gradients:
    dx = dy w with dy by rows, dw = dy^T x with dy and x by columns.

    wq: quant_f8_tiles(w, transposed=True) made earlier, for weights that stay
    (without the transposed half where x needs no gradient, or under no_grad)."""
    if x.dim() < 1 or w.dim() != 2 or x.size(-1) != w.size(1):
        raise ValueError(f"expect x [.., K] and w [N, K], got {tuple(x.shape)} and {tuple(w.shape)}")
    wq = tuple(wq) if wq is not None else ()
    if len(wq) not in (0, 2, 4):
        raise ValueError("wq: what quant_f8_tiles gives, two or four tensors")
    if wq and wq[0].shape != w.shape:
        raise ValueError(f"wq is of another weight: {tuple(wq[0].shape)} and {tuple(w.shape)}")
    return _Linear.apply(x, w, *(wq + (None,) * (4 - len(wq))), torch.is_grad_enabled())


class _SwigluCkpt(torch.autograd.Function):
    @staticmethod
    def forward(ctx, h, grad):
        y, *kept = swiglu_f8(_as_rows(h), keep=grad and ctx.needs_input_grad[0])
        ctx.save_for_backward(*kept)
        ctx.shape = h.shape
        return y.view(*h.shape[:-1], y.size(1))

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        return swiglu_f8_backward(_as_rows(dy), *ctx.saved_tensors).view(ctx.shape), None


def swiglu_ckpt_f8(h: torch.Tensor) -> torch.Tensor:
    """y = silu(g) u for h = [.., g | u] in h's type, differentiable once: its
    backward pass reads an 8-bit checkpoint of h instead of h."""
    if h.dim() < 1 or h.size(-1) % 2:
        raise ValueError(f"expect h as [.., 2 F], got {tuple(h.shape)}")
    return _SwigluCkpt.apply(h, torch.is_grad_enabled())


__all__ = ["quant_f8", "quant_f8_tiles", "mm_f8", "bmm_f8", "swiglu_f8", "swiglu_f8_backward",
           "linear_f8", "swiglu_ckpt_f8"]
