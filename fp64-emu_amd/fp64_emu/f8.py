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

A product's sums are float32: one block of K is summed by the matrix
instruction, scaled by both blocks' scales and added to the running sum.
Products take their operands' rows along K, so a gradient needs its operands
quantised along another dimension; the quantiser's "cols" form gives blocks
along M with the codes laid transposed, in the same pass over x.

No reference counterpart: the reference's products are float64 ones.  The
work runs in hand-written gfx950 kernels; host tensors are refused.
"""
import torch

from ._ops import ops

E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2
BLOCK = 128
_QUANT = (None, "rows", "both")


def _blocks(n):
    return -(-n // BLOCK)


def _codes(like, batch, rows, depth, fmt):
    """Room for codes in rows of a multiple of 16 bytes, which the product copies fastest."""
    q = torch.empty((*batch, rows, -(-depth // 16) * 16), dtype=fmt, device=like.device)
    return q if depth % 16 == 0 else q[..., :depth]


def _scales(like, batch, rows, blocks):
    """Scales stored block by block, in the order the product reads them."""
    s = torch.empty((*batch, blocks, rows), dtype=torch.float32, device=like.device)
    return s.transpose(-1, -2)


def _along_rows(x):
    return x if x.size(-1) <= 1 or x.stride(-1) == 1 else x.contiguous()


def _check_x(x, fmt):
    if x.dim() not in (2, 3):
        raise ValueError(f"expect x as [M, K] or [batch, M, K], got {tuple(x.shape)}")
    if fmt not in (E4M3, E5M2):
        raise ValueError(f"fmt must be float8_e4m3fn or float8_e5m2, got {fmt}")


def quant_f8(x: torch.Tensor, rows: bool = True, cols: bool = False, fmt: torch.dtype = E4M3):
    """x [M, K] or [batch, M, K] (float32, bfloat16, float16) by blocks of 128.

    rows: (q, s) with blocks along K, q [.., M, K]; cols: (qt, st) with blocks
    along M and the codes laid transposed, qt [.., K, M]; with both
    (q, s, qt, st), from one pass over x."""
    _check_x(x, fmt)
    if not (rows or cols):
        raise ValueError("neither rows nor cols are asked for")
    *batch, M, K = x.shape
    q = s = qt = st = None
    if rows:
        q, s = _codes(x, batch, M, K, fmt), _scales(x, batch, M, _blocks(K))
    if cols:
        qt, st = _codes(x, batch, K, M, fmt), _scales(x, batch, K, _blocks(M))
    ops.fp64_emu_quant_f8(_along_rows(x), q, s, qt, st, False)
    return (q, s, qt, st) if rows and cols else (q, s) if rows else (qt, st)


def quant_f8_tiles(x: torch.Tensor, transposed: bool = False, fmt: torch.dtype = E4M3):
    """x [M, K] or [batch, M, K] by tiles of 128 x 128: (q, s), and with
    `transposed` (q, s, qt, st), the same values laid out as x^T.  The form of
    a weight, whose forward product and input gradient read it both ways."""
    _check_x(x, fmt)
    *batch, M, K = x.shape
    q, s = _codes(x, batch, M, K, fmt), _scales(x, batch, _blocks(M), _blocks(K))
    qt = st = None
    if transposed:
        qt, st = _codes(x, batch, K, M, fmt), _scales(x, batch, _blocks(K), _blocks(M))
    ops.fp64_emu_quant_f8(_along_rows(x), q, s, qt, st, True)
    return (q, s, qt, st) if transposed else (q, s)


def _product(dim, A, sA, B, sB, out_dtype, out, accumulate):
    if A.dim() != dim or B.dim() != dim:
        raise ValueError(f"expect {dim}-D operands, got {A.dim()}-D and {B.dim()}-D")
    if out is None:
        if accumulate:
            raise ValueError("accumulate needs out")
        out = torch.empty((*A.shape[:-1], B.size(-2)), dtype=out_dtype, device=A.device)
    ops.fp64_emu_mm_f8(out, A, sA, B, sB, accumulate)
    return out


def mm_f8(A: torch.Tensor, sA: torch.Tensor, B: torch.Tensor, sB: torch.Tensor,
          out_dtype: torch.dtype = torch.bfloat16, out: torch.Tensor = None,
          accumulate: bool = False) -> torch.Tensor:
    """C = A @ B^T of quantised A [M, K] and B [N, K], A's scales by rows, B's by
    rows or tiles.  out: where to (float32, bfloat16 or float16, rows any
    distance apart); accumulate: C is added to it, the sum rounded once."""
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
    if quant not in _QUANT:
        raise ValueError(f"quant must be one of {_QUANT}, got {quant!r}")
    if h.dim() != 2 or h.size(1) % 2:
        raise ValueError(f"expect h as [M, 2 F], got {tuple(h.shape)}")
    M, F = h.size(0), h.size(1) // 2
    y = q = s = qt = st = hq = hs = None
    if quant is None:
        y = torch.empty((M, F), dtype=h.dtype, device=h.device)
    else:
        q, s = _codes(h, (), M, F, E4M3), _scales(h, (), M, _blocks(F))
        if quant == "both":
            qt, st = _codes(h, (), F, M, E4M3), _scales(h, (), F, _blocks(M))
    if keep:
        hq, hs = _codes(h, (), M, 2 * F, E4M3), _scales(h, (), M, 2 * _blocks(F))
    ops.fp64_emu_swiglu_f8(_along_rows(h), y, hq, hs, q, s, qt, st)
    return tuple(t for t in (y, q, s, qt, st, hq, hs) if t is not None)


def swiglu_f8_backward(dy: torch.Tensor, hq: torch.Tensor, hs: torch.Tensor, quant: str = None):
    """The gradient of swiglu_f8 for dy [M, F], taken at the values its checkpoint
    (hq, hs) stands for.  quant None: dh [M, 2 F] in dy's type; "rows": (q, s);
    "both": (q, s, qt, st), quantised from the float32 values."""
    if quant not in _QUANT:
        raise ValueError(f"quant must be one of {_QUANT}, got {quant!r}")
    if dy.dim() != 2:
        raise ValueError(f"expect dy as [M, F], got {tuple(dy.shape)}")
    M, F = dy.shape
    dy = _along_rows(dy)
    if quant is None or F % BLOCK:
        # Blocks of the whole 2 F that straddle the halves are quantised in a pass of
        # their own, from float32 so that nothing is rounded twice.
        dh = torch.empty((M, 2 * F), dtype=dy.dtype if quant is None else torch.float32,
                         device=dy.device)
        ops.fp64_emu_swiglu_f8_backward(dy, hq, hs, dh, None, None, None, None)
        return dh if quant is None else quant_f8(dh, cols=quant == "both")
    q, s = _codes(dy, (), M, 2 * F, E4M3), _scales(dy, (), M, _blocks(2 * F))
    qt = st = None
    if quant == "both":
        qt, st = _codes(dy, (), 2 * F, M, E4M3), _scales(dy, (), 2 * F, _blocks(M))
    ops.fp64_emu_swiglu_f8_backward(dy, hq, hs, None, q, s, qt, st)
    return (q, s) if qt is None else (q, s, qt, st)


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, wq, ws, wqt, wst):
        K = x.size(-1)
        rows = x.reshape(-1, K)
        wants_x, wants_w = ctx.needs_input_grad[:2]
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
    def backward(ctx, dy):
        xqt, xst, wqt, wst = ctx.saved_tensors
        rows = dy.reshape(-1, dy.size(-1))
        dx = dw = None
        got = quant_f8(rows, rows=wqt is not None, cols=xqt is not None)
        if wqt is not None:
            dx = mm_f8(got[0], got[1], wqt, wst, out_dtype=ctx.x_dtype).view(ctx.shape)
        if xqt is not None:
            dw = mm_f8(got[-2], got[-1], xqt, xst, out_dtype=ctx.w_dtype)
        return dx, dw, None, None, None, None


def linear_f8(x: torch.Tensor, w: torch.Tensor, wq: tuple = None) -> torch.Tensor:
    """y = x @ w^T for x [.., K] and w [N, K], in x's type, by 8-bit products:
    x by rows, w by tiles.  Differentiable in x and w; what is kept for w's
    gradient is x in 8 bits (blocks along its rows' direction), not x.  Gradients:
    dx = dy w with dy by rows, dw = dy^T x with dy and x by columns.

    wq: quant_f8_tiles(w, transposed=True) made earlier, for weights that stay
    (without the transposed half where x needs no gradient)."""
    if x.dim() < 1 or w.dim() != 2 or x.size(-1) != w.size(1):
        raise ValueError(f"expect x [.., K] and w [N, K], got {tuple(x.shape)} and {tuple(w.shape)}")
    wq = tuple(wq) if wq is not None else ()
    if len(wq) not in (0, 2, 4):
        raise ValueError("wq: what quant_f8_tiles gives, two or four tensors")
    if wq and wq[0].shape != w.shape:
        raise ValueError(f"wq is of another weight: {tuple(wq[0].shape)} and {tuple(w.shape)}")
    return _Linear.apply(x, w, *(wq + (None,) * (4 - len(wq))))


class _Swiglu(torch.autograd.Function):
    @staticmethod
    def forward(ctx, h):
        y, *kept = swiglu_f8(h.reshape(-1, h.size(-1)), keep=ctx.needs_input_grad[0])
        ctx.save_for_backward(*kept)
        ctx.shape = h.shape
        return y.view(*h.shape[:-1], y.size(1))

    @staticmethod
    def backward(ctx, dy):
        return swiglu_f8_backward(dy.reshape(-1, dy.size(-1)), *ctx.saved_tensors).view(ctx.shape)


def swiglu_ckpt_f8(h: torch.Tensor) -> torch.Tensor:
    """y = silu(g) u for h = [.., g | u] in h's type, differentiable: its
    backward pass reads an 8-bit checkpoint of h instead of h."""
    if h.dim() < 1 or h.size(-1) % 2:
        raise ValueError(f"expect h as [.., 2 F], got {tuple(h.shape)}")
    return _Swiglu.apply(h)


__all__ = ["quant_f8", "quant_f8_tiles", "mm_f8", "bmm_f8", "swiglu_f8", "swiglu_f8_backward",
           "linear_f8", "swiglu_ckpt_f8"]
