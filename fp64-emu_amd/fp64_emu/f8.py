"""Matrices in 8-bit floating point with one float32 scale per block of 128:
the quantiser, products of such matrices with what follows them in their epilogue,
the gated activation whose checkpoint is held so, and what stands around the
products of a block: norms with residual, gate and dropout.

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

A dropout's random bits come from an element's place and rng, two int64 on the GPU: a
seed and an offset (Philox4x32-10, sixteen bits an element).  No mask is stored; the
same rng gives the same one again, and a program that drops anew adds to the offset
(in place, where a captured graph is to read it).  Of elements the share
round(p 2^16) / 2^16 is dropped and the rest scaled by its exact inverse.

Differentiable are linear_f8, swiglu_ckpt_f8, residual_norm_f8 and seeded_dropout_f8, once.
The other functions have no derivative: given tensors that require a gradient, their results raise in a
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
_SUMS = 3                                   # act_f8_backward's form without dh, dbias alone
_ACTS = {None: 0, "relu": 1, "relu2": 2, "silu": 3, "gelu": 4, "gelu_tanh": 5}

# The overloads themselves: resolving a packet's overload costs a microsecond a call.
_quant = ops.fp64_emu_quant_f8.default
_mm = ops.fp64_emu_mm_f8.default
_mm_out = ops.fp64_emu_mm_f8_out.default
_swiglu = ops.fp64_emu_swiglu_f8.default
_swiglu_backward = ops.fp64_emu_swiglu_f8_backward.default
_mm_epilogue = ops.fp64_emu_mm_f8_epilogue.default
_act_backward = ops.fp64_emu_act_f8_backward.default
_dropout = ops.fp64_emu_dropout_f8.default
_norm = ops.fp64_emu_norm_f8.default
_norm_backward = ops.fp64_emu_norm_f8_backward.default


def _check_x(x, fmt):
    if x.dim() not in (2, 3):
        raise ValueError(f"expect x as [M, K] or [batch, M, K], got {tuple(x.shape)}")
    if fmt is not E4M3 and fmt is not E5M2:
        raise ValueError(f"fmt must be float8_e4m3fn or float8_e5m2, got {fmt}")


def _form(quant):
    if quant not in _FORMS:
        raise ValueError(f"quant must be one of {tuple(_FORMS)}, got {quant!r}")
    return _FORMS[quant]


def _act(act):
    if act not in _ACTS:
        raise ValueError(f"act must be one of {tuple(_ACTS)}, got {act!r}")
    return _ACTS[act]


def _drop(p, rng):
    """The share of 65536 that is dropped."""
    drop = round(p * 65536) if 0.0 <= p <= 1.0 else -1
    if not 0 <= drop <= 65535:
        raise ValueError(f"p must be in 0 .. 1 - 2^-16, got {p}")
    if drop and rng is None:
        raise ValueError("a dropout needs rng: two int64 on the GPU, a seed and an offset")
    return drop


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


def _product(dim, A, sA, B, sB, out_dtype, out, accumulate, bias, act, residual, keep):
    if A.dim() != dim or B.dim() != dim:
        raise ValueError(f"expect {dim}-D operands, got {A.dim()}-D and {B.dim()}-D")
    if bias is not None or act is not None or residual is not None or keep:
        if out is not None or accumulate:
            raise ValueError("out and accumulate go without bias, act, residual and keep")
        got = _mm_epilogue(A, sA, B, sB, out_dtype, bias, _act(act), residual, keep)
        return tuple(got) if keep else got[0]
    if out is None:
        if accumulate:
            raise ValueError("accumulate needs out")
        return _mm(A, sA, B, sB, out_dtype)
    _mm_out(out, A, sA, B, sB, accumulate)
    return out


def mm_f8(A: torch.Tensor, sA: torch.Tensor, B: torch.Tensor, sB: torch.Tensor,
          out_dtype: torch.dtype = torch.bfloat16, out: torch.Tensor = None,
          accumulate: bool = False, bias: torch.Tensor = None, act: str = None,
          residual: torch.Tensor = None, keep: bool = False) -> torch.Tensor:
    """C = A @ B^T of quantised A [M, K] and B [N, K], A's scales by rows, B's by
    rows or tiles.  out: where to (float32, bfloat16 or float16, rows any
    distance apart; out_dtype is then out's); accumulate: C is added to it, the
    sum rounded once.  16-bit outputs of more than a few rows take less exact sums of a
    block than float32 ones (the module's notes say how much).

    bias [N], act ("relu", "relu2", "silu", "gelu", "gelu_tanh") and residual [M, N] in
    out_dtype give act(C + bias) + residual instead, from the float32 sums and rounded once;
    keep: then (that, C + bias), the second for act_f8_backward.  Which kernel a product takes follows from its sizes, and
    with it the last bits of a 16-bit output: beside the block sums, the activation's exponential, whose argument is rounded
    once on tiles and exact to float32 elsewhere (2^-17 of itself at most)."""
    return _product(2, A, sA, B, sB, out_dtype, out, accumulate, bias, act, residual, keep)


def bmm_f8(A: torch.Tensor, sA: torch.Tensor, B: torch.Tensor, sB: torch.Tensor,
           out_dtype: torch.dtype = torch.bfloat16, out: torch.Tensor = None,
           accumulate: bool = False, bias: torch.Tensor = None, act: str = None,
           residual: torch.Tensor = None, keep: bool = False) -> torch.Tensor:
    """C[b] = A[b] @ B[b]^T, as mm_f8 for each member; bias [batch, N], or [N] for all."""
    return _product(3, A, sA, B, sB, out_dtype, out, accumulate, bias, act, residual, keep)


def act_f8_backward(dy: torch.Tensor, h: torch.Tensor = None, act: str = None, quant: str = None,
                    bias: bool = False):
    """dh = dy act'(h) for the h that mm_f8 kept, dy and h [M, N] of one type; without act,
    dh = dy.  quant None: (dh,) in dy's type; "rows": (q, s); "both": (q, s, qt, st), quantised from
    the float32 values.  bias: then also dbias [N], their float32 sum over the rows."""
    code, form = _act(act), _form(quant)
    if dy.dim() != 2:
        raise ValueError(f"expect dy as [M, N], got {tuple(dy.shape)}")
    if code and (h is None or h.shape != dy.shape):
        raise ValueError(f"expect h with dy's shape {tuple(dy.shape)}")
    return tuple(_act_backward(dy, h if code else None, code, form, bias))


def dropout_f8(x: torch.Tensor, p: float, rng: torch.Tensor, quant: str = None):
    """x [M, K] with a share p of its elements zero and the others scaled, by rng's bits (the
    module's notes).  quant None: (y,) in x's type; "rows": (q, s); "both": (q, s, qt, st).
    The same call on a gradient is the gradient."""
    form, drop = _form(quant), _drop(p, rng)
    if x.dim() != 2:
        raise ValueError(f"expect x as [M, K], got {tuple(x.shape)}")
    return tuple(_dropout(x, drop, rng, form))


def _check_norm(r, w, y, post, gate, scale, drop, eps=1.0):
    shape = r.shape                         # (a tensor's shape is made anew each time it is asked for)
    width = shape[1:]
    if len(shape) != 2 or w.shape != width or not width[0]:
        raise ValueError(f"expect r [M, D] and w [D], got {tuple(shape)} and {tuple(w.shape)}")
    if y is None:
        if post is not None or gate is not None or drop or scale != 1.0:
            raise ValueError("post, gate, scale and p are of y")
    elif y.shape != shape:
        raise ValueError(f"y must have r's shape {tuple(shape)}, got {tuple(y.shape)}")
    if post is not None and post.shape != width:
        raise ValueError(f"expect post as [D], got {tuple(post.shape)}")
    if gate is not None:
        have = gate.shape
        if have != width and have != shape:
            raise ValueError(f"expect gate as [D] or [M, D], got {tuple(have)}")
    if not eps >= 2.0 ** -126:
        raise ValueError(f"eps must be positive and not denormal, got {eps}")
    return shape


def norm_f8(r: torch.Tensor, w: torch.Tensor, y: torch.Tensor = None, post: torch.Tensor = None,
            gate: torch.Tensor = None, scale: float = 1.0, p: float = 0.0, rng: torch.Tensor = None,
            quant: str = None, keep: bool = False, eps: float = 1e-6):
    """Between two blocks: the block's output y joins the residual stream r, and the norm of
    the new stream is the next block's input.  With i(v) = (mean(v^2) + eps)^-1/2 over a row of D,

      z = y i(y) post,  r' = scale r + gate drop(z),  x = r' i(r') w

    for r and y [M, D], w and post [D], gate [D] or [M, D]; z = y without post, r' = r without y.
    x comes from r' before that is rounded to r's type.  y has r's type, or r is float32; x (and
    a gate [M, D]) have y's.  p, rng: the dropout of z.  post, gate, scale and p are of y: without it they are
    refused, a scale of 1 aside.

    Returns (r',) with y; then quant None: (x,), "rows": (q, s), "both": (q, s, qt, st); then with keep
    (stats,), i(r') and, with post, i(y) of each row, for norm_f8_backward.  Sums of squares are
    float32 ones: rows past about 1e18 give x = 0."""
    form, drop = _form(quant), _drop(p, rng)
    _check_norm(r, w, y, post, gate, scale, drop, eps)
    return tuple(_norm(r, w, y, post, gate, scale, drop, rng, form, keep, eps))


def norm_f8_backward(dx: torch.Tensor, dr: torch.Tensor, r: torch.Tensor, w: torch.Tensor, stats: torch.Tensor,
                     y: torch.Tensor = None, post: torch.Tensor = None, gate: torch.Tensor = None,
                     scale: float = 1.0, p: float = 0.0, rng: torch.Tensor = None):
    """The gradient of norm_f8 for dx (x's) and dr (the new stream's own, or None), from the
    new stream r that it returned (with y None, r itself), its stats and its other arguments.

    Returns (dr, dy, dw, dpost, dgate), None for what is absent: dr in r's type, dy in y's, dw, dpost
    and the gradient of a gate [D] float32, that of a gate [M, D] in its type."""
    return _norm_gradients(dx, dr, r, w, stats, y, post, gate, scale, p, rng, False)


def _norm_gradients(dx, dr, r, w, stats, y, post, gate, scale, p, rng, wide):
    """norm_f8_backward; wide: the gradient of a gate [M, D] in float32."""
    drop = _drop(p, rng)
    shape = _check_norm(r, w, y, post, gate, scale, drop)
    if dx.shape != shape or (dr is not None and dr.shape != shape):
        raise ValueError(f"dx and dr must have r's shape {tuple(shape)}")
    got = _norm_backward(dx, dr, r, w, stats, y, post, gate, scale, drop, rng, wide)
    if y is None:
        return got[0], None, got[1], None, None
    return got[0], got[1], got[2], None if post is None else got[3], None if gate is None else got[-1]


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


# The functions below take and give matrices: flattened and unfolded around them, results are no views made inside,
# which could not be written in place.

def _flat(t):
    return t if t is None or t.dim() == 2 else _as_rows(t)


def _unfold(t, lead):
    return t if len(lead) == 1 else t.view(*lead, t.size(1))


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, wq, ws, wqt, wst, bias, act, residual, grad):
        # (needs_input_grad does not heed no_grad, and in here gradients are always off.)
        wants_x, wants_w, wants_b = (grad and ctx.needs_input_grad[i] for i in (0, 1, 6))
        q, s, *kept = quant_f8(x, cols=wants_w)
        if wq is None:
            wq, ws, *across = quant_f8_tiles(w.detach(), transposed=wants_x)
            wqt, wst = across if wants_x else (None, None)
        elif wants_x and wqt is None:
            raise ValueError("wq lacks the transposed half that x's gradient reads")
        ctx.act, ctx.wants_b = act, wants_b
        ctx.w_dtype, ctx.x_dtype = w.dtype, x.dtype
        ctx.b_dtype = bias.dtype if bias is not None else None
        h = None
        if bias is None and act is None and residual is None:
            y = mm_f8(q, s, wq, ws, out_dtype=x.dtype)
        else:
            keep = act is not None and (wants_x or wants_w or wants_b)
            y = mm_f8(q, s, wq, ws, out_dtype=x.dtype, bias=bias, act=act, residual=residual, keep=keep)
            y, h = y if keep else (y, None)
        ctx.save_for_backward(*(kept if wants_w else (None, None)),
                              *((wqt, wst) if wants_x else (None, None)), h)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        xqt, xst, wqt, wst, h = ctx.saved_tensors
        dx = dw = db = None
        got = ()
        if ctx.wants_b or h is not None:
            form = _FORMS["both"] if xqt is not None else _FORMS["rows"] if wqt is not None else _SUMS
            got = _act_backward(dy, h, _act(ctx.act), form, ctx.wants_b)
            if ctx.wants_b:
                *got, db = got
                db = db.to(ctx.b_dtype)
        elif wqt is not None or xqt is not None:
            got = quant_f8(dy, rows=wqt is not None, cols=xqt is not None)
        if wqt is not None:
            dx = mm_f8(got[0], got[1], wqt, wst, out_dtype=ctx.x_dtype)
        if xqt is not None:
            dw = mm_f8(got[-2], got[-1], xqt, xst, out_dtype=ctx.w_dtype)
        return dx, dw, None, None, None, None, db, None, dy if ctx.needs_input_grad[8] else None, None


def linear_f8(x: torch.Tensor, w: torch.Tensor, wq: tuple = None, bias: torch.Tensor = None, act: str = None,
              residual: torch.Tensor = None) -> torch.Tensor:
    """y = act(x @ w^T + bias) + residual for x [.., K] and w [N, K], in x's type, by 8-bit products:
    x by rows, w by tiles.  Differentiable once, in x, w, bias [N] and residual [.., N] (in x's
    type); what is kept for w's gradient is x in 8 bits (blocks along its rows' direction), not x, and
    with act its argument in x's type.  Gradients: with dh = dy act', dx = dh w with dh by rows,
    dw = dh^T x with dh and x by columns.

    wq: quant_f8_tiles(w, transposed=True) made earlier, for weights that stay
    (without the transposed half where x needs no gradient, or under no_grad)."""
    if x.dim() < 1 or w.dim() != 2 or x.size(-1) != w.size(1):
        raise ValueError(f"expect x [.., K] and w [N, K], got {tuple(x.shape)} and {tuple(w.shape)}")
    wq = tuple(wq) if wq is not None else ()
    if len(wq) not in (0, 2, 4):
        raise ValueError("wq: what quant_f8_tiles gives, two or four tensors")
    if wq and wq[0].shape != w.shape:
        raise ValueError(f"wq is of another weight: {tuple(wq[0].shape)} and {tuple(w.shape)}")
    _act(act)
    if bias is not None and bias.shape != w.shape[:1]:
        raise ValueError(f"expect bias as [N], got {tuple(bias.shape)}")
    if residual is not None and (residual.shape != (*x.shape[:-1], w.size(0)) or residual.dtype != x.dtype):
        raise ValueError(f"expect residual as {(*x.shape[:-1], w.size(0))} in x's type")
    y = _Linear.apply(_flat(x), w, *(wq + (None,) * (4 - len(wq))), bias, act, _flat(residual), torch.is_grad_enabled())
    return _unfold(y, x.shape[:-1])


class _SwigluCkpt(torch.autograd.Function):
    @staticmethod
    def forward(ctx, h, grad):
        y, *kept = swiglu_f8(h, keep=grad and ctx.needs_input_grad[0])
        ctx.save_for_backward(*kept)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        return swiglu_f8_backward(dy, *ctx.saved_tensors), None


def swiglu_ckpt_f8(h: torch.Tensor) -> torch.Tensor:
    """y = silu(g) u for h = [.., g | u] in h's type, differentiable once: its
    backward pass reads an 8-bit checkpoint of h instead of h."""
    if h.dim() < 1 or h.size(-1) % 2:
        raise ValueError(f"expect h as [.., 2 F], got {tuple(h.shape)}")
    return _unfold(_SwigluCkpt.apply(_flat(h), torch.is_grad_enabled()), h.shape[:-1])


def _gate_rows(gate, shape, dtype):
    """A gate that spreads to `shape` [.., D] as norm_f8 takes it: [D] where all rows have one, else a row for each, in dtype."""
    if gate is None or gate.shape == shape[-1:] or (gate.dim() == 1 and gate.numel() != 1):
        return gate
    if gate.shape[-1:] == shape[-1:] and gate.numel() == shape[-1] and gate.dim() <= len(shape):
        return gate.reshape(shape[-1:])
    return _as_rows(gate.to(dtype).expand(shape))


def _column_sums(t):
    """Of float32 [M, N]: by act_f8_backward's kernels, in an order that the sizes say, and without the memset that a library's
    sum leaves in a captured graph."""
    return _act_backward(t, None, 0, _SUMS, True)[0]


def _sum_to(t, shape):
    """Float32 t summed over the dimensions along which a tensor of `shape` spreads to t's."""
    full, lead = t.shape, (1,) * (t.dim() - len(shape)) + tuple(shape)
    over = [i for i in range(len(full) - 1) if lead[i] != full[i]]
    rest = [i for i in range(len(full)) if i not in over]
    if over:
        count = math.prod([full[i] for i in over])
        t = _column_sums(t.permute(over + rest).reshape(count, math.prod([full[i] for i in rest])))
    if lead[-1] != full[-1]:
        t = _column_sums(t.reshape(math.prod([full[i] for i in rest[:-1]]), full[-1]).t())
    return t.reshape(shape)


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, r, w, y, post, gate, shape, scale, p, rng, eps, grad):
        gates = _gate_rows(gate, shape, (r if y is None else y).dtype)
        keep = grad and any(ctx.needs_input_grad[:5])
        got = norm_f8(r, w, y, post, gates, scale, p, rng, keep=keep, eps=eps)
        ctx.shape, ctx.scale, ctx.p, ctx.joined = shape, scale, p, y is not None
        if keep:
            # (rng may go on in place before the backward pass.)
            rng = rng.clone() if p and rng is not None else None
            ctx.save_for_backward(got[0] if ctx.joined else r, w, y, post, gate, got[-1], rng)
        ctx.set_materialize_grads(False)
        return got[:2] if ctx.joined else got[0]

    @staticmethod
    @once_differentiable
    def backward(ctx, *grads):
        r, w, y, post, gate, stats, rng = ctx.saved_tensors
        dr, dx = grads if ctx.joined else (None, grads[0])
        if dr is None and dx is None:
            return (None,) * 11
        if dx is None:
            dx = torch.zeros_like(r if y is None else y)
        shape = ctx.shape
        gates = _gate_rows(gate, shape, (r if y is None else y).dtype)
        # (Of a gate that rows share, or of another type than y, in float32 until it is what is returned.)
        wide = gates is not None and gates.dim() == 2 and (gate.shape != shape or gate.dtype != y.dtype)
        dr, dy, dw, dpost, dgate = _norm_gradients(dx, dr, r, w, stats, y, post, gates, ctx.scale, ctx.p, rng, wide)
        dpost = dpost.to(post.dtype) if post is not None else None
        if gate is not None:
            dgate = (_sum_to(dgate.view(shape), gate.shape) if gates.dim() == 2 else dgate.view(gate.shape)).to(gate.dtype)
        return dr, dw.to(w.dtype), dy, dpost, dgate, None, None, None, None, None, None


def residual_norm_f8(r: torch.Tensor, w: torch.Tensor, y: torch.Tensor = None, post: torch.Tensor = None,
                     gate: torch.Tensor = None, scale: float = 1.0, p: float = 0.0, rng: torch.Tensor = None,
                     eps: float = 1e-6):
    """(r', x) of norm_f8 in their plain forms for r [.., D], x alone without y.  Differentiable once, in r,
    w, y, post and gate: [D], or of a shape that spreads to r's, as a gate for each sequence or
    token does.  A gate that is not one row for all is rounded to y's type, and spread to [.., D] for each
    pass; its gradient is summed in float32 and rounded once to its own type.  What is kept is r', y, w, post, gate as
    it was given, and two floats a row: r' is not to be changed in place before the backward pass, x may be."""
    if r.dim() < 1 or w.dim() != 1:
        raise ValueError(f"expect r [.., D] and w [D], got {tuple(r.shape)} and {tuple(w.shape)}")
    if y is not None and y.shape != r.shape:
        raise ValueError(f"y must have r's shape {tuple(r.shape)}, got {tuple(y.shape)}")
    lead = r.shape[:-1]
    got = _ResidualNorm.apply(_flat(r), w, _flat(y), post, gate, r.shape, scale, p, rng, eps, torch.is_grad_enabled())
    return _unfold(got, lead) if y is None else (_unfold(got[0], lead), _unfold(got[1], lead))


class _SeededDropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, rng, grad):
        if grad and ctx.needs_input_grad[0]:
            ctx.p = p
            # (rng may go on in place before the backward pass.)
            ctx.save_for_backward(rng.clone() if rng is not None else None)
        return dropout_f8(x, p, rng)[0]

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        rng, = ctx.saved_tensors
        return dropout_f8(dy, ctx.p, rng)[0], None, None, None


def seeded_dropout_f8(x: torch.Tensor, p: float, rng: torch.Tensor) -> torch.Tensor:
    """dropout_f8's plain form for x [.., K], differentiable once: the gradient makes the mask again from
    rng's value at the call."""
    if x.dim() < 1:
        raise ValueError(f"expect x as [.., K], got {tuple(x.shape)}")
    return _unfold(_SeededDropout.apply(_flat(x), p, rng, torch.is_grad_enabled()), x.shape[:-1])


__all__ = ["quant_f8", "quant_f8_tiles", "mm_f8", "bmm_f8", "swiglu_f8", "swiglu_f8_backward",
           "linear_f8", "swiglu_ckpt_f8", "act_f8_backward", "dropout_f8", "norm_f8", "norm_f8_backward",
           "residual_norm_f8", "seeded_dropout_f8"]
