"""The 8-bit floating-point operators as timed cases: blocks of 128 that share a float32 scale,
products of such operands, and the gated activation whose checkpoint is held so.

A matrix in 8 bits is a pair (q, s): q holds e4m3 or e5m2 codes and x ~ q s, one scale for a
block of 128 along a row ("rows"), of 128 along a column with q laid transposed ("cols"), or for
a tile of 128 x 128 ("tiles").  With a = max(amax of the block, 2^-110) and F the format's
largest value (448 or 57344): s = a / F and q = x (F / a), rounded to the nearest code.

Fields of a case: `op`; `batch`, `M`, `N`, `K` (M x K operands; N where a product has it, the
halves' width F = K for the activation); `dtype` of the input or of the product; `fmt` of A (of
what is quantised); `scales` of a product's B ("tiles" or "rows"); `form` (what is asked for).
"""
import math
import os
import sys

import torch

own = False

F32, F64 = torch.float32, torch.float64
E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": F32}
FMTS = {"e4m3": E4M3, "e5m2": E5M2}
TOP = {E4M3: 448.0, E5M2: 57344.0}
TINY = 2.0 ** -110
BLOCK = 128


def _case(name, op, M, K, N=0, batch=1, dtype="bf16", fmt="e4m3", scales="tiles", form=""):
    case = {"op": op, "batch": batch, "M": M, "N": N, "K": K, "dtype": dtype, "fmt": fmt,
            "scales": scales, "form": form}
    if name:
        case["name"] = name
    return case


def listed():
    return [
        # One token's activations before a product: launch latency.
        _case("quant_1x8192", "quant", 1, 8192, form="rows"),
        # The input of a linear layer in training: rows for the forward product, columns as the
        # checkpoint that the weight's gradient reads.
        _case("quant_8192x8192", "quant", 8192, 8192, form="both"),
        # Float32 master weights, off the block grid, in both orientations.
        _case("tiles_2049x4097", "tiles", 2049, 4097, dtype="fp32", form="both"),
        # One token through a linear layer: the weight's bytes.
        _case("mm_1x8192x8192", "mm", 1, 8192, 8192),
        # Ragged everywhere, float32 out, scales by rows on both sides.
        _case("mm_333x501x777", "mm", 333, 777, 501, dtype="fp32", scales="rows"),
        # The large square product (the benchmark's n).
        _case("mm_8192", "mm", 8192, 8192, 8192),
        # A weight's gradient added to a float32 buffer: both operands by rows over 8192 tokens,
        # the incoming gradient in e5m2.
        _case("mm_wgrad_4096x4096x8192", "mm", 4096, 8192, 4096, dtype="fp32", fmt="e5m2",
              scales="rows", form="add"),
        # Many members in one call.
        _case("bmm_64x512", "bmm", 512, 512, 512, batch=64),
        # The gated activation of one token, quantised for the next product; nothing is kept.
        _case("swiglu_1x4096", "swiglu", 1, 4096, form="rows"),
        # In training: checkpoint in 8 bits, output quantised in both orientations.
        _case("swiglu_8192x4096", "swiglu", 8192, 4096, form="both"),
        # Its gradient from the checkpoint, a ragged one in the input's type and a large one
        # quantised in both orientations.
        _case("swiglu_grad_333x777", "swiglu_grad", 333, 777, form="plain"),
        _case("swiglu_grad_8192x4096", "swiglu_grad", 8192, 4096, form="both"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: any operator, one token to 8192, odd sizes and multiples of 128."""
    op = rng.choice(["quant", "tiles", "mm", "mm", "mm", "bmm", "swiglu", "swiglu_grad"])
    M, K, N = _log_int(rng, 1, 8192), _log_int(rng, 64, 8192), 0
    if rng.random() < 0.5:
        K = max(128, K // 128 * 128)
        M = max(128, M // 128 * 128) if M > 256 else M
    dtype, fmt = rng.choice(["bf16", "bf16", "fp16", "fp32"]), rng.choice(["e4m3", "e4m3", "e5m2"])
    if op == "quant":
        return _case("", op, M, K, dtype=dtype, fmt=fmt, form=rng.choice(["rows", "cols", "both"]))
    if op == "tiles":
        return _case("", op, max(M, 32), K, dtype=dtype, form=rng.choice(["one", "both"]))
    if op in ("mm", "bmm"):
        N, batch = _log_int(rng, 64, 8192), 1
        if rng.random() < 0.5:
            N = max(128, N // 128 * 128)
        if op == "bmm":
            M, N, K = (max(32, min(v, 1024)) for v in (M, N, K))
            batch = _log_int(rng, 2, 128)
            while batch > 1 and batch * max(M * K, N * K, M * N) > 2 ** 26:
                batch //= 2
        form = rng.choice(["", "", "add"])
        return _case("", op, M, K, N, batch, dtype, fmt, rng.choice(["tiles", "tiles", "rows"]), form)
    K = min(K, 4096)
    form = rng.choice(["plain", "both"] + (["rows"] if op == "swiglu" else []))
    return _case("", op, M, K, dtype=rng.choice(["bf16", "fp16"]), form=form)


def _blocks(x, fmt):
    """(q, s) by blocks of 128 along the last dimension, q as float32 values of the codes."""
    K = x.shape[-1]
    pad = -K % BLOCK
    xb = torch.nn.functional.pad(x.float(), (0, pad)).unflatten(-1, (-1, BLOCK))
    a = xb.abs().amax(-1).clamp_min(TINY)
    q = (xb * (TOP[fmt] / a)[..., None]).to(fmt)
    return q.flatten(-2)[..., :K], a / TOP[fmt]


def _tiles(x, fmt):
    """(q, s) by tiles of 128 x 128 of the last two dimensions."""
    M, K = x.shape[-2:]
    xb = torch.nn.functional.pad(x.float(), (0, -K % BLOCK, 0, -M % BLOCK))
    xb = xb.unflatten(-1, (-1, BLOCK)).unflatten(-3, (-1, BLOCK))       # [.., MB, 128, KB, 128]
    a = xb.abs().amax((-3, -1)).clamp_min(TINY)
    q = (xb * (TOP[fmt] / a)[..., :, None, :, None]).to(fmt)
    return q.flatten(-2).flatten(-3, -2)[..., :M, :K], a / TOP[fmt]


def _values(q, s, K, rows):
    """What (q, s) stand for; s by rows or, with fewer rows than q, by tiles."""
    s = s.repeat_interleave(BLOCK, -1)[..., :K]
    if s.shape[-2] != rows:
        s = s.repeat_interleave(BLOCK, -2)[..., :rows, :]
    return q.to(s.dtype) * s


def _randn(shape, g, scale=1.0):
    return torch.randn(shape, device="cuda", dtype=F32, generator=g) * scale


def _activations(b, M, K, g):
    """Tokens x channels: a few channels many times larger, now and then a row of padding."""
    x = _randn((b, M, K), g)
    loud = torch.rand(K, device="cuda", generator=g) < 0.004
    x = x * torch.where(loud, 25.0, 1.0)
    pad = torch.rand((b, M, 1), device="cuda", generator=g) < 0.01
    return x.masked_fill(pad & (M > 1), 0.0)


def _gradients(b, M, K, g):
    """Small, and of another size from token to token."""
    return _randn((b, M, K), g, 1e-4) * torch.exp(_randn((b, M, 1), g))


def _in_rows(q):
    """q's codes in rows of a multiple of 16 bytes, as the quantiser lays them out."""
    b, M, K = q.shape
    room = torch.zeros((b, M, -(-K // 16) * 16), dtype=torch.uint8, device=q.device)
    room[..., :K] = q.contiguous().view(torch.uint8)
    return room.view(q.dtype)[..., :K]


def _by_blocks(s):
    """Scales stored block by block, as the quantiser lays them out."""
    return s.transpose(-1, -2).contiguous().transpose(-1, -2)


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    b, M, N, K = case["batch"], case["M"], case["N"], case["K"]
    dt, fmt, op = DTYPES[case["dtype"]], FMTS[case["fmt"]], case["op"]
    if op == "quant":
        x = _gradients(1, M, K, g) if fmt == E5M2 else _activations(1, M, K, g)
        return {"x": x[0].to(dt)}
    if op == "tiles":
        return {"x": _randn((M, K), g, 0.02).to(dt)}
    if op in ("mm", "bmm"):
        a = _gradients(b, M, K, g) if fmt == E5M2 else _activations(b, M, K, g)
        qa, sa = _blocks(a, fmt)
        w = _randn((b, N, K), g, 0.02)
        qb, sb = _blocks(w, E4M3) if case["scales"] == "rows" else _tiles(w, E4M3)
        out = {"qa": _in_rows(qa), "sa": _by_blocks(sa), "qb": _in_rows(qb), "sb": _by_blocks(sb)}
        if case["form"] == "add":
            out["acc"] = _randn((b, M, N), g, 1e-4 if fmt == E5M2 else 1.0).to(dt)
        return {k: v[0] for k, v in out.items()} if op == "mm" else out
    h = _activations(1, M, 2 * K, g)[0].to(dt)
    if op == "swiglu":
        return {"h": h}
    hq, hs = _blocks(h.float().view(M, 2, K), E4M3)
    return {"dy": _gradients(1, M, K, g)[0].to(dt), "hq": _in_rows(hq.reshape(1, M, 2 * K))[0],
            "hs": _by_blocks(hs.reshape(M, -1))}


def prepare(case, seed):
    """The operands on the GPU: inputs as a layer gets them, quantised operands as the
    quantiser leaves them."""
    state = _inputs(case, seed)
    state.update(op=case["op"], form=case["form"], dt=DTYPES[case["dtype"]], fmt=FMTS[case["fmt"]])
    return state


def _f8():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "fp64-emu_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import fp64_emu
    return fp64_emu


def _run_own(s):
    f8, op, form = _f8(), s["op"], s["form"]
    if op == "quant":
        return f8.quant_f8(s["x"], rows=form != "cols", cols=form != "rows", fmt=s["fmt"])
    if op == "tiles":
        return f8.quant_f8_tiles(s["x"], transposed=form == "both", fmt=s["fmt"])
    if op in ("mm", "bmm"):
        fn = f8.mm_f8 if op == "mm" else f8.bmm_f8
        if form == "add":
            return fn(s["qa"], s["sa"], s["qb"], s["sb"], out=s["acc"], accumulate=True)
        return fn(s["qa"], s["sa"], s["qb"], s["sb"], out_dtype=s["dt"])
    quant = {"plain": None}.get(form, form)
    if op == "swiglu":
        return f8.swiglu_f8(s["h"], quant=quant, keep=form != "rows")
    return f8.swiglu_f8_backward(s["dy"], s["hq"], s["hs"], quant=quant)


def _both(x, fmt):
    return (*_blocks(x, fmt), *_blocks(x.transpose(-1, -2), fmt))


def run(s):
    """One pass: the framework's operators, or the same from elementary operations."""
    if own:
        return _run_own(s)
    op, form, fmt = s["op"], s["form"], s["fmt"]
    if op == "quant":
        x = s["x"].float()
        got = _blocks(x, fmt) if form != "cols" else ()
        return got + (_blocks(x.t(), fmt) if form != "rows" else ())
    if op == "tiles":
        q, sc = _tiles(s["x"], fmt)
        return (q, sc, q.t().contiguous(), sc.t().contiguous()) if form == "both" else (q, sc)
    if op in ("mm", "bmm"):
        K = s["qa"].shape[-1]
        a = _values(s["qa"], s["sa"], K, s["qa"].shape[-2])
        b = _values(s["qb"], s["sb"], K, s["qb"].shape[-2])
        c = torch.matmul(a, b.transpose(-1, -2).contiguous())
        if form == "add":
            s["acc"].copy_(s["acc"].float() + c)
            return s["acc"]
        return c.to(s["dt"])
    if op == "swiglu":
        h = s["h"].float()
        M, F = h.shape[0], h.shape[1] // 2
        gate, up = h[:, :F], h[:, F:]
        y = gate / (1 + torch.exp(-gate)) * up
        got = (y.to(s["dt"]),) if form == "plain" else _both(y, E4M3) if form == "both" else _blocks(y, E4M3)
        if form == "rows":
            return got
        hq, hs = _blocks(h.view(M, 2, F), E4M3)
        return (*got, hq.reshape(M, 2 * F), hs.reshape(M, -1))
    M, F = s["dy"].shape
    h = _values(s["hq"].reshape(M, 2, F), s["hs"].reshape(M, 2, -1), F, 2)
    gate, up, dy = h[:, 0], h[:, 1], s["dy"].float()
    sig = 1 / (1 + torch.exp(-gate))
    d = torch.cat((dy * up * sig * (1 + gate * (1 - sig)), dy * gate * sig), 1)
    return d.to(s["dt"]) if form == "plain" else _both(d, E4M3)


def work(case):
    """Inputs read once and outputs written once; two operations per multiply-add of a product,
    a few per element elsewhere."""
    b, M, N, K, op, form = (case[k] for k in ("batch", "M", "N", "K", "op", "form"))
    size = {"bf16": 2, "fp16": 2, "fp32": 4}[case["dtype"]]
    MB, NB, KB = (-(-v // BLOCK) for v in (M, N, K))
    rows, cols, tiles = M * K + 4 * M * KB, M * K + 4 * K * MB, M * K + 4 * MB * KB
    if op == "quant":
        out = (rows if form != "cols" else 0) + (cols if form != "rows" else 0)
        return {"bytes": size * M * K + out, "flops": 3 * M * K}
    if op == "tiles":
        return {"bytes": size * M * K + tiles * (2 if form == "both" else 1), "flops": 3 * M * K}
    if op in ("mm", "bmm"):
        wb = N * K + 4 * KB * (N if case["scales"] == "rows" else NB)
        return {"bytes": b * (rows + wb + M * N * size * (2 if form == "add" else 1)),
                "flops": 2 * b * M * N * K}
    keep = 2 * rows
    if op == "swiglu":
        out = {"plain": size * M * K, "rows": rows, "both": rows + cols}[form]
        return {"bytes": 2 * size * M * K + out + (0 if form == "rows" else keep), "flops": 15 * M * K}
    out = 2 * size * M * K if form == "plain" else 2 * (rows + cols)
    return {"bytes": size * M * K + keep + out, "flops": 20 * M * K}


# What the definitions give in 64 bits.

def _round8(v, fmt):
    """v to the nearest value of the format, ties to the even mantissa."""
    mant, least = (3, -6) if fmt == E4M3 else (2, -14)
    _, e = torch.frexp(v)
    step = torch.ldexp(torch.ones_like(v), (e - 1).clamp_min(least) - mant)
    return torch.round(v / step) * step


def _spread(s, M, K, tall, wide):
    """One value of s for each element of an M x K matrix of blocks of tall x wide."""
    i, j = (torch.arange(n, device=s.device) // d for n, d in ((M, tall), (K, wide)))
    return s[..., i, :][..., j]


def _exact_blocks(x, fmt, tall=1):
    """Codes' values and scales of blocks of `tall` x 128 of the matrix x."""
    M, K = x.shape
    a = torch.nn.functional.max_pool2d(x.abs()[None, None], (tall, BLOCK), ceil_mode=True)[0, 0]
    a = torch.where(a < TINY, TINY, a)
    return _round8(x / _spread(a, M, K, tall, BLOCK) * TOP[fmt], fmt), a / TOP[fmt]


def _exact_values(q, s):
    """What codes and scales (rows or tiles) stand for."""
    R, K = q.shape[-2:]
    return q.to(F64) * _spread(s.to(F64), R, K, 1 if s.shape[-2] == R else BLOCK, BLOCK)


def exact(case, seed):
    """The outputs by definition in 64 bits."""
    op, form, fmt, F = case["op"], case["form"], FMTS[case["fmt"]], case["K"]
    s = _inputs(case, seed)

    def asked(v, f):
        got = _exact_blocks(v, f) if form != "cols" else ()
        return got + (_exact_blocks(v.t().contiguous(), f) if form in ("cols", "both") else ())

    if op in ("mm", "bmm"):
        b = _exact_values(s["qb"], s["sb"]).transpose(-1, -2).contiguous()
        c = torch.matmul(_exact_values(s["qa"], s["sa"]), b)
        return c + s["acc"].to(F64) if form == "add" else c
    if op == "quant":
        return asked(s["x"].to(F64), fmt)
    if op == "tiles":
        q, sc = _exact_blocks(s["x"].to(F64), fmt, BLOCK)
        return (q, sc, q.t(), sc.t()) if form == "both" else (q, sc)
    if op == "swiglu":
        h = s["h"].to(F64)
        y = torch.nn.functional.silu(h[:, :F]) * h[:, F:]
        got = (y,) if form == "plain" else asked(y, E4M3)
        if form == "rows":
            return got
        halves = [_exact_blocks(h[:, :F].contiguous(), E4M3), _exact_blocks(h[:, F:].contiguous(), E4M3)]
        return (*got, *(torch.cat(v, 1) for v in zip(*halves)))
    half = s["hs"].shape[1] // 2
    gate = _exact_values(s["hq"][:, :F], s["hs"][:, :half])
    up = _exact_values(s["hq"][:, F:], s["hs"][:, half:])
    sig, dy = torch.special.expit(gate), s["dy"].to(F64)
    d = torch.cat((dy * up * (sig + gate * sig * (1 - sig)), dy * gate * sig), 1)
    return d if form == "plain" else asked(d, E4M3)
