"""What stands around the 8-bit products of a transformer's block as timed cases: the norms before
and after the block with its gate, residual and dropout, products with bias, activation and
residual in their epilogue and their gradient, and dropout from a counter-based generator.

With 1 / rms(v) = (mean(v^2) + eps)^-1/2 over a row:

  norm      z = y / rms(y) post;  r' = scale r + gate drop(z), given in r's type;
            x = r' / rms(r') w of the r' before that rounding, plain or quantised; without y, r' = r
  mm        y = act(A B^T + bias) + residual of quantised operands; h = A B^T + bias
  act_grad  dh = dy act'(h) plain or quantised, and dbias, dh's sum over the rows
  dropout   drop(x), plain or quantised

drop() of an M x D matrix: sixteen random bits for an element, t = round(p 2^16); an element whose
bits are below t becomes 0, any other is multiplied by 2^16 / (2^16 - t).  Element (m, d) has the
half d % 2 (0: the lower) of word d % 8 / 2 that Philox4x32-10 gives for the counter
(c, c >> 32, offset, offset >> 32) with c = m ceil(D / 8) + d / 8, and the key (seed, seed >> 32).

Quantised is by blocks of 128 with a float32 scale each, as pairs (q, s), x ~ q s: "rows" along a
row, "both" also along columns with q laid transposed.  With a = max(amax of the block, 2^-110):
s = a / 448 and q = x (448 / a), rounded to the nearest e4m3 code.

Fields of a case: `op`; `batch`, `M`, `N`, `K` (M x K a matrix or the product's first operand); `dtype`
of the plain matrices or of the product; `form` (plain, rows, both); `parts`: what the call has of
the operator's options, as text; `act`; `p`.
"""
import math
import os
import sys

import numpy
import torch

own = False

F32, F64 = torch.float32, torch.float64
E4M3 = torch.float8_e4m3fn
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": F32}
TOP, TINY, BLOCK = 448.0, 2.0 ** -110, 128
EPS = 1e-6
ACTS = ("relu", "relu2", "silu", "gelu", "gelu_tanh")


def _case(name, op, M, K, N=0, batch=1, dtype="bf16", form="plain", parts="", act="", p=0.0):
    case = {"op": op, "batch": batch, "M": M, "N": N, "K": K, "dtype": dtype, "form": form,
            "parts": parts, "act": act, "p": p}
    if name:
        case["name"] = name
    return case


def listed():
    return [
        # One token between two layers: the block's output joins the residual stream, whose norm the
        # next product takes in 8 bits.  Launch latency.
        _case("norm_1x8192", "norm", 1, 8192, form="rows", parts="y post"),
        # The same in training: both orientations for the products, statistics kept.
        _case("norm_8192x4096", "norm", 8192, 4096, form="both", parts="y post gate keep", p=0.1),
        # Ragged everywhere, a float32 residual stream, another gate for each token.
        _case("norm_grad_333x777", "norm_grad", 333, 777, dtype="fp32", parts="y post gates", p=0.25),
        # The gradient of the training case, all weights' gradients included.
        _case("norm_grad_8192x4096", "norm_grad", 8192, 4096, parts="y post gate", p=0.1),
        # One token through a layer that ends a block: the weight's bytes.
        _case("mm_1x8192x8192", "mm", 1, 8192, 8192, parts="bias residual"),
        # Ragged everywhere, float32 out, scales by rows on both sides, the gradient's input kept.
        _case("mm_333x501x777", "mm", 333, 777, 501, dtype="fp32", parts="bias keep rows", act="gelu"),
        # The large square product (the benchmark's n), with everything.
        _case("mm_8192", "mm", 8192, 8192, 8192, parts="bias residual", act="gelu_tanh"),
        # Many members in one call, a bias for each.
        _case("bmm_64x512", "mm", 512, 512, 512, batch=64, parts="bias", act="silu"),
        # The gradient of a layer's activation and bias, ragged and plain, and large with both
        # orientations for the two products that follow.
        _case("act_grad_333x777", "act_grad", 333, 777, parts="bias", act="silu"),
        _case("act_grad_8192x8192", "act_grad", 8192, 8192, form="both", parts="bias", act="gelu_tanh"),
        # Few tokens' activations, and the input of a layer in training.
        _case("dropout_16x4096", "dropout", 16, 4096, p=0.1),
        _case("dropout_8192x8192", "dropout", 8192, 8192, form="both", p=0.1),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: any operator, one token to 8192, odd sizes and multiples of 128."""
    op = rng.choice(["norm", "norm", "norm_grad", "norm_grad", "mm", "mm", "mm", "bmm", "act_grad", "dropout"])
    M, K, N = _log_int(rng, 1, 8192), _log_int(rng, 64, 8192), 0
    if rng.random() < 0.5:
        K = max(128, K // 128 * 128)
        M = max(128, M // 128 * 128) if M > 256 else M
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    form, p = rng.choice(["plain", "rows", "both"]), rng.choice([0.0, 0.1, 0.5])
    some = lambda *names: " ".join(n for n in names if rng.random() < 0.5)  # noqa: E731
    if op == "norm":
        y = rng.random() < 0.8
        parts = ("y " + some("post", rng.choice(["gate", "gates"])) if y else "") + rng.choice([" keep", ""])
        return _case("", op, M, K, dtype=dtype, form=form, parts=parts, p=p if y else 0.0)
    if op == "norm_grad":
        y = rng.random() < 0.8
        parts = "y " + some("post", rng.choice(["gate", "gates"])) if y else ""
        return _case("", op, M, K, dtype=dtype, parts=parts, p=p if y else 0.0)
    if op in ("mm", "bmm"):
        N, batch = _log_int(rng, 64, 8192), 1
        if rng.random() < 0.5:
            N = max(128, N // 128 * 128)
        if op == "bmm":
            M, N, K = (max(32, min(v, 1024)) for v in (M, N, K))
            batch = _log_int(rng, 2, 128)
            while batch > 1 and batch * max(M * K, N * K, M * N) > 2 ** 26:
                batch //= 2
        while batch * M * N * K > 2 ** 38:
            N = N // 2
        act = rng.choice(["", "", *ACTS])
        parts = some("bias", "residual", "rows") + (rng.choice([" keep", ""]) if act else "")
        return _case("", "mm", M, K, N, batch, dtype, parts=parts, act=act)
    if op == "act_grad":
        return _case("", op, M, K, dtype=dtype, form=form, parts=rng.choice(["bias", ""]), act=rng.choice(ACTS))
    return _case("", op, M, K, dtype=dtype, form=form, p=rng.choice([0.1, 0.5]))


def _blocks(x):
    """(q, s) by blocks of 128 along the last dimension, q as codes."""
    K = x.shape[-1]
    xb = torch.nn.functional.pad(x.float(), (0, -K % BLOCK)).unflatten(-1, (-1, BLOCK))
    a = xb.abs().amax(-1).clamp_min(TINY)
    q = (xb * (TOP / a)[..., None]).to(E4M3)
    return q.flatten(-2)[..., :K], a / TOP


def _asked(x, form, dtype):
    """x in the form asked for."""
    if form == "plain":
        return (x.to(dtype),)
    return _blocks(x) + (_blocks(x.transpose(-1, -2)) if form == "both" else ())


def _values(q, s, K, rows):
    """What (q, s) stand for; s by rows or, with fewer rows than q, by tiles."""
    s = s.repeat_interleave(BLOCK, -1)[..., :K]
    if s.shape[-2] != rows:
        s = s.repeat_interleave(BLOCK, -2)[..., :rows, :]
    return q.to(s.dtype) * s


def _randn(shape, g, scale=1.0):
    return torch.randn(shape, device="cuda", dtype=F32, generator=g) * scale


def _activations(shape, g):
    """Tokens x channels: a few channels many times larger."""
    loud = torch.rand(shape[-1], device="cuda", generator=g) < 0.004
    return _randn(shape, g) * torch.where(loud, 25.0, 1.0)


def _gradients(M, K, g):
    """Small, and of another size from token to token."""
    return _randn((M, K), g, 1e-4) * torch.exp(_randn((M, 1), g))


def _in_rows(q):
    """q's codes in rows of a multiple of 16 bytes, as the quantiser lays them out."""
    K = q.shape[-1]
    room = torch.zeros((*q.shape[:-1], -(-K // 16) * 16), dtype=torch.uint8, device=q.device)
    room[..., :K] = q.contiguous().view(torch.uint8)
    return room.view(q.dtype)[..., :K]


def _by_blocks(s):
    """Scales stored block by block, as the quantiser lays them out."""
    return s.transpose(-1, -2).contiguous().transpose(-1, -2)


def _weight_tiles(w):
    """(q, s) by tiles of 128 x 128 of the last two dimensions."""
    M, K = w.shape[-2:]
    b = torch.nn.functional.pad(w, (0, -K % BLOCK, 0, -M % BLOCK)).unflatten(-1, (-1, BLOCK)).unflatten(-3, (-1, BLOCK))
    a = b.abs().amax((-3, -1)).clamp_min(TINY)
    q = (b * (TOP / a)[..., :, None, :, None]).to(E4M3)
    return q.flatten(-2).flatten(-3, -2)[..., :M, :K], a / TOP


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    M, N, K, op, parts = (case[k] for k in ("M", "N", "K", "op", "parts"))
    dt, has = DTYPES[case["dtype"]], parts.split()
    rng = torch.tensor([(seed * 2654435761 + 12345) % 2 ** 62, seed % 97], device="cuda")
    if op == "mm":
        b = case["batch"]
        qa, sa = _blocks(_activations((b, M, K), g))
        w = _randn((b, N, K), g, 0.02)
        qb, sb = _blocks(w) if "rows" in has else _weight_tiles(w)
        s = {"qa": _in_rows(qa), "sa": _by_blocks(sa), "qb": _in_rows(qb), "sb": _by_blocks(sb)}
        if "bias" in has:
            s["bias"] = _randn((b, N), g, 0.5)
        if "residual" in has:
            s["residual"] = _activations((b, M, N), g).to(dt)
        return s if b > 1 else {k: v[0] for k, v in s.items()}
    if op == "dropout":
        return {"x": _activations((M, K), g).to(dt), "rng": rng}
    if op == "act_grad":
        return {"dy": _gradients(M, K, g).to(dt), "h": _activations((M, K), g).to(dt)}
    s = {"r": (4.0 * _activations((M, K), g)).to(dt), "w": 1.0 + _randn((K,), g, 0.2)}
    if "y" in has:
        # (Beside a float32 residual stream the block computes in 16 bits.)
        s["y"] = _activations((M, K), g).to(torch.bfloat16 if dt == F32 else dt)
        s["rng"] = rng
    if "post" in has:
        s["post"] = 0.5 + _randn((K,), g, 0.1)
    if "gate" in has:
        s["gate"] = 0.3 + _randn((K,), g, 0.1)
    if "gates" in has:
        s["gate"] = (0.3 + _randn((M, K), g, 0.1)).to(s["y"].dtype)
    if op == "norm_grad":
        # (r is then the stream with the block's output in it, as the forward pass left it.)
        s["dx"] = _gradients(M, K, g).to(s.get("y", s["r"]).dtype)
        s["dr"] = _gradients(M, K, g).to(dt)
        kept = (s["r"], s["y"]) if "post" in s else (s["r"],)
        s["stats"] = torch.stack([_inverse_rms(v.float()).squeeze(-1) for v in kept])
    return s


def prepare(case, seed):
    """The operands on the GPU: inputs as a layer gets them, quantised operands as the
    quantiser leaves them, the statistics that the forward pass kept."""
    state = _inputs(case, seed)
    state.update(op=case["op"], form=case["form"], dt=DTYPES[case["dtype"]], act=case["act"] or None,
                 p=case["p"], parts=case["parts"].split(), scale=0.9 if case["parts"] else 1.0)
    return state


def _f8():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "fp64-emu_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import fp64_emu
    return fp64_emu


def _run_own(s):
    f8, op = _f8(), s["op"]
    quant = None if s["form"] == "plain" else s["form"]
    if op == "mm":
        fn = f8.mm_f8 if s["qa"].dim() == 2 else f8.bmm_f8
        return fn(s["qa"], s["sa"], s["qb"], s["sb"], out_dtype=s["dt"], bias=s.get("bias"), act=s["act"],
                  residual=s.get("residual"), keep="keep" in s["parts"])
    if op == "dropout":
        return f8.dropout_f8(s["x"], s["p"], s["rng"], quant=quant)
    if op == "act_grad":
        return f8.act_f8_backward(s["dy"], s["h"], s["act"], quant=quant, bias="bias" in s["parts"])
    # (scale is of the stream that y joins: without y there is none to pass.)
    around = {"y": s["y"], "post": s.get("post"), "gate": s.get("gate"), "scale": s["scale"], "p": s["p"],
              "rng": s["rng"]} if "y" in s else {}
    if op == "norm":
        return f8.norm_f8(s["r"], s["w"], **around, quant=quant, keep="keep" in s["parts"], eps=EPS)
    got = f8.norm_f8_backward(s["dx"], s["dr"], s["r"], s["w"], s["stats"], **around)
    return tuple(t for t in got if t is not None)


def _inverse_rms(v):
    return 1 / torch.sqrt(v.square().mean(-1, keepdim=True) + EPS)


def _drop(rng, p, M, D):
    """What an M x D matrix is multiplied by."""
    t, mask = round(p * 65536), 0xffffffff
    c = torch.arange(M * -(-D // 8), device=rng.device)
    seed, offset = rng[0], rng[1]
    x0, x1 = c & mask, c >> 32
    x2, x3 = (v.expand_as(c) for v in (offset & mask, offset >> 32 & mask))
    k0, k1 = seed & mask, seed >> 32 & mask
    for _ in range(10):
        a, b = x0 * 0xd2511f53, x2 * 0xcd9e8d57
        x0, x1, x2, x3 = (b >> 32 & mask) ^ x1 ^ k0, b & mask, (a >> 32 & mask) ^ x3 ^ k1, a & mask
        k0, k1 = k0 + 0x9e3779b9 & mask, k1 + 0xbb67ae85 & mask
    bits = torch.stack([x0 & 0xffff, x0 >> 16, x1 & 0xffff, x1 >> 16, x2 & 0xffff, x2 >> 16, x3 & 0xffff, x3 >> 16], -1)
    return torch.where(bits.view(M, -1)[:, :D] >= t, 65536.0 / (65536 - t), 0.0)


def _act(h, act):
    if act == "relu":
        return h.clamp_min(0)
    if act == "relu2":
        return h.clamp_min(0).square()
    if act == "silu":
        return h / (1 + torch.exp(-h))
    if act == "gelu":
        return 0.5 * h * (1 + torch.erf(h * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * h * (1 + torch.tanh(math.sqrt(2 / math.pi) * (h + 0.044715 * h * h * h)))
    return h


def _act_slope(h, act):
    if act == "relu":
        return (h > 0).to(h.dtype)
    if act == "relu2":
        return 2 * h.clamp_min(0)
    if act == "silu":
        s = 1 / (1 + torch.exp(-h))
        return s * (1 + h * (1 - s))
    if act == "gelu":
        return 0.5 * (1 + torch.erf(h * math.sqrt(0.5))) + h * torch.exp(-0.5 * h * h) / math.sqrt(2 * math.pi)
    t = torch.tanh(math.sqrt(2 / math.pi) * (h + 0.044715 * h * h * h))
    return 0.5 * (1 + t) + 0.5 * h * (1 - t * t) * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * h * h)


def run(s):
    """One pass: the framework's operators, or the same from elementary operations."""
    if own:
        return _run_own(s)
    op, form, parts = s["op"], s["form"], s["parts"]
    if op == "mm":
        K = s["qa"].shape[-1]
        a = _values(s["qa"], s["sa"], K, s["qa"].shape[-2])
        b = _values(s["qb"], s["sb"], K, s["qb"].shape[-2])
        h = torch.matmul(a, b.transpose(-1, -2).contiguous())
        if "bias" in s:
            h = h + s["bias"].unsqueeze(-2)
        y = _act(h, s["act"])
        if "residual" in s:
            y = y + s["residual"].float()
        return (y.to(s["dt"]), h.to(s["dt"])) if "keep" in parts else y.to(s["dt"])
    if op == "dropout":
        m = _drop(s["rng"], s["p"], *s["x"].shape)
        return _asked(torch.where(m == 0, 0.0, s["x"].float() * m), form, s["dt"])
    if op == "act_grad":
        dh = s["dy"].float() * _act_slope(s["h"].float(), s["act"])
        return _asked(dh, form, s["dt"]) + ((dh.sum(0),) if "bias" in parts else ())
    r, w, scale = s["r"].float(), s["w"], s["scale"]
    one = torch.ones((), device=r.device)
    post, gate = s.get("post", one), s.get("gate", one).float()
    m = _drop(s["rng"], s["p"], *r.shape) if s["p"] else one
    if op == "norm":
        stats, new = [], ()
        if "y" in s:
            y = s["y"].float()
            rms = _inverse_rms(y)
            z = y * rms * post if "post" in s else y
            r = scale * r + gate * torch.where(m == 0, 0.0, z * m)
            new = (r.to(s["dt"]),)
            stats = [rms.squeeze(-1)] if "post" in s else []
        rms = _inverse_rms(r)
        out = new + _asked(r * rms * w, form, s.get("y", s["r"]).dtype)
        return out + ((torch.stack([rms.squeeze(-1), *stats]),) if "keep" in parts else ())
    # The gradient: through the norm of r', then through the joining and the norm of y.
    dx, rms = s["dx"].float(), s["stats"][0].unsqueeze(-1)
    rhat, gw = r * rms, dx * w
    dr = s["dr"].float() + rms * (gw - rhat * (gw * rhat).mean(-1, keepdim=True))
    dw = (dx * rhat).sum(0)
    if "y" not in s:
        return dr.to(s["dt"]), dw
    y, rms = s["y"].float(), s["stats"][-1].unsqueeze(-1)
    yhat = y * rms if "post" in s else y
    dz = torch.where(m == 0, 0.0, dr * gate * m)
    dgate = torch.where(m == 0, 0.0, dr * yhat * post * m)
    dy = rms * (dz * post - yhat * (dz * post * yhat).mean(-1, keepdim=True)) if "post" in s else dz
    got = ((scale * dr).to(s["dt"]), dy.to(s["y"].dtype), dw)
    got += ((dz * yhat).sum(0),) if "post" in s else ()
    if "gate" not in s:
        return got
    return got + ((dgate.sum(0) if s["gate"].dim() == 1 else dgate.to(s["gate"].dtype)),)


def work(case):
    """Inputs read once and outputs written once; two operations per multiply-add of a product, a
    few per element elsewhere (ten rounds of the generator for eight of them)."""
    b, M, N, K, op, form = (case[k] for k in ("batch", "M", "N", "K", "op", "form"))
    size, has = {"bf16": 2, "fp16": 2, "fp32": 4}[case["dtype"]], case["parts"].split()
    MB, NB, KB = (-(-v // BLOCK) for v in (M, N, K))
    rows, cols = M * K + 4 * M * KB, M * K + 4 * K * MB
    asked = lambda size: {"plain": size * M * K, "rows": rows, "both": rows + cols}[form]  # noqa: E731
    drop = 12 * M * K if case["p"] else 0
    if op == "mm":
        wb = N * K + 4 * KB * (N if "rows" in has else NB)
        outs = 1 + ("residual" in has) + ("keep" in has)
        return {"bytes": b * (rows + wb + M * N * size * outs + 4 * N * ("bias" in has)), "flops": 2 * b * M * N * K}
    if op == "dropout":
        return {"bytes": size * M * K + asked(size), "flops": M * K + drop}
    if op == "act_grad":
        return {"bytes": 2 * size * M * K + asked(size) + 4 * K * ("bias" in has), "flops": 20 * M * K}
    half = 2 if "y" in has else size
    weights = 4 * K * (1 + ("post" in has) + ("gate" in has))
    gates = 2 * M * K if "gates" in has else 0
    stats = 4 * M * (1 + ("post" in has))
    if op == "norm":
        y = 2 * M * K + size * M * K if "y" in has else 0
        return {"bytes": size * M * K + y + gates + weights + asked(half) + stats * ("keep" in has),
                "flops": 12 * M * K + drop}
    return {"bytes": M * K * (half + 3 * size) + (4 * M * K if "y" in has else 0) + 2 * gates + 2 * weights + stats,
            "flops": 30 * M * K + drop}


# What the definitions give in 64 bits.

def _round8(v):
    """v to the nearest value of e4m3, ties to the even mantissa."""
    _, e = torch.frexp(v)
    step = torch.ldexp(torch.ones_like(v), (e - 1).clamp_min(-6) - 3)
    return torch.round(v / step) * step


def _spread(s, M, K, tall):
    """One value of s for each element of an M x K matrix of blocks of tall x 128."""
    i, j = (torch.arange(n, device=s.device) // d for n, d in ((M, tall), (K, BLOCK)))
    return s[..., i, :][..., j]


def _exact_blocks(x):
    a = torch.nn.functional.max_pool2d(x.abs()[None, None], (1, BLOCK), ceil_mode=True)[0, 0]
    a = torch.where(a < TINY, TINY, a)
    return _round8(x / _spread(a, *x.shape, 1) * TOP), a / TOP


def _exact_asked(x, form):
    if form == "plain":
        return (x,)
    return _exact_blocks(x) + (_exact_blocks(x.t().contiguous()) if form == "both" else ())


def _exact_values(q, s):
    R, K = q.shape[-2:]
    return q.to(F64) * _spread(s.to(F64), R, K, 1 if s.shape[-2] == R else BLOCK)


def _exact_drop(rng, p, M, D):
    """The factors by unsigned arithmetic on the host."""
    seed, offset = (int(v) % 2 ** 64 for v in rng.tolist())
    low, half = numpy.uint64(0xffffffff), numpy.uint64(32)
    chunk = numpy.arange(M * ((D + 7) // 8), dtype=numpy.uint64)
    word = [chunk & low, chunk >> half, numpy.uint64(offset) & low, numpy.uint64(offset) >> half]
    for i in range(10):
        key = [numpy.uint64((seed % 2 ** 32 + i * 0x9e3779b9) % 2 ** 32),
               numpy.uint64((seed // 2 ** 32 + i * 0xbb67ae85) % 2 ** 32)]
        left, right = word[0] * numpy.uint64(0xd2511f53), word[2] * numpy.uint64(0xcd9e8d57)
        word = [right >> half ^ word[1] ^ key[0], right & low, left >> half ^ word[3] ^ key[1], left & low]
    out = numpy.empty((chunk.size, 8), dtype=numpy.uint16)
    for i in range(8):
        out[:, i] = word[i // 2] >> numpy.uint64(16 * (i % 2)) & numpy.uint64(0xffff)
    kept = torch.from_numpy(out.reshape(M, -1)[:, :D].astype(numpy.int32)).to(rng.device) >= round(p * 2 ** 16)
    return kept.to(F64) / (1 - round(p * 2 ** 16) / 2 ** 16)


def _exact_act(h, act):
    F = torch.nn.functional
    return {None: lambda: h, "relu": lambda: F.relu(h), "relu2": lambda: F.relu(h) ** 2, "silu": lambda: F.silu(h),
            "gelu": lambda: F.gelu(h), "gelu_tanh": lambda: F.gelu(h, approximate="tanh")}[act]()


def exact(case, seed):
    """The outputs by definition in 64 bits (gradients of activations by torch's own derivatives)."""
    s = prepare(case, seed)
    op, form, parts, act = s["op"], s["form"], s["parts"], s["act"]
    wide = {k: v.to(F64) for k, v in s.items() if torch.is_tensor(v) and v.is_floating_point() and v.dtype != E4M3}
    if op == "mm":
        b = _exact_values(s["qb"], s["sb"]).transpose(-1, -2).contiguous()
        h = torch.matmul(_exact_values(s["qa"], s["sa"]), b)
        h = h + wide["bias"][..., None, :] if "bias" in wide else h
        y = _exact_act(h, act) + wide.get("residual", 0.0)
        return (y, h) if "keep" in parts else y
    if op == "dropout":
        return _exact_asked(wide["x"] * _exact_drop(s["rng"], s["p"], *s["x"].shape), form)
    if op == "act_grad":
        h = wide["h"].requires_grad_()
        dh, = torch.autograd.grad(_exact_act(h, act), h, wide["dy"])
        return _exact_asked(dh, form) + ((dh.sum(0),) if "bias" in parts else ())
    M, D = s["r"].shape
    m = _exact_drop(s["rng"], s["p"], M, D) if s["p"] else 1.0
    norm = lambda v: (v * v).sum(-1, keepdim=True).div(D).add(EPS).pow(-0.5)  # noqa: E731
    post, gate = wide.get("post", 1.0), wide.get("gate", 1.0)
    if op == "norm":
        r, new, stats = wide["r"], (), ()
        if "y" in wide:
            z = wide["y"] * norm(wide["y"]) * post if "post" in wide else wide["y"]
            r = s["scale"] * r + gate * m * z
            new = (r,)
            stats = (norm(wide["y"])[:, 0],) if "post" in wide else ()
        x = _exact_asked(r * norm(r) * wide["w"], form)
        return new + x + ((torch.stack((norm(r)[:, 0], *stats)),) if "keep" in parts else ())
    i1, i2 = wide["stats"][0][:, None], wide["stats"][-1][:, None]
    r, dx = wide["r"], wide["dx"]
    total = wide["dr"] + i1 * wide["w"] * dx - r * i1 ** 3 / D * (dx * wide["w"] * r).sum(-1, keepdim=True)
    dw = torch.einsum("md,md,mi->d", dx, r, i1)
    if "y" not in wide:
        return total, dw
    y = wide["y"]
    f = i2 if "post" in wide else torch.ones_like(i2)
    dz = total * gate * m
    dy = dz
    if "post" in wide:
        dy = f * post * dz - y * f ** 3 / D * (dz * post * y).sum(-1, keepdim=True)
    out = (s["scale"] * total, dy, dw) + (((dz * y * f).sum(0),) if "post" in wide else ())
    if "gate" in wide:
        dgate = total * m * y * f * post
        out += (dgate.sum(0) if gate.dim() == 1 else dgate,)
    return out
