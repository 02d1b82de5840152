"""GPU tier: the norms around a block and their gradient against float64, at row lengths around every
launch shape (16 threads a row up to rows that do not stay in registers), ragged and odd ones, all
types, and a run of both through autograd."""
import ctypes

import pytest
import torch

import fp64_emu
from fp64_emu import capi
from f8_block_util import F64, close, close_codes, factors, inverse_rms, norm, norm_grad, randn, rng
from f8_util import quantised, same_codes

pytestmark = pytest.mark.gpu

BF16, FP16, F32 = torch.bfloat16, torch.float16, torch.float32
EPS = 1e-6
TYPES = [(BF16, BF16), (FP16, FP16), (F32, F32), (F32, BF16), (F32, FP16)]
# M, D: each launch shape whole and ragged; one row and many.
SHAPES = [(1, 1), (3, 5), (37, 100), (300, 128), (2, 129), (70, 512), (9, 700), (5, 1024), (33, 1500), (6, 2048),
          (1, 4096), (130, 3001), (3, 5000), (2, 8192), (1, 8200), (3, 20001)]
OPTIONS = ["plain", "y", "y post", "y gate", "y gates", "y post gate p", "y post gates p", "y post p"]


def _inputs(M, D, types, options, dev, seed=0):
    rt, yt = types
    has = options.split()
    s = {"r": randn(M, D, seed=seed + 1, scale=3.0, dtype=rt).to(dev), "w": (1 + randn(D, seed=seed + 2, scale=0.3)).to(dev)}
    if "y" in has:
        s["y"] = randn(M, D, seed=seed + 3, dtype=yt).to(dev)
        s["scale"] = 0.75
    if "post" in has:
        s["post"] = (0.5 + randn(D, seed=seed + 4, scale=0.1)).to(dev)
    if "gate" in has:
        s["gate"] = (0.3 + randn(D, seed=seed + 5, scale=0.2)).to(dev, BF16)       # (any type)
    if "gates" in has:
        s["gate"] = randn(M, D, seed=seed + 6, scale=0.3, dtype=yt).to(dev)
    if "p" in has:
        s["p"], s["rng"] = 0.25, rng(77 + seed, 2 ** 40 + seed, dev)
    return s


def _wide(s):
    M, D = s["r"].shape
    out = {k: s[k].to(F64) for k in ("r", "w", "y", "post", "gate") if k in s}
    out["scale"] = s.get("scale", 1.0)
    if "p" in s:
        out["drop"] = factors(*s["rng"].tolist(), s["p"], M, D).to(s["r"].device)
    return out


def _call(s, **kw):
    rest = {k: v for k, v in s.items() if k not in ("r", "w")}
    return fp64_emu.norm_f8(s["r"], s["w"], **rest, eps=EPS, **kw)


@pytest.mark.parametrize("options", OPTIONS)
@pytest.mark.parametrize("M,D", SHAPES)
def test_norm(dev, M, D, options):
    """Plain, with the statistics; the types take turns over the shapes."""
    types = TYPES[(M + D + OPTIONS.index(options)) % len(TYPES)]
    print("case norm", M, D, options, types, flush=True)
    s = _inputs(M, D, types, options, dev)
    out = _call(s, keep=True)
    v, x, iv, iy, verr, xerr = norm(**_wide(s), eps=EPS)
    new = out[:-2]
    assert len(new) == ("y" in s) and out[-2].dtype == (s["y"] if "y" in s else s["r"]).dtype
    if new:
        close(new[0], v, verr)
    close(out[-2], x, xerr)
    stats = out[-1]
    assert stats.shape == (2 if "post" in s else 1, M)
    rel = xerr.abs().amax(-1) / (x.abs().amax(-1)).clamp_min(1e-300)
    assert ((stats[0].to(F64) - iv[:, 0]).abs() <= iv[:, 0] * (rel * 4 + 2.0 ** -18)).all()
    if "post" in s:
        assert ((stats[1].to(F64) - iy[:, 0]).abs() <= iy[:, 0] * 2.0 ** -18).all()


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("M,D", [(1, 8), (5, 130), (129, 256), (300, 1000), (64, 4096), (140, 5000), (3, 20001)])
def test_norm_quantised(dev, M, D, types):
    print("case norm quantised", M, D, types, flush=True)
    s = _inputs(M, D, types, "y post gate p", dev, seed=9)
    _, x, *_, xerr = norm(**_wide(s), eps=EPS)
    new, q, sc = _call(s, quant="rows")
    both = _call(s, quant="both", keep=True)
    assert torch.equal(new, both[0]) and torch.equal(new, _call(s)[0])
    close_codes(q, sc, x, xerr)
    close_codes(both[1], both[2], x, xerr)
    close_codes(both[3], both[4], x.t().contiguous(), xerr.t().contiguous())
    if types == (F32, F32):                 # x is then seen as it is quantised
        plain = _call(s)[1]
        for got, want in ((q, quantised(plain, q.dtype)), (both[3], quantised(plain.t(), q.dtype))):
            assert same_codes(got, want[0])
        assert torch.equal(sc.cpu(), quantised(plain, q.dtype)[1])


def _grad(s, stats, new, dx, dr):
    rest = {k: v for k, v in s.items() if k not in ("r", "w")}
    return fp64_emu.norm_f8_backward(dx, dr, new, s["w"], stats, **rest)


@pytest.mark.parametrize("options", OPTIONS)
@pytest.mark.parametrize("M,D", SHAPES + [(700, 96), (600, 2000)])
def test_norm_gradient(dev, M, D, options):
    """At the new stream and the statistics that it is given."""
    types = TYPES[(M + 2 * D + OPTIONS.index(options)) % len(TYPES)]
    print("case norm gradient", M, D, options, types, flush=True)
    s = _inputs(M, D, types, options, dev, seed=20)
    yt = s["y"].dtype if "y" in s else types[0]
    stats = [inverse_rms(s["r"].to(F64), EPS)] + ([inverse_rms(s["y"].to(F64), EPS)] if "post" in s else [])
    stats = torch.stack([t[:, 0] for t in stats]).float()
    dx = randn(M, D, seed=31, dtype=yt, scale=0.5).to(dev)
    dr = randn(M, D, seed=32, dtype=types[0], scale=0.5).to(dev) if M % 3 else None
    got = dict(zip(("dr", "dy", "dw", "dpost", "dgate"), _grad(s, stats, s["r"], dx, dr)))
    wide = _wide(s)
    wide.pop("scale")
    zero = torch.zeros(M, D, dtype=F64, device=dev)
    want = norm_grad(dx.to(F64), zero if dr is None else dr.to(F64), wide.pop("r"), wide.pop("w"), stats[0][:, None].to(F64),
                     iy=stats[-1][:, None].to(F64) if "post" in s else None, scale=s.get("scale", 1.0), **wide)
    if "gate" in s and s["gate"].dim() == 1:
        want["dgate"] = want["dgate sum"]
    assert (got["dy"] is None) == ("y" not in s) and (got["dpost"] is None) == ("post" not in s)
    assert (got["dgate"] is None) == ("gate" not in s)
    for name, t in got.items():
        if t is not None:
            close(t, *want[name])
    assert got["dr"].dtype == types[0] and got["dw"].dtype == F32


def test_norm_gradient_differences(dev):
    """Against central differences of the float32 forward pass, along random directions: a step of h along a
    unit direction changes the loss by h g; curvature takes h^2 of it, rounding 2^-22 |loss terms| / h."""
    print("case norm differences", flush=True)
    M, D, h = 6, 300, 1e-2
    s = _inputs(M, D, (F32, F32), "y post gate p", dev, seed=40)
    s["gate"] = s["gate"].float()
    a, b = randn(M, D, seed=50).to(dev), randn(M, D, seed=51).to(dev)

    def loss(t):
        new, x = _call(t)
        return (new.double() * a.double()).sum() + (x.double() * b.double()).sum()

    new, x, stats = _call(s, keep=True)
    got = dict(zip(("r", "y", "w", "post", "gate"), _grad(s, stats, new, b, a)))
    for i, name in enumerate(got):
        u = randn(*s[name].shape, seed=60 + i).to(dev)
        u = u / u.norm()
        up, down = loss({**s, name: s[name] + h * u}), loss({**s, name: s[name] - h * u})
        want = ((up - down) / (2 * h)).item()
        have = (got[name].double() * u.double()).sum().item()
        # the loss has 3600 terms of size 1, off by at most 2^-20 each, as a random sum; third derivatives of size 10
        assert abs(have - want) <= 60 * 2.0 ** -20 / h + 10 * h * h + 1e-3 * abs(want), (name, have, want)


@pytest.mark.parametrize("options", ["plain", "y gate", "y post gate p", "y post gates p"])
@pytest.mark.parametrize("D", [4097, 5003, 8191])
def test_norm_ragged_long_rows(dev, D, options):
    """Rows of two chunks a thread whose last eight elements overlap another chunk's, forward and back."""
    test_norm(dev, 3, D, options)
    test_norm_gradient(dev, 2, D, options)
    test_norm_gradient(dev, 530, D, options)        # more than a row to a work group


@pytest.mark.parametrize("D,each", [(1003, 8), (4096, 8), (8192, 16), (20001, 24)])
def test_norm_gradient_cancels(dev, D, each):
    """The stream mostly the branch's output, dx along it: dr + i(v) dx w and what is taken off it are large beside what is
    left.  dy has no part along y but what c2's error and the elements' roundings leave.

    Sum dy y over a row, against the formula's: an element's term of magnitude m = i(y) |gate post y| (|dr + i(v) dx w| +
    i(v) |vh c1|) has eight roundings, uniform within U m, so of deviation U m / 3^1/2; a thread's sum of `each` terms as many
    of its partial sums, which grow evenly: (each / 9)^1/2 U of the thread's sum of m, at most each^1/2 times the root of
    its m^2, twice.  Sums over threads in 64 bits have none.  c2 has five of itself.  Over 64 rows the root mean square of
    the errors in deviations is below 1.4 (1 + 5 (2 / 64)^1/2 is its square's fifth deviation).  Sums joined in 32 bits
    give 3 to 4 from 4096 on."""
    print("case norm gradient cancels", D, flush=True)
    M, U = 64, 2.0 ** -24
    y = randn(M, D, seed=1).to(dev)
    r = 4 * y + randn(M, D, seed=2, scale=0.01).to(dev)
    dx = 0.5 * r + randn(M, D, seed=3, scale=0.01).to(dev)
    dr = randn(M, D, seed=4, scale=0.01).to(dev)
    w, post, gate = ((a + b * randn(D, seed=5 + i)).to(dev) for i, (a, b) in enumerate([(1, 0.1), (1, 0.1), (0.3, 0.05)]))
    stats = torch.stack([inverse_rms(v.to(F64), EPS)[:, 0] for v in (r, y)]).float()
    got = fp64_emu.norm_f8_backward(dx, dr, r, w, stats, y, post, gate)[1]
    r, y, dx, dr, w, post, gate, iv, iy = (t.to(F64) for t in (r, y, dx, dr, w, post, gate, stats[0][:, None], stats[1][:, None]))
    want = norm_grad(dx, dr, r, w, iv, y, iy, post, gate)["dy"][0]
    mean = lambda t: t.mean(-1, keepdim=True)  # noqa: E731
    back = iv * iv * iv * mean(dx * w * r) * r
    m = iy * (gate * post * y).abs() * ((dr + iv * dx * w).abs() + back.abs())
    c2 = mean((dr + iv * dx * w - back) * gate * post * y * iy)
    roundings = (8 / 3) ** 0.5 + 2 ** 0.5 * (each / 9) ** 0.5 * each ** 0.5
    deviation = U * (roundings ** 2 * m.square().sum(-1) + 5 / 3 * (iy * c2 * (y * y * iy).sum(-1, keepdim=True))[:, 0] ** 2).sqrt()
    off = ((got.to(F64) - want) * y).sum(-1) / deviation
    rms = off.square().mean().sqrt().item()
    print("root mean square", rms, flush=True)
    assert rms <= 1.4


@pytest.mark.parametrize("what", ["rows apart", "odd start", "transposed", "expanded gate", "one row of many"])
def test_norm_layouts(dev, what):
    print("case norm layouts", what, flush=True)
    M, D = 13, 200
    s = _inputs(M, D, (BF16, BF16), "y post gates", dev, seed=70)
    dx, dr = randn(M, D, seed=71, dtype=BF16).to(dev), randn(M, D, seed=72, dtype=BF16).to(dev)
    t = dict(s)
    moved = lambda x, pad, at: torch.nn.functional.pad(x, (at, pad - at))[:, at:at + D]  # noqa: E731
    if what == "rows apart":
        t["r"], t["y"], t["gate"] = (moved(s[k], 56, 0) for k in ("r", "y", "gate"))
        dx2, dr2 = moved(dx, 8, 0), moved(dr, 24, 0)
    elif what == "odd start":
        t["r"], t["y"], t["gate"] = (moved(s[k], 7, 3) for k in ("r", "y", "gate"))
        dx2, dr2 = moved(dx, 5, 1), moved(dr, 9, 3)
    elif what == "transposed":
        t["r"], t["y"], t["gate"] = (s[k].t().contiguous().t() for k in ("r", "y", "gate"))
        t["w"] = torch.stack([s["w"], s["w"]], 1)[:, 0]
        dx2, dr2 = dx.t().contiguous().t(), dr.t().contiguous().t()
    elif what == "expanded gate":
        s["gate"] = s["gate"][:1].expand(M, D).contiguous()
        t["gate"] = s["gate"][:1].expand(M, D)
        dx2, dr2 = dx[:1].expand(M, D), dr
        dx = dx2.contiguous()
    else:
        s, dx, dr = {k: v[4:5] if torch.is_tensor(v) and v.dim() == 2 else v for k, v in s.items()}, dx[4:5], dr[4:5]
        t, dx2, dr2 = dict(s), dx, dr
        s = {k: v.clone() if torch.is_tensor(v) else v for k, v in s.items()}
    for quant in (None, "rows", "both"):
        for a, b in zip(_call(s, quant=quant, keep=True), _call(t, quant=quant, keep=True)):
            assert torch.equal(a.float(), b.float())
    new, _, stats = _call(s, keep=True)
    for a, b in zip(_grad(s, stats, new, dx, dr), _grad(t, stats, new, dx2, dr2)):
        assert torch.equal(a, b)


def test_norm_empty_and_zero_rows(dev):
    print("case norm empty", flush=True)
    w = torch.ones(300, device=dev)
    none = torch.empty(0, 300, device=dev, dtype=BF16)
    assert [tuple(t.shape) for t in fp64_emu.norm_f8(none, w, none, w, w, quant="both", keep=True)] == [
        (0, 300), (0, 300), (0, 3), (300, 0), (300, 0), (2, 0)]
    dr, dy, dw, dpost, dgate = fp64_emu.norm_f8_backward(none, none, none, w, torch.empty(2, 0, device=dev), none, w, w)
    assert dr.shape == dy.shape == (0, 300) and not dw.any() and not dpost.any() and not dgate.any()
    # Rows of zeros: 1 / sqrt(eps), finite; x and its codes are zero.
    z = torch.zeros(3, 300, device=dev)
    new, x, stats = fp64_emu.norm_f8(z, w, z, w, keep=True, eps=1e-6)
    assert not x.any() and torch.allclose(stats, torch.full_like(stats, 1e3), rtol=1e-5)
    assert not fp64_emu.norm_f8(z, w, quant="rows")[0].float().any()


def test_norm_not_finite(dev):
    """A NaN or an infinity stays in its row; an element that is dropped is zero whatever it was."""
    print("case norm not finite", flush=True)
    M, D = 40, 260
    r, y, w = randn(M, D, seed=80).to(dev), randn(M, D, seed=81).to(dev), torch.ones(D, device=dev)
    clean = fp64_emu.norm_f8(r, w, y, w, quant="rows")
    r2, y2 = r.clone(), y.clone()
    r2[3, 5], y2[7, 200], r2[9, 0] = float("nan"), float("inf"), float("-inf")
    new, q, s = fp64_emu.norm_f8(r2, w, y2, w, quant="rows")
    rows = [i for i in range(M) if i not in (3, 7, 9)]
    assert torch.equal(new[rows], clean[0][rows]) and torch.equal(q[rows].float(), clean[1][rows].float())
    assert torch.isnan(q[[3, 7]].float()).all() and not torch.isfinite(q[9].float()).all()
    state = rng(5, 0, dev)
    gone = fp64_emu.dropout_f8(torch.ones(M, D, device=dev), 0.5, state)[0] == 0
    y3 = torch.where(gone, float("nan"), y)
    a, b = (fp64_emu.norm_f8(r, w, t, p=0.5, rng=state) for t in (y3, y))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    st = torch.ones(1, M, device=dev)
    a, b = (fp64_emu.norm_f8_backward(r, r, r, w, st, t, gate=w, p=0.5, rng=state) for t in (y3, y))
    for u, v in zip(a, b):
        assert (u is None and v is None) or torch.equal(u, v)


def test_norm_same_bits_again(dev):
    print("case norm same bits", flush=True)
    s = _inputs(777, 1024, (BF16, BF16), "y post gate p", dev, seed=90)
    dx, dr = randn(777, 1024, seed=91, dtype=BF16).to(dev), randn(777, 1024, seed=92, dtype=BF16).to(dev)
    new, _, stats = _call(s, keep=True)
    a, b = _grad(s, stats, new, dx, dr), _grad(s, stats, new, dx, dr)
    assert all(torch.equal(u, v) for u, v in zip(a, b))
    # A row's outputs do not go by the rows beside it (without dropout, whose bits go by the row's place).
    s = _inputs(777, 1024, (BF16, BF16), "y post gate", dev, seed=90)
    few = {k: v[100:103] if torch.is_tensor(v) and v.dim() == 2 else v for k, v in s.items()}
    assert all(torch.equal(u[100:103], v) for u, v in zip(_call(s), _call(few)))


def test_norm_far_offsets(dev):
    """Rows whose elements lie past 2^31 elements (and 2^32 bytes) from the first."""
    print("case norm far offsets", flush=True)
    D, ld = 264, 2 ** 30 + 8
    buf = torch.zeros(2 * ld + D, dtype=BF16, device=dev)
    far = buf.as_strided((3, D), (ld, 1))
    near = randn(3, D, seed=95, dtype=BF16).to(dev)
    far.copy_(near)
    w = torch.ones(D, device=dev)
    for quant in (None, "both"):
        for a, b in zip(fp64_emu.norm_f8(far, w, far, w, quant=quant, keep=True),
                        fp64_emu.norm_f8(near, w, near, w, quant=quant, keep=True)):
            assert torch.equal(a.float(), b.float())
    stats = torch.ones(2, 3, device=dev)
    for a, b in zip(fp64_emu.norm_f8_backward(far, far, far, w, stats, far, w, far),
                    fp64_emu.norm_f8_backward(near, near, near, w, stats, near, w, near)):
        assert torch.equal(a, b)


def test_norm_many_rows(dev):
    """More rows than a launch has work groups, of each launch shape of several rows a group."""
    print("case norm many rows", flush=True)
    for M, D in ((70000, 40), (20000, 136), (9000, 600)):
        s = _inputs(M, D, (BF16, BF16), "y post gate", dev, seed=M)
        v, x, iv, iy, verr, xerr = norm(**_wide(s), eps=EPS)
        new, got, stats = _call(s, keep=True)
        close(new, v, verr)
        close(got, x, xerr)
        dx = randn(M, D, seed=3, dtype=BF16).to(dev)
        dw = _grad(s, stats, new, dx, dx)[2]
        vh = new.to(F64) * stats[0][:, None].to(F64)
        want = (dx.to(F64) * vh).sum(0)
        # sums of at most M / 512 + 16 + 512 / 16 + 16 terms one after the other
        close(dw, want, (M / 512 + 64 + 8) * 2.0 ** -24 * (dx.to(F64) * vh).abs().sum(0))


@pytest.mark.parametrize("lead", [(7,), (2, 3), ()])
def test_residual_norm(dev, lead):
    """Through autograd, against float64 autograd of the formulas, with a gate for each sequence."""
    print("case residual norm", lead, flush=True)
    D = 96
    make = lambda *s, seed: randn(*s, seed=seed).to(dev).requires_grad_()  # noqa: E731
    gate_shape = (lead[0], *[1] * (len(lead) - 1), D) if lead else (D,)
    t = {"r": make(*lead, D, seed=1), "w": make(D, seed=2), "y": make(*lead, D, seed=3), "post": make(D, seed=4),
         "gate": make(*gate_shape, seed=5)}
    state = rng(11, 4, dev)
    new, x = fp64_emu.residual_norm_f8(**t, scale=0.5, p=0.25, rng=state)
    state += 1                              # the backward pass has the call's own bits
    a, b = randn(*lead, D, seed=6).to(dev), randn(*lead, D, seed=7).to(dev)
    got = torch.autograd.grad((new, x), list(t.values()), (a, b))
    wide = {k: v.detach().double().requires_grad_() for k, v in t.items()}
    M = new.numel() // D
    drop = factors(11, 4, 0.25, M, D).to(dev).view(new.shape)
    spread = {**wide, "gate": wide["gate"].expand(new.shape)}
    v, wx, *_ = norm(**spread, scale=0.5, drop=drop, eps=EPS)
    want = torch.autograd.grad((v, wx), list(wide.values()), (a.double(), b.double()))
    for name, u, o in zip(t, got, want):
        # float32 throughout: sums of at most 96 + 6 terms of cancelling signs, 2^-14 of the gradient's norm
        assert u.shape == t[name].shape and (u.double() - o).norm() <= 2.0 ** -14 * o.norm() + 1e-12, name


@pytest.mark.parametrize("shape", [(), (1,), (3, 1), (1, 64), (64,)])
def test_residual_norm_gate_spreads(shape, dev):
    """A gate of any shape that spreads to r's does what the spread one does, and its gradient is the sum."""
    print("case residual norm gate", shape, flush=True)
    r, y, w, a, b = (randn(*s, seed=i).to(dev) for i, s in enumerate([(3, 64), (3, 64), (64,), (3, 64), (3, 64)]))
    gate = randn(*shape, seed=9).to(dev).requires_grad_()
    whole = gate.detach().expand(3, 64).contiguous().requires_grad_()
    got, want = (fp64_emu.residual_norm_f8(r, w, y, gate=g) for g in (gate, whole))
    assert all(torch.equal(u, v) for u, v in zip(got, want))
    g, = torch.autograd.grad(got, gate, (a, b))
    each, = torch.autograd.grad(want, whole, (a, b))
    o = each.double().sum_to_size(shape)
    # two orders of sums of at most 192 float32 terms
    assert g.shape == gate.shape
    assert ((g.double() - o).abs() <= 192 * 2.0 ** -24 * each.double().abs().sum_to_size(shape)).all()


def test_residual_norm_parts(dev):
    """x alone, only one of the results used, nothing kept without gradients, no second derivative."""
    print("case residual norm parts", flush=True)
    r, y, w = (randn(*s, seed=i).to(dev).requires_grad_() for i, s in enumerate([(4, 64), (4, 64), (64,)]))
    x = fp64_emu.residual_norm_f8(r, w)
    dr, dw = torch.autograd.grad(x.sum(), (r, w))
    new, x = fp64_emu.residual_norm_f8(r, w, y)
    assert torch.equal(torch.autograd.grad(new.sum(), y, retain_graph=True)[0], torch.ones_like(y))
    assert torch.autograd.grad(x.sum(), w, allow_unused=True)[0] is not None
    with torch.no_grad():
        assert all(t.grad_fn is None for t in fp64_emu.residual_norm_f8(r, w, y))
    new, x = fp64_emu.residual_norm_f8(r, w, y)
    g, = torch.autograd.grad(x.sum(), r, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), r)
    with pytest.raises(RuntimeError):
        fp64_emu.norm_f8(r, w)[0].sum().backward()


def test_norm_refusals(dev):
    x = torch.zeros(4, 64, device=dev)
    w, h = x[0], x.half()
    for call in (lambda: fp64_emu.norm_f8(h, w, x), lambda: fp64_emu.norm_f8(x.double(), w), lambda: fp64_emu.norm_f8(x, w.double()),
                 lambda: fp64_emu.norm_f8(x, w.cpu()), lambda: fp64_emu.norm_f8(x, w, x.cpu()),
                 lambda: fp64_emu.norm_f8(x, w, h, gate=x), lambda: fp64_emu.norm_f8(x, w, x, p=0.5, rng=torch.zeros(2, device=dev)),
                 lambda: fp64_emu.norm_f8(x, w, x, p=0.5, rng=torch.zeros(3, dtype=torch.int64, device=dev)),
                 lambda: fp64_emu.norm_f8(x, w, x, p=0.5, rng=torch.zeros(2, dtype=torch.int64)),
                 lambda: fp64_emu.norm_f8_backward(h, None, x, w, x[:1, :4]),
                 lambda: fp64_emu.norm_f8_backward(x, h, x, w, x[:1, :4].contiguous()),
                 lambda: fp64_emu.norm_f8_backward(x, None, x, w, x[:1, :3].contiguous()),
                 lambda: fp64_emu.norm_f8_backward(x, None, x, w, x[:2, :4].contiguous())):
        with pytest.raises(RuntimeError):
            call()


# ---- The C entry points by themselves.

CODE = {F32: 0, BF16: 1, FP16: 2}


def _c_norm(r, w, y=None, scale=1.0, gate=None):
    M, D = r.shape
    at = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    kind = lambda t: CODE[(r if t is None else t).dtype]  # noqa: E731
    return capi.Norm(at(r), at(y), at(w), None, at(gate), None, M, D, r.stride(0), 0 if y is None else y.stride(0),
                     0 if gate is None else gate.stride(0), kind(r), kind(y), CODE[w.dtype], 0, kind(gate), 0, scale, EPS)


def _stream():
    return torch.cuda.current_stream().cuda_stream


@pytest.mark.parametrize("D", [5, 300, 8200])
def test_norm_alone_has_no_scale(dev, D):
    """Without y the stream is r, whatever scale the structure holds: forward and backward give scale 1's bits."""
    print("case norm alone, scale", D, flush=True)
    L, M = capi.lib(), 9
    r, w, dx, dr = randn(M, D, seed=1).to(dev), randn(D, seed=2).to(dev), randn(M, D, seed=3).to(dev), randn(M, D, seed=4).to(dev)
    want = None
    for scale in (1.0, 0.75, 0.0):
        p = _c_norm(r, w, scale=scale)
        x, stats = torch.empty(M, D, device=dev), torch.empty(M, device=dev)
        out, dw = torch.empty(M, D, device=dev), torch.empty(D, device=dev)
        assert L.fp64emu_norm_f8(ctypes.byref(p), None, 0, x.data_ptr(), D, stats.data_ptr(), None, None, _stream()) == 0
        d = capi.NormGrad(dx=dx.data_ptr(), dr=dr.data_ptr(), dr_out=out.data_ptr(), dw=dw.data_ptr(), ld_dx=D, ld_dr=D, ld_dr_out=D)
        need = L.fp64emu_norm_f8_backward_workspace(ctypes.byref(p))
        ws = torch.empty(max(need, 1), dtype=torch.uint8, device=dev)
        assert L.fp64emu_norm_f8_backward(ctypes.byref(p), stats.data_ptr(), ctypes.byref(d), ws.data_ptr(), need, _stream()) == 0
        got = (x, stats, out, dw)
        want = want or [t.clone() for t in got]
        assert all(torch.equal(a, b) for a, b in zip(got, want)), scale


@pytest.mark.parametrize("form", ["x", "rows"])
@pytest.mark.parametrize("D", [40, 300, 5000, 8200])
def test_norm_in_place(dev, D, form):
    """The new stream in r's, y's or the gates' place, x in y's, the new stream beside r in one buffer: the bits of
    outputs of their own."""
    print("case norm in place", D, form, flush=True)
    L, M = capi.lib(), 70
    w = randn(D, seed=1).to(dev)
    fresh = [randn(M, D, seed=i, dtype=BF16).to(dev) for i in (2, 3, 4)]
    want = fp64_emu.norm_f8(fresh[0], w, fresh[1], gate=fresh[2], scale=0.5, eps=EPS, quant=None if form == "x" else "rows")

    def run(r, y, gate, out, x=None):
        p = _c_norm(r, w, y, 0.5, gate)
        q, s = torch.empty(M, D, device=dev, dtype=torch.uint8), torch.empty(M, -(-D // 128), device=dev)
        rows = capi.F8(q.data_ptr(), s.data_ptr(), D, 0, s.stride(0), 1, 0, 0, 0)
        st = L.fp64emu_norm_f8(ctypes.byref(p), out.data_ptr(), out.stride(0), None if x is None else x.data_ptr(), D, None,
                               None if x is not None else ctypes.byref(rows), None, _stream())
        assert st == 0, L.fp64emu_last_error()
        assert torch.equal(out, want[0])
        if x is not None:
            assert torch.equal(x, want[1])
        else:
            assert torch.equal(q, want[1].view(torch.uint8)) and torch.equal(s, want[2])

    for at in range(3):
        t = [v.clone() for v in fresh]
        x = None if form == "rows" else t[1] if at != 1 else torch.empty(M, D, dtype=BF16, device=dev)
        run(*t, t[at], x)
    both = torch.cat([fresh[0], torch.zeros_like(fresh[0])], 1)
    run(both[:, :D], fresh[1], fresh[2], both[:, D:], torch.empty(M, D, dtype=BF16, device=dev) if form == "x" else None)
    assert torch.equal(both[:, :D], fresh[0])


# ---- Gates that rows share.

GATES = [(), (1,), (1, 1, 96), (96,), (3, 1, 96), (1, 700, 96), (3, 700, 1), (3, 1, 1), (1, 1, 1), (700, 96), (3, 700, 96)]


@pytest.mark.parametrize("gate_type", [F32, BF16, FP16])
@pytest.mark.parametrize("shape", GATES)
def test_shared_gates(dev, shape, gate_type):
    """Beside a bfloat16 branch a gate of any shape and type: what it gives is what its spread rows in bfloat16 (or the one row
    for all as it is) give, its gradient the float32 sum of theirs, rounded once to its own type."""
    print("case shared gates", shape, gate_type, flush=True)
    lead, D = (3, 700), 96
    M, U = 2100, 2.0 ** -24
    r, y = randn(*lead, D, seed=1).to(dev), randn(*lead, D, seed=2, dtype=BF16).to(dev)
    w, post = (1 + 0.1 * randn(D, seed=3)).to(dev), (1 + 0.1 * randn(D, seed=4)).to(dev)
    gate = (0.3 + randn(*shape, seed=5, scale=0.2)).to(dev, gate_type).requires_grad_()
    a, b = randn(*lead, D, seed=6).to(dev), randn(*lead, D, seed=7, dtype=BF16).to(dev)
    state = rng(3, 1, dev)
    got = fp64_emu.residual_norm_f8(r, w, y, post, gate, 0.75, 0.25, state)
    grad, = torch.autograd.grad(got, gate, (a, b))
    one = shape in ((1, 1, 96), (96,))
    rows = gate.detach().reshape(D) if one else gate.detach().to(BF16).expand(*lead, D).reshape(M, D).contiguous()
    new, x, stats = fp64_emu.norm_f8(r.view(M, D), w, y.view(M, D), post, rows, 0.75, 0.25, state, keep=True)
    assert torch.equal(got[0].view(M, D), new) and torch.equal(got[1].view(M, D), x)
    wide = [t.to(F64) for t in (b.view(M, D), a.view(M, D), new, w, stats[0][:, None], y.view(M, D), stats[1][:, None], post, rows)]
    each, err = norm_grad(*wide, scale=0.75, drop=factors(3, 1, 0.25, M, D).to(dev))["dgate"]
    to = lambda t: t.view(*lead, D).sum_to_size(shape)  # noqa: E731
    assert grad.shape == shape and grad.dtype == gate_type
    # Of a sum of n rows: a thread's (16), two exchanges of lanes, four waves, and of the n / 16 groups' parts a sixteenth and then
    # 16 waves' one after the other, 40 + n / 256 and for columns 40 more: at most 120 roundings of what is summed so far.  (With
    # terms rounded to bfloat16 those of 700 rows would be off by 700^1/2 2^-9 / 3^1/2 = 0.03 of one; this is 700 200 U = 0.008.)
    close(grad, to(each), to(err) + 120 * U * to(each.abs() + err))


def test_shared_gate_keeps_the_gate_alone(dev):
    """For the backward pass the gate is kept as it was given, not spread."""
    print("case shared gate kept", flush=True)
    r, y, w = randn(4, 500, 256, seed=1).to(dev), randn(4, 500, 256, seed=2).to(dev), torch.ones(256, device=dev)
    gate = randn(4, 1, 256, seed=3).to(dev).requires_grad_()
    kept = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t) or t, lambda t: t):
        fp64_emu.residual_norm_f8(r, w, y, gate=gate)
    assert sum(t.numel() for t in kept) == 2 * r.numel() + 2000 + w.numel() + gate.numel()


def test_shared_gates_captured(dev):
    """Forward and backward in a graph, with gates whose gradients are sums over rows, columns and both: each replay gives the
    eager bits."""
    print("case shared gates captured", flush=True)
    B, S, D = 3, 900, 320
    t = {"r": randn(B, S, D, seed=1, dtype=BF16).to(dev), "w": randn(D, seed=2).to(dev), "y": randn(B, S, D, seed=3, dtype=BF16).to(dev),
         "post": randn(D, seed=4).to(dev)}
    gates = [randn(*s, seed=5 + i).to(dev) for i, s in enumerate([(B, 1, D), (B, S, 1), (1, S, D), ()])]
    a, b = randn(B, S, D, seed=9, dtype=BF16).to(dev), randn(B, S, D, seed=10, dtype=BF16).to(dev)
    state = rng(1, 2, dev)

    def step():
        out = []
        for gate in gates:
            leaves = [v.detach().requires_grad_() for v in (*t.values(), gate)]
            got = fp64_emu.residual_norm_f8(*leaves, 0.5, 0.25, state)
            out += [*(v.detach() for v in got), *torch.autograd.grad(got, leaves, (a, b))]
        return out

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for turn in range(3):
        t["y"].mul_(0.5)
        gates[turn].add_(0.25)
        state += 1
        graph.replay()
        torch.cuda.synchronize()
        seen = [v.clone() for v in got]
        assert all(torch.equal(u, v) for u, v in zip(seen, step())), turn
        torch.cuda.synchronize()


@pytest.mark.parametrize("lead,shape", [((0,), ()), ((0,), (1, 64)), ((0, 5), (0, 1, 64)), ((3, 0), (3, 1, 64)), ((3, 0), (3, 1, 1)), ((3, 0), (1,))])
def test_shared_gates_of_no_rows(dev, lead, shape):
    print("case shared gates of no rows", lead, shape, flush=True)
    r, w, gate = torch.ones(*lead, 64, device=dev), torch.ones(64, device=dev), torch.ones(shape, device=dev).requires_grad_()
    new, x = fp64_emu.residual_norm_f8(r, w, r, gate=gate)
    grad, = torch.autograd.grad((new, x), gate, (new, x))
    assert x.shape == r.shape and grad.shape == gate.shape and not grad.any()
