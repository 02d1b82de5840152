"""Plain forms of the 8-bit operators for the tests: codes and scales step by
step in float32 on the host (the definition names every rounding), products
and the activation in float64, and the error bounds that follow from the
formats."""
import torch

E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2
TOP = {E4M3: 448.0, E5M2: 57344.0}
BLOCK = 128
F32, F64 = torch.float32, torch.float64


def _grouped(x, tall):
    """x [.., M, K] padded to whole blocks, as [.., MB, tall, KB, 128]."""
    M, K = x.shape[-2:]
    x = torch.nn.functional.pad(x, (0, -K % BLOCK, 0, -M % tall))
    return x.reshape(*x.shape[:-2], x.shape[-2] // tall, tall, x.shape[-1] // BLOCK, BLOCK)


def quantised(x, fmt, tall=1):
    """(q, s) of x by blocks of tall x 128, q as its codes."""
    M, K = x.shape[-2:]
    b = _grouped(x.detach().cpu().to(F32), tall)
    a = torch.maximum(b.abs().amax((-3, -1)), torch.tensor(2.0 ** -110))
    r = (torch.ones_like(a) / a) * torch.tensor(TOP[fmt])
    q = (b * r[..., :, None, :, None]).to(fmt)
    q = q.reshape(*x.shape[:-2], b.shape[-4] * tall, b.shape[-2] * BLOCK)[..., :M, :K]
    return q, a / torch.tensor(TOP[fmt])


def values(q, s):
    """What codes and scales (by rows or tiles) stand for, in float64."""
    R, K = q.shape[-2:]
    s = s.to(F64)
    i = torch.arange(R, device=s.device) // (1 if s.shape[-2] == R else BLOCK)
    j = torch.arange(K, device=s.device) // BLOCK
    return q.to(F64) * s[..., i, :][..., j]


def same_codes(got, want):
    """Equal codes, any NaN equal to any."""
    got, want = got.detach().cpu(), want.detach().cpu()
    if got.dtype != want.dtype or got.shape != want.shape:
        return False
    g, w = got.to(F32), want.to(F32)
    return bool((torch.isnan(g) == torch.isnan(w)).all()) and torch.equal(
        g.nan_to_num(0.0), w.nan_to_num(0.0))


def operand(shape, seed, fmt=E4M3, tiles=False, device="cuda", spread=True):
    """A quantised matrix with values that a few columns dominate."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g)
    if spread:
        x = x * torch.exp2(torch.randint(-3, 4, shape[-1:], generator=g).float())
    q, s = quantised(x, fmt, BLOCK if tiles else 1)
    return q.to(device), s.to(device)


def rounding(dtype):
    """(relative, absolute) error of one rounding to dtype: 2^-p for significands of p bits
    (24, 8 and 11), half of the least denormal."""
    return {torch.float32: (2.0 ** -24, 2.0 ** -150), torch.bfloat16: (2.0 ** -8, 2.0 ** -134),
            torch.float16: (2.0 ** -11, 2.0 ** -25)}[dtype]


def product_bound(A, B, want, out_dtype, exact):
    """Elementwise error bound of a product of values A [.., M, K], B [.., N, K].

    Every float32 operation (128 of a block's sum, two on the scales, one per
    block on the running sum, and at most 32 joining partial sums) errs by at
    most 2^-23 of the absolute sum (rounding or truncation).  Matrix
    instructions on the codes themselves also cut each product at 2^-13 of the
    largest of its eight neighbours: at most 8 2^-13 of the absolute sum."""
    total = A.abs() @ B.abs().transpose(-1, -2)
    K = A.shape[-1]
    rel = (128 + 2 + -(-K // BLOCK) + 32) * 2.0 ** -23 + (0.0 if exact else 8 * 2.0 ** -13)
    r, a = rounding(out_dtype)
    return total * rel * (1 + r) + want.abs() * r + a
