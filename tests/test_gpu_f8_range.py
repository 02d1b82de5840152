"""GPU tier: products of 8-bit operands whose scales lie near the ends of float32's range.
The product of two blocks' scales may leave that range while the block's sum does not: an
ordinary result must come out as one, and a sum of zero as zero."""
import pytest
import torch

import fp64_emu
from f8_util import E4M3, E5M2, F64, BLOCK, product_bound, quantised, values

pytestmark = pytest.mark.gpu

BF16, FP16, F32 = torch.bfloat16, torch.float16, torch.float32

# Few rows (16, 32 and 64 of A), 128 x 128 tiles, 256 x 256 or 128 x 256 tiles, split depths.
SHAPES = [(1, 200, 1024), (20, 96, 1024), (50, 130, 1000), (300, 260, 200), (2048, 2048, 1024),
          (4096, 4096, 1024), (2000, 2100, 8200), (3, 64, 40000)]


def _like(shape, seed, power):
    """Values of one sign within 2^power [1, 2): no cancellation, so a block's sum is far above
    its scales' product."""
    g = torch.Generator().manual_seed(seed)
    return torch.ldexp(1 + torch.rand(shape, generator=g), torch.tensor(power))


@pytest.mark.parametrize("fa,fb", [(E4M3, E4M3), (E5M2, E4M3)])
@pytest.mark.parametrize("tiles", [True, False])
@pytest.mark.parametrize("shape", SHAPES)
def test_small_scales(dev, shape, tiles, fa, fb):
    """Elements of 2^-100 and 2^-30 (and the other way): scales whose product is a denormal or zero,
    results of 2^-120 and more, which are normal numbers of float32 and bfloat16."""
    M, N, K = shape
    for pa, pb in ((-100, -30), (-40, -90), (-109, -15)):
        qa, sa = (t.to(dev) for t in quantised(_like((M, K), 1, pa), fa))
        qb, sb = (t.to(dev) for t in quantised(_like((N, K), 2, pb), fb, BLOCK if tiles else 1))
        A, B = values(qa, sa), values(qb, sb)
        want = A @ B.t().contiguous()
        for out_dtype in (F32, BF16):
            print("case small scales", shape, tiles, fa, fb, pa, pb, out_dtype, flush=True)
            got = fp64_emu.mm_f8(qa, sa, qb, sb, out_dtype=out_dtype).to(F64)
            bound = product_bound(A, B, want, out_dtype, out_dtype == F32)
            assert ((got - want).abs() <= bound).all(), ((got - want).abs() / bound).max().item()


@pytest.mark.parametrize("tiles", [True, False])
@pytest.mark.parametrize("shape", SHAPES)
def test_large_scales(dev, shape, tiles):
    """Scales whose product is infinite beside codes of zero: those sums are zero, not NaN; small beside large
    ones give their ordinary results."""
    M, N, K = shape
    x, w = _like((M, K), 3, 120), torch.zeros(N, K)
    w[0] = _like((K,), 4, 100)                   # its tile's scale, and its own row's
    if not tiles:
        w[1:] = 0.0
    qa, sa = (t.to(dev) for t in quantised(x, E4M3))
    qb, sb = (t.to(dev) for t in quantised(w, E4M3, BLOCK if tiles else 1))
    if not tiles:
        sb[1:] = sb[:1]                          # a row of zero codes with a large scale
    for out_dtype in (F32, BF16, FP16):
        print("case large scales", shape, tiles, out_dtype, flush=True)
        got = fp64_emu.mm_f8(qa, sa, qb, sb, out_dtype=out_dtype)
        assert torch.isinf(got[:, 0]).all() and (got[:, 0] > 0).all() and (got[:, 1:] == 0).all()
    qb, sb = (t.to(dev) for t in quantised(_like((N, K), 5, -118), E4M3, BLOCK if tiles else 1))
    A, B = values(qa, sa), values(qb, sb)
    want = A @ B.t().contiguous()
    for out_dtype in (F32, BF16):
        got = fp64_emu.mm_f8(qa, sa, qb, sb, out_dtype=out_dtype).to(F64)
        assert ((got - want).abs() <= product_bound(A, B, want, out_dtype, out_dtype == F32)).all()


@pytest.mark.parametrize("tiles", [True, False])
@pytest.mark.parametrize("shape", SHAPES)
def test_scales_grow_along_the_depth(dev, shape, tiles):
    """Blocks of ordinary size, then one far larger in a few rows of A or of B: what was summed before it counts in
    the rows that stay small, and rows of zeros stay zero."""
    M, N, K = shape
    g = torch.Generator().manual_seed(7)
    x, w = torch.randn(M, K, generator=g), torch.randn(N, K, generator=g)
    x[::5, K // 2:] *= 2.0 ** 70
    x[1::7] = 0.0
    w[N // 2:N // 2 + 3, K // 4:] *= 2.0 ** 40
    qa, sa = (t.to(dev) for t in quantised(x, E4M3))
    qb, sb = (t.to(dev) for t in quantised(w, E4M3, BLOCK if tiles else 1))
    A, B = values(qa, sa), values(qb, sb)
    want = A @ B.t().contiguous()
    for out_dtype in (F32, BF16):
        print("case growing scales", shape, tiles, out_dtype, flush=True)
        got = fp64_emu.mm_f8(qa, sa, qb, sb, out_dtype=out_dtype).to(F64)
        bound = product_bound(A, B, want, out_dtype, out_dtype == F32)
        assert ((got - want).abs() <= bound).all(), ((got - want).abs() / bound).max().item()


@pytest.mark.parametrize("shape", SHAPES)
def test_callers_own_scales(dev, shape):
    """Scales that the quantiser never gives: negative, zero and denormal ones act as the factors they are."""
    M, N, K = shape
    g = torch.Generator().manual_seed(6)
    qa, _ = quantised(torch.randn(M, K, generator=g), E4M3)
    qb, _ = quantised(torch.randn(N, K, generator=g), E4M3)
    kb = -(-K // BLOCK)
    sa = torch.rand(M, kb, generator=g) - 0.5
    sa[:, ::3] = 0.0
    sb = torch.ldexp(torch.rand(N, kb, generator=g) - 0.5, torch.tensor(3))
    for factor_a, factor_b in ((1.0, 1.0), (2.0 ** -130, 2.0 ** 40), (2.0 ** 126, 2.0 ** -126)):
        s1, s2 = (sa * factor_a).to(dev), (sb * factor_b).to(dev)
        q1, q2 = qa.to(dev), qb.to(dev)
        A, B = values(q1, s1), values(q2, s2)
        want = A @ B.t().contiguous()
        for out_dtype in (F32, BF16):
            print("case own scales", shape, factor_a, out_dtype, flush=True)
            got = fp64_emu.mm_f8(q1, s1, q2, s2, out_dtype=out_dtype).to(F64)
            bound = product_bound(A, B, want, out_dtype, out_dtype == F32)
            assert ((got - want).abs() <= bound).all(), ((got - want).abs() / bound).max().item()
