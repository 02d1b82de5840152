"""GPU tier: every kernel of the 8-bit products against float64, each case with the kernel it is there for
(capi.mm_f8_plan), so that a change of the rule cannot move a test off its kernel unseen."""
import math

import pytest
import torch

import fp64_emu
from fp64_emu import capi
from f8_util import E4M3, E5M2, F64, operand, product_bound, values

pytestmark = pytest.mark.gpu

BF16, FP16, F32 = torch.bfloat16, torch.float16, torch.float32
CODE = {F32: 0, BF16: 1, FP16: 2}
SPLIT = "split"

# (tile_m, tile_n, whole depth or split), members, M, N, K: ragged in every direction but where it says whole.
CASES16 = [((16, 16, 1), 1, 5, 130, 1000), ((16, 16, SPLIT), 1, 16, 64, 65536), ((32, 32, 1), 1, 20, 97, 1023),
           ((32, 32, SPLIT), 1, 20, 96, 20000), ((64, 32, SPLIT), 1, 64, 512, 16384), ((64, 32, SPLIT), 1, 257, 513, 1025),
           ((128, 128, 1), 1, 1000, 1101, 300), ((128, 128, 1), 1, 2048, 2048, 2048),       # (whole)
           ((128, 128, SPLIT), 1, 1000, 1001, 8000), ((128, 128, SPLIT), 1, 200, 301, 100000),
           ((128, 128, 1), 5, 513, 700, 600), ((128, 128, SPLIT), 3, 1100, 1100, 16000),
           ((256, 256, 1), 1, 4096, 4096, 1024),                                           # (whole)
           ((256, 256, 1), 1, 3001, 3010, 2900), ((256, 256, 1), 1, 4000, 4001, 700), ((256, 256, SPLIT), 1, 2000, 2101, 8200),
           ((256, 256, 1), 8, 1000, 1100, 500), ((256, 256, 1), 64, 512, 512, 512)]
CASES32 = [((16, 16, 1), 1, 5, 130, 1000), ((32, 32, SPLIT), 1, 20, 96, 20000), ((64, 32, 1), 1, 300, 301, 256),
           ((128, 128, 1), 1, 1000, 1101, 300), ((128, 128, SPLIT), 1, 1000, 1001, 8000),
           ((128, 128, SPLIT), 3, 1100, 1100, 16000), ((128, 128, 1), 5, 513, 700, 600),
           ((128, 256, 1), 1, 2000, 2101, 8200), ((128, 256, 1), 1, 4096, 4096, 8192),       # (whole)
           ((128, 256, SPLIT), 1, 260, 8200, 16500), ((128, 256, 1), 2, 1500, 1501, 6000)]


def _plan(case, dtype, ld=None):
    form, batch, M, N, K = case
    p = capi.mm_f8_plan(M, N, K, CODE[dtype], batch, ld)
    assert (p.tile_m, p.tile_n, p.splits if form[2] == 1 else SPLIT) == form and (form[2] == 1) == (p.splits == 1)
    return p


def _in_norm(dtype, exact):
    """The largest error in norm: roundings of at most half a last place, uniformly (2^-p / sqrt 3 where every
    significand is near 1), beside block sums that lose up to 4e-5 of theirs (1e-4 taken) or float32 sums (2^-20)."""
    return {F32: 0.0, BF16: 2.0 ** -8, FP16: 2.0 ** -11}[dtype] / math.sqrt(3) + (2.0 ** -20 if exact else 1e-4)


def _check(got, want, A, B, dtype, exact):
    err = got.to(F64) - want
    bound = product_bound(A, B, want, dtype, exact)
    assert (err.abs() <= bound).all(), ((err.abs() / bound).max().item(), (err.abs() > bound).sum().item())
    assert err.norm() <= want.norm() * _in_norm(dtype, exact), (err.norm() / want.norm()).item()


def _run(case, dtype, tiles, accumulate, fa, fb, dev, seed=0):
    form, batch, M, N, K = case
    plan = _plan(case, dtype)
    lead = (batch,) if batch > 1 else ()
    qa, sa = operand((*lead, M, K), seed + 1, fa, device=dev)
    qb, sb = operand((*lead, N, K), seed + 2, fb, tiles, device=dev)
    A, B = values(qa, sa), values(qb, sb)
    want = A @ B.transpose(-1, -2).contiguous()
    out = None
    if accumulate:
        out = (torch.randn(want.shape, device=dev, generator=torch.Generator(dev).manual_seed(seed)) * want.std()).to(dtype)
        want = want + out.to(F64)
    fn = fp64_emu.bmm_f8 if lead else fp64_emu.mm_f8
    got = fn(qa, sa, qb, sb, out_dtype=dtype, out=out, accumulate=accumulate)
    _check(got, want, A, B, dtype, bool(plan.exact))


@pytest.mark.parametrize("tiles", [True, False])
@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("case", CASES16, ids=str)
def test_16_bit_outputs(dev, case, accumulate, tiles):
    print("case 16 bits", case, accumulate, tiles, flush=True)
    _run(case, BF16, tiles, accumulate, E4M3, E4M3, dev)
    if case[0][2] == 1 and case[1] == 1:
        _run(case, FP16, tiles, accumulate, E4M3, E5M2 if accumulate else E4M3, dev, 3)


@pytest.mark.parametrize("tiles", [True, False])
@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("case", CASES32, ids=str)
def test_float32_outputs(dev, case, accumulate, tiles):
    print("case 32 bits", case, accumulate, tiles, flush=True)
    _run(case, F32, tiles, accumulate, E5M2 if accumulate else E4M3, E4M3, dev, 5)


@pytest.mark.parametrize("case,dtype", [(((128, 128, 1), 1, 1000, 1101, 300), BF16), (((128, 128, 1), 1, 1000, 1101, 300), F32),
                                        (((128, 128, SPLIT), 1, 1000, 1001, 8000), BF16),
                                        (((128, 128, SPLIT), 1, 1000, 1001, 8000), F32),
                                        (((256, 256, 1), 1, 3001, 3010, 2900), BF16),
                                        (((128, 256, 1), 1, 2000, 2101, 8200), F32)], ids=str)
def test_rows_laid_out_again(dev, case, dtype):
    """Rows that do not start at 16 bytes, on tiles: the same bits as from the quantiser's own layout."""
    _, _, M, N, K = case
    plan = _plan(case, dtype, K + 3)
    assert plan.relaid_a and plan.relaid_b and not _plan(case, dtype).relaid_a
    print("case laid out again", case, dtype, flush=True)
    qa, sa = operand((M, K), 1, device=dev)
    qb, sb = operand((N, K), 2, tiles=True, device=dev)

    def rows(q, ld):
        room = torch.full((q.shape[0], ld), 0x7f, dtype=torch.uint8, device=dev).view(q.dtype)[:, :q.shape[1]]
        room.copy_(q)
        return room

    want = fp64_emu.mm_f8(rows(qa, -(-K // 16) * 16), sa, rows(qb, -(-K // 16) * 16), sb, out_dtype=dtype)
    assert torch.equal(fp64_emu.mm_f8(rows(qa, K + 3), sa, rows(qb, K + 3), sb, out_dtype=dtype), want)


@pytest.mark.parametrize("M,N,K", [(1000, 1001, 8001), (200, 301, 100001)])
def test_captured_with_splits_and_rows_laid_out_again(dev, M, N, K):
    """A captured product that lays its operands out again and joins partial sums replays to the eager bits, with eager
    work between the replays."""
    plan = _plan(((128, 128, SPLIT), 1, M, N, K), BF16, K)
    assert plan.splits > 1 and plan.relaid_a and plan.relaid_b
    print("case captured", M, N, K, flush=True)
    qa, sa = operand((M, K), 1, device=dev)
    qb, sb = operand((N, K), 2, tiles=True, device=dev)
    want = fp64_emu.mm_f8(qa, sa, qb, sb)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = fp64_emu.mm_f8(qa, sa, qb, sb)
    for r in range(4):
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want), r
        fp64_emu.mm_f8(qa, sa, qb, sb)
        torch.cuda.synchronize()


def test_rows_of_b_by_rows_and_nan(dev):
    """A NaN in one row of B's scales or codes on 256 x 256 tiles by rows: its column and no other."""
    case = ((256, 256, 1), 1, 3001, 3010, 2900)
    _plan(case, BF16)
    print("case NaN", case, flush=True)
    qa, sa = operand((3001, 2900), 1, device=dev)
    qb, sb = operand((3010, 2900), 2, device=dev)
    clean = fp64_emu.mm_f8(qa, sa, qb, sb)
    sb[3009, 22] = math.nan
    qa.view(torch.uint8)[3000, 2899] = 0x7f
    got = fp64_emu.mm_f8(qa, sa, qb, sb)
    hit = torch.zeros_like(got, dtype=torch.bool)
    hit[3000] = True
    hit[:, 3009] = True
    assert torch.isnan(got[hit]).all() and torch.equal(got[~hit], clean[~hit])
