"""CPU tier: which kernel a product of 8-bit operands takes, and what it asks for: the rule runs on
the host.  And calls with nothing to do."""
import ctypes

import pytest

from fp64_emu import capi

BF16 = 1


def _product(M, N, K, batch=1, dtype=BF16, ld=None):
    a, b = (capi.F8(0x1000, 0x1000, K if ld is None else ld, 0, 1, r, 0, 0, 0) for r in (M, N))
    return capi.MmF8(0x1000, N, 0, dtype, 0, a, b, batch, M, N, K)


def test_plan():
    """The rule as the library tells it: one kernel for one token, tiles for large products, rows laid out again
    where a tile kernel cannot copy them."""
    p = capi.mm_f8_plan(1, 8192, 8192, BF16)
    assert (p.tile_m, p.splits, p.exact, p.relaid_a, p.relaid_b) == (16, 1, 1, 0, 0)
    p = capi.mm_f8_plan(8192, 8192, 8192, BF16)
    assert (p.tile_m, p.tile_n, p.splits, p.exact, p.relaid_a) == (256, 256, 1, 0, 0)
    p = capi.mm_f8_plan(8192, 8192, 8192, 0)
    assert (p.tile_m, p.tile_n, p.splits, p.exact) == (128, 256, 1, 1)
    p = capi.mm_f8_plan(8192, 8192, 8191, BF16, ld=8191)
    assert (p.relaid_a, p.relaid_b) == (1, 1)
    assert capi.mm_f8_plan(0, 8192, 8192, BF16).splits == 0
    for a in ((-1, 8, 8, BF16), (8, 8, 8, 7), (1 << 31, 8, 8, BF16)):
        with pytest.raises(capi.CapiError):
            capi.mm_f8_plan(*a)
    assert capi.lib().fp64emu_mm_f8_plan(ctypes.byref(_product(8, 8, 8)), None) == 1


def test_any_width_has_a_kernel():
    """More few-row work groups than a launch takes: tiles, or a refusal before any room is asked for."""
    p = capi.mm_f8_plan(1, 2 ** 27, 128, BF16)
    assert p.tile_m == 128 and p.splits == 1
    L = capi.lib()
    p = _product(1, 1, 128, batch=2 ** 25)
    assert L.fp64emu_mm_f8_workspace(ctypes.byref(p)) == 0
    assert L.fp64emu_mm_f8(ctypes.byref(p), None, 0, None) == 1 and b"too large for one launch" in L.fp64emu_last_error()


def test_any_depth_has_a_kernel():
    """Tile kernels hold a row's offset in 32 bits (2^24 codes); deeper products take few rows, whatever their
    other sizes, and ask for no room to lay their operands out again: partial sums alone, 32 of them at most."""
    L = capi.lib()
    for K in (2 ** 24 - 300, 2 ** 24 - 256, 2 ** 24, 17_000_000, 2 ** 31 - 256):
        for M, N in ((1, 1000), (1000, 1000), (4096, 8192)):
            for dtype in (0, 1, 2):
                p = _product(M, N, K, dtype=dtype, ld=-(-K // 16) * 16)
                need = L.fp64emu_mm_f8_workspace(ctypes.byref(p))
                assert need <= 32 * 4 * M * N + 256, (M, N, K, need)
                # Short of its room, the call says so; no depth is refused for itself.
                p.out = 0x1000
                if need:
                    assert L.fp64emu_mm_f8(ctypes.byref(p), None, 0, None) == 2
                    assert b"workspace too small" in L.fp64emu_last_error()


def test_empty_activation():
    """No rows or no columns: nothing to do, whatever of the outputs is NULL (an empty tensor's memory is)."""
    L = capi.lib()
    for M, F in ((0, 256), (4, 0), (0, 0)):
        assert L.fp64emu_swiglu_f8(None, BF16, M, F, 2 * F, None, F, None, None, None, None) == 0
        keep = capi.F8(None, None, 2 * F, 0, 1, M, 0, 0, 0)
        assert L.fp64emu_swiglu_f8_backward(None, BF16, M, F, F, ctypes.byref(keep), None, BF16, 2 * F, None, None, None) == 0
