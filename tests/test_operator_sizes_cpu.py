"""Widths at which 32-bit column and item numbers would run out are refused before anything is launched."""
import ctypes as C

import pytest

ONE = C.c_void_p(256)      # never dereferenced


@pytest.fixture(scope="module")
def lib():
    import __graft_entry__
    __graft_entry__.build()
    from momoe import _lib
    return _lib


@pytest.mark.parametrize("wide", [2 ** 31 - 16, 2 ** 30 + 16])
def test_widths_beyond_32_bits(lib, wide):
    L = lib.lib
    assert L.momoe_quantize_rows(ONE, wide, 0, 1, wide, ONE, ONE, None) == -4
    assert L.momoe_fp8_quantize_weights(ONE, 0, 1, wide, 1, 128, ONE, ONE, None) == -4
    assert L.momoe_fp8_quantize_weights(ONE, 0, 1, 128, 1, wide, ONE, ONE, None) == -4
    assert L.momoe_fp8_dispatch_rows(ONE, None, ONE, ONE, 4, 8, 2, wide, ONE, ONE, ONE, ONE, ONE, ONE, ONE, 128 * 9, ONE, 0,
                                     ONE, ONE, ONE, None) == -4
    for D, H in ((wide, 32), (32, wide)):
        plan = lib.Plan(M=4, N=8, K=2, D=D, H=H, reserved=0, rows_capacity=128 * 9, sched=16, tile_expert=16, pad_off=16,
                        row_token=16, row_weight=16, pos_MK=16, status=16, pair_info=16)
        for f in (L.momoe_fp8_up_swiglu, L.momoe_fp8_up_swiglu_decode, L.momoe_fp8_down_scale, L.momoe_fp8_down_scale_decode):
            assert f(C.byref(plan), ONE, ONE, ONE, ONE, ONE, ONE, ONE, None) == -4
        assert L.momoe_fp8_experts_forward(ONE, None, ONE, ONE, 4, 8, 2, D, H, ONE, ONE, ONE, ONE, 16, ONE, ONE, ONE, 1 << 62,
                                           ONE, None) == -4
