"""Flags of the 4-bit products that there are none of, without a GPU."""
import ctypes

from mkernel_b200 import _lib
from tests.test_w4_cpu import view


def test_unknown_flags_are_refused():
    lib = _lib.lib()
    ok = ctypes.byref(view(data=4096))
    assert lib.mk_w4_gemm_ex(4096, 128, ok, 4096, 64, 1, 2, None) == -1 and "flags" in _lib.last_error()
    assert lib.mk_w4_gemm_ex(4096, 127, ok, 4096, 64, 2, _lib.MK_W4_EXACT, None) == -1
    assert lib.mk_w4_gemm_ex(None, 0, ok, None, 0, 0, _lib.MK_W4_EXACT, None) == 0
    turned = ctypes.byref(view(form=2, head_dim=64, rotary_dim=64, rotated=1, data=4096))
    assert lib.mk_w4_gemm_rotary_ex(4096, 128, turned, 4096, 64, 1, 4096, 0, 4096, 1.0, -1, None) == -1
    assert "flags" in _lib.last_error()


def test_plan_refusals():
    lib, out = _lib.lib(), _lib.W4Plan()
    assert lib.mk_w4_plan_product(ctypes.byref(view()), 0, 0, ctypes.byref(out)) == -1
    assert lib.mk_w4_plan_product(ctypes.byref(view()), 1, 4, ctypes.byref(out)) == -1
    assert lib.mk_w4_plan_product(ctypes.byref(view()), 1, 0, None) == -1
    assert lib.mk_w4_plan_product(ctypes.byref(view(group=5)), 1, 0, ctypes.byref(out)) == -1
