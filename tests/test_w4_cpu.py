"""What the 4-bit products and rotary positions refuse, and their host arithmetic, without a GPU."""
import ctypes
import math

import pytest
import torch

from mkernel_b200 import _lib, ops
from oracle import w4_oracle as orc


def view(N=64, K=128, group=128, dtype=0, zeros=0, form=0, head_dim=0, rotary_dim=0, rotated=0, data=None):
    return _lib.W4View(data, N, K, group, dtype, zeros, form, head_dim, rotary_dim, rotated, 0)


@pytest.mark.parametrize("N,K,group,zeros", [(64, 128, 128, 0), (1, 1, 32, 1), (65, 129, 64, 1), (8192, 8192, 128, 0),
                                             (131072, 65536, 32, 1)])
def test_bytes_are_the_chunks(N, K, group, zeros):
    """64 x 128 codes a chunk, half a byte each, and 2 bytes a scale (and a zero point) per row and group."""
    chunks = -(-N // 64) * -(-K // 128)
    want = chunks * (4096 + 128 // group * 128 * (1 + zeros))
    assert _lib.lib().mk_w4_bytes(ctypes.byref(view(N, K, group, zeros=zeros))) == want


@pytest.mark.parametrize("bad", [
    dict(N=0), dict(K=0), dict(N=-5), dict(group=48), dict(group=256), dict(dtype=2), dict(form=3), dict(form=1, N=63),
    dict(form=2), dict(form=2, head_dim=64, rotary_dim=65), dict(form=2, head_dim=64, rotary_dim=66),
    dict(form=2, head_dim=60, rotary_dim=8), dict(form=2, head_dim=32, rotary_dim=32, rotated=3),
    dict(form=2, head_dim=32, rotary_dim=32, rotated=-1), dict(N=2 ** 31 - 1, K=64),
])
def test_bad_weights_are_refused(bad):
    v = view(**bad)
    assert _lib.lib().mk_w4_bytes(ctypes.byref(v)) == -1
    assert "mk_w4_bytes" in _lib.last_error()
    v.data = 256
    assert _lib.lib().mk_w4_gemm(256, 10 ** 10, ctypes.byref(v), 256, 10 ** 10, 1, None) == -1


def test_bad_operands_are_refused():
    lib = _lib.lib()
    ok = ctypes.byref(view(data=4096))
    assert lib.mk_w4_bytes(None) == -1
    assert lib.mk_w4_gemm(None, 128, ok, 4096, 64, 1, None) == -1
    assert lib.mk_w4_gemm(4096, 127, ok, 4096, 64, 2, None) == -1       # row strides below the row
    assert lib.mk_w4_gemm(4096, 128, ok, 4096, 63, 2, None) == -1
    assert lib.mk_w4_gemm(4097, 128, ok, 4096, 64, 1, None) == -1       # half an element
    assert lib.mk_w4_gemm(4096, 128, ok, 4096, 64, -1, None) == -1
    assert lib.mk_w4_gemm(4096, 128, ctypes.byref(view(data=4100)), 4096, 64, 1, None) == -1
    assert lib.mk_w4_gemm(4096, 128, ctypes.byref(view()), 4096, 64, 1, None) == -1
    assert lib.mk_w4_gemm_swiglu(4096, 128, ok, 4096, 64, 1, None) == -1   # another form
    assert "form" in _lib.last_error()
    turned = ctypes.byref(view(form=2, head_dim=64, rotary_dim=64, rotated=1, data=4096))
    assert lib.mk_w4_gemm_rotary(4096, 128, turned, 4096, 64, 1, None, 0, 4096, 1.0, None) == -1
    assert lib.mk_w4_gemm_rotary(4096, 128, turned, 4096, 64, 1, 4100, 1, 4096, 1.0, None) == -1
    assert lib.mk_w4_pack(ok, None, 4096, None, None) == -1
    assert lib.mk_w4_pack(ok, 4096, 4096, 4096, None) == -1              # zero points that are not stored
    assert lib.mk_w4_pack(ctypes.byref(view(zeros=1, data=4096)), 4096, 4096, None, None) == -1
    assert lib.mk_w4_quantize(ok, 4096, 127, 0, None) == -1
    assert lib.mk_w4_quantize(ok, 4096, 128, 3, None) == -1
    assert lib.mk_w4_quantize(ok, 4098, 128, 2, None) == -1
    assert lib.mk_w4_dequantize(ok, None, 128, 0, None) == -1
    assert lib.mk_w4_dequantize(ok, 4096, 128, 7, None) == -1
    assert lib.mk_w4_bytes(ctypes.byref(view(N=65536 * 64, K=64))) == -1
    assert lib.mk_w4_bytes(ctypes.byref(view(N=64, K=(1 << 30) + 1))) == -1
    assert lib.mk_w4_bytes(ctypes.byref(view(N=64, K=1 << 30))) == (1 << 23) * (4096 + 128 * 128 // view().group)
    assert lib.mk_w4_gemm(4098, 128, ok, 4096, 64, 17, None) == -1      # rows that start on no 16 bytes
    assert lib.mk_w4_gemm(4096, 132, ok, 4096, 64, 17, None) == -1
    assert "mk_align_rows" in _lib.last_error()
    assert lib.mk_align_rows(4096, 100, 2, 101, 8192, 104, None) == -1
    assert lib.mk_align_rows(4096, 100, 2, 100, 8192, 100, None) == -1
    assert lib.mk_align_rows(4096, 100, 2, 100, 8200, 104, None) == -1
    assert lib.mk_align_rows(None, 100, 2, 100, 8192, 104, None) == -1
    assert lib.mk_align_rows(None, 100, 0, 100, None, 104, None) == 0
    assert lib.mk_w4_gemm(None, 0, ok, None, 0, 0, None) == 0             # no rows, nothing to do


def test_rotary_refusals():
    lib = _lib.lib()

    def call(x=4096, xr=32, xh=16, y=8192, yr=32, yh=16, rows=4, heads=2, dim=16, rot=8, dtype=0, pos=4096, pos64=1,
             freq=4096):
        return lib.mk_rotary(x, xr, xh, y, yr, yh, rows, heads, dim, rot, dtype, pos, pos64, freq, 1.0, 0, 0, None)

    for bad in (dict(rot=0), dict(rot=7), dict(rot=18), dict(dtype=3), dict(rows=-1), dict(heads=-1), dict(dim=0),
                dict(x=None), dict(y=None), dict(pos=None), dict(freq=None), dict(x=4097), dict(y=8193), dict(pos=4100),
                dict(freq=4098), dict(y=4096, yr=64)):
        assert call(**bad) == -1, bad
    assert call(rows=0) == 0 and call(heads=0, x=None) == 0


def test_tensors_on_the_host_are_refused():
    t = torch.zeros((4, 128), dtype=torch.bfloat16)
    for call in (lambda: ops.w4_quantize(t), lambda: ops.w4_pack(t.byte(), t, K=256),
                 lambda: ops.rotary(t.view(4, 8, 16), torch.zeros(4, dtype=torch.int64), torch.ones(8))):
        with pytest.raises(RuntimeError):
            call()


def test_oracle_quantiser_and_nibbles():
    w = torch.tensor([[-7.0, 3.5, 0.4, -0.5, 7.0]])
    q, s, z = orc.quantize(w, 32, False, torch.bfloat16)
    assert s.tolist() == [[1.0]] and q.tolist() == [[1, 12, 8, 8, 15]]       # 3.5 and -0.5 go to even
    q, s, z = orc.quantize(torch.tensor([[-5.0, 10.0, 0.0]]), 32, True, torch.bfloat16)
    assert s.tolist() == [[1.0]] and z.tolist() == [[5]] and q.tolist() == [[0, 15, 5]]
    assert orc.pack_nibbles(torch.tensor([[1, 2, 3]])).tolist() == [[0x21, 0x03]]


def test_oracle_rotary_turns_by_the_angle():
    x = torch.tensor([[[1.0, 0.0, 5.0]]])
    y = orc.rotary(x, torch.tensor([1]), torch.tensor([math.pi / 2]))
    assert torch.allclose(y, torch.tensor([[[0.0, 1.0, 5.0]]], dtype=torch.float64), atol=1e-7)


def test_frequencies():
    plain, one = ops.rotary_frequencies(8, base=10000.0, device="cpu")
    want = torch.tensor([10000.0 ** (-2 * i / 8) for i in range(4)], dtype=torch.float64)
    assert one == 1.0 and plain.dtype == torch.float32 and torch.equal(plain, want.float())
    lin, one = ops.rotary_frequencies(8, scaling="linear", factor=4.0, device="cpu")
    assert one == 1.0 and torch.equal(lin, (want / 4).float())
    base, _ = ops.rotary_frequencies(8, scaling="base", factor=4.0, device="cpu")
    assert base[0] == 1.0 and math.isclose(base[-1].item(), want[-1].item() / 4, rel_tol=1e-6)
    d, length, factor = 64, 4096, 8.0
    plain64 = 10000.0 ** (-2 * torch.arange(d // 2, dtype=torch.float64) / d)
    turns = length * plain64 / (2 * math.pi)
    for scaling, low, high in (("parts", 1.0, 32.0), ("wavelength", 1.0, 4.0)):
        f, scale = ops.rotary_frequencies(d, scaling=scaling, factor=factor, original_length=length, low=low, high=high,
                                          device="cpu")
        ratio = (f.double() / plain64)
        assert ((ratio <= 1 + 1e-6) & (ratio >= 1 / factor - 1e-6)).all()
        assert (ratio[turns > high * 1.5] > 1 - 1e-6).all() and (ratio[turns < low / 1.5] < 1 / factor + 1e-6).all()
        assert (ratio[1:] <= ratio[:-1] + 1e-6).all()
        assert math.isclose(scale, 0.1 * math.log(factor) + 1 if scaling == "parts" else 1.0)
    for bad in (dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=8, scaling="other"),
                dict(rotary_dim=8, scaling="parts", factor=2.0), dict(rotary_dim=2, scaling="base", factor=2.0),
                dict(rotary_dim=8, factor=0.5), dict(rotary_dim=8, base=1.0)):
        with pytest.raises(RuntimeError):
            ops.rotary_frequencies(**bad, device="cpu")
