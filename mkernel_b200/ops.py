"""Host-side operator functions with the reference's Python-callable signatures.

Each function checks shapes the way the reference's pybind lambdas do and forwards raw pointers
to the C ABI on the current torch CUDA stream.  References:
  ag_gemm_warp_specialized_prepare/_launch  include/operators/ag_gemm/ag_gemm_warp_specialized_session.cuh:12-47
  gemm_rs_blackwell_prepare/_launch         include/operators/gemm_rs/gemm_rs_blackwell_session.cuh:11-40
  gemm_ar_intranode_blackwell               include/operators/gemm_ar/gemm_ar_blackwell.cuh:205-246
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .dist_buffer import DistBuffer

ag_gemm_warp_specialized_ready_words = _lib.MK_AG_READY_WORDS
gemm_rs_blackwell_sync_shape = (_lib.MK_RS_SYNC_WORDS,)
gemm_ar_blackwell_barrier_shape = (2, 1024, 1024)


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream() -> ctypes.c_void_p:
    """The current torch CUDA stream of the current device as a raw cudaStream_t."""
    if _raw_stream is not None:
        return ctypes.c_void_p(_raw_stream(torch.cuda.current_device()))
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


# Moves the version counters of tensors that a kernel has written through their addresses.
_count_as_changed = getattr(torch._C, "_increment_version", None) or torch.autograd.graph.increment_version

_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _raw_stream_of(index: int):
    """The current torch stream of device `index` as an address."""
    if _raw_stream is not None:
        return _raw_stream(index)
    return torch.cuda.current_stream(index).cuda_stream


def _call_on(index: int, call, *args) -> None:
    """call(*args, stream) on device `index` and its current stream; raises what the library reports."""
    if _current_device() != index:
        with _on_device(index):
            rc = call(*args, _raw_stream_of(index))
    else:
        rc = call(*args, _raw_stream_of(index))
    if rc < 0:
        _lib.check(rc)


class _on_device:
    """Make `index` the current CUDA device for the duration of a call; free when it already is
    (the common case: one process per GPU), since these wrappers sit on latency-bound paths."""

    __slots__ = ("index", "prev")

    def __init__(self, index):
        self.index = index.index if isinstance(index, torch.device) else int(index)
        self.prev = None

    def __enter__(self):
        cur = torch.cuda.current_device()
        if cur != self.index:
            self.prev = cur
            torch.cuda.set_device(self.index)

    def __exit__(self, *exc):
        if self.prev is not None:
            torch.cuda.set_device(self.prev)
        return False


def _require(cond: bool, msg: str) -> None:
    if not cond:
        raise RuntimeError(msg)


def _bf16_matrix(t: torch.Tensor, name: str) -> None:
    _require(isinstance(t, torch.Tensor) and t.is_cuda, f"{name} must be a CUDA tensor")
    _require(t.dtype == torch.bfloat16, f"{name} must be bfloat16")
    _require(t.is_contiguous(), f"{name} must be contiguous")


def gemm_bf16(A: torch.Tensor, B: torch.Tensor, C: torch.Tensor, b_layout: int = _lib.MK_B_NK,
              status: torch.Tensor | None = None) -> None:
    """C[M,N] = A[M,K] @ B on one GPU; B is [N,K] (MK_B_NK) or [K,N] (MK_B_KN)."""
    for t, n in ((A, "A"), (B, "B"), (C, "C")):
        _bf16_matrix(t, n)
    M, K = A.shape
    N = B.shape[0] if b_layout == _lib.MK_B_NK else B.shape[1]
    kb = B.shape[1] if b_layout == _lib.MK_B_NK else B.shape[0]
    _require(kb == K, f"A and B disagree on K: {K} vs {kb}")
    _require(tuple(C.shape) == (M, N), f"C must be [{M},{N}]")
    with _on_device(A.device):
        _lib.check(_lib.lib().mk_gemm_bf16(A.data_ptr(), B.data_ptr(), C.data_ptr(), M, N, K,
                                           b_layout, status.data_ptr() if status is not None else None,
                                           _stream()))


def ag_gemm_warp_specialized_prepare(A_copy_ready: DistBuffer, M: int = 0, N: int = 0) -> None:
    """All-rank entry barrier + epoch bump on the current stream (M, N kept for compatibility)."""
    _require(isinstance(A_copy_ready, DistBuffer), "A_copy_ready must be a DistBuffer")
    with _on_device(A_copy_ready.local_rank_):
        _lib.check(_lib.lib().mk_ag_gemm_prepare(A_copy_ready.view_ref(), _stream()))


def ag_gemm_warp_specialized_launch(A: DistBuffer, A_copy_ready: DistBuffer, B: torch.Tensor,
                                    C: torch.Tensor) -> None:
    """C[d] = A_shard[d] @ B^T for every shard d.  A: DistBuffer [W, M/W, K]; B: [N, K];
    C: [W, M/W, N]."""
    _require(isinstance(A, DistBuffer) and isinstance(A_copy_ready, DistBuffer),
             "A and A_copy_ready must be DistBuffers")
    _require(A.dtype == torch.bfloat16 and len(A.shape) == 3, "A must be bf16 [W, M/W, K]")
    _bf16_matrix(B, "B")
    _require(C.dtype == torch.bfloat16 and C.is_cuda and C.is_contiguous() and C.dim() == 3,
             "C must be a contiguous bf16 CUDA tensor [W, M/W, N]")
    W, Ms, K = A.shape
    _require(W == A.local_world_size_, "A.shape[0] must equal the local world size")
    N = B.size(0)
    _require(B.size(1) == K, f"B must be [N, K] with K={K}")
    _require(tuple(C.shape) == (W, Ms, N), f"C must be [{W},{Ms},{N}]")
    with _on_device(A.local_rank_):
        _lib.check(_lib.lib().mk_ag_gemm_launch(A.view_ref(), A_copy_ready.view_ref(),
                                                B.data_ptr(), C.data_ptr(), W * Ms, N, K,
                                                _stream()))


def interleave_gate_up(w_gate: torch.Tensor, w_up: torch.Tensor) -> torch.Tensor:
    """Weight layout of ``ag_gemm_swiglu_launch``: per block of 256 rows, 128 rows of the gate
    projection followed by the 128 rows of the up projection of the same outputs.
    w_gate, w_up: [I, K] with I a multiple of 128 -> [2 I, K]."""
    I, K = w_gate.shape
    _require(tuple(w_up.shape) == (I, K) and I % 128 == 0,
             "w_gate and w_up must both be [I, K] with I a multiple of 128")
    return torch.stack((w_gate.view(I // 128, 128, K), w_up.view(I // 128, 128, K)),
                       dim=1).reshape(2 * I, K).contiguous()


def ag_gemm_swiglu_launch(A: DistBuffer, A_copy_ready: DistBuffer, B_gate_up: torch.Tensor,
                          H: torch.Tensor) -> None:
    """H[d] = silu(A_shard[d] @ G^T) * (A_shard[d] @ U^T) for every shard d: AllGather+GEMM of
    the gate and up projections with the activation fused into the epilogue (the gated
    activation never crosses HBM as [M, 2I]).  A: DistBuffer [W, M/W, K]; B_gate_up: [2I, K] from
    ``interleave_gate_up``; H: [W, M/W, I].  No counterpart call in the reference's TP modules;
    its MoE kernel fuses the same epilogue (src/dispatch_gemm_glu_combine.cu:21-25)."""
    _require(isinstance(A, DistBuffer) and isinstance(A_copy_ready, DistBuffer),
             "A and A_copy_ready must be DistBuffers")
    _require(A.dtype == torch.bfloat16 and len(A.shape) == 3, "A must be bf16 [W, M/W, K]")
    _bf16_matrix(B_gate_up, "B_gate_up")
    W, Ms, K = A.shape
    N2 = B_gate_up.size(0)
    _require(B_gate_up.size(1) == K and N2 % 256 == 0,
             f"B_gate_up must be [2I, K] with K={K} and 2I a multiple of 256")
    _require(H.dtype == torch.bfloat16 and H.is_cuda and H.is_contiguous() and
             tuple(H.shape) == (W, Ms, N2 // 2), f"H must be a contiguous bf16 [{W},{Ms},{N2 // 2}]")
    with _on_device(A.local_rank_):
        _lib.check(_lib.lib().mk_ag_gemm_swiglu_launch(A.view_ref(), A_copy_ready.view_ref(),
                                                       B_gate_up.data_ptr(), H.data_ptr(),
                                                       W * Ms, N2, K, _stream()))


_W4_FORMS = {"plain": _lib.MK_W4_PLAIN, "gate_up": _lib.MK_W4_GATE_UP, "rotary": _lib.MK_W4_ROTARY}
_DTYPES = {torch.bfloat16: _lib.MK_BF16, torch.float16: _lib.MK_FP16, torch.float32: _lib.MK_FP32}


class W4Weight:
    """A matrix [N, K] of 4-bit weights in the library's layout, made once by ``w4_quantize`` or
    ``w4_pack`` and taken by ``w4_gemm``, ``w4_gemm_swiglu`` or ``w4_gemm_rotary`` (according to
    ``form``).  ``data`` is the packed buffer, ``dtype`` the type of its scales and of the activations."""

    def __init__(self, N: int, K: int, group: int, dtype: torch.dtype, zero_points: bool, device,
                 form: str = "plain", head_dim: int = 0, rotary_dim: int = 0, rotated_heads: int = 0,
                 interleaved: bool = False):
        if not (0 < N <= 0x7fffffff and 0 < K <= 0x7fffffff):
            _require(False, f"bad shape [{N}, {K}]")
        if form not in _W4_FORMS:
            _require(False, f"form must be one of {sorted(_W4_FORMS)}")
        if dtype is not torch.bfloat16 and dtype is not torch.float16:
            _require(False, "4-bit weights have bfloat16 or float16 scales")
        if form != "rotary" and (head_dim or rotary_dim or rotated_heads or interleaved):
            _require(False, "head_dim, rotary_dim, rotated_heads and interleaved belong to form 'rotary'")
        self.shape, self.K, self.group, self.dtype, self.form = (N, K), K, group, dtype, form
        self.n_out = N // 2 if form == "gate_up" else N
        self.zero_points, self.rotary_dim = bool(zero_points), rotary_dim
        view = _lib.W4View(None, N, K, group, _DTYPES[dtype], self.zero_points, _W4_FORMS[form], head_dim,
                           rotary_dim, rotated_heads, bool(interleaved))
        self.view, self.view_ref = view, ctypes.byref(view)
        nbytes = _lib.lib().mk_w4_bytes(self.view_ref)
        if nbytes < 0:
            _lib.check(nbytes)
        self.data = data = torch.empty(nbytes, dtype=torch.uint8, device=device)
        self.device, self.index = data.device, data.get_device()
        view.data = data.data_ptr()

    def dequantize(self, out: torch.Tensor | None = None) -> torch.Tensor:
        """The matrix these weights stand for, rows in the order given to ``w4_quantize`` or
        ``w4_pack``, in ``out``'s type (by default a new tensor of this weight's type)."""
        if out is None:
            out = torch.empty(self.shape, dtype=self.dtype, device=self.device)
        (N, K), (ld, step) = self.shape, out.stride() if out.dim() == 2 else (0, 0)
        if out.get_device() != self.index or out.dtype not in _DTYPES or out.shape != self.shape or \
                (step != 1 and K > 1) or (ld < K and N > 1):
            _require(False, f"out must be {self.shape} on {self.device}, bfloat16, float16 or float32, rows contiguous")
        _call_on(self.index, _lib.lib().mk_w4_dequantize, self.view_ref, out.data_ptr(), ld if N > 1 else K,
                 _DTYPES[out.dtype])
        return out


def w4_quantize(weight: torch.Tensor, group: int = 128, zero_points: bool = False,
                dtype: torch.dtype | None = None, **form) -> W4Weight:
    """Round ``weight`` [N, K] (bfloat16, float16 or float32, rows contiguous) to 4 bits with one
    scale, and with ``zero_points`` one whole zero point, per row and ``group`` (32, 64 or 128) columns.
    ``dtype``: type of the scales and of the products' activations, by default the weight's.
    ``form``: nothing for ``w4_gemm``; ``form="gate_up"`` for ``w4_gemm_swiglu`` (gate rows, then up
    rows); ``form="rotary", head_dim=, rotary_dim=, rotated_heads=, interleaved=`` for
    ``w4_gemm_rotary``."""
    if not isinstance(weight, torch.Tensor) or not weight.is_cuda or weight.dim() != 2 or weight.dtype not in _DTYPES:
        _require(False, "weight must be a CUDA matrix of bfloat16, float16 or float32")
    src_dtype, (N, K), (ld, step) = weight.dtype, weight.shape, weight.stride()
    if (step != 1 and K > 1) or (ld < K and N > 1):
        _require(False, "weight's rows must be contiguous and not overlap")
    if dtype is None:
        dtype = src_dtype if src_dtype is not torch.float32 else torch.bfloat16
    W = W4Weight(N, K, group, dtype, zero_points, weight.device, **form)
    _call_on(W.index, _lib.lib().mk_w4_quantize, W.view_ref, weight.data_ptr(), ld if N > 1 else K, _DTYPES[src_dtype])
    return W


def w4_pack(codes: torch.Tensor, scales: torch.Tensor, zero_points: torch.Tensor | None = None, *,
            K: int, **form) -> W4Weight:
    """Lay out weights that are in 4 bits already: ``codes`` uint8 [N, (K + 1) // 2], two per byte, the even
    column in the low half; ``scales`` [N, ceil(K / group)] bfloat16 or float16; ``zero_points`` uint8 of
    the same shape (without: 8), any byte: a weight is (code - zero point) * scale.  The group (32, 64 or 128)
    follows from the shapes.  ``form`` as in
    ``w4_quantize``."""
    for t, n in ((codes, "codes"), (scales, "scales")) + (((zero_points, "zero_points"),) if zero_points is not None else ()):
        _require(isinstance(t, torch.Tensor) and t.is_cuda and t.dim() == 2 and t.is_contiguous()
                 and t.device == codes.device, f"{n} must be a contiguous CUDA matrix on the codes' device")
    _require(codes.dtype == torch.uint8, "codes must be uint8")
    _require(zero_points is None or zero_points.dtype == torch.uint8, "zero_points must be uint8")
    N, K = codes.shape[0], int(K)
    _require(tuple(codes.shape) == (N, (K + 1) // 2), f"codes must be [N, {(K + 1) // 2}] for K={K}")
    # where two groups give as many scales there is one scale a row, and it means the same
    group = next((g for g in (128, 64, 32) if -(-K // g) == scales.shape[1]), 0)
    _require(group > 0 and scales.shape[0] == N,
             f"scales must be [N, ceil(K / group)] with a group of 32, 64 or 128 (K={K})")
    _require(zero_points is None or zero_points.shape == scales.shape, "zero_points must have the scales' shape")
    W = W4Weight(N, K, group, scales.dtype, zero_points is not None, codes.device, **form)
    _call_on(W.index, _lib.lib().mk_w4_pack, W.view_ref, codes.data_ptr(), scales.data_ptr(),
             zero_points.data_ptr() if zero_points is not None else None)
    return W


def _w4_launch(call, A: torch.Tensor, W: W4Weight, C: torch.Tensor, form: str, *more) -> None:
    """Checks A [M, K] and C [M, outputs of W] and calls a product.  On the path of every token: each
    property of a tensor is read once, and what a message needs only when there is one."""
    if not isinstance(W, W4Weight) or W.form != form:
        _require(False, f"W must be a W4Weight of form '{form}' (w4_quantize, w4_pack)")
    a_shape, c_shape, a_stride, c_stride = A.shape, C.shape, A.stride(), C.stride()
    index, dtype = W.index, W.dtype
    if A.get_device() != index or C.get_device() != index:
        _require(False, f"A and C must be on the weights' device cuda:{index}")
    if A.dtype is not dtype or C.dtype is not dtype:
        _require(False, f"A and C must be {dtype} like the weights' scales")
    K, n_out = W.K, W.n_out
    if len(a_shape) != 2 or a_shape[1] != K:
        _require(False, f"A must be [M, {K}]")
    M = a_shape[0]
    if len(c_shape) != 2 or c_shape[0] != M or c_shape[1] != n_out:
        _require(False, f"C must be [{M}, {n_out}]")
    if (a_stride[1] != 1 and K != 1) or (c_stride[1] != 1 and n_out != 1):
        _require(False, "rows of A and C must be contiguous")
    lda, ldc = (a_stride[0], c_stride[0]) if M > 1 else (K, n_out)     # one row may have any stride
    if M > 1 and (ldc < n_out or M > 0x7fffffff):
        _require(False, "rows of C overlap, or are more than 2^31 - 1")
    a = A.data_ptr()
    if (a & 15 or (lda & 7 and M > 1)) and (M > 16 or M * K > 32768):
        # Rows that no 16-byte access can start on: more than 16 are copied, and few where a launch more costs less
        # than reading them element by element (8 rows of 8191, 1024 outputs: 6.4 us copied, 8.4 not; 2 rows of
        # 1023: 3.6 and 2.5; in between it gains less than the launch costs the host).
        lda = (K + 7) // 8 * 8
        rows = torch.empty((M, lda), dtype=dtype, device=W.device)
        if M:
            _call_on(index, _lib.lib().mk_align_rows, a, a_stride[0] if M > 1 else K, M, K, rows.data_ptr(), lda)
        a = rows.data_ptr()
    _call_on(index, call, a, lda, W.view_ref, C.data_ptr(), ldc, M, *more)


def w4_gemm(A: torch.Tensor, W: W4Weight, C: torch.Tensor, exact: bool = False) -> None:
    """C[M, N] = A[M, K] @ W^T with 4-bit weights: the single-token and small-batch form of
    ``gemm_bf16``.  A and C in the type of W's scales, rows that do not overlap at any stride, sharing no memory;
    fp32 sums, rounded once.
    For more than 16 rows the weights are rounded to that type first, as ``W.dequantize()`` gives them, which
    adds to the error less than the rounding of C (against 64 bits 1.3 times as much in all).  ``exact``: never, so
    a token's result is as good in a batch as alone; up to twice the tensor core's work."""
    if exact:
        _w4_launch(_lib.lib().mk_w4_gemm_ex, A, W, C, "plain", _lib.MK_W4_EXACT)
    else:
        _w4_launch(_lib.lib().mk_w4_gemm, A, W, C, "plain")


def w4_gemm_swiglu(A: torch.Tensor, W: W4Weight, H: torch.Tensor) -> None:
    """H[M, N/2] = silu(A @ G^T) * (A @ U^T), W of form "gate_up": the single-token form of
    ``ag_gemm_swiglu_launch``."""
    _w4_launch(_lib.lib().mk_w4_gemm_swiglu, A, W, H, "gate_up")


def _device_index(device) -> int:
    """The index of a device; of the current one for None and for "cuda" alone."""
    index = torch.device("cuda" if device is None else device).index
    return torch.cuda.current_device() if index is None else index


def w4_status(device=None) -> tuple[int, int, int, int]:
    """Status words of the 4-bit products on a device (by default the current one); raises MkError if a device wait of
    one of them has run out since ``w4_status_clear`` (its outputs hold NaN).  Synchronises the device."""
    out = (ctypes.c_uint32 * 4)()
    with _on_device(_device_index(device)):
        torch.cuda.synchronize()
        _lib.check(_lib.lib().mk_w4_status(out))
    return tuple(int(x) for x in out)


def w4_status_clear(device=None) -> None:
    """Clears what ``w4_status`` reads, on the current stream of the device."""
    with _on_device(_device_index(device)):
        _lib.check(_lib.lib().mk_w4_status_clear(_stream()))


def _rotary_operands(positions: torch.Tensor, inv_freq: torch.Tensor, rows: int, pairs: int, index: int) -> int:
    """Checks the operands that say how far to turn; returns whether positions have 64 bits."""
    if positions.get_device() != index or inv_freq.get_device() != index:
        _require(False, f"positions and inv_freq must be on cuda:{index}")
    wide = positions.dtype is torch.int64
    shape = positions.shape
    if not (wide or positions.dtype is torch.int32) or len(shape) != 1 or shape[0] != rows or \
            (rows > 1 and positions.stride(0) != 1):
        _require(False, f"positions must be contiguous int32 or int64 [{rows}]")
    shape = inv_freq.shape
    if inv_freq.dtype is not torch.float32 or len(shape) != 1 or (pairs >= 0 and shape[0] != pairs) or \
            (shape[0] > 1 and inv_freq.stride(0) != 1):
        _require(False, "inv_freq must be contiguous float32 [rotary_dim / 2]")
    return wide


def w4_gemm_rotary(A: torch.Tensor, W: W4Weight, C: torch.Tensor, positions: torch.Tensor,
                   inv_freq: torch.Tensor, scale: float = 1.0, exact: bool = False) -> None:
    """C[M, N] = A @ W^T, W of form "rotary": the query/key/value projection of M tokens with the
    rotated heads of row m turned by positions[m] before the rounding (see ``rotary``).  ``exact`` as in ``w4_gemm``."""
    if not isinstance(W, W4Weight) or W.form != "rotary":
        _require(False, "W must be a W4Weight of form 'rotary' (w4_quantize, w4_pack)")
    wide = _rotary_operands(positions, inv_freq, A.shape[0] if A.dim() else 0, W.rotary_dim // 2, W.index)
    if exact:
        _w4_launch(_lib.lib().mk_w4_gemm_rotary_ex, A, W, C, "rotary", positions.data_ptr(), wide, inv_freq.data_ptr(),
                   scale, _lib.MK_W4_EXACT)
    else:
        _w4_launch(_lib.lib().mk_w4_gemm_rotary, A, W, C, "rotary", positions.data_ptr(), wide, inv_freq.data_ptr(),
                   scale)


def _share_memory(x: int, xs, y: int, ys, rows: int, heads: int, dim: int, size: int) -> bool:
    """Whether [rows, heads, dim] at address x with strides xs and at y with strides ys may have an element in common.
    They have none where their address ranges do not meet, or where both step by one stride from window to
    window and the windows lie beside one another: two ranges of heads in the rows of one projection."""
    if not (rows and heads and x < y + size * ((rows - 1) * ys[0] + (heads - 1) * ys[1] + dim) and
            y < x + size * ((rows - 1) * xs[0] + (heads - 1) * xs[1] + dim)):
        return False
    for outer, inner, n in ((0, 1, heads), (1, 0, rows)):
        step, (apart, rest) = xs[outer], divmod(x - y, size)
        if step > 0 and step == ys[outer] and rest == 0 and (n - 1) * ys[inner] + dim <= apart % step and \
                apart % step + (n - 1) * xs[inner] + dim <= step:
            return False
    return True


def rotary(X: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor,
           Y: torch.Tensor | None = None, *, interleaved: bool = False, inverse: bool = False,
           scale: float = 1.0) -> torch.Tensor:
    """Turn the first 2 * len(inv_freq) features of every head of X [rows, heads, head_dim] by
    positions[row] * inv_freq (radians) and multiply them by ``scale``; pairs are (i, i + rotary_dim / 2),
    or neighbours with ``interleaved``.  Into Y, or in place without one; Y shares no memory with X unless
    it is X; the two may be ranges of heads of one buffer.  ``inverse`` turns back, which is the gradient: dX = rotary(dY, ..., inverse=True).  No graph is
    recorded: what is written must not require a gradient (X in place: call it on X.detach(), or under
    torch.no_grad()), and it counts as changed, so a backward pass that needs its old value says so.
    Features contiguous, any row and head strides: the queries and keys of a projection
    [rows, (heads + ...) * head_dim] are a view of its output."""
    shape, index, dtype = (X.shape, X.get_device(), X.dtype) if isinstance(X, torch.Tensor) else ((), -1, None)
    if index < 0 or dtype not in _DTYPES or len(shape) != 3:
        _require(False, "X must be a CUDA tensor [rows, heads, head_dim] of bfloat16, float16 or float32")
    xs, x = X.stride(), X.data_ptr()
    rows, heads, dim = shape
    if heads > 0x7fffffff or dim > 0x7fffffff:
        _require(False, "too many heads or features")
    if Y is None or Y is X:
        Y, ys, y = X, xs, x
    else:
        if Y.get_device() != index or Y.dtype is not dtype or Y.shape != shape:
            _require(False, "Y must have X's device, type and shape")
        ys, y = Y.stride(), Y.data_ptr()
        if (y != x or ys != xs) and _share_memory(x, xs, y, ys, rows, heads, dim, 4 if dtype is torch.float32 else 2):
            _require(False, "Y must be X, share no memory with it, or lie beside it in rows of the same stride")
    if dim > 1 and (xs[2] != 1 or ys[2] != 1):
        _require(False, "features of X and Y must be contiguous")
    # No two elements of Y at one address: one of the outer dimensions steps over all inside it.
    if not ((heads < 2 or ys[1] >= dim) and (rows < 2 or ys[0] >= (heads - 1) * ys[1] + dim) or
            (rows < 2 or ys[0] >= dim) and (heads < 2 or ys[1] >= (rows - 1) * ys[0] + dim)):
        _require(False, "two elements of Y share memory")
    if Y.requires_grad and torch.is_grad_enabled():
        _require(False, "no graph is recorded of rotary: what it writes must not require a gradient "
                        "(detach it, or call under torch.no_grad())")
    wide = _rotary_operands(positions, inv_freq, rows, -1, index)
    _call_on(index, _lib.lib().mk_rotary, x, xs[0], xs[1], y, ys[0], ys[1], rows, heads, dim, 2 * inv_freq.shape[0],
             _DTYPES[dtype], positions.data_ptr(), wide, inv_freq.data_ptr(), scale, interleaved, inverse)
    _count_as_changed((Y,))
    return Y


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: str | None = None,
                       factor: float = 1.0, original_length: int = 0, low: float = 1.0,
                       high: float = 32.0, device="cuda") -> tuple[torch.Tensor, float]:
    """(inv_freq, scale) for ``rotary`` and ``w4_gemm_rotary``: base ** (-2 i / rotary_dim), changed for
    contexts ``factor`` times longer than the ``original_length`` that a model was trained on:
      None          as they are
      "linear"      every frequency divided by factor
      "base"        the base raised by factor ** (d / (d - 2)): the last pair is divided by factor, the
                    first one kept
      "parts"       by how many turns a pair makes over original_length: above ``high`` kept, below
                    ``low`` divided by factor, linear in the pair's index between; scale is
                    0.1 ln(factor) + 1
      "wavelength"  the same ends, linear in the number of turns between them; scale 1
    Computed in 64 bits, returned as float32."""
    import math
    d = int(rotary_dim)
    _require(d >= 2 and d % 2 == 0, "rotary_dim must be even and positive")
    _require(base > 1.0 and factor >= 1.0, "base must be above 1, factor at least 1")
    _require(scaling in (None, "linear", "base", "parts", "wavelength"), f"unknown scaling {scaling!r}")
    scale = 1.0
    if scaling == "base":
        _require(d > 2, "scaling 'base' needs more than one pair")
        base = base * factor ** (d / (d - 2))
    i = torch.arange(d // 2, dtype=torch.float64)
    freq = float(base) ** (-2.0 * i / d)
    if scaling == "linear":
        freq = freq / factor
    elif scaling in ("parts", "wavelength"):
        _require(original_length > 0 and high > low > 0, "needs original_length > 0 and high > low > 0")
        if scaling == "parts":
            def index(turns):     # of the pair that makes so many turns over the original length
                return d * math.log(original_length / (turns * 2 * math.pi)) / (2 * math.log(base))
            first, last = max(math.floor(index(high)), 0), min(math.ceil(index(low)), d - 1)
            keep = 1 - ((i - first) / max(last - first, 1e-3)).clamp(0, 1)
            scale = 0.1 * math.log(factor) + 1.0
        else:
            keep = ((original_length * freq / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
        freq = freq * keep + freq / factor * (1 - keep)
    return freq.to(torch.float32).to(device), scale


class TpMlp:
    """The tensor-parallel MLP as two fused launches on one stream:
    AllGather+GEMM(gate, up) with the SwiGLU epilogue -> H, then GEMM+ReduceScatter(down) on H.
    Both kernels are launched with programmatic stream serialization (the default), so the
    second one's set-up overlaps the first one's tail; captured in a CUDA graph they are two
    nodes.  All buffers are allocated once, collectively (same order on every rank):
      x:    DistBuffer [W, M/W, K]    rank r fills x.data_[r]
      out:  rows [rank*M/W, (rank+1)*M/W) of y.data_ (the reduced slice)
    A decode step's few tokens take ``forward_tokens`` with weights in 4 bits."""

    def __init__(self, M: int, K: int, I_local: int, N_out: int, local_rank: int,
                 local_world_size: int):
        W = int(local_world_size)
        _require(M % W == 0, "M must be divisible by the world size")
        dev = torch.device("cuda", local_rank)
        self.M, self.K, self.I, self.N, self.W, self.rank = M, K, I_local, N_out, W, local_rank
        self.x = DistBuffer((W, M // W, K), torch.bfloat16, local_rank, W)
        self.ready = DistBuffer((ag_gemm_warp_specialized_ready_words,), torch.int32, local_rank, W)
        self.ready.data_.zero_()
        self.h = torch.empty((W, M // W, I_local), device=dev, dtype=torch.bfloat16)
        self.y = DistBuffer((M, N_out), torch.bfloat16, local_rank, W)
        self.sync = DistBuffer(gemm_rs_blackwell_sync_shape, torch.int32, local_rank, W)
        gemm_rs_blackwell_prepare(None, None, self.y, self.sync)
        self.w_gate_up = None
        self.w_down = None
        self.w4_gate_up = None
        self.w4_down = None

    def load_weights(self, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor) -> None:
        """w_gate, w_up: [I_local, K]; w_down: [N_out, I_local] (this rank's shards)."""
        self.w_gate_up = interleave_gate_up(w_gate, w_up)
        _bf16_matrix(w_down, "w_down")
        _require(tuple(w_down.shape) == (self.N, self.I), f"w_down must be [{self.N},{self.I}]")
        self.w_down = w_down

    def forward(self) -> torch.Tensor:
        """Enqueue both launches on the current stream; returns the view of this rank's output
        rows (valid when the stream has completed)."""
        ag_gemm_warp_specialized_prepare(self.ready, self.M, 2 * self.I)
        ag_gemm_swiglu_launch(self.x, self.ready, self.w_gate_up, self.h)
        gemm_rs_blackwell_launch(self.h.view(self.M, self.I), self.w_down, self.y, self.sync)
        Ms = self.M // self.W
        return self.y.data_[self.rank * Ms:(self.rank + 1) * Ms]

    def load_weights_w4(self, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor,
                        group: int = 128, zero_points: bool = False) -> None:
        """Round this rank's shards (shapes as in ``load_weights``, any I_local) to 4 bits for
        ``forward_tokens``; independent of the weights of ``forward``."""
        _require(tuple(w_gate.shape) == tuple(w_up.shape) == (self.I, self.K),
                 f"w_gate and w_up must be [{self.I},{self.K}]")
        _require(tuple(w_down.shape) == (self.N, self.I), f"w_down must be [{self.N},{self.I}]")
        self.w4_gate_up = w4_quantize(torch.cat((w_gate, w_up)), group, zero_points, form="gate_up")
        self.w4_down = w4_quantize(w_down, group, zero_points)

    def forward_tokens(self, x: torch.Tensor, out: torch.Tensor | None = None, exact: bool = False) -> torch.Tensor:
        """The MLP of a few tokens x [m, K] (any m; a decode step) with the 4-bit weights: two launches
        on the current stream.  Returns out [m, N_out], this rank's part of the sum over ranks -- the
        whole result when there is one rank; with more the caller sums it over them.  ``exact`` as in ``w4_gemm``."""
        _require(self.w4_gate_up is not None, "call load_weights_w4 first")
        m = x.shape[0]
        h = torch.empty((m, self.I), device=x.device, dtype=x.dtype)
        if out is None:
            out = torch.empty((m, self.N), device=x.device, dtype=x.dtype)
        w4_gemm_swiglu(x, self.w4_gate_up, h)
        w4_gemm(h, self.w4_down, out, exact)
        return out

    def free(self) -> None:
        for b in (self.x, self.ready, self.y, self.sync):
            b.free()


def gemm_rs_blackwell_prepare(A, B, C: DistBuffer, sync: DistBuffer) -> None:
    """Zero the synchronisation words once; the caller then synchronises and barriers."""
    _require(isinstance(sync, DistBuffer), "sync must be a DistBuffer")
    with _on_device(sync.local_rank_):
        _lib.check(_lib.lib().mk_gemm_rs_prepare(sync.view_ref(), _stream()))


def gemm_rs_blackwell_launch(A: torch.Tensor, B: torch.Tensor, C: DistBuffer,
                             sync: DistBuffer) -> None:
    """Partial C = A @ B^T, then rows [rank*M/W, (rank+1)*M/W) of C.data_ hold the sum over ranks."""
    _bf16_matrix(A, "A")
    _bf16_matrix(B, "B")
    _require(isinstance(C, DistBuffer) and isinstance(sync, DistBuffer),
             "C and sync must be DistBuffers")
    M, K = A.shape
    N = B.size(0)
    _require(B.size(1) == K, f"B must be [N, K] with K={K}")
    _require(C.dtype == torch.bfloat16 and tuple(C.shape) == (M, N), f"C must be bf16 [{M},{N}]")
    with _on_device(C.local_rank_):
        _lib.check(_lib.lib().mk_gemm_rs_launch(A.data_ptr(), B.data_ptr(), C.view_ref(),
                                                sync.view_ref(), M, N, K, _stream()))


def gemm_ar_intranode_blackwell(A: torch.Tensor, B: torch.Tensor, C: DistBuffer,
                                barrier: DistBuffer, C_final: DistBuffer, epoch: int,
                                b_layout: int = _lib.MK_B_KN) -> None:
    """C_final = sum over ranks of A_r @ B_r on every rank; C receives this rank's partial."""
    _bf16_matrix(A, "A")
    _bf16_matrix(B, "B")
    for d, n in ((C, "C"), (barrier, "barrier"), (C_final, "C_final")):
        _require(isinstance(d, DistBuffer), f"{n} must be a DistBuffer")
    M, K = A.shape
    if b_layout == _lib.MK_B_KN:
        _require(B.size(0) == K, f"B must be [K, N] with K={K}")
        N = B.size(1)
    else:
        _require(B.size(1) == K, f"B must be [N, K] with K={K}")
        N = B.size(0)
    for d, n in ((C, "C"), (C_final, "C_final")):
        _require(d.dtype == torch.bfloat16 and tuple(d.shape) == (M, N), f"{n} must be bf16 [{M},{N}]")
    _require(int(epoch) >= 0, "epoch starts at 1 and must increase by one per call "
                              "(0 = keep the epoch on the device; graph-replayable)")
    with _on_device(C.local_rank_):
        _lib.check(_lib.lib().mk_gemm_ar_launch(A.data_ptr(), B.data_ptr(), C.view_ref(),
                                                barrier.view_ref(), C_final.view_ref(), M, N, K,
                                                int(epoch), b_layout, _stream()))


def op_status(sync: DistBuffer) -> tuple[int, int, int, int]:
    """Status words of an operator's synchronisation buffer; raises MkError if a device wait
    expired.  Synchronises the device."""
    out = (ctypes.c_uint32 * 4)()
    with _on_device(sync.local_rank_):
        _lib.check(_lib.lib().mk_op_status(sync.view_ref(), out))
    return tuple(int(x) for x in out)


def op_status_clear(sync: DistBuffer) -> None:
    with _on_device(sync.local_rank_):
        _lib.check(_lib.lib().mk_op_status_clear(sync.view_ref(), _stream()))
