"""CPU oracle of the products with 4-bit weights and of rotary positions: the definitions in plain
torch, products and angles in 64 bits.  Imported by tests only."""
from __future__ import annotations

import torch


def quantize(w: torch.Tensor, group: int, zero_points: bool, dtype: torch.dtype):
    """(codes [N, K] int64, scales [N, G] of dtype, zeros [N, G] int64) of a CPU matrix.  The divisions
    are fp32 because that is the definition: which code is nearest depends on it at ties."""
    N, K = w.shape
    G = -(-K // group)
    wf = torch.zeros((N, G * group), dtype=torch.float32)
    wf[:, :K] = w.float()
    wf = wf.view(N, G, group)
    lo, hi = wf.amin(-1).clamp(max=0), wf.amax(-1).clamp(min=0)
    if zero_points:
        s = ((hi - lo) / 15).to(dtype)
    else:
        s = (wf.abs().amax(-1) / 7).to(dtype)
    bad = ~torch.isfinite(wf).all(-1)
    s = torch.where(bad, torch.full_like(s, float("nan")), s)
    d = torch.where(s.float() == 0, torch.ones(()), s.float())
    z = (-lo / d).round().clamp(0, 15) if zero_points else torch.full((N, G), 8.0)
    q = ((wf / d.unsqueeze(-1)).round() + z.unsqueeze(-1)).clamp(0, 15).nan_to_num(0)
    return q.long().view(N, G * group)[:, :K], s, z.nan_to_num(0).long()


def pack_nibbles(codes: torch.Tensor) -> torch.Tensor:
    """uint8 [N, (K + 1) / 2], the even column in the low half."""
    N, K = codes.shape
    c = torch.zeros((N, K + K % 2), dtype=torch.uint8)
    c[:, :K] = codes.to(torch.uint8)
    return (c[:, 0::2] | (c[:, 1::2] << 4)).contiguous()


def dequantize(codes: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor, group: int) -> torch.Tensor:
    """fp64 [N, K]."""
    K = codes.shape[1]
    s = scales.double().repeat_interleave(group, 1)[:, :K]
    z = zeros.double().repeat_interleave(group, 1)[:, :K]
    return (codes.double() - z) * s


def silu_mul(y: torch.Tensor) -> torch.Tensor:
    gate, up = y.chunk(2, dim=1)
    return gate * torch.sigmoid(gate) * up


def rotary(x: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, interleaved: bool = False,
           inverse: bool = False, scale: float = 1.0) -> torch.Tensor:
    """x [rows, heads, dim] -> fp64."""
    x = x.double().clone()
    angle = positions.double()[:, None] * inv_freq.double()[None, :] * (-1 if inverse else 1)
    n = inv_freq.numel()
    for i in range(n):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + n)
        c, s = angle[:, i].cos()[:, None] * scale, angle[:, i].sin()[:, None] * scale
        u, v = x[:, :, a] * c - x[:, :, b] * s, x[:, :, b] * c + x[:, :, a] * s
        x[:, :, a], x[:, :, b] = u, v
    return x
