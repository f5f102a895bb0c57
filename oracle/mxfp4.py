"""MXFP4 oracle in 64-bit torch — TEST INFRASTRUCTURE ONLY.

Written from the format's definition (OCP microscaling formats, MXFP4: e2m1
elements, one e8m0 scale per 32), device-agnostic, without the library. The
functions mirror ``dsmoe.mxfp4``: quantise, dequantise, product, ragged
products by expert, and the routed FFN.
"""
from __future__ import annotations

import torch

GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def quantize(x: torch.Tensor, scale_inv: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes uint8 [..., K/2], scales uint8 [..., K/32])."""
    v = x.double()
    if scale_inv is not None:
        rows, cols = x.shape[-2:]
        r, c = torch.arange(rows, device=x.device) // 128, torch.arange(cols, device=x.device) // 128
        v = v * scale_inv.double()[..., r, :][..., c]
    b = v.reshape(*v.shape[:-1], v.shape[-1] // 32, 32)
    a = b.abs().amax(-1)
    bad = ~torch.isfinite(b).all(-1)
    e = torch.frexp(torch.where(bad, torch.ones_like(a), a)).exponent.long() - 1
    byte = torch.where(a > 0, (e - 2).clamp(-127, 127) + 127, torch.zeros_like(e))
    q = torch.ldexp(torch.where(bad.unsqueeze(-1), torch.zeros_like(b), b), 127 - byte.unsqueeze(-1))
    d = (q.abs().unsqueeze(-1) - GRID.to(x.device)).abs()
    near = d.amin(-1, keepdim=True)
    codes = torch.arange(8, device=x.device)
    # of the nearest grid points (two at a tie) the one with the even code
    code = torch.where((d == near) & (codes % 2 == 0), codes, -1).amax(-1)
    odd = torch.where(d == near, codes, -1).amax(-1)
    code = torch.where(code >= 0, code, odd)
    code = code + 8 * torch.signbit(q).long()
    byte = torch.where(bad, torch.full_like(byte, 255), byte)
    code = torch.where(bad.unsqueeze(-1), torch.zeros_like(code), code)
    code = code.reshape(*v.shape[:-1], v.shape[-1] // 2, 2).to(torch.uint8)
    return code[..., 0] | (code[..., 1] << 4), byte.to(torch.uint8)


def dequantize(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    n = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()
    v = GRID.to(codes.device)[n & 7] * (1 - 2 * (n >> 3)).double()
    s = torch.ldexp(torch.ones_like(scales, dtype=torch.float64), scales.long() - 127)
    s = torch.where(scales == 255, torch.full_like(s, float("nan")), s)
    return (v.reshape(*scales.shape, 32) * s.unsqueeze(-1)).flatten(-2)


def linear(x: torch.Tensor, w: torch.Tensor) -> torch.Tensor:
    """x @ w.T in 64 bits."""
    return x.double() @ w.double().T


def grouped_linear(x: torch.Tensor, w: torch.Tensor, offsets) -> torch.Tensor:
    """w [E, out, in]; rows outside every segment are zero."""
    off = [int(v) for v in offsets]
    out = torch.zeros(x.shape[0], w.shape[1], dtype=torch.float64, device=x.device)
    for e in range(w.shape[0]):
        if off[e + 1] > off[e]:
            out[off[e]:off[e + 1]] = linear(x[off[e]:off[e + 1]], w[e])
    return out


def ffn(x: torch.Tensor, gate: torch.Tensor, up: torch.Tensor, down: torch.Tensor) -> torch.Tensor:
    g = linear(x, gate)
    return linear(g * torch.sigmoid(g) * linear(x, up), down)


def moe(x, idx, w, gate, up, down, shared: bool, scale: float) -> torch.Tensor:
    """gate, up, down: dequantised stacks, the shared expert first if ``shared``."""
    base = int(shared)
    out = ffn(x, gate[0], up[0], down[0]) if shared else torch.zeros_like(x, dtype=torch.float64)
    for e in range(gate.shape[0] - base):
        t, k = (idx == e).nonzero(as_tuple=True)
        if t.numel():
            y = ffn(x[t], gate[base + e], up[base + e], down[base + e])
            out.index_add_(0, t, scale * w[t, k].double().unsqueeze(1) * y)
    return out
