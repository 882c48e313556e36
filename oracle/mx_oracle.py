"""The microscaled (MX) operators from their definitions, in 64 bits, with PyTorch.

The formats are those of include/b200moe.h: blocks of 32 elements with one power-of-two
scale (the smallest one, 2^-127 at least, with which the largest magnitude does not pass
the element type's largest value), elements rounded to the nearest with ties to even.  The
grids of the element types are written out here from their bit layouts."""
from __future__ import annotations

import torch

BLOCK = 32
E2M1 = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
# e4m3: 3 mantissa bits, exponent bias 7, code 0x7f is NaN
E4M3 = torch.tensor([m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
                     for e in range(16) for m in range(8)][:-1], dtype=torch.float64)


def quantize(x: torch.Tensor, four_bit: bool):
    """x [..., K] -> (codes [..., K] uint8 with the sign in the top bit of the type, scale
    bytes [..., K/32] uint8)."""
    grid = (E2M1 if four_bit else E4M3).to(x.device)
    b = x.double().unflatten(-1, (-1, BLOCK))
    amax = b.abs().amax(-1)
    bad = ~torch.isfinite(b).all(-1)
    safe = torch.where(bad, torch.ones_like(amax), amax)
    # smallest e with amax <= max * 2^e: start one below the logarithm's answer and step up
    e = torch.floor(torch.log2(torch.where(safe > 0, safe, torch.ones_like(safe)) / grid[-1])) - 1
    for _ in range(3):
        e = torch.where(safe > grid[-1] * torch.exp2(e), e + 1, e)
    e = torch.where(safe > 0, e.clamp_min(-127), torch.full_like(e, -127.0))
    v = torch.where(bad[..., None], torch.zeros_like(b), b) / torch.exp2(e)[..., None]
    a = v.abs()
    hi = torch.searchsorted(grid, a.contiguous()).clamp_max(grid.numel() - 1)   # first point >= a
    lo = (hi - 1).clamp_min(0)
    up, down = grid[hi] - a, a - grid[lo]
    even_hi = hi % 2 == 0                     # the code's last bit is the mantissa's last bit
    code = torch.where((up < down) | ((up == down) & even_hi), hi, lo)
    code = code | (torch.signbit(v).long() << (3 if four_bit else 7))
    if not four_bit:
        code = torch.where(bad[..., None], torch.full_like(code, 0x7F), code)
    byte = torch.where(bad, torch.full_like(e, 255.0), e + 127)
    return code.flatten(-2).to(torch.uint8), byte.to(torch.uint8)


def scale_values(byte: torch.Tensor) -> torch.Tensor:
    v = torch.exp2(byte.double() - 127)
    return torch.where(byte == 255, torch.full_like(v, float("nan")), v)


def values(codes: torch.Tensor, byte: torch.Tensor, four_bit: bool) -> torch.Tensor:
    """The numbers that codes and scale bytes stand for, in 64 bits."""
    grid = (E2M1 if four_bit else torch.cat([E4M3, torch.tensor([float("nan")], dtype=torch.float64)])).to(codes.device)
    sign, top = (3, 7) if four_bit else (7, 127)
    c = codes.long()
    v = grid[c & top] * (1 - 2 * (c >> sign).double())
    return (v.unflatten(-1, (-1, BLOCK)) * scale_values(byte)[..., None]).flatten(-2)


def unpack4(data: torch.Tensor) -> torch.Tensor:
    """[..., K/2] bytes -> [..., K] codes, the even element in the low half."""
    return torch.stack([data & 15, data >> 4], -1).flatten(-2)


def pack4(codes: torch.Tensor) -> torch.Tensor:
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


def grouped(x: torch.Tensor, offsets, w: torch.Tensor) -> torch.Tensor:
    """y[r] = x[r] w[e]^T for the rows of every expert (64 bits)."""
    y = torch.zeros(x.shape[0], w.shape[1], dtype=torch.float64, device=x.device)
    for e in range(w.shape[0]):
        a, b = int(offsets[e]), int(offsets[e + 1])
        y[a:b] = x[a:b].double() @ w[e].double().T
    return y


def swiglu(gu: torch.Tensor) -> torch.Tensor:
    g, u = gu.chunk(2, -1)
    return g / (1 + torch.exp(-g)) * u


def add_rmsnorm(residual, hidden, weight, eps):
    """(residual', normed) with a rounding to the type after the add, after the
    normalisation and after the weight."""
    dt = residual.dtype
    r = residual.double() + (0 if hidden is None else hidden.double())
    r = r.to(dt)
    d = r.double()
    unit = (d / torch.sqrt(d.square().mean(-1, keepdim=True) + eps)).to(dt)
    return r, (unit.double() * weight.double()).to(dt)
