"""Microscaled numbers in plain 64-bit torch, from the format's definition: what the tests compare with."""

from __future__ import annotations

import torch

GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
EMAX = {"fp4": 2, "int8": 0}


def quantize64(x: torch.Tensor, fmt: str):
    """(byte of each block [rows, blocks], signed codes [rows, 32 * blocks], values [rows, cols]) of ``x`` [rows, cols]."""
    rows, cols = x.shape
    blocks = (cols + 31) // 32
    v = torch.zeros(rows, blocks * 32, dtype=torch.float64)
    v[:, :cols] = x.detach().cpu().double()
    v = v.view(rows, blocks, 32)
    bad = ~v.isfinite().all(-1)
    v = torch.where(bad[..., None], torch.zeros_like(v), v)
    top = v.abs().amax(-1)
    e = torch.where(top > 0, torch.frexp(top)[1].double() - 1 - EMAX[fmt], torch.full_like(top, -127.0)).clamp(min=-127)
    a = v.abs() * torch.exp2(-e)[..., None]
    if fmt == "int8":
        code = torch.round(a * 64).clamp(max=127)              # half to even
        value = code / 64
        code = torch.where(v < 0, -code, code)
    else:
        middle = (GRID[1:] + GRID[:-1]) / 2
        code = sum((a > m if i % 2 == 0 else a >= m).double() for i, m in enumerate(middle))   # a tie goes to the even code
        value = GRID[code.long()]
        code = torch.where(v < 0, code + 8, code)
    value = torch.where(v < 0, -value, value) * torch.exp2(e)[..., None]
    value = torch.where(bad[..., None], torch.full_like(value, float("nan")), value)
    byte = torch.where(bad, torch.full_like(e, 255.0), e + 127).to(torch.uint8)
    return byte, code.view(rows, -1), value.view(rows, -1)[:, :cols]


def rounding(y: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """What rounding ``y`` to ``dtype`` may be off by: half a step, of the smallest numbers at least."""
    info = torch.finfo(dtype)
    return torch.clamp(y.abs() * (info.eps / 2), min=info.smallest_normal * info.eps / 2)


def product_bound(a: torch.Tensor, b: torch.Tensor, terms: int) -> torch.Tensor:
    """Error bound of ``a @ b`` with products and sums in fp32: ``terms`` additions, each off by at most a step of 2^-23
    (the tensor cores may cut instead of rounding) of a partial sum that is at most sum |a| |b|."""
    return (terms + 1) * 2.0 ** -23 * (a.abs() @ b.abs())


def check(y: torch.Tensor, want: torch.Tensor, bound: torch.Tensor, what: str = "") -> None:
    y = y.detach().cpu().double()
    assert y.shape == want.shape, (y.shape, want.shape)
    nan = want.isnan()
    assert torch.equal(y.isnan(), nan), f"{what}: NaN in other places"
    off = torch.where(nan | (y == want), torch.zeros_like(y), (y - want).abs() - bound)
    worst = int(off.argmax()) if off.numel() else 0
    assert off.numel() == 0 or float(off.max()) <= 0, (
        f"{what}: {float(y.flatten()[worst])} instead of {float(want.flatten()[worst])} (bound {float(bound.flatten()[worst])})"
        f" at {worst} of {tuple(y.shape)}; {int((off > 0).sum())} values are off")
