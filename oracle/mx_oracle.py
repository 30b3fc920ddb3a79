"""CPU restatement, in float64, of the microscaled formats and of what is computed with them (test infrastructure only).

A block of 32 elements shares 2^(s - 127); the largest magnitude's exponent gives s, the elements are rounded to nearest
even on the format's grid and held at its largest value."""
from __future__ import annotations

import torch

BLOCK = 32
EMAX = {"mxfp4": 2, "mxfp8": 8, "mxint8": 0}
GRID4 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def grid8() -> list:
    """The 127 magnitudes of e4m3 by their codes."""
    out = []
    for c in range(127):
        e, m = c >> 3, c & 7
        out.append(m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10))
    return out


def _nearest_even(m: torch.Tensor, grid: list) -> torch.Tensor:
    """Codes of the grid values nearest to m >= 0, ties to the even code."""
    g = torch.tensor(grid, dtype=torch.float64)
    half = (g[1:] + g[:-1]) / 2
    down = torch.searchsorted(half, m.contiguous(), right=False)
    up = torch.searchsorted(half, m.contiguous(), right=True)
    return torch.where(down % 2 == 0, down, up)


def quantise(x: torch.Tensor, fmt: str):
    """(codes uint8 [..., bytes], scales uint8 [..., blocks]) of x [..., d]."""
    x = x.detach().cpu().double()
    d = x.shape[-1]
    v = torch.nn.functional.pad(x, (0, -d % BLOCK)).unflatten(-1, (-1, BLOCK))
    bad = ~torch.isfinite(v).all(-1)
    v = torch.where(bad.unsqueeze(-1), torch.zeros_like(v), v)
    top = torch.frexp(v.abs().amax(-1))[1].to(torch.int64) - 1
    zero = v.abs().amax(-1) == 0
    s = (top - EMAX[fmt] + 127).clamp(0, 254)
    s = torch.where(zero, torch.zeros_like(s), s)
    v = torch.ldexp(v, (127 - s).unsqueeze(-1))
    sign = (torch.signbit(v)).to(torch.int64)
    m = v.abs()
    if fmt == "mxint8":
        c = torch.sign(v).to(torch.int64) * torch.round(m * 64).clamp(max=127).to(torch.int64)
        codes = (c & 255).to(torch.uint8).flatten(-2)
    elif fmt == "mxfp8":
        codes = (_nearest_even(m.clamp(max=448.0), grid8()) | (sign << 7)).to(torch.uint8).flatten(-2)
    else:
        c = (_nearest_even(m, GRID4) | (sign << 3)).flatten(-2)
        codes = (c[..., 0::2] | (c[..., 1::2] << 4)).to(torch.uint8)
    return codes, torch.where(bad, torch.full_like(s, 255), s).to(torch.uint8)


def dequantise(codes: torch.Tensor, scales: torch.Tensor, fmt: str, d: int) -> torch.Tensor:
    """float64 [..., d]."""
    c = codes.cpu().to(torch.int64)
    if fmt == "mxint8":
        q = torch.where(c >= 128, c - 256, c).double() / 64
    elif fmt == "mxfp8":
        g = torch.tensor(grid8() + [float("nan")], dtype=torch.float64)
        q = torch.where(c >= 128, -1.0, 1.0) * g[c & 127]
    else:
        g = torch.tensor(GRID4 + [-v for v in GRID4], dtype=torch.float64)
        q = g[torch.stack((c & 15, c >> 4), dim=-1).flatten(-2)]
    s = scales.cpu().to(torch.int64)
    scale = torch.where(s == 255, torch.full((), float("nan"), dtype=torch.float64),
                        torch.ldexp(torch.ones((), dtype=torch.float64), s - 127))
    return (q.unflatten(-1, (-1, BLOCK)) * scale.unsqueeze(-1)).flatten(-2)[..., :d]


def round_trip(x: torch.Tensor, fmt: str) -> torch.Tensor:
    return dequantise(*quantise(x, fmt), fmt, x.shape[-1])
