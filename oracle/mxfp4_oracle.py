"""MXFP4 in fp64 torch operations: the oracle of the 4-bit kernels.

Format: 32 consecutive values of a row share the scale 2^max(floor(log2 A) - 2, -127), A their largest
magnitude; a value is the nearest of 0, .5, 1, 1.5, 2, 3, 4, 6 times the scale (ties to the code whose
last bit is 0, saturating at 6).  A block with an infinity or a NaN is NaN throughout.
"""
from __future__ import annotations

import torch

LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def scale_exponents(x: torch.Tensor) -> torch.Tensor:
    """The E8M0 byte of every block of 32 along the rows of x (255 where a value is not finite)."""
    r, c = x.shape
    xp = torch.nn.functional.pad(x.double(), (0, (-c) % 32)).reshape(r, -1, 32)
    amax = xp.abs().amax(2)
    bad = ~torch.isfinite(xp).all(2)
    safe = torch.where(bad | (amax == 0), torch.ones_like(amax), amax)
    e = (torch.frexp(safe).exponent - 1 - 2).clamp(min=-127) + 127
    e = torch.where(amax == 0, torch.zeros_like(e), e)
    return torch.where(bad, torch.full_like(e, 255), e).to(torch.uint8)


def values(x: torch.Tensor) -> torch.Tensor:
    """fp64 values that the MXFP4 codes of x stand for."""
    r, c = x.shape
    s = scale_exponents(x)
    xp = torch.nn.functional.pad(x.double(), (0, (-c) % 32)).reshape(r, -1, 32)
    scale = torch.exp2(s.double() - 127)[..., None]
    a = torch.where(torch.isfinite(xp), xp.abs(), torch.zeros_like(xp)) / scale
    code = torch.zeros_like(a, dtype=torch.int64)
    for t in (0.25, 1.25, 2.5, 5.0):   # ties go down
        code += a > t
    for t in (0.75, 1.75, 3.5):        # ties go up
        code += a >= t
    v = torch.copysign(torch.tensor(LEVELS, dtype=torch.float64, device=x.device)[code], xp) * scale
    return torch.where((s == 255)[..., None], torch.full_like(v, float("nan")), v).reshape(r, -1)[:, :c]


def product(a: torch.Tensor, b: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``a·bᵀ`` of two value matrices and the sum of the magnitudes of its terms."""
    return a @ b.t(), a.abs() @ b.abs().t()


def bf16(x: torch.Tensor) -> torch.Tensor:
    return x.to(torch.bfloat16).double()


def swiglu(g: torch.Tensor, u: torch.Tensor) -> torch.Tensor:
    return g * torch.sigmoid(g) * u


def swiglu_grad(dh, g, u):
    s = torch.sigmoid(g)
    return dh * u * (s * (1 + g * (1 - s))), dh * (g * s)
