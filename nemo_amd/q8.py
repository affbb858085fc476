"""Feature rows held in 8 bits: the type, and the encoding on the host (what the GPU calls of PoseEngine compute, for feature
records written and read where there is no GPU).

A row of C channels is C e4m3 codes and one power of two per block of 128 channels; its numbers are code * scale.
Per block, scale = 2^e with the smallest e >= -117 for which max |x| <= 448 * 2^e over the finite numbers; codes are the nearest,
ties to even; what is not finite becomes NaN.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

BLOCK = 128
LOWEST = -117  # the smallest code times the smallest scale is still a normal 32-bit number


class Q8(NamedTuple):
    codes: torch.Tensor   # float8_e4m3fn [..., C]
    scale: torch.Tensor   # float8_e8m0fnu [..., ceil(C / 128)]


def n_blocks(channels: int) -> int:
    return -(-channels // BLOCK)


def empty(shape, device) -> Q8:
    """Room for rows of shape[-1] channels."""
    return Q8(torch.empty(tuple(shape), dtype=torch.float8_e4m3fn, device=device),
              torch.empty(tuple(shape[:-1]) + (n_blocks(shape[-1]),), dtype=torch.float8_e8m0fnu, device=device))


def quantize_host(x: torch.Tensor) -> Q8:
    """Rows [..., C] on the CPU; bit for bit what PoseEngine.quantize writes, but for the sign of a NaN."""
    if x.device.type != 'cpu':
        raise ValueError('quantize_host: tensor on %s (PoseEngine.quantize works on the GPU)' % x.device)
    c = x.shape[-1]
    nb = n_blocks(c)
    y = x.to(torch.float32)
    y = torch.where(torch.isfinite(y), y, torch.full_like(y, float('nan')))
    y = torch.nn.functional.pad(y, (0, nb * BLOCK - c)).unflatten(-1, (nb, BLOCK))
    part, two = torch.frexp(y.nan_to_num(0.0).abs().amax(-1))       # amax = part * 2^two, 1/2 <= part < 1; 448 = 0.875 * 2^9
    e = torch.where(part > 0, two - 9 + (part > 0.875).to(two.dtype), torch.full_like(two, LOWEST)).clamp(min=LOWEST)
    codes = (y * torch.ldexp(torch.ones_like(part), -e)[..., None]).to(torch.float8_e4m3fn).flatten(-2)
    return Q8(codes.view(torch.uint8)[..., :c].contiguous().view(torch.float8_e4m3fn), (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu))


def dequantize_host(q: Q8, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    c = q.codes.shape[-1]
    return (q.codes.to(torch.float32) * q.scale.to(torch.float32).repeat_interleave(BLOCK, -1)[..., :c]).to(dtype)
