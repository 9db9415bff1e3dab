"""Rows in 4 bits by their definition, for the tests: 64-bit arithmetic on the CPU,
a table of the sixteen values, no code of the package."""
from __future__ import annotations

import torch

LEVELS = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
VALUES = torch.cat([LEVELS, -LEVELS])


def quantise(x):
    """(codes, two to a byte; scale bytes) of rows [..., d]."""
    x = x.detach().cpu().double().unflatten(-1, (-1, 32))
    finite = torch.isfinite(x).all(-1, keepdim=True)
    top = torch.where(finite, x.abs().amax(-1, keepdim=True), 0.0)
    live = top >= 2.0 ** -100
    e = torch.ceil(torch.log2(torch.where(live, top, 1.0) / 7.0))
    e = torch.where(top > 7.0 * torch.exp2(e), e + 1, e)
    e = torch.where(top <= 7.0 * torch.exp2(e - 1), e - 1, e).clamp(max=125)
    y = torch.where(finite & live, x.abs() / torch.exp2(e), 0.0)
    # the nearest level, of two as near the even code
    gap = (y[..., None] - LEVELS).abs()
    best = gap.amin(-1, keepdim=True)
    near = gap == best
    code = torch.where(near.sum(-1) > 1,
                       (near & (torch.arange(8) % 2 == 0)).int().argmax(-1),
                       near.int().argmax(-1))
    code = code + 8 * (torch.signbit(x) & finite & live)
    code = code.flatten(-2).to(torch.uint8)
    scale = torch.where(finite, torch.where(live, e + 127, 0.0), 255.0)
    return code[..., 0::2] | code[..., 1::2] << 4, scale.squeeze(-1).to(torch.uint8)


def values(codes, scales):
    """The float64 values of codes (bytes) and their blocks' scale bytes."""
    codes, scales = codes.cpu().long(), scales.cpu()
    x = torch.stack([VALUES[codes & 15], VALUES[codes >> 4]], -1).flatten(-2)
    factor = torch.where(scales == 255, torch.nan, torch.exp2(scales.double() - 127))
    return (x.unflatten(-1, (-1, 32)) * factor[..., None]).flatten(-2)
