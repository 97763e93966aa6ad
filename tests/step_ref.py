"""float64 restatements of the step operators (not collected)."""

from __future__ import annotations

import torch


def rotate64(x, positions, freqs, interleaved, factor):
    """x [rows, heads, dim] rotated, float64 on the CPU."""
    x = x.detach().cpu().double().clone()
    a = positions.cpu().double()[:, None] * freqs.cpu()[None]
    cos, sin = torch.cos(a)[:, None] * factor, torch.sin(a)[:, None] * factor
    n = freqs.numel()
    i = torch.arange(n)
    ia, ib = (2 * i, 2 * i + 1) if interleaved else (i, i + n)
    u, w = x[..., ia].clone(), x[..., ib].clone()
    x[..., ia], x[..., ib] = u * cos - w * sin, w * cos + u * sin
    return x


def rotate_tolerance(x, positions, freqs, factor, want):
    """Per element: half a step of the type and of fp32 (a value is rounded to
    fp32, then to the type; below the type's smallest normal a step is fixed),
    and what 64-bit angles leave: p f is off by half a step of itself, and so
    are cos, sin and each product (8 such, generously)."""
    fi = torch.finfo(x.dtype)
    angle = positions.cpu().double().abs().max() * freqs.cpu().abs().max() if len(positions) else 0
    size = 2 * float(x.double().abs().max()) * abs(factor) if x.numel() else 0.0
    return (want.abs() * (fi.eps / 2 + 2.0 ** -23) + fi.tiny * fi.eps
            + size * (8 + 2 * float(angle)) * 2.0 ** -53)
