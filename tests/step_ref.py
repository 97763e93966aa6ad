"""float64 restatements of the step operators (not collected)."""

from __future__ import annotations

import math

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


HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def rows64(q, k, v, pos, scale, k_scale=1.0, v_scale=1.0, ok=None):
    """float64 causal attention of q [n, Hq, D] at positions `pos` over k, v
    [tokens, H, D], those with ok[t] only.  Returns (out, weights @ |v|), on the CPU."""
    q, k, v = q.cpu().double(), k.cpu().double(), v.cpu().double()
    n, Hq, D = q.shape
    G = Hq // k.shape[1]
    out, mass = torch.zeros(n, Hq, D, dtype=torch.float64), torch.zeros(n, Hq, D,
                                                                        dtype=torch.float64)
    seen = torch.arange(k.shape[0])[None] <= torch.as_tensor(pos)[:, None]
    if ok is not None:
        seen = seen & ok[None]
    for j in range(n):  # only what the row sees takes part
        t = torch.nonzero(seen[j])[:, 0]
        if not len(t):
            continue
        for h in range(k.shape[1]):
            x = q[j, h * G:(h + 1) * G] @ k[t, h].t() * (scale * k_scale)
            w = torch.softmax(x, -1)
            out[j, h * G:(h + 1) * G] = w @ v[t, h] * v_scale
            mass[j, h * G:(h + 1) * G] = w @ v[t, h].abs() * abs(v_scale)
    return out, mass


def rows_tolerance(q, k, want, mass, tokens, scale, weight, k_scale=1.0):
    """Per element.  A score is a sum of D exact products in fp32, off by at most
    (D + 4) 2^-24 of |q| |k|, and its weight by twice that (its own and the
    sum's), by half a step of the type that it is multiplied in, and by the 2^x and
    the sum over tokens (2^-21, 2 (tokens / 32 + 64) 2^-24); what a weight is off by
    reaches the output by weight * |v|, which `mass` sums.  fp16 weights are held
    2^7 times as large or more, of the row's largest, so their smallest step, 2^-24,
    rounds a weight off by at most 2^-25 / 2^7 of that: 2^-32 each.  Then the output's own rounding."""
    if not k.numel():
        return mass + torch.finfo(q.dtype).tiny  # no token: zeros
    # |q| |k|, by their largest elements where norms overflow
    clean = [torch.nan_to_num(x.float(), 0, 0, 0) for x in (q, k)]
    top = min(math.prod(float(x.norm(dim=-1).max()) for x in clean),
              math.prod(float(x.abs().max()) for x in clean) * q.shape[-1])
    rel = (2 * (q.shape[-1] + 4) * 2.0 ** -24 * top * abs(scale * k_scale)
           + HALF_STEP[weight] + 2.0 ** -21 + 2 * (tokens / 32 + 64) * 2.0 ** -24)
    fi = torch.finfo(q.dtype)
    big = torch.nan_to_num(mass, 0, 0, 0).max() if mass.numel() else 0.0
    return (mass * rel * (1 + HALF_STEP[q.dtype]) + tokens * 2.0 ** -32 * big
            + want.abs() * HALF_STEP[q.dtype] * 1.01 + fi.tiny * fi.eps)
