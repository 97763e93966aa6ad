"""Attention of several rows where the softmax weights' own bits show: values that cancel."""

from __future__ import annotations

import pytest
import torch

import step_ref
from paged_ref import DEV, make_cache, make_tables
from test_gpu_paged_rows import _check, _i32, _pool

pytestmark = pytest.mark.gpu

BF16, F16, FP8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn

# A weight enters the second product as two terms of the type beside V: bf16, its first 8 bits
# and what is left (and 2^-23 of it), at most 2^-7 of the leading bit and rounded to 8 bits, so
# off by at most 2^-16 + 2^-23; fp16, a step less than its first 11 bits and what is left, at
# most 2^-9 of the leading bit and rounded to 11 bits: 2^-21.
TWO = {BF16: "two bf16 terms", F16: "two fp16 terms"}
step_ref.HALF_STEP[TWO[BF16]] = 2.0 ** -16 + 2.0 ** -23
step_ref.HALF_STEP[TWO[F16]] = 2.0 ** -21


def _gen(seed):
    return torch.Generator().manual_seed(seed)


@pytest.mark.parametrize("dtype,cache", [(BF16, BF16), (F16, F16), (BF16, FP8), (F16, FP8),
                                         (BF16, "int4"), (F16, "int4")])
@pytest.mark.parametrize("hq,hkv,D", [(8, 2, 128), (14, 2, 64), (4, 1, 256)])
@pytest.mark.parametrize("rows,ctx", [([1, 1, 1], [2, 40, 1500]), ([5, 9, 20], [6, 300, 2001]),
                                      ([130], [200])])
def test_cancelling_values(dtype, cache, hq, hkv, D, rows, ctx):
    """Neighbours of nearly equal keys (two dims a step of 16 bits apart) and opposite values:
    what is left of their weights is some 2^-9 of them, of which a weight of 8 bits has none."""
    from korith_vllm_ext.codecs import get_codec

    g = _gen(hq + D + len(rows))
    table, pool = make_tables(ctx, 16, g)
    kv = make_cache(pool, 16, hkv, D, dtype, g).contiguous()
    kv[0, :, 1::2] = kv[0, :, 0::2]
    kv[0, :, 1::2, :, 3:5] *= 1 + 2 * torch.finfo(dtype).eps
    kv[1] = 1.0
    kv[1, :, 1::2] = -1.0
    values = kv
    if cache == "int4":
        kv = _pool(kv)
        values = get_codec("int4_asym_g32").decompress_to(kv, dtype)
    elif cache is FP8:
        kv = kv.to(FP8)
        values = kv.cpu().float()
    q = torch.randn(sum(rows), hq, D, generator=g).to(dtype).to(DEV)
    _check(q, kv, values, table, rows, ctx, 16,
           TWO[BF16 if dtype is BF16 and cache is not FP8 else F16])


def test_one_row_is_as_exact_as_the_decode_attention():
    from korith_vllm_ext.kernels import paged_attention, paged_decode_attention

    g = _gen(41)
    ctx = [700, 33, 2, 2048]
    table, pool = make_tables(ctx, 16, g)
    for dtype in (BF16, F16):
        kv = make_cache(pool, 16, 2, 128, dtype, g)
        kv[1] = torch.where(torch.rand(kv[1].shape, generator=g) < 0.5, 1.0, -1.0).to(dtype).to(DEV)
        q = torch.randn(4, 8, 128, generator=g).to(dtype).to(DEV)
        kw = dict(block_tables=table.to(DEV), context_lens=_i32(ctx))
        a = paged_attention(q, kv, query_start=_i32([0, 1, 2, 3, 4]), **kw).double()
        b = paged_decode_attention(q, kv, **kw, out_dtype=torch.float32).double()
        # the output's half step, the terms' (of weights that add up to 1, beside values of 1),
        # and what 32-bit scores (of at most |q| |k| scale), powers and sums leave on either side
        top = float(q.float().norm(dim=-1).max() * kv[0].float().norm(dim=-1).max()) / 128 ** 0.5
        tol = (b.abs() * torch.finfo(dtype).eps / 2 * 1.01 + step_ref.HALF_STEP[TWO[dtype]]
               + 2 * (2 * 132 * 2.0 ** -24 * top + 2.0 ** -21 + 2 * (2048 / 32 + 64) * 2.0 ** -24))
        assert ((a - b).abs() <= tol).all()


@pytest.mark.parametrize("rows", [1, 9, 40])
@pytest.mark.parametrize("rise", [5.0, 29.0, 60.0])
def test_large_finite_values_and_rising_scores(rows, rise):
    """Weights are at most 1 whatever tile the largest score lies in: values of 1e30 to 1e35 stay
    finite where their average is."""
    ctx = [448, 6000]
    g = _gen(3)
    table, pool = make_tables(ctx, 16, g)
    for D in (64, 128, 256):
        kv = make_cache(pool, 16, 1, D, BF16, g)
        kv[0] = 0.0
        for s, c in enumerate(ctx):  # scores in powers of two: flat, then higher by `rise`
            for t in range(c):
                kv[0, int(table[s, t // 16]), t % 16, 0, 0] = rise if t % 448 >= 128 else 0.0
        for big in (1e30, 1e35):
            kv[1].normal_().mul_(big)
            q = torch.zeros(2 * rows, 4, D)
            q[..., 0] = 1.0
            got = _check(q.to(BF16).to(DEV), kv, kv, table, [rows, rows], ctx, 16, TWO[BF16],
                         scale=0.6931471805599453)
            assert torch.isfinite(got).all()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rows", [1, 12, 40])
def test_infinite_values_of_any_weight(dtype, rows):
    """An infinite value far from the diagonal stays one, not NaN, whether its token has the largest
    weight, one that a term holds exactly, or 2^-20 of the largest; NaN, and both infinities, give NaN."""
    g = _gen(8)
    ctx = [512]
    for D in (64, 128, 256):
        table, pool = make_tables(ctx, 16, g)
        kv = make_cache(pool, 16, 1, D, dtype, g)
        kv[0] = 0.0
        place = lambda t: (int(table[0, t // 16]), t % 16, 0)  # noqa: E731
        for t, score in ((5, 0.0), (70, -1.0), (140, -7.25), (200, -20.0), (300, 6.0)):
            kv[(0, *place(t), 0)] = score
        # (dim, token): each alone; then NaN, and infinities of both signs
        for d, t in ((0, 5), (1, 70), (2, 140), (3, 200), (4, 300)):
            kv[(1, *place(t), d)] = float("inf") if d % 2 else -float("inf")
        kv[(1, *place(140), 5)] = float("nan")
        kv[(1, *place(5), 6)], kv[(1, *place(300), 6)] = float("inf"), -float("inf")
        q = torch.zeros(rows, 4, D)
        q[..., 0] = 1.0
        got = _check(q.to(dtype).to(DEV), kv, kv, table, [rows], ctx, 16, TWO[dtype],
                     scale=0.6931471805599453)
        assert torch.isinf(got[..., :5]).all() and torch.isnan(got[..., 5:7]).all()
        assert torch.isfinite(got[..., 7:]).all()
