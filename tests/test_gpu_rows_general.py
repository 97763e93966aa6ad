"""Attention of several rows on both of its kernels: what query_start may hold, and limits."""

from __future__ import annotations

import pytest
import torch

from paged_ref import DEV, make_cache, make_tables
from test_gpu_paged_rows import _check, _i32

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _call(D, dtype, start, ctx, rows=40):
    from korith_vllm_ext.kernels import paged_attention

    g = _gen(D)
    table, pool = make_tables(ctx, 16, g)
    kv = make_cache(pool, 16, 2, D, dtype, g)
    q = torch.randn(rows, 4, D, generator=g).to(dtype).to(DEV)
    out = torch.full_like(q, 7.0)
    flag = torch.zeros(1, dtype=torch.int32, device=DEV)
    paged_attention(q, kv, query_start=_i32(start), block_tables=table.to(DEV),
                    context_lens=_i32(ctx), out=out, err_flag=flag)
    return q, kv, table, out, int(flag)


@pytest.mark.parametrize("D,dtype", [(64, F16), (48, F16), (64, F32), (7, F32)])
@pytest.mark.parametrize("start,ctx", [([3, 9, 41], [20, 50]), ([-1, 9, 29], [20, 50]),
                                       ([9, 3, 29], [20, 50])])
def test_malformed_starts_are_flagged(D, dtype, start, ctx):
    """Rows outside the step, or that end before they begin."""
    assert _call(D, dtype, start, ctx)[-1] == 2


@pytest.mark.parametrize("D,dtype", [(64, F16), (48, F16), (64, F32)])
def test_short_tables_are_flagged_and_rows_of_nobody_are_not(D, dtype):
    assert _call(D, dtype, [0, 6, 26], [20, 50])[-1] == 0
    # no rows, so nothing is asked of the table
    from korith_vllm_ext.kernels import paged_attention

    q, kv, table, _, _ = _call(D, dtype, [0, 6, 26], [20, 50])
    for start, want in (([0, 6, 6], 0), ([0, 6, 7], 2)):
        flag = torch.zeros(1, dtype=torch.int32, device=DEV)
        paged_attention(q, kv, query_start=_i32(start), block_tables=table.to(DEV),
                        context_lens=_i32([20, 500]), err_flag=flag)
        assert int(flag) == want


@pytest.mark.parametrize("D,dtype", [(64, F16), (48, F16), (64, F32)])
def test_sequences_behind_a_malformed_one_get_their_rows(D, dtype):
    """Starts that do not ascend: the sequences whose own two are in order have their rows."""
    start, ctx = [0, 5, 41, 20, 30], [9, 50, 70, 33]
    q, kv, table, out, flag = _call(D, dtype, start, ctx)
    assert flag == 2
    assert (out[5:20] == 7.0).all() and (out[30:] == 7.0).all()
    w = F16 if dtype is F16 and D == 64 else F32
    got = _check(q[20:30], kv, kv, table[3:], [10], [33], 16, w)
    assert torch.equal(out[20:30], got)
    assert torch.equal(out[:5], _check(q[:5], kv, kv, table[:1], [5], [9], 16, w))


def test_the_most_rows_that_a_call_takes():
    """2^26 rows of one head on the general kernel: more waves than one dimension of a grid has."""
    from korith_vllm_ext.kernels import paged_attention

    n = 1 << 26
    g = _gen(2)
    table, pool = make_tables([n], 1 << 20, g, spare=0)
    kv = torch.randn(2, pool, 1 << 20, 1, 1, generator=g).to(DEV)
    q = torch.zeros(n, 1, 1, device=DEV)  # scores of 0: averages of the values
    seqs = n // 2  # two rows each, of two tokens
    start = torch.arange(0, n + 1, 2, dtype=torch.int32, device=DEV)
    bt = torch.randint(0, pool, (seqs, 1), dtype=torch.int32, device=DEV)
    lens = torch.full((seqs,), 2, dtype=torch.int32, device=DEV)
    out = paged_attention(q, kv, query_start=start, block_tables=bt, context_lens=lens)
    v = kv[1][bt[:, 0].long(), :2, 0, 0]
    want = torch.stack((v[:, 0], v.double().mean(1).float()), 1).view(-1)
    # halves are exact: one rounding of the sum, one of the quotient
    assert ((out.view(-1) - want).abs() <= 2.0 ** -22 * v.abs().max()).all()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("bad,wild", [(0, 1), (1, 0), (2, 3), (3, 2), (0, 4)])
def test_int4_infinite_values_beside_a_bad_page(D, bad, wild):
    """Pages that one wave takes out of their codes together: one is none, all rows see an infinite
    zero point of the other, far from the diagonal."""
    from korith_vllm_ext.codecs import get_codec
    from test_gpu_paged_rows import _pool

    g = _gen(D)
    for rows in (1, 20):
        table, pool = make_tables([200], 16, g)
        kv = _pool(make_cache(pool, 16, 2, D, BF16, g))
        # V params [page][head][groups][16 tokens]
        words = kv.scales[1, int(table[0, wild])].view(2, D // 32, 16)
        words[1, 1, 3] = (0x7C00 << 16) | (int(words[1, 1, 3]) & 0xFFFF)
        values = get_codec("int4_asym_g32").decompress_to(kv, BF16)
        table[0, bad] = -1
        q = torch.randn(rows, 4, D, generator=g).to(BF16).to(DEV)
        flag = torch.zeros(1, dtype=torch.int32, device=DEV)
        got = _check(q, kv, values, table, [rows], [200], 16, BF16, err_flag=flag)
        assert torch.isinf(got[:, 2:, 32:64]).all() and int(flag) == 1
