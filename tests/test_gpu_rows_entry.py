"""The entry points of a step's operators: what they take and refuse beside the plain calls."""

from __future__ import annotations

import pytest
import torch

from paged_ref import DEV, make_cache, make_tables
from test_gpu_paged_rows import _i32, _pool

pytestmark = pytest.mark.gpu

BF16, F16, F32, FP8 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn


def _gen(seed):
    return torch.Generator().manual_seed(seed)


@pytest.mark.parametrize("kind", ["cache", "planes", "pool"])
def test_lists_and_host_tensors(kind):
    """hip_decode_attention converts tables, lengths and starts, as without query_start."""
    from korith_vllm_ext import int4_decode_attention as entry

    g = _gen(1)
    ctx, start = [40, 100, 7], [0, 5, 6, 9]
    table, pool = make_tables(ctx, 16, g, fill=0)
    kv = make_cache(pool, 16, 2, 64, BF16, g)
    q = torch.randn(9, 4, 64, generator=g).to(BF16).to(DEV)
    kv = _pool(kv) if kind == "pool" else kv
    k, v = (kv[0], kv[1]) if kind == "planes" else (kv, None)
    call = entry.int4_decode_attention
    want = call(q, k, v, block_tables=table.to(DEV), context_lens=_i32(ctx),
                query_start=_i32(start))
    wide = torch.zeros(3, 50, dtype=torch.int32, device=DEV)
    wide[:, :table.shape[1]] = table.to(DEV)
    for bt, cl, st in ((table.tolist(), ctx, start), (table, torch.tensor(ctx), _i32(start)),
                       (table.to(DEV).long(), _i32(ctx).long(), _i32(start).long()),
                       (wide[:, :table.shape[1]], ctx, torch.tensor(start)),
                       (table.t().contiguous().t().to(DEV), _i32(ctx), start)):
        got = call(q, k, v, block_tables=bt, context_lens=cl, query_start=st,
                   max_context_len=100)  # a hint that this form does not need
        assert torch.equal(got, want)
    for bad in (dict(block_tables=None), dict(context_lens=None), dict(algo="valu"),
                dict(mask=torch.zeros(1, device=DEV)), dict(out_dtype=F32),
                dict(context_lens=[1, 2])):
        kw = dict(block_tables=table.tolist(), context_lens=ctx, query_start=start) | bad
        with pytest.raises((ValueError, TypeError)):
            call(q, k, v, **kw)
    with pytest.raises(TypeError):
        call(q, "cache", block_tables=table.tolist(), context_lens=ctx, query_start=start)


@pytest.mark.parametrize("D,kind", [(64, BF16), (128, F16), (256, BF16), (128, FP8),
                                    (128, "pool")])
def test_misaligned_queries_take_the_same_kernel(D, kind):
    """Rows that are not of whole 16-byte vectors are copied: the same bits as aligned ones."""
    from korith_vllm_ext.kernels import paged_attention

    g = _gen(D)
    ctx, start = [400, 100, 7], [0, 50, 51, 54]
    table, pool = make_tables(ctx, 16, g)
    dtype = BF16 if kind in (FP8, "pool") else kind
    kv = make_cache(pool, 16, 2, D, dtype if kind == "pool" else kind, g)
    kv = _pool(kv) if kind == "pool" else kv
    q = torch.randn(54, 4, D, generator=g).to(dtype).to(DEV)
    kw = dict(query_start=_i32(start), block_tables=table.to(DEV), context_lens=_i32(ctx))
    want = paged_attention(q, kv, **kw)
    n = q.numel()
    shifted = torch.empty(n + 3, dtype=dtype, device=DEV)[3:].view(q.shape)
    rows = torch.empty(54, 4 * D + 4, dtype=dtype, device=DEV)[:, :4 * D].view(54, 4, D)
    heads = torch.empty(54, 4, D + 2, dtype=dtype, device=DEV)[..., :D]
    for x in (shifted, rows, heads):
        x.copy_(q)
        assert torch.equal(paged_attention(x, kv, **kw), want)
    one = torch.empty(4 * D + 3, dtype=dtype, device=DEV)[3:].view(1, 4, D)
    one.copy_(q[50:51])
    kw = dict(query_start=_i32([0, 1]), block_tables=table[1:2].to(DEV), context_lens=_i32([100]))
    assert torch.equal(paged_attention(one, kv, **kw), paged_attention(q[50:51].clone(), kv, **kw))
    # an output that is not aligned is written by the other kernel
    from test_gpu_paged_rows import _check

    out = torch.empty(4 * D + 1, dtype=dtype, device=DEV)[1:].view(1, 4, D)
    values = kv if kind != "pool" else None
    if values is not None:
        _check(one, kv, values.cpu().float(), table[1:2], [1], [100], 16, F32, out=out)
