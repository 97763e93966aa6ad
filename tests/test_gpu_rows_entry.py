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
