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


def test_what_lies_in_the_cache_is_refused():
    """Rows, outputs and indices that lie in what the call writes otherwise, or reads."""
    from korith_vllm_ext.kernels import (int4_page_pool, paged_attention, read_kv_cache,
                                         rotary_embedding, rotary_frequencies, write_kv_cache)

    g = _gen(5)
    kv, pool = make_cache(8, 16, 2, 64, BF16, g), int4_page_pool(8, 2, 64)
    blob = pool.meta["_blob"]
    k, q = (torch.randn(4, h, 64, generator=g).to(BF16).to(DEV) for h in (2, 4))
    slots = torch.arange(4, device=DEV)
    r = rotary_frequencies(64)
    inside = kv[0, 3, :4]                                   # rows of the cache
    wide = kv[1, 2].reshape(4, 8, 64)[:, :4]                # [4, 4, 64] there, a view
    assert wide.data_ptr() == kv[1, 2].data_ptr()
    tokens = blob[:4 * 4 * 64 * 2].view(BF16).view(4, 4, 64)
    ints = blob[:32].view(torch.int64)
    at = dict(slot_mapping=slots)
    rot = at | dict(rotary=r, positions=slots)
    flag = kv[0, 0, 0, 0, :2].view(torch.int32)
    bad = [
        lambda: write_kv_cache(inside, k, kv, **at),
        lambda: write_kv_cache(k, inside, kv[0], kv[1], **at),
        lambda: write_kv_cache(k, k, kv, q=wide, **rot),
        lambda: write_kv_cache(k, k, kv, q=q, q_out=wide, **rot),
        lambda: write_kv_cache(tokens[:, :2], k, pool, **at),
        lambda: write_kv_cache(k, tokens[:, 2:], pool, **at),
        lambda: write_kv_cache(k, k, pool, q=q, q_out=tokens, **rot),
        lambda: write_kv_cache(k, k, pool, slot_mapping=ints),
        lambda: write_kv_cache(k, k, pool, slot_mapping=slots, rotary=r, positions=ints),
        lambda: write_kv_cache(k, k, kv, err_flag=flag, **at),
        lambda: write_kv_cache(k, k, kv, q=q[:, :2], q_out=q.view(-1)[:512].view(4, 2, 64),
                               **rot),
        lambda: write_kv_cache(k, k, kv, slot_mapping=q.view(-1)[:16].view(torch.int64), rotary=r,
                               positions=slots, q=q, q_out=q),
        lambda: read_kv_cache(kv, out=(inside, k), **at),
        lambda: read_kv_cache(kv, out=(k, inside), **at),
        lambda: read_kv_cache(kv[0], kv[1], out=(k, wide[:, :2]), **at),
        lambda: read_kv_cache(pool, out=(k, tokens[:, 2:]), **at),
        lambda: read_kv_cache(pool, slot_mapping=k.view(-1)[:16].view(torch.int64),
                              out=(k, k.clone())),
        lambda: rotary_embedding(q, None, q.view(-1)[:16].view(torch.int64), r, out=(q, None)),
    ]
    a = dict(query_start=_i32([0, 4]), block_tables=_i32([[0, 1]]), context_lens=_i32([20]))
    ws = torch.empty(140 << 20, dtype=torch.uint8, device=DEV)
    bad += [
        lambda: paged_attention(q, kv, out=kv[0, 3].view(-1)[:1024].view(4, 4, 64), **a),
        lambda: paged_attention(q, pool, out=tokens, **a),
        lambda: paged_attention(q, kv, out=torch.empty_like(q), workspace=ws, err_flag=ws[:4].view(
            torch.int32), **a),
        lambda: paged_attention(q, kv, workspace=ws, out=ws[:2048].view(BF16).view(4, 4, 64), **a),
        lambda: paged_attention(ws[:2048].view(BF16).view(4, 4, 64), kv, workspace=ws, **a),
        lambda: paged_attention(q, kv, workspace=ws, **a | dict(
            block_tables=ws[:8].view(torch.int32).view(1, 2))),
    ]
    state = [t.clone() for t in (q, k, kv, blob)]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            raise AssertionError(f"call {i} was taken")
    torch.cuda.synchronize()
    for x, y in zip(state, (q, k, kv, blob)):
        assert torch.equal(x, y)
    # rows beside each other, pages of K and V in turn, and a copy of what lies in the cache
    pages = torch.zeros(8, 2, 16, 2, 64, dtype=BF16, device=DEV)
    write_kv_cache(inside.clone(), k, pages[:, 0], pages[:, 1], **at)
    got = read_kv_cache(pages[:, 0], pages[:, 1], **at)
    assert torch.equal(got[0], inside) and torch.equal(got[1], k)
    qkv = torch.randn(4, 8, 64, generator=g).to(BF16).to(DEV)
    want, _ = rotary_embedding(qkv[:, :4], None, slots, r)
    write_kv_cache(qkv[:, 4:6], qkv[:, 6:], pages[:, 0], pages[:, 1], q=qkv[:, :4],
                   q_out=qkv[:, :4], **rot)
    assert torch.equal(qkv[:, :4], want)
    out = torch.empty_like(q)
    assert paged_attention(q, kv, out=out, workspace=ws, **a) is out


def test_one_row_in_place():
    from korith_vllm_ext.kernels import rotary_embedding, rotary_frequencies

    g = _gen(6)
    x = torch.randn(1, 8 * 64, generator=g).to(BF16).to(DEV)
    pos, r = torch.full((1,), 1234, device=DEV), rotary_frequencies(64)
    want, _ = rotary_embedding(x[:, :256].view(1, 4, 64), None, pos, r)
    q, out = x.view(1, 8, 64)[:, :4], x[0, :256].view(1, 4, 64)
    assert q.stride() != out.stride()
    rest = x[:, 256:].clone()
    assert rotary_embedding(q, None, pos, r, out=(out, None))[0] is out
    assert torch.equal(q, want) and torch.equal(x[:, 256:], rest)


def test_scales_that_fp32_does_not_hold_are_refused():
    from korith_vllm_ext.kernels import paged_attention

    g = _gen(7)
    kv = make_cache(4, 16, 2, 64, BF16, g)
    q = torch.randn(2, 4, 64, generator=g).to(BF16).to(DEV)
    kw = dict(query_start=_i32([0, 2]), block_tables=_i32([[0, 1]]), context_lens=_i32([20]))
    for bad in (1e39, 1e300, float("inf"), 1e-39, 0.0, -0.1, float("nan")):
        with pytest.raises(ValueError, match="scale"):
            paged_attention(q, kv, scale=bad, **kw)
    paged_attention(q, kv, scale=1e-30, **kw)


@pytest.mark.parametrize("dtype,n,H", [(BF16, 4100, 2), (F32, 40, 2), (F16, 4100, 3)])
def test_int4_rows_of_512_dims(dtype, n, H):
    """The widest heads, rotated whole: the most LDS that a write asks for, and the codec's bytes."""
    from korith_vllm_ext.codecs import get_codec
    from korith_vllm_ext.kernels import (read_kv_cache, rotary_embedding, rotary_frequencies,
                                         write_kv_cache)

    g = _gen(n)
    pages, D = -(-n // 16) + 2, 512
    mirror = make_cache(pages, 16, H, D, dtype, g)
    slots = torch.arange(5, n + 5, device=DEV)
    k, v = (torch.randn(n, H, D, generator=g).to(dtype).to(DEV) for _ in range(2))
    pos = torch.randint(0, 40000, (n,), generator=g).to(DEV)
    r = rotary_frequencies(D)
    pool = _pool(mirror)
    write_kv_cache(k, v, pool, slot_mapping=slots, rotary=r, positions=pos)
    mirror[0].view(-1, H, D)[slots] = rotary_embedding(k, None, pos, r)[0]
    mirror[1].view(-1, H, D)[slots] = v
    want = _pool(mirror)
    assert torch.equal(pool.meta["_blob"], want.meta["_blob"])
    got = read_kv_cache(pool, slot_mapping=slots, dtype=dtype)
    full = get_codec("int4_asym_g32").decompress_to(want, dtype)
    for i in range(2):
        assert torch.equal(got[i], full[i].view(-1, H, D)[slots])


@pytest.mark.parametrize("D,kind", [(64, F16), (128, BF16), (256, BF16), (128, FP8), (128, "pool")])
def test_a_workspace_of_the_call_s_size(D, kind):
    """No byte behind it is written, and what it held before does not matter."""
    import amf_hip
    from korith_vllm_ext.kernels import paged_attention

    g = _gen(D)
    size = amf_hip.load().amf_paged_attn_rows_call_bytes
    dtype = BF16 if kind in (FP8, "pool") else kind
    for rows, ctx in (([1], [1]), ([1], [3000]), ([5] * 3, [40, 900, 5000]), ([200, 1], [700, 9]),
                      ([1] * 40, [100 + 37 * i for i in range(40)]), ([2500], [2500])):
        table, pool = make_tables(ctx, 16, g)
        kv = make_cache(pool, 16, 2, D, dtype if kind == "pool" else kind, g)
        kv = _pool(kv) if kind == "pool" else kv
        q = torch.randn(sum(rows), 8, D, generator=g).to(dtype).to(DEV)
        start = [0] + torch.cumsum(torch.tensor(rows), 0).tolist()
        kw = dict(query_start=_i32(start), block_tables=table.to(DEV), context_lens=_i32(ctx))
        need = size(sum(rows), len(rows), table.shape[1], 16, 8, 2, D)
        ws = torch.full((need + (1 << 20),), 0xFF, dtype=torch.uint8, device=DEV)
        got = paged_attention(q, kv, workspace=ws[:need], **kw)
        assert torch.equal(got, paged_attention(q, kv, **kw))
        assert (ws[need:] == 0xFF).all()
        with pytest.raises(ValueError, match="workspace"):
            paged_attention(q, kv, workspace=ws[:need - 16], **kw)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("pages", [3, 700])
def test_int4_rows_of_odd_values_are_the_codec_s(dtype, pages):
    """Zeros of both signs, constants, subnormals, infinities and NaN in a group of 32."""
    from korith_vllm_ext.kernels import int4_page_pool, write_kv_cache

    g = _gen(pages)
    H, D, n = 2, 128, pages * 16
    x = torch.randn(2, n, H, D // 32, 32, generator=g)
    kinds = torch.randint(0, 8, (2, n, H, D // 32), generator=g)
    sign = torch.where(torch.rand(x.shape, generator=g) < 0.5, -1.0, 1.0)
    x = torch.where((kinds == 1)[..., None], 0.0 * sign, x)
    x = torch.where((kinds == 2)[..., None], torch.full_like(x, 1.25), x)
    x = torch.where((kinds == 3)[..., None], x * torch.finfo(dtype).tiny, x)
    x = torch.where((kinds == 4)[..., None], x * 1e4, x)
    at = torch.randint(0, 32, kinds.shape, generator=g)[..., None] == torch.arange(32)
    for k, v in ((5, float("inf")), (6, -float("inf")), (7, float("nan"))):
        x = torch.where((kinds == k)[..., None] & at, v, x)
    mirror = x.view(2, pages, 16, H, D).to(dtype).to(DEV)
    want = _pool(mirror).meta["_blob"]
    pool = int4_page_pool(pages, H, D)
    write_kv_cache(mirror[0].view(n, H, D), mirror[1].view(n, H, D), pool,
                   slot_mapping=torch.arange(n, device=DEV))
    assert torch.equal(pool.meta["_blob"], want)
    order = torch.randperm(n, generator=g).to(DEV)
    one = int4_page_pool(pages, H, D)
    for part in order.split(n // 3 + 1):
        write_kv_cache(mirror[0].view(n, H, D)[part], mirror[1].view(n, H, D)[part], one,
                       slot_mapping=part)
    assert torch.equal(one.meta["_blob"], want)
