"""Attention of several rows per sequence over caches and INT4 pools against
float64, where it can go wrong: tiles and shares, empty rows, masks, values that
are not finite, bad pages, strides."""

from __future__ import annotations

import math

import pytest
import torch

from paged_ref import DEV, make_cache, make_tables
from step_ref import rows64, rows_tolerance

pytestmark = pytest.mark.gpu

BF16, F16, F32, FP8 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _i32(x):
    return torch.as_tensor(x, dtype=torch.int32).to(DEV)


def _starts(rows):
    return _i32([0] + torch.cumsum(torch.tensor(rows), 0).tolist())


def _pool(kv):
    from korith_vllm_ext.codecs import get_codec

    return get_codec("int4_asym_g32").compress(kv)


def _tokens(kv, values, table, s, n, block):
    """(K, V, good) of the first n tokens of sequence s, from the values."""
    t = torch.arange(n)
    ids = table[s, t // block].long()
    ok = (ids >= 0) & (ids < values.shape[1])
    ids = ids.clamp(0, values.shape[1] - 1)
    return values[0][ids, t % block], values[1][ids, t % block], ok


def _check(q, kv, values, table, rows, ctx, block, weight, scale=None, ks=1.0, vs=1.0, out=None,
           start=None, **kw):
    """Runs the call and compares every row."""
    from korith_vllm_ext.kernels import paged_attention

    st = _starts(rows) if start is None else start
    got = paged_attention(q, kv, query_start=st, block_tables=table.to(DEV),
                          context_lens=_i32(ctx), scale=scale, k_scale=ks, v_scale=vs, out=out,
                          **kw)
    values = values.cpu()
    scale = scale or 1 / math.sqrt(q.shape[2])
    at = st.tolist()
    for s, (n, c) in enumerate(zip(rows, ctx)):
        if n == 0:
            continue
        held = min(c, table.shape[1] * block)
        k, v, ok = _tokens(kv, values, table, s, held, block)
        qs = q[at[s]:at[s] + n]
        pos = [c - n + j for j in range(n)]
        want, mass = rows64(qs, k, v, pos, scale, ks, vs, ok)
        r = got[at[s]:at[s] + n].cpu().double()
        assert torch.equal(torch.isnan(r), torch.isnan(want)), (s, n, c)
        inf = torch.isinf(want)
        assert torch.equal(r[inf], want[inf]), (s, n, c)
        tol = rows_tolerance(qs.cpu(), k, want, mass, max(held, 1), scale, weight, ks)
        fine = torch.isfinite(want)
        bad = (r - want).abs()[fine] > tol[fine]
        assert not bad.any(), (s, n, c, int(bad.sum()), float((r - want).abs()[fine].max()),
                               float(tol[fine].max()))
    return got


MIXES = {
    "ones": ([1, 1, 1], [1, 100, 17]),
    "chunk": ([100], [100]),
    "tail": ([70], [333]),
    "mixed": ([1, 0, 37, 5, 1, 130], [64, 9, 37, 300, 1, 131]),
    "edges": ([1, 64, 65, 2, 31, 33], [63, 64, 65, 128, 129, 200]),
}
HEADS = [(8, 2, 128), (32, 8, 64), (4, 1, 256), (14, 2, 64), (3, 3, 128)]


@pytest.mark.parametrize("mix", list(MIXES))
@pytest.mark.parametrize("hq,hkv,D", HEADS)
@pytest.mark.parametrize("dtype,cache", [(BF16, BF16), (F16, F16), (BF16, FP8), (F16, FP8),
                                         (BF16, "int4"), (F16, "int4")])
def test_matrix_tiles(mix, hq, hkv, D, dtype, cache):
    rows, ctx = MIXES[mix]
    g = _gen(hq + D + len(rows))
    block, order = (16, "thd") if cache == "int4" else (16, "htd") if hkv == 2 else (32, "thd")
    table, pool = make_tables(ctx, block, g, extra=2)
    q = torch.randn(sum(rows), hq, D, generator=g).to(dtype).to(DEV)
    if cache == "int4":
        from korith_vllm_ext.codecs import get_codec

        kv = _pool(make_cache(pool, 16, hkv, D, dtype, g))
        values = get_codec("int4_asym_g32").decompress_to(kv, dtype)
        ks = vs = 1.0
    else:
        kv = values = make_cache(pool, block, hkv, D, cache, g, order, 1.0)
        values = values.cpu().float()
        ks, vs = (0.7, 1.3) if cache is FP8 else (1.0, 1.0)
    _check(q, kv, values, table, rows, ctx, block, BF16 if dtype is BF16 and cache is not FP8
           else F16, None, ks, vs)


@pytest.mark.parametrize("dtype,cache,hq,hkv,D,block", [
    (F32, F32, 4, 2, 64, 16), (F32, F32, 2, 1, 7, 5), (BF16, BF16, 4, 2, 80, 16),
    (F16, FP8, 3, 1, 96, 16), (BF16, "int4", 4, 2, 96, 16), (F16, "int4", 2, 2, 32, 16),
    (BF16, BF16, 260, 2, 64, 16), (BF16, BF16, 4, 2, 250, 1), (F16, F16, 4, 4, 129, 3)])
def test_general_kernel(dtype, cache, hq, hkv, D, block):
    from korith_vllm_ext.codecs import get_codec

    rows, ctx = [1, 0, 9, 66, 3], [200, 4, 30, 66, 2]
    g = _gen(D)
    table, pool = make_tables(ctx, block, g)
    q = torch.randn(sum(rows), hq, D, generator=g).to(dtype).to(DEV)
    if cache == "int4":
        kv = _pool(make_cache(pool, 16, hkv, D, dtype, g))
        values = get_codec("int4_asym_g32").decompress_to(kv, dtype)
    else:
        kv = make_cache(pool, block, hkv, D, cache, g)
        values = kv.cpu().float()
    _check(q, kv, values, table, rows, ctx, block, F32)


@pytest.mark.parametrize("hq,hkv,D,dtype,block", [
    (64, 8, 128, BF16, 16), (128, 1, 64, F16, 16), (9, 1, 128, BF16, 48), (8, 2, 128, F16, 1),
    (4, 4, 256, F16, 64)])
def test_shares_of_long_and_many(hq, hkv, D, dtype, block):
    """Contexts that many shares cut, and more sequences than threads."""
    g = _gen(hq * D)
    for rows, ctx in (([3], [20011]), ([1] * 300, [(7 * i) % 90 + 1 for i in range(300)]),
                      ([40, 1, 1], [2600, 9000, 0 + 5])):
        table, pool = make_tables(ctx, block, g)
        kv = make_cache(pool, block, hkv, D, dtype, g)
        q = torch.randn(sum(rows), hq, D, generator=g).to(dtype).to(DEV) * 2
        _check(q, kv, kv, table, rows, ctx, block, dtype, scale=0.2)


def test_int4_shares():
    from korith_vllm_ext.codecs import get_codec

    g = _gen(5)
    rows, ctx = [5, 1, 200], [9000, 4001, 3000]
    table, pool = make_tables(ctx, 16, g)
    kv = _pool(make_cache(pool, 16, 2, 128, BF16, g))
    values = get_codec("int4_asym_g32").decompress_to(kv, BF16)
    q = torch.randn(sum(rows), 8, 128, generator=g).to(BF16).to(DEV)
    _check(q, kv, values, table, rows, ctx, 16, BF16)


@pytest.mark.parametrize("D,dtype", [(128, BF16), (64, F16), (256, BF16), (80, BF16)])
def test_what_is_not_attended_is_not_used(D, dtype):
    """NaN and inf behind contexts, in pages of nobody, and in a later row's K and V."""
    rows, ctx = [50, 3, 1], [90, 70, 33]
    g = _gen(D)
    table, pool = make_tables(ctx, 16, g, fill=0)
    kv = make_cache(pool, 16, 2, D, dtype, g)
    used = torch.zeros(pool, 16, dtype=torch.bool)
    for s, c in enumerate(ctx):
        t = torch.arange(c)
        used[table[s, t // 16].long(), t % 16] = True
    kv[:, ~used.to(DEV)] = float("nan")
    q = torch.randn(sum(rows), 4, D, generator=g).to(dtype).to(DEV)
    _check(q, kv, kv, table, rows, ctx, 16, dtype)
    # token 60 of sequence 0 is the 21st row's own: its V, some of it, is not finite
    page, at = int(table[0, 60 // 16]), 60 % 16
    kv[1, page, at, 0, 3], kv[1, page, at, 0, 5] = float("inf"), float("nan")
    kv[1, page, at, 1, D - 1] = -float("inf")
    kv[1, int(table[0, 5]), 9, 1, 0] = float("nan")  # token 89, the last row's
    got = _check(q, kv, kv, table, rows, ctx, 16, dtype)
    assert torch.isfinite(got[:20]).all() and not torch.isfinite(got[20:50]).all()
    kv[1, page, at] = 0.0
    kv[0, page, at, 0] = float("nan")  # and K: rows from the 21st on are NaN, none before
    got = _check(q, kv, kv, table, rows, ctx, 16, dtype)
    assert torch.isnan(got[20:50, :2]).all() and torch.isfinite(got[:20]).all()


@pytest.mark.parametrize("cache", [FP8, "int4"])
def test_wild_values_of_quantised_caches(cache):
    from korith_vllm_ext.codecs import get_codec

    rows, ctx = [40], [100]
    g = _gen(77)
    table, pool = make_tables(ctx, 16, g)
    q = torch.randn(40, 4, 64, generator=g).to(BF16).to(DEV)
    page, at = int(table[0, 75 // 16]), 75 % 16
    if cache is FP8:
        kv = make_cache(pool, 16, 2, 64, FP8, g)
        kv.view(torch.uint8)[1, page, at, 1, 7] = 0x7F
        values = kv.cpu().float()
    else:
        kv = _pool(make_cache(pool, 16, 2, 64, BF16, g))
        # V params [page][head][2 groups][16 tokens]: an infinite zero point
        words = kv.scales[1, page].view(2, 2, 16)
        words[1, 1, at] = (0x7C00 << 16) | (int(words[1, 1, at]) & 0xFFFF)
        values = get_codec("int4_asym_g32").decompress_to(kv, BF16)
        assert torch.isinf(values[1, page, at, 1, 32:]).all()
    got = _check(q, kv, values, table, rows, ctx, 16, F16 if cache is FP8 else BF16)
    assert torch.isfinite(got[:15]).all() and not torch.isfinite(got[15:]).all()


def test_scores_of_minus_infinity_and_huge():
    g = _gen(21)
    rows, ctx = [20, 1], [20, 700]
    table, pool = make_tables(ctx, 16, g)
    kv = make_cache(pool, 16, 1, 64, F16, g)
    q = torch.rand(21, 4, 64, generator=g).to(F16).to(DEV) + 0.5
    kv[0, table[0, 0].item(), :4] = -float("inf")  # all that rows 0 .. 3 see: NaN there
    got = _check(q, kv, kv, table, rows, ctx, 16, F16)
    assert torch.isnan(got[:4]).all() and torch.isfinite(got[4:]).all()
    kv[0, table[1, 7].item(), 3] = float("inf")  # one score of +inf: NaN
    got = _check(q, kv, kv, table, rows, ctx, 16, F16)
    assert torch.isnan(got[20]).all()
    kv = make_cache(pool, 16, 1, 64, F16, g, scale=200.0)  # scores of thousands
    _check(q * 10, kv, kv, table, rows, ctx, 16, F16, scale=1.0)


@pytest.mark.parametrize("D", [128, 40])
def test_bad_pages_short_tables_and_rows(D):
    g = _gen(D)
    rows, ctx = [30, 2, 6, 1], [100, 40, 3, 0]
    table, pool = make_tables([128, 48, 16, 1], 16, g, fill=-1)
    kv = make_cache(pool, 16, 2, D, BF16, g)
    q = torch.randn(sum(rows), 4, D, generator=g).to(BF16).to(DEV)
    flag = torch.zeros(1, dtype=torch.int32, device=DEV)
    # the third sequence has more rows than tokens: three of them see none; the fourth has none
    got = _check(q, kv, kv, table, rows, ctx, 16, BF16 if D == 128 else F32, err_flag=flag)
    assert not got[32:35].any() and not got[38].any() and int(flag) == 0
    table[0, 2], table[0, 5], table[1, :] = pool, -5, 1 << 30
    got = _check(q, kv, kv, table, rows, ctx, 16, BF16 if D == 128 else F32, err_flag=flag)
    assert not got[30:32].any() and int(flag) == 1
    flag.zero_()
    _check(q, kv, kv, table[:, :4], [30, 2, 6, 1], [100, 40, 3, 0], 16,
           BF16 if D == 128 else F32, err_flag=flag)
    assert int(flag) == 1 | 2


@pytest.mark.parametrize("D", [64, 48])
def test_rows_of_nobody_stay(D):
    from korith_vllm_ext.kernels import paged_attention

    g = _gen(D)
    ctx = [20, 50]
    table, pool = make_tables(ctx, 16, g)
    kv = make_cache(pool, 16, 2, D, F16, g)
    q = torch.randn(40, 4, D, generator=g).to(F16).to(DEV)
    out = torch.full_like(q, 7.0)
    _check(q, kv, kv, table, [6, 20], ctx, 16, F16, out=out, start=_i32([3, 9, 29]))
    assert (out[:3] == 7.0).all() and (out[29:] == 7.0).all()
    # rows outside the step, or that end before they begin: no rows
    flag = torch.zeros(1, dtype=torch.int32, device=DEV)
    for start in ([3, 9, 41], [-1, 9, 29], [9, 3, 29]):
        flag.zero_()
        out.fill_(7.0)
        paged_attention(q, kv, query_start=_i32(start), block_tables=table.to(DEV),
                        context_lens=_i32(ctx), out=out, err_flag=flag)
        a, b = (3, 9) if start[2] == 41 else (9, 29) if start[0] == -1 else (3, 29)
        assert (out[:a] == 7.0).all() and (out[b:] == 7.0).all() and not (out[a:b] == 7.0).all()
        if D == 64:
            assert int(flag) == 2
    e = paged_attention(q[:0], kv, query_start=_i32([0, 0, 0]), block_tables=table.to(DEV),
                        context_lens=_i32(ctx))
    assert e.shape == (0, 4, D)
    out.fill_(7.0)
    paged_attention(q, kv, query_start=_i32([0]), block_tables=table.to(DEV)[:0],
                    context_lens=_i32([]), out=out)
    assert (out == 7.0).all()


@pytest.mark.parametrize("heads,D", [((8, 2), 64), ((8, 2), 128), ((64, 2), 128), ((4, 1), 256)])
def test_infinite_values_before_the_end_of_a_short_table(heads, D):
    """Every row sees all that the table holds, which ends inside a tile."""
    g = _gen(heads[0] + D)
    rows, ctx = [2, 1], [100, 333]
    table, pool = make_tables([48, 48], 16, g)
    kv = make_cache(pool, 16, heads[1], D, BF16, g)
    kv[1, int(table[0, 2]), 8, 0, 3] = float("inf")   # token 40
    kv[1, int(table[1, 0]), 5, -1, 1] = -float("inf")
    q = torch.randn(3, heads[0], D, generator=g).to(BF16).to(DEV)
    flag = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = _check(q, kv, kv, table, rows, ctx, 16, BF16, err_flag=flag)
    assert torch.isinf(got[:2, 0, 3]).all() and torch.isinf(got[2, -1, 1]) and int(flag) == 2


@pytest.mark.parametrize("cache", [BF16, FP8, "int4"])
@pytest.mark.parametrize("n,group", [(1, 4), (5, 4), (12, 4), (20, 4), (3, 16)])
def test_few_columns(cache, n, group):
    """Tiles of 4 to 80 columns: waves share tokens and dims; bad pages in either half of a tile,
    values that are not finite beside the diagonal, contexts that shares cut."""
    from korith_vllm_ext.codecs import get_codec

    g = _gen(n * group)
    ctx = [n, 40 + n, 2500, 7001]
    rows, H = [n] * 4, 2
    for D in (64, 128, 256):
        table, pool = make_tables(ctx, 16, g, extra=1)
        q = torch.randn(4 * n, H * group, D, generator=g).to(BF16).to(DEV)
        if cache == "int4":
            kv = _pool(make_cache(pool, 16, H, D, BF16, g))
            values = get_codec("int4_asym_g32").decompress_to(kv, BF16)
        else:
            kv = values = make_cache(pool, 16, H, D, cache, g)
            if cache is BF16:
                t = ctx[1] - 1 - n // 2
                kv[1, int(table[1, t // 16]), t % 16, 1, D - 1] = float("inf")
            else:
                values = values.cpu().float()
        weight = F16 if cache is FP8 else BF16
        _check(q, kv, values, table, rows, ctx, 16, weight)
        table[2, 3], table[2, 5], table[3, 100] = -1, pool, -7
        flag = torch.zeros(1, dtype=torch.int32, device=DEV)
        _check(q, kv, values, table, rows, ctx, 16, weight, err_flag=flag)
        assert int(flag) == 1


def test_strided_rows_and_planes():
    g = _gen(31)
    rows, ctx = [9, 30], [100, 64]
    table, pool = make_tables(ctx, 16, g)
    kv = make_cache(pool, 16, 2, 128, BF16, g)
    qkv = torch.randn(39, 12, 128, generator=g).to(BF16).to(DEV)
    a = _check(qkv[:, :8], kv, kv, table, rows, ctx, 16, BF16)
    b = _check(qkv[:, :8].clone(), kv, kv, table, rows, ctx, 16, BF16)
    assert torch.equal(a, b)
    from korith_vllm_ext.kernels import paged_attention

    wide = torch.full((2, 200), -1, dtype=torch.int32)
    wide[:, :table.shape[1]] = table
    kw = dict(query_start=_starts(rows), context_lens=_i32(ctx))
    c = paged_attention(qkv[:, :8], kv[0], kv[1], block_tables=wide.to(DEV)[:, :table.shape[1]],
                        **kw)
    assert torch.equal(a, c)
    t = qkv[:, :8].transpose(1, 2).contiguous().transpose(1, 2)  # dims not contiguous
    assert torch.equal(a, paged_attention(t, kv, block_tables=table.to(DEV), **kw))
    # misaligned rows take the general kernel
    odd = torch.empty(39 * 8 * 128 + 1, dtype=BF16, device=DEV)[1:].view(39, 8, 128)
    odd.copy_(qkv[:, :8])
    _check(odd, kv, kv, table, rows, ctx, 16, BF16)


def test_one_row_is_the_decode_attention():
    from korith_vllm_ext import int4_decode_attention as entry
    from korith_vllm_ext.kernels import paged_attention, paged_decode_attention

    g = _gen(41)
    ctx = [700, 33, 1, 2048]
    table, pool = make_tables(ctx, 16, g)
    kv = make_cache(pool, 16, 2, 128, BF16, g)
    q = torch.randn(4, 8, 128, generator=g).to(BF16).to(DEV)
    kw = dict(block_tables=table.to(DEV), context_lens=_i32(ctx))
    a = paged_attention(q, kv, query_start=_i32([0, 1, 2, 3, 4]), **kw).float()
    b = paged_decode_attention(q, kv, **kw, out_dtype=torch.float32)
    # half a step of the weights and of the output, of values whose mass is at most max |v|
    assert float((a - b).abs().max()) <= 2 * 2.0 ** -8 * float(kv[1].float().abs().max())
    c = entry.int4_decode_attention(q, kv, query_start=_i32([0, 1, 2, 3, 4]), **kw)
    assert torch.equal(a, c.float())


def test_captured_and_side_by_side():
    """Replays with other lengths, two captured calls, and two streams at once."""
    from korith_vllm_ext.kernels import paged_attention

    g = _gen(51)
    table, pool = make_tables([3000, 500], 16, g)
    kv = make_cache(pool, 16, 2, 128, BF16, g)
    pool4 = _pool(kv.contiguous())
    q = torch.randn(12, 8, 128, generator=g).to(BF16).to(DEV)
    lens, start, bt = _i32([3000, 500]), _i32([0, 4, 12]), table.to(DEV)

    def both():
        kw = dict(query_start=start, block_tables=bt, context_lens=lens)
        return paged_attention(q, kv, **kw), paged_attention(q, pool4, **kw)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both()
    for i in range(4):
        q.normal_()
        lens.copy_(_i32([2900 - 700 * i, 400 + i]))
        start.copy_(_i32([0, 1 + i, 12 - i]))
        graph.replay()
        want = both()
        torch.cuda.synchronize()
        n = int(start[2])
        assert torch.equal(got[0][:n], want[0][:n]) and torch.equal(got[1][:n], want[1][:n])
    n = int(start[2])
    for _ in range(5):
        with torch.cuda.stream(side):
            a = both()
        b = both()
        torch.cuda.synchronize()
        for x, y, z in zip(a, b, want):
            assert torch.equal(x[:n], z[:n]) and torch.equal(y[:n], z[:n])


def test_a_step_from_lengths_to_attention():
    """Slot maps, rotation and write, then attention over the pages: the whole
    step of a batch of prompts and decoding sequences, in FP8, INT4 and bf16."""
    from korith_vllm_ext.codecs import get_codec
    from korith_vllm_ext.kernels import (build_slot_maps, int4_page_pool, paged_attention,
                                         read_kv_cache, rotary_frequencies, write_kv_cache)

    g = _gen(61)
    H, Hq, D, pool = 2, 8, 128, 64
    r = rotary_frequencies(D, base=500000.0)
    free = torch.randperm(pool, generator=g).int().to(DEV)
    for kind in ("fp8", "int4", "bf16"):
        cache = int4_page_pool(pool, H, D) if kind == "int4" else torch.zeros(
            2, pool, 16, H, D, dtype=FP8 if kind == "fp8" else BF16, device=DEV)
        lens, used = _i32([0, 0, 0]), _i32([0])
        table = torch.full((3, 20), -1, dtype=torch.int32, device=DEV)
        ks, vs = (0.02, 0.02) if kind == "fp8" else (1.0, 1.0)
        for new in ([40, 7, 100], [1, 1, 1], [5, 0, 1], [1, 60, 3]):
            n = sum(new)
            rows = -(-n // 8) * 8  # padded, as a captured step is
            qkv = torch.randn(rows, Hq + 2 * H, D, generator=g).to(BF16).to(DEV)
            m = build_slot_maps(lens, _i32(new), table, block_size=16, num_tokens=rows,
                                free_pages=free, free_used=used, pool_pages=pool)
            q = write_kv_cache(qkv[:, Hq:Hq + H], qkv[:, Hq + H:], cache,
                               slot_mapping=m.slot_mapping, positions=m.positions, rotary=r,
                               q=qkv[:, :Hq], k_scale=ks, v_scale=vs)
            lens, used = m.context_lens, m.free_used
            if kind == "int4":
                values = get_codec("int4_asym_g32").decompress_to(cache, BF16)
            else:
                values = cache.cpu().float()
            _check(q, cache, values, table.cpu(), new, lens.tolist(), 16,
                   F16 if kind == "fp8" else BF16, None, ks, vs, start=m.query_start)
            k, _ = read_kv_cache(cache, slot_mapping=m.slot_mapping, dtype=BF16, k_scale=ks,
                                 v_scale=vs)
            assert not k[n:].any() and k[:n].any()


def test_refusals():
    from korith_vllm_ext import int4_decode_attention as entry
    from korith_vllm_ext.kernels import int4_page_pool, paged_attention

    g = _gen(71)
    kv = make_cache(4, 16, 2, 64, BF16, g)
    pool = int4_page_pool(4, 2, 64)
    q = torch.randn(6, 4, 64, generator=g).to(BF16).to(DEV)
    kw = dict(query_start=_i32([0, 2, 6]), block_tables=_i32([[0, 1], [2, 3]]),
              context_lens=_i32([20, 30]))
    ws = torch.empty(64, dtype=torch.uint8, device=DEV)
    bad = [
        lambda: paged_attention(q.float(), kv, **kw),
        lambda: paged_attention(q.float(), pool, **kw),
        lambda: paged_attention(q[:, :3], kv, **kw),
        lambda: paged_attention(q[..., :32], kv, **kw),
        lambda: paged_attention(q[0], kv, **kw),
        lambda: paged_attention(q.cpu(), kv, **kw),
        lambda: paged_attention(q, kv[0], **kw),
        lambda: paged_attention(q, pool, kv, **kw),
        lambda: paged_attention(q, pool, k_scale=2.0, **kw),
        lambda: paged_attention(q, kv, k_scale=0.0, **kw),
        lambda: paged_attention(q, kv, scale=-1.0, **kw),
        lambda: paged_attention(q, kv, scale=float("nan"), **kw),
        lambda: paged_attention(q, kv, out=q, **kw),
        lambda: paged_attention(q, kv, out=torch.empty(6, 4, 64, device=DEV), **kw),
        lambda: paged_attention(q, kv, workspace=ws, **kw),
        lambda: paged_attention(q, kv, **kw | dict(query_start=_i32([0, 6]))),
        lambda: paged_attention(q, kv, **kw | dict(query_start=_i32([0, 2, 6]).long())),
        lambda: paged_attention(q, kv, **kw | dict(context_lens=_i32([20]))),
        lambda: paged_attention(q, kv, **kw | dict(block_tables=_i32([0, 1]))),
        lambda: entry.int4_decode_attention(q, kv, query_start=kw["query_start"]),
        lambda: entry.int4_decode_attention(q, kv, algo="mfma", **kw),
        lambda: entry.int4_decode_attention(q, kv, out_dtype=torch.float32, **kw),
    ]
    for i, call in enumerate(bad):
        with pytest.raises((ValueError, TypeError)):
            call()
            raise AssertionError(f"call {i} was taken")
