"""page_key_bounds and select_pages against float64 restatements, and a decode
loop of the paged operators together."""

from __future__ import annotations

import pytest
import torch

from paged_ref import (DEV, attend64, attend_tolerance, bounds64, make_cache, make_tables,
                       select64)

pytestmark = pytest.mark.gpu

F8 = torch.float8_e4m3fn
BF, FP = torch.bfloat16, torch.float16


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("dtype,H,D,block,lens,order", [
    (BF, 8, 128, 16, [1, 16, 17, 100, 0], "thd"),
    (FP, 2, 64, 16, [33, 500], "htd"),
    (F8, 4, 128, 32, [31, 32, 33, 200], "thd"),
    (F8, 1, 256, 16, [77], "htd"),
    (BF, 3, 8, 7, [20, 6], "thd"),
    (FP, 1, 80, 1, [9], "thd"),
])
@pytest.mark.parametrize("step", [None, "exact", "grid"])
def test_bounds(dtype, H, D, block, lens, order, step):
    """All pages, or those that a step touched; others keep what they held."""
    from korith_vllm_ext.kernels import page_key_bounds

    g = torch.Generator().manual_seed(H + D)
    table, pool = make_tables(lens, block, g)
    kv = make_cache(pool, block, H, D, dtype, g, order)
    bdt = BF if dtype == F8 else dtype
    held = torch.full((pool, H, 2, D), 5.0, dtype=bdt, device=DEV)
    first = new = None
    if step:
        first = [max(0, c - 1 - 3 * i) for i, c in enumerate(lens)]
        new = max(c - f for c, f in zip(lens, first)) if step == "grid" else None
    want = held.clone()
    for i, b in bounds64(kv[0].float(), table, lens, block, first).items():
        want[i] = b.to(bdt)
    got = page_key_bounds(kv, table.to(DEV), _i32(lens), bounds=held,
                          first_tokens=_i32(first) if step else None, max_new_tokens=new)
    assert got is held and torch.equal(got, want)
    if step is None:
        want = torch.where(want == 5.0, 0.0, want)
        assert torch.equal(page_key_bounds(kv[0], table.to(DEV), _i32(lens)), want)


def test_bounds_leave_stale_tokens_out_and_show_nan():
    from korith_vllm_ext.kernels import page_key_bounds

    g = torch.Generator().manual_seed(1)
    table, pool = make_tables([20, 40], 16, g)
    kv = make_cache(pool, 16, 2, 64, BF, g)
    kv[0, int(table[0, 1]), 4:] = float("nan")    # behind the context
    kv[0, int(table[1, 0]), 3, 1, 5] = float("nan")
    flag = torch.zeros(1, dtype=torch.int32, device=DEV)
    b = page_key_bounds(kv, table.to(DEV), _i32([20, 40]), err_flag=flag)
    nan = torch.isnan(b)
    assert int(nan.sum()) == 2 and nan[int(table[1, 0]), 1, :, 5].all() and int(flag) == 0
    table[0, 0], table[1, 1] = -2, pool
    want = bounds64(kv[0].float(), table, [20, 40], 16)
    b = page_key_bounds(kv, table.to(DEV), _i32([20, 40]), err_flag=flag)
    assert int(flag) == 1
    assert set(torch.nonzero(b.float().abs().sum((1, 2, 3)) != 0).flatten().tolist()) == set(want)
    flag.zero_()
    page_key_bounds(kv, table[:, :1].to(DEV), _i32([20, 8]), err_flag=flag)
    assert int(flag) == 1 | 2


@pytest.mark.parametrize("lens,width,first,new,want", [
    ([33], 2, None, None, 2), ([32], 2, None, None, 0),
    ([33], 2, [0], None, 2), ([33], 2, [0], 33, 2), ([33], 2, [15], 18, 2),
    ([33], 2, [33], 1, 2), ([20, 40, 7], 2, None, None, 2), ([20, 32, 7], 2, [3, 3, 3], 29, 0),
    ([5], 0, None, None, 2), ([0, -2], 0, None, None, 0), ([5], 0, [2], 3, 2),
])
def test_bounds_flag_a_context_that_the_table_does_not_hold(lens, width, first, new, want):
    """Whatever part of the pages the call writes; 8 heads of 128 fill the
    grid's workgroups, so that no thread lies behind the table's pages."""
    from korith_vllm_ext.kernels import page_key_bounds

    g = torch.Generator().manual_seed(3)
    kv = make_cache(8, 16, 8, 128, BF, g)
    table = torch.arange(len(lens) * width, dtype=torch.int32).view(len(lens), width)
    flag = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = page_key_bounds(kv, table.to(DEV), _i32(lens), max_new_tokens=new, err_flag=flag,
                          first_tokens=None if first is None else _i32(first))
    assert int(flag) == want
    ref = torch.zeros_like(got)
    for i, b in bounds64(kv[0].float(), table, lens, 16, first).items():
        ref[i] = b.to(BF)
    assert torch.equal(got, ref)


def _selection(dtype, Hq, H, D, block, lens, seed=0):
    g = torch.Generator().manual_seed(seed + D + Hq)
    table, pool = make_tables(lens, block, g)
    b = torch.randn(pool, H, 2, D, generator=g).to(dtype)
    b = torch.stack((b.amin(2), b.amax(2)), 2).contiguous().to(DEV)
    q = torch.randn(len(lens), Hq, D, generator=g).to(dtype).to(DEV)
    return q, b, table


def _select(q, b, table, lens, block, keep, first=1, last=1, **kw):
    from korith_vllm_ext.kernels import select_pages

    return select_pages(q, b, table.to(DEV), _i32(lens), block_size=block, num_pages=keep,
                        first_pages=first, last_pages=last, **kw)


@pytest.mark.parametrize("dtype,Hq,H,D,block,lens,keep,first,last", [
    (BF, 32, 8, 128, 16, [1000, 16, 0, 33, 528, 529, 545], 33, 1, 1),
    (FP, 14, 2, 64, 16, [3000, 100], 8, 0, 0),
    (BF, 64, 8, 128, 32, [5000], 20, 2, 3),
    (FP, 16, 2, 256, 16, [900, 901], 17, 1, 1),
    (BF, 3, 3, 80, 16, [400], 1, 0, 0),
    (BF, 3, 3, 80, 16, [400], 1, 0, 1),
    (FP, 17, 1, 8, 5, [333, 14], 4, 2, 2),
    (BF, 8, 1, 128, 1, [1500], 64, 1, 1),          # one-token pages
    (BF, 8, 4, 64, 16, [30000], 100, 1, 1),
    (BF, 2, 1, 64, 1, [33000], 1025, 0, 7),        # more pages than LDS holds keys
])
def test_select(dtype, Hq, H, D, block, lens, keep, first, last):
    q, b, table = _selection(dtype, Hq, H, D, block, lens)
    pages, counts = _select(q, b, table, lens, block, keep, first, last)
    want = select64(q, b, table, lens, block, keep, first, last)
    assert torch.equal(counts.cpu(), want[1]) and torch.equal(pages.cpu(), want[0])


@pytest.mark.parametrize("n", [1023, 1024, 1025, 4095, 4096, 4097, 8191, 8192, 8193, 16385])
def test_select_around_the_choices_row_sizes(n):
    """Rows that the choice keeps in registers of 256 and 1024 threads, and
    reads again for each pass; half of the pages have equal scores."""
    lens = [n * 4, n * 4 - 3, (n - 1) * 4, n]
    q, b, table = _selection(BF, 4, 1, 8, 4, lens, seed=n)
    even = torch.randperm(b.shape[0], generator=torch.Generator().manual_seed(n))[::2].to(DEV)
    b[even] = b[int(table[0, 1])].clone()  # in the middle of the scores: ties at the cut
    for keep in (1, n // 4, n // 2, n - 1):
        first, last = (0, 0) if keep == 1 else (1, 2)
        pages, counts = _select(q, b, table, lens, 4, keep, first, last)
        want = select64(q, b, table, lens, 4, keep, first, last)
        assert torch.equal(counts.cpu(), want[1]) and torch.equal(pages.cpu(), want[0]), keep


@pytest.mark.parametrize("kind", ["equal", "few", "near", "zero"])
def test_select_ties(kind):
    """Equal scores go to the lowest places; scores one step apart in the last
    bits of a sum that fp32 would not tell apart do not tie."""
    lens, H, D = [9000, 700], 2, 128
    q, b, table = _selection(BF, 8, H, D, 16, lens, seed=1)
    if kind == "equal":
        b[:] = b[:1]
    elif kind == "few":
        b[:] = b[torch.arange(b.shape[0], device=DEV) % 3]
    elif kind == "zero":
        q.zero_()
    else:
        b[:] = b[:1]  # one channel differs by 2^-30 of the sum
        q.fill_(1.0)
        b[:, :, :, 0] = 0
        b[:, :, :, 1] = 4096.0
        b[:, :, 1, 0] = (2.0 ** -17 * torch.randint(1, 90, (b.shape[0], H), device=DEV)).to(BF)
    pages, counts = _select(q, b, table, lens, 16, 24)
    want = select64(q, b, table, lens, 16, 24, 1, 1)
    assert torch.equal(pages.cpu(), want[0]) and torch.equal(counts.cpu(), want[1])


def test_select_non_finite_and_bad_pages():
    """Pages with NaN or infinite bounds come first, pages outside the pool
    last; a q that is not finite makes every page equal."""
    lens = [1600, 1600]
    q, b, table = _selection(FP, 4, 2, 64, 16, lens, seed=2)
    b[int(table[0, 50]), 0, 0, 3] = float("nan")
    b[int(table[0, 60]), 1, 1, 9] = float("inf")
    b[int(table[0, 61]), 1, 0, 9] = float("-inf")
    q[1, 3, 5] = float("nan")
    table[0, 20:90:2] = -1
    table[0, 33] = b.shape[0]
    flag = torch.zeros(1, dtype=torch.int32, device=DEV)
    pages, counts = _select(q, b, table, lens, 16, 80, err_flag=flag)
    want = select64(q, b, table, lens, 16, 80, 1, 1)
    assert int(flag) == 1
    assert torch.equal(pages.cpu(), want[0]) and torch.equal(counts.cpu(), want[1])
    flag.zero_()
    pages, counts = _select(q, b, table, [1600, 800], 16, 10, max_context_len=800, err_flag=flag)
    assert int(flag) & 2
    want = select64(q, b, table, [800, 800], 16, 10, 1, 1)
    assert torch.equal(pages.cpu(), want[0])


def test_select_score_bounds_every_key():
    """The kept pages hold the best token of all whenever it beats the bound of
    every page left out (it always does not exceed its own page's)."""
    from korith_vllm_ext.kernels import page_key_bounds, select_pages

    g = torch.Generator().manual_seed(6)
    lens, H, D = [4000], 2, 64
    table, pool = make_tables(lens, 16, g)
    kv = make_cache(pool, 16, H, D, BF, g)
    q = torch.randn(1, 4, D, generator=g).to(BF).to(DEV)
    at = int(table[0, 100])
    kv[0, at, 7] = 0
    kv[0, at, 7, :, :] = torch.sign(q[0, ::2].float()).to(BF) * 8  # along head 0 of each group
    b = page_key_bounds(kv, table.to(DEV), _i32(lens))
    pages, _ = select_pages(q, b, table.to(DEV), _i32(lens), block_size=16, num_pages=3)
    assert (pages == 100).any(-1).all()


def test_select_refusals():
    lens = [100, 50]
    q, b, table = _selection(BF, 8, 2, 64, 16, lens)
    bad = [
        dict(q=q.half()), dict(q=q[:, :3]), dict(q=q[..., :32]), dict(q=q[:1]), dict(b=b[0]),
        dict(b=b.float()), dict(b=b.transpose(0, 1)), dict(b=b.cpu()), dict(keep=0),
        dict(keep=2, first=2, last=1), dict(first=-1), dict(block=0), dict(max_context_len=-1),
        dict(workspace=torch.empty(8, dtype=torch.uint8, device=DEV)),
        dict(out=(torch.empty(2, 2, 3, dtype=torch.int32, device=DEV),
                  torch.empty(2, 2, dtype=torch.int32, device=DEV))),
    ]
    for kw in bad:
        args = dict(q=q, b=b, table=table, lens=lens, block=16, keep=4) | kw
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            _select(**args)
    from korith_vllm_ext.kernels import page_key_bounds

    kv = torch.zeros(2, 20, 16, 2, 64, dtype=BF, device=DEV)
    bt, cl = table.to(DEV), _i32(lens)
    bad = [
        dict(k_cache=kv.float()), dict(k_cache=kv[..., :12]), dict(k_cache=kv.cpu()),
        dict(context_lens=cl.long()), dict(context_lens=cl[:1]), dict(first_tokens=cl[:1]),
        dict(max_new_tokens=4), dict(first_tokens=cl, max_new_tokens=0), dict(dtype=FP),
        dict(bounds=torch.zeros(20, 2, 2, 64, device=DEV)),
        dict(bounds=torch.zeros(19, 2, 2, 64, dtype=BF, device=DEV)),
        dict(k_cache=torch.zeros(2, 20, 16, 2, 65, dtype=BF, device=DEV)[..., 1:]),
    ]
    for kw in bad:
        args = dict(k_cache=kv, block_tables=bt, context_lens=cl) | kw
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            page_key_bounds(**args)


@pytest.mark.parametrize("dtype,Hq,H,D", [(BF, 8, 2, 128), (FP, 14, 2, 64), (F8, 8, 2, 128)])
def test_decode_loop(dtype, Hq, H, D):
    """Prompts of three sequences, then steps of one token each: slots built on
    the device, rows written through amf_kv_scatter_slots, bounds kept up, pages
    selected and attended; against float64 over what the cache then holds."""
    import amf_hip
    from korith_vllm_ext.kernels import (build_slot_maps, page_key_bounds, paged_decode_attention,
                                         select_pages)

    g = torch.Generator().manual_seed(8)
    bs, pool, keep = 16, 64, 6
    kv = torch.zeros(2, pool, bs, H, D, dtype=dtype, device=DEV)
    planes = amf_hip.address_table([kv[0].data_ptr(), kv[1].data_ptr()], DEV)
    table = torch.full((3, 20), -1, dtype=torch.int32, device=DEV)
    free = torch.randperm(pool, generator=g).int().to(DEV)
    used = torch.zeros(1, dtype=torch.int32, device=DEV)
    bdt = BF if dtype == F8 else dtype
    bounds = torch.zeros(pool, H, 2, D, dtype=bdt, device=DEV)
    lens = [0, 0, 0]
    cl = _i32(lens)
    for new in ([40, 200, 0], [1, 1, 5], [1, 1, 1], [0, 1, 70], [1, 1, 1]):
        n = sum(new)
        m = build_slot_maps(cl, _i32(new), table, block_size=bs, num_tokens=n + 3,
                            free_pages=free, free_used=used, pool_pages=pool)
        rows = (torch.randn(2, n + 3, H, D, generator=g)).to(dtype).to(DEV)
        src = amf_hip.address_table([rows[0].data_ptr(), rows[1].data_ptr()], DEV)
        rb = H * D * kv.element_size()
        amf_hip.call("amf_kv_scatter_slots", src.data_ptr(), rb, planes.data_ptr(), bs * rb, bs,
                     m.slot_mapping.data_ptr(), pool * bs, 2, n + 3, rb, None,
                     amf_hip.stream_handle(DEV))
        page_key_bounds(kv, table, m.context_lens, first_tokens=cl, max_new_tokens=max(new),
                        bounds=bounds)
        q = torch.randn(3, Hq, D, generator=g).to(bdt).to(DEV)
        pages, counts = select_pages(q, bounds, table, m.context_lens, block_size=bs,
                                     num_pages=keep)
        out = paged_decode_attention(q, kv, block_tables=table, context_lens=m.context_lens,
                                     pages=pages, page_counts=counts, out_dtype=torch.float32)
        full = paged_decode_attention(q, kv, block_tables=table, context_lens=m.context_lens,
                                      out_dtype=torch.float32)
        before, lens = lens, [c + k for c, k in zip(lens, new)]
        assert m.context_lens.tolist() == lens and m.query_start.tolist()[-1] == n
        cl, used = m.context_lens, m.free_used
        # every token of the step sits in its sequence's page
        tab, start = table.cpu(), m.query_start.tolist()
        for s in range(3):
            for j in range(new[s]):
                t = before[s] + j
                assert torch.equal(kv[:, int(tab[s, t // bs]), t % bs].float(),
                                   rows[:, start[s] + j].float())
        for i, b in bounds64(kv[0].float(), tab, lens, bs).items():
            assert torch.equal(bounds[i], b.to(bdt))
        wp, wc = select64(q, bounds, tab, lens, bs, keep, 1, 1)
        assert torch.equal(pages.cpu(), wp) and torch.equal(counts.cpu(), wc)
        tol = attend_tolerance(q, kv, lens, D ** -0.5)
        ref = attend64(q, kv, tab, lens, D ** -0.5, pages=wp, counts=wc)
        assert float((out.cpu().double() - ref).abs().max()) <= tol
        ref = attend64(q, kv, tab, lens, D ** -0.5)
        assert float((full.cpu().double() - ref).abs().max()) <= tol


def test_captured_bounds_are_the_graphs_own():
    """A captured bounds launch writes what the eager one does, over whatever
    the buffer held before the replay."""
    from korith_vllm_ext.kernels import page_key_bounds

    g = torch.Generator().manual_seed(14)
    table, pool = make_tables([300, 90, 16], 16, g)
    kv = make_cache(pool, 16, 2, 64, BF, g)
    bt, cl, ft = table.to(DEV), _i32([300, 90, 16]), _i32([0, 0, 0])
    held = torch.zeros(pool, 2, 2, 64, dtype=BF, device=DEV)

    def call(bounds):
        return page_key_bounds(kv, bt, cl, first_tokens=ft, bounds=bounds)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(held)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(held)
    for lens, first in (([300, 90, 16], [0, 0, 0]), ([299, 33, 0], [250, 32, 0]),
                        ([17, 90, 5], [0, 89, 0])):
        cl.copy_(_i32(lens))
        ft.copy_(_i32(first))
        held.fill_(9.0)
        graph.replay()
        torch.cuda.synchronize()
        want = call(torch.full_like(held, 9.0))
        assert torch.equal(held, want)
        for i, b in bounds64(kv[0].float(), table, lens, 16, first).items():
            assert torch.equal(held[i], b.to(BF).to(DEV))
            want[i] = 9.0
        assert bool((want == 9.0).all())


def test_captured_step():
    """Maps, bounds, choice and attention in one graph, replayed as sequences
    grow; the eager calls give the same bits."""
    from korith_vllm_ext.kernels import (build_slot_maps, page_key_bounds, paged_decode_attention,
                                         select_pages)

    g = torch.Generator().manual_seed(12)
    lens = [1000, 333, 16]
    table, pool = make_tables(lens, 16, g, spare=40, extra=8)
    kv = make_cache(pool, 16, 2, 128, BF, g)
    left = sorted(set(range(pool)) - set(table[table >= 0].tolist()))
    free = torch.tensor(left, dtype=torch.int32, device=DEV)
    q = torch.randn(3, 8, 128, generator=g).to(BF).to(DEV)
    bounds = torch.zeros(pool, 2, 2, 128, dtype=BF, device=DEV)

    def fresh():
        return table.to(DEV), _i32(lens), torch.zeros(1, dtype=torch.int32, device=DEV)

    def step(bt, cl, used, new):
        m = build_slot_maps(cl, new, bt, block_size=16, num_tokens=8, free_pages=free,
                            free_used=used)
        page_key_bounds(kv, bt, m.context_lens, bounds=bounds)
        pages, counts = select_pages(q, bounds, bt, m.context_lens, block_size=16, num_pages=12)
        out = paged_decode_attention(q, kv, block_tables=bt, context_lens=m.context_lens,
                                     pages=pages, page_counts=counts)
        keep = [t.clone() for t in (*m, pages, counts, out, bt)]
        cl.copy_(m.context_lens)
        used.copy_(m.free_used)
        return keep

    new = _i32([1, 1, 1])
    eager_state = fresh()
    eager = [step(*eager_state, new) for _ in range(1)]
    state = fresh()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*fresh(), new)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(*state, new)
    for i in range(20):
        new.copy_(torch.tensor([1, i % 3, 2], dtype=torch.int32))
        if i == 0:
            eager_state = fresh()
        want = step(*eager_state, new)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b), i
    assert len(eager) == 1
