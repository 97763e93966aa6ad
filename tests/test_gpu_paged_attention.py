"""paged_decode_attention against float64 attention over the same pages: every
element type and page order, context lengths at the edges of its pages, chunks
and shares, page lists, stale and non-finite values, streams and graphs."""

from __future__ import annotations

import pytest
import torch

from paged_ref import DEV, attend64, attend_tolerance, make_cache, make_tables

pytestmark = pytest.mark.gpu

F8 = torch.float8_e4m3fn
BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


def _run(q, kv, table, lens, **kw):
    from korith_vllm_ext.kernels import paged_decode_attention

    return paged_decode_attention(q, kv, block_tables=table.to(DEV),
                                  context_lens=torch.tensor(lens, dtype=torch.int32, device=DEV),
                                  **kw)


def _case(dtype, Hq, Hkv, D, block, lens, order="thd", qdt=None, seed=0, scale=1.0, **kw):
    print(f"paged case {dtype} {Hq}/{Hkv} D={D} block={block} {order} seqs={len(lens)} "
          f"max={max(lens)}", flush=True)
    g = torch.Generator().manual_seed(seed + 31 * D + len(lens))
    table, pool = make_tables(lens, block, g)
    kv = make_cache(pool, block, Hkv, D, dtype, g, order, scale)
    qdt = qdt or (BF if dtype == F8 else dtype)
    q = torch.randn(len(lens), Hq, D, generator=g).to(qdt).to(DEV)
    return q, kv, table


def _check(out, ref, tol):
    err = (out.cpu().double() - ref).abs()
    assert float(err.max()) <= tol, f"max abs {float(err.max()):.3e}, allowed {tol:.3e}"
    # D roundings of a score, independent, each at most 2^-24 of its partial
    # sums (below 64 before the scale of at least 1/16): some 2e-6 of a weight
    assert float(err.norm()) <= 1e-5 * float(ref.norm()) + 1e-30


SHAPES = [
    (BF, 32, 8, 128, 16, [1, 15, 16, 17, 31, 32, 33, 127, 128, 129, 300], "thd"),
    (BF, 64, 8, 128, 16, [700, 5, 2000], "htd"),
    (BF, 8, 1, 128, 32, [4099], "thd"),
    (BF, 14, 2, 64, 16, [40, 1000, 0, 3], "thd"),
    (FP, 32, 8, 128, 32, [257, 64, 65], "htd"),
    (FP, 8, 8, 64, 16, [513, 100], "thd"),
    (FP, 16, 2, 256, 16, [90, 1, 640], "thd"),
    (BF, 16, 2, 256, 64, [333], "htd"),
    (F8, 64, 8, 128, 16, [900, 31, 0, 16], "thd"),
    (F8, 14, 2, 64, 16, [500, 129], "htd"),
    (F8, 8, 4, 256, 32, [100, 77], "thd"),
    (BF, 40, 2, 128, 16, [200, 33], "thd"),    # a group of 20: two head tiles of the matrix kernel
    (FP, 17, 1, 64, 16, [150], "thd"),         # 17: a tile of one head
    (BF, 4, 2, 128, 1, [70, 3], "thd"),        # pages of one token
    (FP, 4, 2, 128, 5, [71, 10], "thd"),       # pages of five
    (BF, 4, 4, 64, 528, [1000, 529], "htd"),   # pages of 33 x 16
    (F32, 12, 4, 96, 16, [100, 0, 33], "thd"),
    (F32, 8, 8, 128, 16, [260], "htd"),
    (BF, 8, 8, 80, 16, [100, 31], "thd"),
    (FP, 5, 1, 33, 16, [50, 7], "thd"),        # odd head_dim
    (F8, 6, 3, 24, 8, [44], "thd"),
    (BF, 3, 3, 1, 4, [9], "thd"),
    (FP, 8, 4, 112, 16, [200, 31], "thd"),     # multiples of 16 below a tile's dims
    (BF, 8, 8, 16, 16, [300], "htd"),
    (F8, 8, 8, 96, 16, [500, 3], "thd"),
    (F8, 6, 2, 48, 32, [130], "htd"),
    (BF, 16, 1, 144, 16, [90, 700], "thd"),
    (F8, 4, 2, 240, 16, [65], "thd"),
    (F32, 4, 4, 250, 16, [40, 600], "thd"),
    (F32, 9, 1, 64, 16, [1000], "thd"),        # three tiles of a group
]


@pytest.mark.parametrize("dtype,Hq,Hkv,D,block,lens,order", SHAPES)
def test_matches_f64(dtype, Hq, Hkv, D, block, lens, order):
    q, kv, table = _case(dtype, Hq, Hkv, D, block, lens, order)
    ks, vs = (0.5, 1.5) if dtype == F8 else (1.0, 1.0)
    s = D ** -0.5
    ref = attend64(q, kv, table, lens, s, ks, vs)
    out = _run(q, kv, table, lens, k_scale=ks, v_scale=vs, out_dtype=F32)
    _check(out, ref, attend_tolerance(q, kv, lens, s, ks, vs))
    # a 16-bit output is the fp32 one rounded once
    if q.dtype != F32:
        assert torch.equal(_run(q, kv, table, lens, k_scale=ks, v_scale=vs), out.to(q.dtype))


@pytest.mark.parametrize("dtype", [BF, FP])
def test_fp8_cache_takes_either_query_type(dtype):
    q, kv, table = _case(F8, 16, 4, 128, 16, [300, 41], qdt=dtype, seed=3)
    ref = attend64(q, kv, table, [300, 41], 128 ** -0.5)
    out = _run(q, kv, table, [300, 41], out_dtype=F32)
    _check(out, ref, attend_tolerance(q, kv, [300, 41], 128 ** -0.5))


@pytest.mark.parametrize("seqs,lo,hi,D", [(300, 0, 40, 64), (700, 0, 3, 128), (1500, 1, 9, 64)])
def test_many_sequences(seqs, lo, hi, D):
    """More sequences than a workgroup has threads, many of them empty."""
    g = torch.Generator().manual_seed(seqs)
    lens = torch.randint(lo, hi + 1, (seqs,), generator=g).tolist()
    lens[-1] = 0
    q, kv, table = _case(BF, 4, 2, D, 16, lens)
    ref = attend64(q, kv, table, lens, 0.3)
    out = _run(q, kv, table, lens, scale=0.3, out_dtype=F32)
    _check(out, ref, attend_tolerance(q, kv, lens, 0.3))
    assert not out[-1].any()


def test_no_sequence_and_no_tokens():
    q, kv, table = _case(BF, 4, 2, 128, 16, [5])
    assert _run(q[:0], kv, table[:0], []).shape == (0, 4, 128)
    out = torch.full((1, 4, 128), 7.0, dtype=BF, device=DEV)
    assert not _run(q, kv, table, [0], out=out).any()
    out.fill_(7.0)
    assert not _run(q, kv, table, [-3], out=out).any()


@pytest.mark.parametrize("dtype,lens", [(BF, [40000, 100, 9000]), (FP, [20011]), (F8, [30000])])
def test_long_contexts_split(dtype, lens):
    """One sequence over many workgroups, and a small one beside it."""
    q, kv, table = _case(dtype, 8, 1, 128, 16, lens, seed=9)
    ref = attend64(q, kv, table, lens, 128 ** -0.5)
    out = _run(q, kv, table, lens, out_dtype=F32, max_context_len=max(lens))
    _check(out, ref, attend_tolerance(q, kv, lens, 128 ** -0.5))


@pytest.mark.parametrize("dtype,D", [(BF, 128), (FP, 128), (F8, 128), (BF, 80), (F32, 64)])
def test_stale_tokens_never_count(dtype, D):
    """NaN and infinities behind the context, in other pages and under table
    entries that no token uses."""
    lens = [5, 33, 1, 130]
    q, kv, table = _case(dtype, 8, 2, D, 16, lens)
    ref = attend64(q, kv, table, lens, 0.2)
    bad = float("nan")
    used = torch.zeros(kv.shape[1], 16, dtype=torch.bool)
    for s, c in enumerate(lens):
        for t in range(c):
            used[int(table[s, t // 16]), t % 16] = True
    gone = ~used.to(DEV)[None, :, :, None, None]
    dirty = kv.float().masked_fill(gone, bad)
    if dtype != F8:
        dirty[:, :, :, :, ::2] = dirty[:, :, :, :, ::2].masked_fill(gone, float("inf"))
    dirty = dirty.to(dtype)
    table[:, -1:] = torch.where(table[:, -1:] < 0, 1 << 30, table[:, -1:])
    out = _run(q, dirty, table, lens, scale=0.2, out_dtype=F32)
    _check(out, ref, attend_tolerance(q, kv, lens, 0.2))


@pytest.mark.parametrize("dtype,D", [(BF, 128), (FP, 64), (BF, 256), (F32, 96)])
def test_non_finite_tokens_show(dtype, D):
    """NaN in K, inf in V, scores that are all -inf or hold +inf: as float64
    attention shows them."""
    lens = [40, 40, 40, 40, 40]
    q, kv, table = _case(dtype, 4, 2, D, 16, lens, seed=5)
    q[:, :, 0] = 1.0

    def row(s, t):
        return int(table[s, t // 16]), t % 16

    i, t = row(0, 37)
    kv[0, i, t, 1, 3] = float("nan")
    i, t = row(1, 20)
    kv[1, i, t, 0, 2] = float("inf")
    for tok in range(40):
        i, t = row(2, tok)
        kv[0, i, t, 0, 0] = float("-inf")
    i, t = row(3, 8)
    kv[0, i, t, 1, 0] = float("inf")
    i, t = row(4, 39)
    kv[0, i, t, 0, 0] = float("-inf")  # this token weighs nothing
    ref = attend64(q, kv, table, lens, 0.1)
    out = _run(q, kv, table, lens, scale=0.1, out_dtype=F32).cpu().double()
    assert torch.equal(torch.isnan(out), torch.isnan(ref))
    assert torch.equal(torch.isinf(out), torch.isinf(ref)) and torch.isinf(ref).any()
    ok = torch.isfinite(ref)
    assert float((out - ref)[ok].abs().max()) <= attend_tolerance(q, kv, lens, 0.1)


@pytest.mark.parametrize("dtype,Hq,D", [(BF, 8, 128), (FP, 8, 64), (BF, 8, 256), (FP, 8, 80),
                                        (F32, 8, 96), (BF, 6, 33)])
@pytest.mark.parametrize("lists", [False, True])
def test_runs_of_minus_infinity_weigh_nothing(dtype, Hq, D, lists):
    """Scores of -inf for whole steps and shares of a context, beside finite
    ones; NaN only where a head has no other."""
    lens = [40, 300, 5000, 70]
    q, kv, table = _case(dtype, Hq, 2, D, 16, lens, seed=6)
    q[:, :, 0] = 1.0

    def gone(s, h, tokens):
        t = torch.tensor(tokens)
        kv[0, table[s, t // 16].long().to(DEV), (t % 16).to(DEV), h, 0] = float("-inf")

    gone(0, 0, range(32))           # the first step of a wave
    gone(0, 1, range(39))           # all but the last token
    gone(1, 0, range(64, 300))      # all behind the first tokens
    gone(1, 1, [t for t in range(300) if t % 16 != 5])
    gone(2, 0, range(4000))         # whole shares
    gone(2, 1, range(1, 5000))
    gone(3, 0, range(70))           # all of them: NaN, as softmax gives
    kw, ref_kw = {}, {}
    if lists:
        n = table.shape[1]
        pages = torch.arange(n, dtype=torch.int32).expand(4, 2, n).contiguous()
        counts = torch.tensor([[-(-c // 16)] * 2 for c in lens], dtype=torch.int32)
        kw = dict(pages=pages.to(DEV), page_counts=counts.to(DEV))
        ref_kw = dict(pages=pages, counts=counts)
    ref = attend64(q, kv, table, lens, D ** -0.5, **ref_kw)
    out = _run(q, kv, table, lens, out_dtype=F32, **kw).cpu().double()
    nan = torch.isnan(ref)
    assert nan[3, :Hq // 2].all() and int(nan.sum()) == Hq // 2 * D
    assert torch.equal(torch.isnan(out), nan)
    assert float((out - ref)[~nan].abs().max()) <= attend_tolerance(q, kv, lens, D ** -0.5)


@pytest.mark.parametrize("dtype", [BF, FP])
def test_small_weights_keep_their_bits(dtype):
    """One token with V = 0 holds nearly all of the softmax; the output is what
    weights of about 2^-20 give the others."""
    D, T = 128, 200
    kv = torch.zeros(2, 13, 16, 1, D, dtype=dtype, device=DEV)
    g = torch.Generator().manual_seed(2)
    kv[1] = (torch.rand(13, 16, 1, D, generator=g) + 0.5).to(dtype).to(DEV)
    table = torch.arange(13, dtype=torch.int32)[None]
    kv[0, 0, 3, 0, 0] = 14.0  # score 14, the others 0: weights e^-14
    kv[1, 0, 3] = 0.0
    q = torch.zeros(1, 4, D, dtype=dtype, device=DEV)
    q[..., 0] = 1.0
    out = _run(q, kv, table, [T], scale=1.0, out_dtype=F32).cpu().double()
    ref = attend64(q, kv, table, [T], 1.0)
    # 2^x at |x| < 21 rounds its argument by 2^-20, and 200 positive terms are summed
    assert float(((out - ref).abs() / ref).max()) <= 2e-5


@pytest.mark.parametrize("dtype,Hkv,D,block", [(BF, 2, 128, 16), (FP, 8, 64, 32), (F8, 4, 128, 16),
                                               (F32, 2, 80, 16), (BF, 1, 256, 7)])
def test_page_lists(dtype, Hkv, D, block):
    """Lists per KV head: none, one page, the last (partial) page, gaps, places
    behind the context, one place twice."""
    lens = [500, 90, 33, 1, 0, 900]
    q, kv, table = _case(dtype, 4 * Hkv, Hkv, D, block, lens, seed=11)
    g = torch.Generator().manual_seed(1)
    S, n = len(lens), 9
    pages = torch.full((S, Hkv, n), -1, dtype=torch.int32)
    counts = torch.zeros(S, Hkv, dtype=torch.int32)
    for s, c in enumerate(lens):
        m = -(-c // block)
        for h in range(Hkv):
            k = min(n, m)
            pages[s, h, :k] = torch.randperm(max(m, 1), generator=g)[:k].sort()[0].int()
            counts[s, h] = k if (s + h) % 3 else max(k - 2, 0)
    pages[0, 0] = torch.tensor([0, -1, 2, 2, 1 << 20, 3, -1, -(-500 // block) - 1, 4])
    counts[0, 0] = 9
    pages[1, 0, 0] = table.shape[1] - 1  # behind this sequence's context
    counts[1, 0] = 1
    ref = attend64(q, kv, table, lens, 0.15, pages=pages, counts=counts)
    # the place outside the table is skipped, as every entry that holds no page
    out = _run(q, kv, table, lens, scale=0.15, out_dtype=F32, pages=pages.to(DEV),
               page_counts=counts.to(DEV))
    _check(out, ref, attend_tolerance(q, kv, lens, 0.15))
    assert not out[1, :4].any() and not out[4].any()


@pytest.mark.parametrize("dtype,Hq,Hkv,D,block,seqs,n", [
    (BF, 8, 2, 128, 16, 1, 300),      # one sequence over many workgroups
    (BF, 32, 8, 128, 16, 9, 110),
    (FP, 16, 8, 64, 32, 90, 70),      # more sequences than shares
    (F8, 8, 4, 128, 16, 150, 70),
    (F8, 6, 2, 48, 5, 40, 260),       # pages that end inside a step
    (BF, 40, 2, 256, 16, 6, 100),     # two head tiles of a group, one workgroup a CU
    (F32, 12, 4, 96, 16, 3, 150),
    (F32, 8, 1, 64, 16, 60, 80),      # the general kernel, two tiles
    (BF, 3, 3, 33, 1, 5, 1500),       # pages of one token, odd head_dim
])
def test_page_lists_cut_between_workgroups(dtype, Hq, Hkv, D, block, seqs, n):
    """Lists long enough to be cut: KV heads with full, short and empty lists
    in one sequence (partials that saw no token), gaps, repeats, places behind
    the context and outside the table, empty sequences."""
    g = torch.Generator().manual_seed(n + seqs)
    top = (n + n // 4) * block
    lens = torch.randint(1, top + 1, (seqs,), generator=g).tolist()
    lens[0] = top
    for s in range(2, seqs, 7):
        lens[s] = 0
    q, kv, table = _case(dtype, Hq, Hkv, D, block, lens, seed=4)
    pages = torch.full((seqs, Hkv, n), -1, dtype=torch.int32)
    counts = torch.zeros(seqs, Hkv, dtype=torch.int32)
    for s, c in enumerate(lens):
        m = -(-c // block)
        for h in range(Hkv):
            k = min(n, m)
            pages[s, h, :k] = torch.randperm(max(m, 1), generator=g)[:k].sort()[0].int()
            counts[s, h] = (k, 0, min(k, 1), n, k // 2)[(s + h) % 5]
            if k > 8:
                pages[s, h, 3], pages[s, h, 5] = -1, pages[s, h, 4]
                pages[s, h, 6], pages[s, h, 7] = 1 << 20, table.shape[1] - 1
    if seqs > 3:
        counts[3] = 0  # tokens, but no list
    ref = attend64(q, kv, table, lens, 0.15, pages=pages, counts=counts)
    out = _run(q, kv, table, lens, scale=0.15, out_dtype=F32, pages=pages.to(DEV),
               page_counts=counts.to(DEV))
    _check(out, ref, attend_tolerance(q, kv, lens, 0.15))
    none = (ref == 0).all(-1)
    assert torch.equal((out == 0).all(-1).cpu(), none) and (seqs < 4 or none[3].all())


@pytest.mark.parametrize("what", ["lists", "tables", "hint"])
def test_many_sequences_and_no_tokens_that_the_host_knows_of(what):
    """More pairs than a workgroup each is for, and nothing to cut: zeros, or with a
    max_context_len that is too small for the lengths still their attention."""
    lens, kw = [3 + s % 60 for s in range(420)], {}
    q, kv, table = _case(BF, 8, 4, 64, 16, lens)
    ref = torch.zeros(len(lens), 8, 64, dtype=torch.float64)
    if what == "lists":
        kw = dict(pages=torch.empty((len(lens), 4, 0), dtype=torch.int32, device=DEV),
                  page_counts=torch.zeros((len(lens), 4), dtype=torch.int32, device=DEV))
    elif what == "tables":
        table = table[:, :0].contiguous()
    else:
        kw = dict(max_context_len=0)
        ref = attend64(q, kv, table, lens, 64 ** -0.5)
    out = _run(q, kv, table, lens, out_dtype=F32, **kw)
    if what == "hint":
        _check(out, ref, attend_tolerance(q, kv, lens, 64 ** -0.5))
    else:
        assert torch.equal(out.cpu().double(), ref)


def test_lists_without_room_hold_nothing():
    lens = [40, 100]
    q, kv, table = _case(BF, 8, 2, 128, 16, lens)
    out = torch.full_like(q, 5.0)
    _run(q, kv, table, lens, out=out, pages=torch.zeros(2, 2, 0, dtype=torch.int32, device=DEV),
         page_counts=torch.full((2, 2), 3, dtype=torch.int32, device=DEV))
    assert not out.any()


@pytest.mark.parametrize("dtype,Hq,Hkv,D,seqs,hi", [
    (BF, 8, 4, 64, 300, 3000),     # more sequences than shares, four KV heads a workgroup
    (FP, 4, 2, 128, 40, 5000),     # two KV heads a workgroup
    (F8, 6, 3, 128, 30, 4000),     # one
    (BF, 40, 1, 64, 20, 3000),     # three head tiles
    (F8, 68, 2, 64, 9, 5000),      # four tiles: two of each KV head
    (BF, 4, 4, 256, 12, 2500),
    (F32, 8, 2, 64, 25, 2000),     # the general kernel, two tiles of a group
    (FP, 16, 2, 256, 30, 2500),    # one workgroup a CU
    (F8, 8, 4, 256, 30, 2500),
    (BF, 6, 1, 80, 270, 1500),
    (F32, 4, 4, 100, 300, 1200),
])
def test_shares_cut_sequences_anywhere(dtype, Hq, Hkv, D, seqs, hi):
    """Many sequences of any length, most of them cut between workgroups, some
    empty; a hint that is too small changes nothing but the cut."""
    g = torch.Generator().manual_seed(seqs + D)
    lens = torch.randint(1, hi + 1, (seqs,), generator=g)
    lens[torch.rand(seqs, generator=g) < 0.2] = 0
    lens[-1] = hi
    lens = lens.tolist()
    q, kv, table = _case(dtype, Hq, Hkv, D, 16, lens, seed=2)
    ref = attend64(q, kv, table, lens, D ** -0.5)
    out = _run(q, kv, table, lens, out_dtype=F32)
    _check(out, ref, attend_tolerance(q, kv, lens, D ** -0.5))
    out = _run(q, kv, table, lens, out_dtype=F32, max_context_len=1)
    _check(out, ref, attend_tolerance(q, kv, lens, D ** -0.5))


@pytest.mark.parametrize("dtype", [BF, FP])
def test_every_fp8_code(dtype):
    """All finite codes as keys and as values: exact in either query type."""
    codes = torch.tensor([c for c in range(256) if c & 0x7F != 0x7F], dtype=torch.uint8)
    D, T = 64, 256
    kv = torch.zeros(2, 16, 16, 1, D, dtype=torch.uint8)
    kv[0].view(T, D)[:254, 0] = codes
    kv[1].view(T, D)[:254] = codes[:, None]
    kv = kv.view(F8).to(DEV)
    table = torch.arange(16, dtype=torch.int32)[None]
    q = torch.zeros(1, 2, D, dtype=dtype, device=DEV)
    q[0, 0, 0], q[0, 1, 0] = 0.0, 2.0 ** -7  # all weights equal; weights of e^-3.5 to e^3.5
    ref = attend64(q, kv, table, [254], 1.0)
    out = _run(q, kv, table, [254], scale=1.0, out_dtype=F32)
    # 254 terms of at most 448 in fp32, weights off by 2^-22
    assert float((out.cpu().double() - ref).abs().max()) <= 448 * 256 * 2.0 ** -24


def test_every_page_listed_equals_no_list():
    lens = [300, 47]
    q, kv, table = _case(BF, 8, 2, 128, 16, lens)
    n = table.shape[1]
    pages = torch.arange(n, dtype=torch.int32).expand(2, 2, n).contiguous().to(DEV)
    counts = torch.tensor([[19, 19], [3, 3]], dtype=torch.int32, device=DEV)
    ref = attend64(q, kv, table, lens, 128 ** -0.5)
    out = _run(q, kv, table, lens, pages=pages, page_counts=counts, out_dtype=F32)
    _check(out, ref, attend_tolerance(q, kv, lens, 128 ** -0.5))


@pytest.mark.parametrize("dtype,D", [(BF, 128), (F32, 64)])
def test_bad_pages_are_skipped_and_flagged(dtype, D):
    """Ids outside the pool are left out of the softmax; a context that its
    table does not hold is cut to it."""
    lens = [100, 64, 40]
    q, kv, table = _case(dtype, 4, 2, D, 16, lens)
    flag = torch.zeros(1, dtype=torch.int32, device=DEV)
    _run(q, kv, table, lens, err_flag=flag)
    assert int(flag) == 0
    table[0, 2], table[1, 1], table[2, 0] = -1, kv.shape[1], (1 << 31) - 1
    ref = attend64(q, kv, table, lens, 0.2)
    out = _run(q, kv, table, lens, scale=0.2, err_flag=flag, out_dtype=F32)
    assert int(flag) == 1
    _check(out, ref, attend_tolerance(q, kv, lens, 0.2))
    flag.zero_()
    out = _run(q, kv, table[:, :2], [100, 16, 20], scale=0.2, err_flag=flag, out_dtype=F32)
    assert int(flag) == 1 | 2
    ref = attend64(q, kv, table[:, :2], [100, 16, 20], 0.2)
    _check(out, ref, attend_tolerance(q, kv, lens, 0.2))


def test_strided_inputs_and_separate_planes():
    """q as a slice of a fused projection, a block table as a slice of a wider
    one, K and V as views of a [pages, 2, block, H, D] cache."""
    lens = [77, 300]
    q, kv, table = _case(BF, 8, 2, 128, 16, lens)
    ref = attend64(q, kv, table, lens, 0.1)
    wide = torch.zeros(2, 12 * 128, dtype=BF, device=DEV)
    wide[:, :1024] = q.reshape(2, 1024)
    qv = wide[:, :1024].view(2, 8, 128)
    both = kv.transpose(0, 1).contiguous()
    tab = torch.full((2, table.shape[1] + 5), -1, dtype=torch.int32)
    tab[:, :table.shape[1]] = table
    from korith_vllm_ext.kernels import paged_decode_attention

    out = paged_decode_attention(
        qv, both[:, 0], both[:, 1], block_tables=tab.to(DEV)[:, :table.shape[1]],
        context_lens=torch.tensor(lens, dtype=torch.int32, device=DEV), scale=0.1, out_dtype=F32)
    _check(out, ref, attend_tolerance(q, kv, lens, 0.1))
    # rows that no 16-byte load can take
    odd = torch.zeros(2, kv.shape[1], 16, 2, 129, dtype=BF, device=DEV)
    odd[..., 1:] = kv
    out = _run(q, odd[..., 1:], table, lens, scale=0.1, out_dtype=F32)
    _check(out, ref, attend_tolerance(q, kv, lens, 0.1))


def test_plane_alone_is_refused():
    """A K plane without its V plane; one plane that is both has to be said."""
    from korith_vllm_ext.int4_decode_attention import int4_decode_attention

    lens = [77, 300]
    q, kv, table = _case(BF, 8, 2, 128, 16, lens)
    with pytest.raises(ValueError, match="V plane"):
        _run(q, kv[0], table, lens)
    with pytest.raises(ValueError, match="V plane"):
        int4_decode_attention(q, kv[0], block_tables=table.to(DEV),
                              context_lens=torch.tensor(lens, dtype=torch.int32, device=DEV))
    both = torch.stack((kv[0], kv[0]))
    out = _run(q, kv[0], table, lens, v_cache=kv[0], out_dtype=F32)
    _check(out, attend64(q, both, table, lens, 128 ** -0.5),
           attend_tolerance(q, both, lens, 128 ** -0.5))


@pytest.mark.parametrize("lens,block,H", [([77, 300], 16, 1), ([9, 4], 1, 2), ([5], 16, 2)])
def test_planes_with_other_strides_where_a_dim_has_one_element(lens, block, H):
    """One KV head (or token, or page): its stride is never used."""
    g = torch.Generator().manual_seed(2)
    table, pool = make_tables(lens, block, g, spare=0)
    kv = make_cache(pool, block, H, 64, BF, g)
    k, v = kv[0], kv[1].clone()
    v = v.as_strided(v.shape, [7 if n == 1 else st for n, st in zip(v.shape, v.stride())])
    assert k.stride() != v.stride() and torch.equal(v, kv[1])
    from korith_vllm_ext.kernels import page_key_bounds

    bt, cl = table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV)
    assert torch.equal(page_key_bounds(v, bt, cl), page_key_bounds(kv[1], bt, cl))
    q = torch.randn(len(lens), 4, 64, generator=g).to(BF).to(DEV)
    out = _run(q, k, table, lens, v_cache=v, out_dtype=F32)
    _check(out, attend64(q, kv, table, lens, 0.125), attend_tolerance(q, kv, lens, 0.125))


def test_far_pages():
    """Byte offsets past 32 bits: pages at the end of a 5 GB plane."""
    pool, lens = 160000, [90, 40]
    g = torch.Generator().manual_seed(4)
    kv = torch.empty(2, pool, 16, 8, 128, dtype=BF, device=DEV)
    table = torch.tensor([[pool - 1, 3, pool - 7, 70001, 0, pool - 2],
                          [131072, 65536, pool - 3, 0, 0, 0]], dtype=torch.int32)
    ids = table.unique().long()
    small = torch.randn(2, len(ids), 16, 8, 128, generator=g).to(BF)
    kv[:, ids.to(DEV)] = small.to(DEV)
    q = torch.randn(2, 32, 128, generator=g).to(BF).to(DEV)
    near = torch.searchsorted(ids, table.long()).int()
    ref = attend64(q, small, near, lens, 0.1)
    out = _run(q, kv, table, lens, scale=0.1, out_dtype=F32)
    _check(out, ref, attend_tolerance(q, small, lens, 0.1))


def test_reached_through_the_dispatch():
    from korith_vllm_ext.int4_decode_attention import int4_decode_attention
    from korith_vllm_ext.kernels import dispatch_kernel

    lens = [200, 18]
    q, kv, table = _case(BF, 8, 2, 128, 16, lens)
    want = _run(q, kv, table, lens)
    kw = dict(block_tables=table.to(DEV),
              context_lens=torch.tensor(lens, dtype=torch.int32, device=DEV))
    assert torch.equal(dispatch_kernel("bf16", "bf16")(q, kv, **kw), want)
    assert torch.equal(int4_decode_attention(q[:, :, None], kv[0], kv[1], **kw), want[:, :, None])
    with pytest.raises(ValueError):
        int4_decode_attention(q, kv, mask=torch.zeros(1, device=DEV), **kw)
    with pytest.raises(ValueError):
        int4_decode_attention(q, kv, algo="valu", **kw)


@pytest.mark.parametrize("how", ["lists", "int64", "host", "slices", "strided"])
def test_dispatch_takes_tables_as_over_an_int4_pool(how):
    from korith_vllm_ext.kernels import hip_decode_attention

    lens = [200, 18]
    q, kv, table = _case(BF, 8, 2, 128, 16, lens)
    want = _run(q, kv, table, lens)
    cl = torch.tensor(lens, dtype=torch.int32)
    if how == "lists":
        bt, cl = table.tolist(), lens
    elif how == "int64":
        bt, cl = table.long().to(DEV), cl.long().to(DEV)
    elif how == "host":
        bt = table
    elif how == "strided":
        bt = table.t().contiguous().to(DEV).t()
        cl = torch.stack((cl, cl), 1).to(DEV)[:, 0]
    else:
        bt = torch.cat((table, table), 1).to(DEV)[:, :table.shape[1]]
        cl = cl.to(DEV)
    assert torch.equal(hip_decode_attention(q, kv, block_tables=bt, context_lens=cl), want)


def test_dispatch_reports_bad_pages():
    from korith_vllm_ext.int4_decode_attention import int4_decode_attention

    q, kv, table = _case(BF, 8, 2, 128, 16, [100, 18])
    table[0, 2] = kv.shape[1]
    flag = torch.zeros(1, dtype=torch.int32, device=DEV)
    cl = torch.tensor([100, 500], dtype=torch.int32, device=DEV)
    out = int4_decode_attention(q, kv, block_tables=table.to(DEV), context_lens=cl, err_flag=flag)
    assert int(flag) == 1 | 2
    assert torch.equal(out, _run(q, kv, table, [100, 500]))


def test_other_stream_and_shared_scratch():
    """Two streams at once, each with its own scratch; the same bits."""
    lens = [5000, 300]
    q, kv, table = _case(BF, 8, 2, 128, 16, lens)
    want = _run(q, kv, table, lens)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for _ in range(4):
        for st in streams:
            with torch.cuda.stream(st):
                outs.append(_run(q, kv, table, lens))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_threads_on_one_stream():
    """Calls of several host threads on the same stream, whose launches may
    fall between each other."""
    import threading

    cases = [_case(BF, 8, 2, 128, 16, [5000 - 900 * i, 2000], seed=i) + ([5000 - 900 * i, 2000],)
             for i in range(4)]
    want = [_run(*c) for c in cases]
    bad, gate = [], threading.Barrier(4)
    stream = torch.cuda.current_stream()

    def work(i):
        with torch.cuda.stream(stream):
            gate.wait()
            outs = [_run(*cases[i]) for _ in range(40)]
            torch.cuda.synchronize()
            bad.extend(i for o in outs if not torch.equal(o, want[i]))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


@pytest.mark.parametrize("dtype,D", [(BF, 128), (F32, 80)])
def test_captured_graph_replays(dtype, D):
    """A captured step replayed with other lengths and pages, eager work
    between the replays."""
    from korith_vllm_ext.kernels import paged_decode_attention

    lens = [3000, 40, 700]
    q, kv, table = _case(dtype, 8, 2, D, 16, lens)
    bt = table.to(DEV)
    cl = torch.tensor(lens, dtype=torch.int32, device=DEV)
    out = torch.empty_like(q)

    def call():
        return paged_decode_attention(q, kv, block_tables=bt, context_lens=cl, out=out)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for now in ([3000, 40, 700], [17, 0, 701], [2048, 1, 1], [3000, 48, 640]):
        cl.copy_(torch.tensor(now, dtype=torch.int32))
        out.fill_(3.0)
        graph.replay()
        got = out.clone()
        torch.cuda.synchronize()
        assert torch.equal(got, _run(q, kv, table, now)), now


def test_refusals():
    from korith_vllm_ext.kernels import paged_decode_attention

    lens = [20, 5]
    q, kv, table = _case(BF, 8, 2, 128, 16, lens)
    bt, cl = table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV)

    def call(q=q, k=kv, v=None, bt=bt, cl=cl, **kw):
        return paged_decode_attention(q, k, v, block_tables=bt, context_lens=cl, **kw)

    pages = torch.zeros(2, 2, 3, dtype=torch.int32, device=DEV)
    counts = torch.zeros(2, 2, dtype=torch.int32, device=DEV)
    three = torch.zeros(3, 8, 128, dtype=BF, device=DEV)
    bad = [
        dict(q=q.half()), dict(q=q.float()), dict(q=q[:, :7]), dict(q=q[..., :64]),
        dict(q=q[0]), dict(q=torch.stack([q, q], 2)), dict(q=q.cpu()), dict(k=kv[0, 0]),
        dict(k=kv.cpu()), dict(k=kv.double()), dict(k=kv.unflatten(0, (1, 2))),
        dict(k=torch.cat([kv, kv])), dict(k=kv[0], v=kv[1, :-1]), dict(k=kv[0], v=kv[1].half()),
        dict(k=kv.transpose(3, 4)), dict(bt=bt.long()), dict(bt=bt.cpu()), dict(bt=bt[:1]),
        dict(bt=bt.t().contiguous().t()), dict(bt=None), dict(cl=cl.long()), dict(cl=cl[:1]),
        dict(cl=cl.cpu()), dict(cl=lens), dict(scale=0.0), dict(scale=-1.0),
        dict(scale=float("nan")), dict(pages=pages), dict(page_counts=counts),
        dict(pages=pages[:1], page_counts=counts), dict(pages=pages.long(), page_counts=counts),
        dict(pages=pages, page_counts=counts[:, :1]), dict(pages=pages[:, :, ::2], page_counts=counts),
        dict(out=torch.empty(2, 8, 64, dtype=BF, device=DEV)),
        dict(out=torch.empty(2, 8, 128, dtype=BF)),
        dict(out=torch.empty(2, 8, 256, dtype=BF, device=DEV)[..., ::2]),
        dict(out=torch.empty_like(q), out_dtype=F32), dict(out=q), dict(scale=1e-60),
        dict(max_context_len=-1), dict(q=three[:2], out=three[1:]),
        dict(scale=float("inf")), dict(out_dtype=F8),
        dict(workspace=torch.empty(16, device=DEV)),
        dict(err_flag=torch.zeros(1, device=DEV)),
    ]
    for kw in bad:
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            call(**kw)
    big = torch.zeros(2, 4, 16, 1, 264, dtype=BF, device=DEV)
    with pytest.raises(RuntimeError, match="head_dim"):
        call(q=torch.zeros(2, 1, 264, dtype=BF, device=DEV), k=big)
    call()  # and the good call still runs
