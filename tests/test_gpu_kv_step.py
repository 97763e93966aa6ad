"""Rotary positions, K/V written to and read from caches and INT4 pools, against
plain float64 forms, the page codec's bytes and each other."""

from __future__ import annotations

import pytest
import torch

from paged_ref import DEV, make_cache
from step_ref import rotate64, rotate_tolerance

pytestmark = pytest.mark.gpu

BF16, F16, F32, FP8 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _rotary(pairs, interleaved=False, factor=1.0, base=10000.0):
    from korith_vllm_ext.kernels import Rotary

    f = base ** (-torch.arange(pairs, dtype=torch.float64) / max(pairs, 1))
    return Rotary(f.to(DEV), interleaved, factor)


def _rows(n, heads, dim, dtype, g, wide=0, shift=0):
    """Rows of a wider tensor of `wide` more heads, `shift` elements in."""
    x = torch.randn(n * (heads + wide) * dim + shift, generator=g).to(dtype).to(DEV)
    return x[shift:].view(n, heads + wide, dim)[:, :heads]


def _close(got, x, pos, r, label=""):
    want = rotate64(x, pos, r.frequencies, r.interleaved, r.factor)
    tol = rotate_tolerance(x.cpu(), pos, r.frequencies, r.factor, want)
    bad = (got.cpu().double() - want).abs() > tol
    assert not bad.any(), (label, int(bad.sum()), got.cpu().double()[bad][:3], want[bad][:3])


# ---------------------------------------------------------------- rotation --


@pytest.mark.parametrize("dim,pairs,inter", [
    (128, 64, False), (128, 64, True), (64, 16, False), (64, 16, True), (96, 48, False),
    (80, 40, False), (256, 128, False), (256, 32, True), (512, 256, False), (7, 3, False),
    (7, 3, True), (20, 5, False), (2, 1, True), (128, 4, False), (24, 8, False)])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_rotation(dim, pairs, inter, dtype):
    from korith_vllm_ext.kernels import rotary_embedding

    g = _gen(dim + pairs)
    r = _rotary(pairs, inter, 1.13)
    for n, hq, hk in ((1, 3, 1), (5, 4, 2), (1031, 2, 1)):
        q, k = _rows(n, hq, dim, dtype, g), _rows(n, hk, dim, dtype, g)
        pos = torch.randint(0, 1 << 20, (n,), generator=g).to(DEV)
        qo, ko = rotary_embedding(q, k, pos, r)
        _close(qo, q, pos, r, "q")
        _close(ko, k, pos, r, "k")


def test_rotation_of_fused_rows_in_place_and_misaligned():
    from korith_vllm_ext.kernels import rotary_embedding

    g = _gen(3)
    r = _rotary(32)
    for shift in (0, 1, 3):
        qkv = _rows(37, 12, 64, BF16, g, wide=0, shift=shift)
        q, k, v = qkv[:, :8], qkv[:, 8:10], qkv[:, 10:]
        pos = torch.arange(1000, 1037, device=DEV)
        q0, k0, v0 = q.clone(), k.clone(), v.clone()
        qo, ko = rotary_embedding(q, k, pos, r, out=(q, k))
        assert qo is q and ko is k and torch.equal(v, v0)
        _close(q, q0, pos, r)
        _close(k, k0, pos, r)
        alone, none = rotary_embedding(q0, None, pos, r)
        assert none is None and torch.equal(alone, q)
    # heads before rows, and dims that are not contiguous
    q = torch.randn(6, 9, 64, generator=g).to(DEV).transpose(0, 1)
    pos = torch.arange(9, device=DEV)
    out = torch.empty(6, 9, 64, device=DEV).transpose(0, 1)
    assert rotary_embedding(q, None, pos, r, out=(out, None))[0] is out
    _close(out, q, pos, r)
    t = torch.randn(9, 64, 6, generator=g).to(DEV).transpose(1, 2)
    _close(rotary_embedding(t, None, pos, r)[0], t, pos, r)


def test_rotation_far_back_and_empty():
    from korith_vllm_ext.kernels import rotary_embedding

    g = _gen(4)
    r = _rotary(64, False, 1.0)
    q = _rows(40, 2, 128, F32, g)
    far = torch.randint(-(1 << 31), 1 << 31, (40,), generator=g).to(DEV)
    y = rotary_embedding(q, None, far, r)[0]
    _close(y, q, far, r)
    # turned back by the same angles: 2^-24 of values up to sqrt(2) max |q| each way
    back = rotary_embedding(y, None, -far, r)[0]
    assert float((back - q).abs().max()) <= 4 * 2.0 ** -24 * float(q.abs().max())
    e = q[:0]
    qo, ko = rotary_embedding(e, e, far[:0], r)
    assert qo.shape == e.shape and ko.shape == e.shape
    inf = q.clone()
    inf[0, 0, 5], inf[1, 1, 7] = float("inf"), float("nan")
    z = rotary_embedding(inf, None, far, r)[0]
    hit = torch.zeros(40, 2, 128, dtype=torch.bool, device=DEV)
    hit[0, 0, [5, 69]] = hit[1, 1, [7, 71]] = True
    assert torch.equal(z[~hit], y[~hit]) and not torch.isfinite(z[hit]).any()


def test_frequencies():
    from korith_vllm_ext.kernels import rotary_frequencies as f

    plain = f(64, base=500000.0).frequencies
    assert plain.dtype == torch.float64 and plain.is_cuda
    want = 500000.0 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64)
    assert torch.allclose(plain.cpu(), want, rtol=1e-14, atol=0)


# -------------------------------------------------------------- 16 bits, FP8 --


def _slots(n, pool, block, g, drop=0):
    s = torch.randperm(pool * block, generator=g)[:n]
    s[torch.randperm(n, generator=g)[:drop]] = -1
    return s.to(DEV)


@pytest.mark.parametrize("dtype,cache", [(BF16, BF16), (F16, F16), (F32, F32), (BF16, FP8),
                                         (F16, FP8), (F32, FP8)])
@pytest.mark.parametrize("n,H,D,block,order,pairs", [
    (1, 8, 128, 16, "thd", 64), (50, 2, 64, 16, "htd", 16), (1500, 1, 128, 32, "thd", 0),
    (33, 3, 80, 5, "thd", 40), (20, 2, 7, 16, "thd", 2), (9, 4, 256, 1, "htd", 128)])
def test_write_and_read(dtype, cache, n, H, D, block, order, pairs):
    from korith_vllm_ext.kernels import read_kv_cache, rotary_embedding, write_kv_cache

    g = _gen(n + D)
    pool = -(-n // block) + 4
    kv = make_cache(pool, block, H, D, cache, g, order, 3.0)
    k, v = _rows(n, H, D, dtype, g, wide=2), _rows(n, H, D, dtype, g)
    slots = _slots(n, pool, block, g, drop=n // 5)
    pos = torch.randint(0, 9000, (n,), generator=g).to(DEV)
    ks, vs = (0.017, 0.4) if cache is FP8 else (1.0, 1.0)
    was = kv.clone()
    r = _rotary(pairs) if pairs else None
    flag = torch.zeros(1, dtype=torch.int32, device=DEV)
    assert write_kv_cache(k, v, kv, slot_mapping=slots, rotary=r, positions=pos if r else None,
                          k_scale=ks, v_scale=vs, err_flag=flag) is None
    kr = rotary_embedding(k, None, pos, r)[0] if r else k
    want, ok = was.cpu(), slots.cpu() >= 0
    for i, (x, sc) in enumerate(((kr, ks), (v, vs))):
        x = x.cpu()
        if cache is FP8:  # quotients correctly rounded: 53 bits hold twice 24 and 2 more
            sc = float(torch.tensor(sc, dtype=F32))
            x = (x.double() / sc).float().clamp(-448, 448).to(FP8)
        for j in torch.nonzero(ok)[:, 0].tolist():
            s = int(slots[j])
            want[i, s // block, s % block] = x[j]
    assert torch.equal(kv.cpu().view(torch.uint8) if cache is FP8 else kv.cpu(),
                       want.view(torch.uint8) if cache is FP8 else want)
    out = read_kv_cache(kv, slot_mapping=slots, dtype=dtype, k_scale=ks, v_scale=vs,
                        err_flag=flag)
    for i, sc in enumerate((ks, vs)):
        s = slots.clamp_min(0).cpu()
        rows = want[i][s // block, s % block] if cache is not FP8 else \
            want[i].view(torch.uint8)[s // block, s % block].view(FP8)
        rows = (rows.float() * torch.tensor(sc, dtype=F32)).to(dtype)
        rows[~ok] = 0
        assert torch.equal(out[i].cpu(), rows), i
    assert int(flag) == 0


def test_fp8_edges():
    from korith_vllm_ext.kernels import read_kv_cache, write_kv_cache

    x = torch.tensor([0.0, -0.0, 1e30, -1e30, float("inf"), -float("inf"), float("nan"), 448.0,
                      449.0, 463.9, 465.0, 2.0 ** -9, 2.0 ** -10, 1.5 * 2.0 ** -9, 1e-30, 17.0])
    k = x.view(1, 1, 16).to(DEV)
    kv = torch.zeros(2, 1, 1, 1, 16, dtype=FP8, device=DEV)
    write_kv_cache(k, -k, kv, slot_mapping=torch.zeros(1, dtype=torch.int64, device=DEV))
    a, b = read_kv_cache(kv, slot_mapping=torch.zeros(1, dtype=torch.int64, device=DEV), dtype=F32)
    want = x.clamp(-448, 448).to(FP8).float()
    assert torch.equal(torch.nan_to_num(a.cpu().view(-1), nan=-7.0),
                       torch.nan_to_num(want, nan=-7.0))
    assert torch.equal(torch.nan_to_num(b.cpu().view(-1), nan=7.0),
                       torch.nan_to_num(-want, nan=7.0))


def test_slots_outside_the_pool():
    from korith_vllm_ext.kernels import int4_page_pool, read_kv_cache, write_kv_cache

    g = _gen(9)
    k = _rows(6, 2, 64, BF16, g)
    slots = torch.tensor([3, -1, 64, 5, -(1 << 40), 1 << 40], device=DEV)
    for cache in (make_cache(4, 16, 2, 64, BF16, g), int4_page_pool(4, 2, 64)):
        flag = torch.zeros(1, dtype=torch.int32, device=DEV)
        write_kv_cache(k, k, cache, slot_mapping=slots, err_flag=flag)
        assert int(flag) == 1
        a, b = read_kv_cache(cache, slot_mapping=slots, err_flag=flag)
        gone = torch.tensor([1, 2, 4, 5], device=DEV)
        assert not a[gone].any() and not b[gone].any()
        step = 0 if isinstance(cache, torch.Tensor) else 1
        err = (a[[0, 3]].float() - k[[0, 3]].float()).abs().max()
        assert float(err) <= step * 0.5  # a step is a fifteenth of the range, below 8
        write_kv_cache(k, k, cache, slot_mapping=slots)  # nobody asks


# ---------------------------------------------------------------------- INT4 --


def _pool(mirror):
    from korith_vllm_ext.codecs import get_codec

    return get_codec("int4_asym_g32").compress(mirror)


CHUNKS = {
    "one": [(0, 5, 1)],
    "aligned": [(0, 0, 64)],
    "ragged": [(0, 3, 50), (53, 70, 3), (56, 95, 17), (73, 128, 8)],
    "steps": [(i, 7 * i + 1, 1) for i in range(17)],
}


@pytest.mark.parametrize("case", ["one", "aligned", "ragged", "steps", "shuffled", "gaps"])
@pytest.mark.parametrize("H,D,dtype", [(8, 128, BF16), (2, 64, F16), (1, 32, F32), (3, 96, BF16),
                                       (2, 256, F32), (1, 160, F16), (5, 128, F32)])
def test_int4_write_is_the_codec_s(case, H, D, dtype):
    """A pool written by rows holds the bytes of a pool saved from a cache that
    got the same rows."""
    from korith_vllm_ext.kernels import read_kv_cache, rotary_embedding, write_kv_cache

    g = _gen(D + H)
    pool = 9
    mirror = make_cache(pool, 16, H, D, dtype, g)
    if case in CHUNKS:
        slots = torch.cat([torch.arange(a, a + n) for _, a, n in CHUNKS[case]])
    else:
        slots = torch.randperm(pool * 16, generator=g)[:61]
        if case == "gaps":
            slots = slots.sort()[0]
    n = len(slots)
    k, v = _rows(n, H, D, dtype, g, wide=1), _rows(n, H, D, dtype, g, shift=D % 3)
    pos = torch.randint(0, 40000, (n,), generator=g).to(DEV)
    q = _rows(n, 2 * H, D, dtype, g)
    r = _rotary(D // 4, D == 64)
    kv = _pool(mirror)
    qo = write_kv_cache(k, v, kv, slot_mapping=slots.to(DEV), rotary=r, positions=pos, q=q)
    qr, kr = rotary_embedding(q, k, pos, r)
    assert torch.equal(qo, qr)
    mirror[0].view(-1, H, D)[slots] = kr
    mirror[1].view(-1, H, D)[slots] = v
    want = _pool(mirror)
    assert torch.equal(kv.meta["_blob"], want.meta["_blob"])
    # and what is read back is what the codec restores
    some = torch.randperm(pool * 16, generator=g)[:70]
    for at in (slots, some, some.sort()[0], torch.arange(pool * 16)):
        for out in (BF16, F16, F32):
            got = read_kv_cache(kv, slot_mapping=at.to(DEV), dtype=out)
            from korith_vllm_ext.codecs import get_codec

            full = get_codec("int4_asym_g32").decompress_to(want, out)
            for i in range(2):
                assert torch.equal(got[i], full[i].view(-1, H, D)[at])


def test_int4_unaligned_rows_and_strided_outputs():
    from korith_vllm_ext.kernels import int4_page_pool, read_kv_cache, write_kv_cache

    g = _gen(11)
    k = _rows(21, 2, 64, BF16, g, shift=1)
    v = _rows(21, 2, 64, BF16, g, shift=5)
    slots = torch.arange(7, 28, device=DEV)
    a, b = int4_page_pool(3, 2, 64), int4_page_pool(3, 2, 64)
    write_kv_cache(k, v, a, slot_mapping=slots)
    write_kv_cache(k.contiguous().clone(), v.contiguous().clone(), b, slot_mapping=slots)
    assert torch.equal(a.meta["_blob"], b.meta["_blob"])
    wide = torch.full((21, 5, 64), 9.0, dtype=BF16, device=DEV)
    kv = read_kv_cache(a, slot_mapping=slots, out=(wide[:, :2], wide[:, 3:]))
    plain = read_kv_cache(a, slot_mapping=slots, dtype=BF16)
    assert torch.equal(kv[0], plain[0]) and torch.equal(wide[:, 3:], plain[1])
    assert (wide[:, 2] == 9.0).all()
    odd = torch.full((21 * 128 + 1,), 9.0, dtype=BF16, device=DEV)[1:].view(21, 2, 64)
    other = torch.empty_like(plain[1])
    read_kv_cache(a, slot_mapping=slots, out=(odd, other))
    assert torch.equal(odd, plain[0]) and torch.equal(other, plain[1])


def test_pool_over_a_blob_and_empty_rows():
    from korith_vllm_ext.codecs import get_codec
    from korith_vllm_ext.kernels import int4_page_pool, read_kv_cache, write_kv_cache

    g = _gen(12)
    kv = _pool(make_cache(5, 16, 2, 64, BF16, g))
    again = int4_page_pool(5, 2, 64, blob=kv.meta["_blob"])
    assert again.shape == kv.shape and torch.equal(
        get_codec("int4_asym_g32").decompress_to(again, BF16),
        get_codec("int4_asym_g32").decompress_to(kv, BF16))
    none = torch.zeros(0, dtype=torch.int64, device=DEV)
    e = torch.zeros(0, 2, 64, dtype=BF16, device=DEV)
    was = again.meta["_blob"].clone()
    write_kv_cache(e, e, again, slot_mapping=none)
    assert torch.equal(was, again.meta["_blob"])
    assert read_kv_cache(again, slot_mapping=none)[0].shape == (0, 2, 64)


def test_captured_and_on_another_stream():
    """A captured step replayed on new data, with eager work between."""
    from korith_vllm_ext.kernels import int4_page_pool, read_kv_cache, write_kv_cache

    g = _gen(13)
    r = _rotary(64)
    n, H, D = 19, 4, 128
    k, v, q = (_rows(n, h, D, BF16, g) for h in (H, H, 8))
    slots, pos = torch.arange(30, 30 + n, device=DEV), torch.arange(n, device=DEV)
    pools = [int4_page_pool(6, H, D) for _ in range(2)]
    cache = torch.zeros(2, 6, 16, H, D, dtype=FP8, device=DEV)
    eager = torch.zeros_like(cache)

    def step(pool, c):
        a = write_kv_cache(k, v, pool, slot_mapping=slots, rotary=r, positions=pos, q=q)
        b = write_kv_cache(k, v, c, slot_mapping=slots, rotary=r, positions=pos, q=q, k_scale=0.1)
        return a, b, *read_kv_cache(pool, slot_mapping=slots), *read_kv_cache(
            c, slot_mapping=slots, k_scale=0.1)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(pools[0], cache)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(pools[0], cache)
    for i in range(4):
        k.normal_()
        v.normal_()
        slots.add_(3 if i else 0)
        pos.add_(1000)
        graph.replay()
        want = step(pools[1], eager)
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b), i
    # the pools differ where the warm-up wrote what the first replay wrote over
    assert torch.equal(pools[0].meta["_blob"], pools[1].meta["_blob"])


def test_refusals():
    from korith_vllm_ext.kernels import (Rotary, int4_page_pool, read_kv_cache, rotary_embedding,
                                         rotary_frequencies, write_kv_cache)

    g = _gen(14)
    q, k = _rows(4, 4, 64, BF16, g), _rows(4, 2, 64, BF16, g)
    pos = torch.arange(4, device=DEV)
    r = _rotary(32)
    cache, pool = make_cache(3, 16, 2, 64, BF16, g), int4_page_pool(3, 2, 64)
    bad = [
        lambda: rotary_embedding(q, k[:3], pos, r),
        lambda: rotary_embedding(q, k, pos[:3], r),
        lambda: rotary_embedding(q, k, pos.int(), r),
        lambda: rotary_embedding(q, k, pos.cpu(), r),
        lambda: rotary_embedding(q, k.half(), pos, r),
        lambda: rotary_embedding(q, k, pos, None),
        lambda: rotary_embedding(q, k, pos, _rotary(33)),
        lambda: rotary_embedding(q, k, pos, Rotary(r.frequencies.float())),
        lambda: rotary_embedding(q, k, pos, Rotary(r.frequencies, False, float("nan"))),
        lambda: rotary_embedding(q, k, pos, r, out=(q[:, [1, 0, 2, 3]], None)),
        lambda: rotary_embedding(q, k, pos, r, out=(torch.empty_like(q), k.expand(4, 2, 64)[:2])),
        lambda: rotary_embedding(q[:, :2], None, pos, r, out=(q[:, 1:3], None)),
        lambda: rotary_embedding(q[1:], None, pos[1:], r, out=(q[:3], None)),
        lambda: rotary_embedding(q, k, pos, r, out=(torch.empty_like(q),
                                                    torch.empty_like(k[:, :1]).expand(4, 2, 64))),
        lambda: rotary_embedding(_rows(2, 1, 513, BF16, g), None, pos[:2], r),
        lambda: write_kv_cache(k, k[:, :1], cache, slot_mapping=pos),
        lambda: write_kv_cache(k, k, cache, slot_mapping=pos.int()),
        lambda: write_kv_cache(k.half(), k.half(), cache, slot_mapping=pos),
        lambda: write_kv_cache(k, k, cache, slot_mapping=pos, q=q),
        lambda: write_kv_cache(k, k, cache, slot_mapping=pos, positions=pos),
        lambda: write_kv_cache(k, k, cache, slot_mapping=pos, k_scale=0.5),
        lambda: write_kv_cache(k, k, pool, slot_mapping=pos, v_scale=0.5),
        lambda: write_kv_cache(k, k, cache.view(torch.int16).float().to(FP8), slot_mapping=pos,
                               k_scale=0.0),
        lambda: write_kv_cache(q, q, cache, slot_mapping=pos),
        lambda: write_kv_cache(q, q, pool, slot_mapping=pos),
        lambda: write_kv_cache(k, k, cache[0], cache[0], slot_mapping=pos),
        lambda: write_kv_cache(k, k, pool, cache, slot_mapping=pos),
        lambda: write_kv_cache(k, k, cache, slot_mapping=pos, q_out=q),
        lambda: read_kv_cache(cache, slot_mapping=pos, dtype=torch.float16),
        lambda: read_kv_cache(pool, slot_mapping=pos, dtype=FP8),
        lambda: read_kv_cache(pool, slot_mapping=pos.view(2, 2)),
        lambda: read_kv_cache(pool, slot_mapping=pos, out=(k, k)),
        lambda: read_kv_cache(pool, slot_mapping=pos, out=(k, q)),
        lambda: int4_page_pool(3, 2, 48),
        lambda: int4_page_pool(0, 2, 64),
        lambda: int4_page_pool(3, 2, 64, blob=pool.meta["_blob"][:-1]),
        lambda: rotary_frequencies(63),
        lambda: rotary_frequencies(64, scaling="other"),
        lambda: rotary_frequencies(64, scaling="pairs", pair_factors=[1.0]),
        lambda: rotary_frequencies(64, scaling="pairs", pair_factors=[0.0] * 32),
    ]
    state = [t.clone() for t in (q, k, cache, pool.meta["_blob"])]
    for i, call in enumerate(bad):
        with pytest.raises((ValueError, TypeError)):
            call()
            raise AssertionError(f"call {i} was taken")
    for a, b in zip(state, (q, k, cache, pool.meta["_blob"])):
        assert torch.equal(a, b)
