"""Argument checks of the step operators' C entry points, and the rotary
frequencies, on the CPU: every call fails validation (or has nothing to do)
before any HIP call."""

from __future__ import annotations

import math

import pytest
import torch

import amf_hip

FAKE = 1 << 20  # never dereferenced

pytestmark = pytest.mark.skipif(torch.cuda.is_available(),
                                reason="argument-validation calls run on the CPU only")

Q = dict(q=FAKE, q_row=512, q_head=64, qo=FAKE, qo_row=512, qo_head=64, hq=8)
ROT = dict(pos=FAKE, freqs=FAKE, pairs=32, inter=0, factor=1.0)
KV = dict(k=FAKE, k_row=128, k_head=64, v=FAKE, v_row=128, v_head=64, dtype=2, rows=4, hkv=2,
          dim=64, slots=FAKE)
CACHE = dict(kc=FAKE, vc=FAKE, kv_dtype=2, page=2048, token=128, head=64, pool=8, block=16,
             ks=1.0, vs=1.0)
POOL = dict(kc=FAKE, kp=FAKE, vc=FAKE, vp=FAKE, pool=8)
END = dict(err=None, stream=None)
OUT = dict(slots=FAKE, k=FAKE, k_row=128, k_head=64, v=FAKE, v_row=128, v_head=64, dtype=2,
           rows=4, hkv=2, dim=64)
CALLS = {
    "amf_rotary_embedding": Q | dict(k=FAKE, k_row=128, k_head=64, ko=FAKE, ko_row=128, ko_head=64,
                                     hkv=2, dtype=2, rows=4, dim=64) | ROT | dict(stream=None),
    "amf_kv_write": KV | CACHE | ROT | Q | END,
    "amf_int4_kv_write": KV | POOL | ROT | Q | END,
    "amf_kv_read": CACHE | OUT | END,
    "amf_int4_kv_read": POOL | OUT | END,
}
ROWS = dict(q=FAKE, q_dtype=2, q_row=512, q_head=64, out=FAKE, rows=4, start=FAKE)
TABLES = dict(bt=FAKE, bt_stride=4, table=4, cl=FAKE, seqs=2, hq=8, hkv=2, dim=64)
WORK = dict(ws=FAKE, wsb=1 << 30, err=None, stream=None)
ATTEND = {
    "amf_paged_attn_rows": ROWS | dict(k=FAKE, v=FAKE, kv_dtype=2, page=2048, token=128, head=64,
                                       pool=8) | TABLES | dict(block=16, scale=0.0, ks=1.0, vs=1.0)
    | WORK,
    "amf_int4_paged_attn_rows": ROWS | POOL | TABLES | dict(scale=0.0) | WORK,
}
INV, UNS = amf_hip.ERR_INVALID_ARG, amf_hip.ERR_UNSUPPORTED
ALL = [(n, c, w, d) for n in CALLS for c, w, d in (
    (INV, "dtype", dict(dtype=3)), (INV, "n_rows", dict(rows=-1)), (UNS, "n_rows",
                                                                   dict(rows=(1 << 25) + 1)),
    (UNS, "head_dim", dict(dim=544)), (INV, "heads", dict(hkv=-1)), (INV, "null", dict(k=None)))]


@pytest.mark.parametrize("name,code,word,change", ALL + [
    ("amf_rotary_embedding", INV, "pairs", dict(pairs=33)),
    ("amf_rotary_embedding", INV, "pairs", dict(pos=None)),
    ("amf_rotary_embedding", INV, "null", dict(qo=None)),
    ("amf_rotary_embedding", INV, "heads", dict(hq=0, hkv=0)),
    ("amf_kv_write", INV, "pairs", dict(freqs=None)),
    ("amf_kv_write", UNS, "type", dict(kv_dtype=0)),
    ("amf_kv_write", INV, "block_size", dict(block=0)),
    ("amf_kv_write", INV, "pool_pages", dict(pool=0)),
    ("amf_kv_write", INV, "scales", dict(ks=0.0)),
    ("amf_kv_write", INV, "scales", dict(vs=float("nan"))),
    ("amf_kv_write", INV, "null", dict(slots=None)),
    ("amf_kv_write", INV, "null", dict(q=None)),
    ("amf_int4_kv_write", UNS, "multiple", dict(dim=80)),
    ("amf_int4_kv_write", INV, "aligned", dict(vp=FAKE + 4)),
    ("amf_int4_kv_write", INV, "pool_pages", dict(pool=0)),
    ("amf_kv_read", UNS, "type", dict(kv_dtype=1)),
    ("amf_kv_read", INV, "block_size", dict(block=-1)),
    ("amf_int4_kv_read", UNS, "multiple", dict(dim=40)),
    ("amf_int4_kv_read", INV, "aligned", dict(kc=FAKE + 8)),
    ("amf_int4_kv_read", INV, "null", dict(kp=None)),
])
def test_refused(name, code, word, change):
    with pytest.raises(amf_hip.AmfHipError) as e:
        amf_hip.call(name, *(CALLS[name] | change).values())
    assert e.value.code == code and word in e.value.message


@pytest.mark.parametrize("name", list(CALLS))
def test_nothing_to_do(name):
    amf_hip.call(name, *(CALLS[name] | dict(rows=0, k=None)).values())


def _turns(f, context):
    return context * f / (2 * math.pi)


def test_frequencies():
    """Each scaling against its definition, pair by pair."""
    from korith_vllm_ext.kernels import rotary_frequencies as make

    def freqs(**kw):
        r = make(64, base=10000.0, device="cpu", **kw)
        return r.frequencies.tolist(), r.factor

    plain = [10000.0 ** (-2 * i / 64) for i in range(32)]
    f, factor = freqs()
    assert factor == 1.0 and all(math.isclose(a, b, rel_tol=1e-14) for a, b in zip(f, plain))
    f, _ = freqs(scaling="linear", factor=4.0)
    assert all(math.isclose(4 * a, b, rel_tol=1e-14) for a, b in zip(f, plain))
    f, _ = freqs(scaling="ntk", factor=4.0)  # the slowest pair is interpolated, the first stays
    assert f[0] == 1.0 and math.isclose(4 * f[-1], plain[-1], rel_tol=1e-12)
    f, _ = freqs(scaling="bands", factor=8.0, original_context=512)
    for a, b in zip(f, plain):
        t = _turns(b, 512)
        keep = 1.0 if t > 4 else 0.0 if t < 1 else (t - 1) / 3
        assert math.isclose(a, b * keep + b / 8 * (1 - keep), rel_tol=1e-12)
    f, factor = freqs(scaling="yarn", factor=4.0, original_context=4096)
    assert math.isclose(factor, 0.1 * math.log(4) + 1)
    for i, (a, b) in enumerate(zip(f, plain)):
        assert b / 4 * (1 - 1e-12) <= a <= b
        if _turns(plain[max(i - 1, 0)], 4096) < 1:
            assert math.isclose(4 * a, b, rel_tol=1e-12)
        if _turns(plain[min(i + 1, 31)], 4096) > 32:
            assert math.isclose(a, b, rel_tol=1e-12)
    f, factor = freqs(scaling="pairs", pair_factors=[1.0 + i for i in range(32)],
                      attention_factor=1.25)
    assert factor == 1.25
    assert all(math.isclose(a * (1 + i), b, rel_tol=1e-14)
               for i, (a, b) in enumerate(zip(f, plain)))


def test_tensors_on_the_host_are_refused():
    from korith_vllm_ext.kernels import (Rotary, int4_page_pool, read_kv_cache, rotary_embedding,
                                         write_kv_cache)

    x = torch.zeros(1, 2, 64)
    i = torch.zeros(1, dtype=torch.int64)
    cache = torch.zeros(2, 1, 16, 2, 64)
    with pytest.raises(RuntimeError, match="GPU"):
        rotary_embedding(x, x, i, Rotary(torch.ones(32, dtype=torch.float64)))
    with pytest.raises(RuntimeError, match="GPU"):
        write_kv_cache(x, x, cache, slot_mapping=i)
    with pytest.raises(RuntimeError, match="GPU"):
        read_kv_cache(cache, slot_mapping=i)
    with pytest.raises(RuntimeError, match="GPU"):
        read_kv_cache(int4_page_pool(1, 2, 64, device="cpu"), slot_mapping=i)


BOTH = [(n, c, w, d) for n in ATTEND for c, w, d in (
    (INV, "heads", dict(hq=7)), (INV, "num_seqs", dict(seqs=-1)), (INV, "n_rows", dict(rows=-1)),
    (INV, "bt_stride", dict(bt_stride=3)), (INV, "pool_pages", dict(pool=0)),
    (UNS, "head_dim", dict(dim=288)), (UNS, "rows", dict(rows=1 << 24)),
    (UNS, "block tables", dict(table=1 << 27, bt_stride=1 << 27)),
    (UNS, "dtype", dict(q_dtype=3)), (INV, "null", dict(q=None)), (INV, "null", dict(start=None)),
    (INV, "null", dict(bt=None)), (INV, "aligned", dict(out=FAKE + 1)),
    (amf_hip.ERR_WORKSPACE, "workspace", dict(ws=None)),
    (amf_hip.ERR_WORKSPACE, "workspace", dict(wsb=1000)),
    (amf_hip.ERR_WORKSPACE, "workspace", dict(ws=FAKE + 8)))]


@pytest.mark.parametrize("name,code,word,change", BOTH + [
    ("amf_paged_attn_rows", UNS, "type", dict(kv_dtype=0)),
    ("amf_paged_attn_rows", UNS, "type", dict(q_dtype=1, kv_dtype=3)),
    ("amf_paged_attn_rows", INV, "scales", dict(ks=0.0)),
    ("amf_paged_attn_rows", INV, "block_size", dict(block=0)),
    ("amf_paged_attn_rows", INV, "aligned", dict(v=FAKE + 1)),
    ("amf_int4_paged_attn_rows", UNS, "multiple", dict(dim=80)),
    ("amf_int4_paged_attn_rows", UNS, "dtype", dict(q_dtype=1)),
    ("amf_int4_paged_attn_rows", INV, "null", dict(vp=None)),
    ("amf_int4_paged_attn_rows", INV, "aligned", dict(kp=FAKE + 4)),
])
def test_attention_refused(name, code, word, change):
    with pytest.raises(amf_hip.AmfHipError) as e:
        amf_hip.call(name, *(ATTEND[name] | change).values())
    assert e.value.code == code and word in e.value.message


@pytest.mark.parametrize("name", list(ATTEND))
def test_no_rows_to_attend(name):
    amf_hip.call(name, *(ATTEND[name] | dict(rows=0)).values())
    amf_hip.call(name, *(ATTEND[name] | dict(seqs=0)).values())


def test_workspace_of_the_attention():
    f = amf_hip.load().amf_paged_attn_rows_workspace_bytes
    assert f(32, 8, 128) % 16 == 0 and f(64, 8, 256) > f(32, 8, 128) > f(32, 8, 64) > 0
    assert f(32, 8, 80) == 16 and f(7, 2, 64) == f(8, 0, 64) == f(8, 8, 300) == 0


def test_overlaps():
    """Address ranges of rows and planes, and which are refused."""
    from korith_vllm_ext.kernels import step

    x = torch.zeros(5, 6, 8, dtype=torch.bfloat16)
    what, lo, hi = step._span(x[1:, 2:4], "rows")
    assert (what, lo - x.data_ptr(), hi - lo) == ("rows", (48 + 16) * 2, (3 * 48 + 8 + 8) * 2)
    assert step._span(x[:0], "none")[1:] == (0, 0) or step._span(x[:0], "none")[1] == \
        step._span(x[:0], "none")[2]
    # planes of 3 pages of 4 tokens of 2 heads of 8 dims, pages of K and V in turn
    k, v = step._planes_spans(1000, 1128, 128, 16, 8, 3, 4, 2, 8, 2)
    assert k[1:] == (1000, 1000 + (256 + 48 + 8 + 8) * 2) and v[1] - v[2] == k[1] - k[2]
    step._apart([("a", 10, 20)], [("b", 20, 30), ("c", 0, 10), ("d", 15, 15 - 15), ("e", 0, 0)])
    step._apart([], [("b", 20, 30)])
    for lo, hi in ((0, 11), (19, 25), (12, 13), (0, 100), (10, 20)):
        with pytest.raises(ValueError, match="a must not overlap b"):
            step._apart([("z", 200, 300), ("a", 10, 20)], [("c", 0, 5), ("b", lo, hi)][lo < 5:])


def test_outputs_in_place():
    """The same elements at the same places, whatever the strides of dims of one element."""
    from korith_vllm_ext.kernels import step

    x = torch.zeros(6, 4, 64, dtype=torch.bfloat16)
    wide = torch.zeros(1, 8 * 64, dtype=torch.bfloat16)
    for like, out in ((x, x), (x, x.view(6, 4, 64)),
                      (wide[:, :256].view(1, 4, 64), wide[0, :256].view(1, 4, 64)),
                      (wide.view(1, 8, 64)[:, :4], wide[0, :256].view(1, 4, 64)),
                      (x[:1].expand(1, 4, 64), x[:1]), (x[:, 1:2], x[:, 1].unsqueeze(1)),
                      (x[:, :1], x.as_strided((6, 1, 64), (256, 7, 1)))):
        step._output(out, "out", like, ())
        with pytest.raises(ValueError, match="overlap"):
            step._output(out, "out", like, (like,))
    for like, out in ((x[:3], x[1:4]), (x[:, :2], x[:, 1:3]), (x[:1], x.view(-1)[1:257].view(1, 4, 64)),
                      (x[:, :1, :32], x.as_strided((6, 1, 32), (32, 32, 1)))):
        with pytest.raises(ValueError, match="overlap"):
            step._output(out, "out", like, ())


def test_workspace_of_a_call():
    """Grows with rows, sequences and tables up to what is enough for any; too little is refused."""
    lib = amf_hip.load()
    f, most = lib.amf_paged_attn_rows_call_bytes, lib.amf_paged_attn_rows_workspace_bytes
    for heads in ((32, 8, 128), (14, 2, 64), (4, 1, 256)):
        last = 0
        for rows, seqs, pages in ((1, 1, 1), (1, 1, 64), (8, 8, 64), (8, 8, 8192),
                                  (4096, 8, 8192), (1 << 20, 1000, 1 << 20)):
            n = f(rows, seqs, pages, 16, *heads)
            assert n % 16 == 0 and last <= n <= most(*heads)
            last = n
        # (one workgroup a CU at 256 dims, two otherwise)
        assert last == most(*heads) // (1 + heads[2] // 256)
        assert f(1, 1, 1, 16, *heads) * 16 <= last
    assert f(5, 1, 9, 16, 32, 8, 80) == 16 and f(5, 1, 9, 16, 7, 2, 64) == 0
    for odd in ((-1, 1, 1, 16), (1, -1, 1, 16), (1, 1, -1, 16), (1, 1, 1, 0), (1 << 40, 1, 1, 16),
                (1, 1, 1 << 30, 1 << 20)):
        assert f(*odd, 32, 8, 128) == most(32, 8, 128)
    for name in ATTEND:
        at = ATTEND[name]
        need = f(at["rows"], at["seqs"], at["table"], 16, at["hq"], at["hkv"], at["dim"])
        with pytest.raises(amf_hip.AmfHipError) as e:
            amf_hip.call(name, *(at | dict(wsb=need - 16)).values())
        assert e.value.code == amf_hip.ERR_WORKSPACE and str(need) in e.value.message
