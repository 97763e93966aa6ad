"""Argument checks of the paged operators' C entry points, on the CPU: every
call fails validation (or has nothing to do) before any HIP call."""

from __future__ import annotations

import pytest
import torch

import amf_hip

FAKE = 1 << 20  # never dereferenced

pytestmark = pytest.mark.skipif(torch.cuda.is_available(),
                                reason="argument-validation calls run on the CPU only")

ATTN = dict(q=FAKE, q_dtype=2, q_seq=1024, q_head=128, out=FAKE, out_dtype=2, k=FAKE, v=FAKE,
            kv_dtype=2, page=4096, token=256, head=128, pool=8, bt=FAKE, bt_stride=4, table=4,
            cl=FAKE, pages=None, counts=None, max_pages=0, seqs=1, hq=8, hkv=2, dim=128, block=16,
            max_ctx=64, scale=0.0, ks=1.0, vs=1.0, ws=FAKE, wsb=1 << 30, err=None, stream=None)
BOUNDS = dict(k=FAKE, dtype=2, page=4096, token=256, head=128, pool=8, bt=FAKE, bt_stride=4,
              table=4, cl=FAKE, first=None, new=0, seqs=1, hkv=2, dim=128, block=16, bounds=FAKE,
              bdt=2, err=None, stream=None)
SELECT = dict(q=FAKE, dtype=2, q_seq=1024, q_head=128, bounds=FAKE, pool=8, bt=FAKE, bt_stride=4,
              table=4, cl=FAKE, max_ctx=64, seqs=1, hq=8, hkv=2, dim=128, block=16, keep=2,
              first=1, last=1, pages=FAKE, counts=FAKE, ws=FAKE, wsb=1 << 20, err=None,
              stream=None)
SLOTS = dict(cl=FAKE, new=FAKE, seqs=1, bt=FAKE, bt_stride=4, table=4, block=16, pool=8,
             free=FAKE, n_free=3, used=None, tokens=4, slots=FAKE, pos=FAKE, start=FAKE,
             out=FAKE, used_out=None, err=None, stream=None)
CALLS = {"amf_paged_decode_attn": ATTN, "amf_page_key_bounds": BOUNDS, "amf_select_pages": SELECT,
         "amf_build_slot_maps": SLOTS}
INV, UNS, WSP = (amf_hip.ERR_INVALID_ARG, amf_hip.ERR_UNSUPPORTED, amf_hip.ERR_WORKSPACE)


@pytest.mark.parametrize("name,code,word,change", [
    ("amf_paged_decode_attn", INV, "multiple", dict(hq=7)),
    ("amf_paged_decode_attn", INV, "num_seqs", dict(seqs=-1)),
    ("amf_paged_decode_attn", INV, "block_size", dict(block=0)),
    ("amf_paged_decode_attn", INV, "bt_stride", dict(bt_stride=3)),
    ("amf_paged_decode_attn", INV, "pool_pages", dict(pool=0)),
    ("amf_paged_decode_attn", UNS, "head_dim", dict(dim=257)),
    ("amf_paged_decode_attn", UNS, "dtype", dict(kv_dtype=4)),
    ("amf_paged_decode_attn", INV, "type", dict(q_dtype=0)),
    ("amf_paged_decode_attn", INV, "type", dict(q_dtype=1, kv_dtype=3)),
    ("amf_paged_decode_attn", INV, "type", dict(out_dtype=3)),
    ("amf_paged_decode_attn", INV, "null", dict(k=None)),
    ("amf_paged_decode_attn", INV, "null", dict(bt=None)),
    ("amf_paged_decode_attn", INV, "null", dict(pages=FAKE, max_pages=2)),
    ("amf_paged_decode_attn", INV, "aligned", dict(v=FAKE + 1)),
    ("amf_paged_decode_attn", WSP, "workspace", dict(ws=None)),
    ("amf_paged_decode_attn", WSP, "workspace", dict(wsb=64)),
    ("amf_page_key_bounds", UNS, "fp32", dict(dtype=1, bdt=1)),
    ("amf_page_key_bounds", UNS, "head_dim", dict(dim=12)),
    ("amf_page_key_bounds", UNS, "sequences", dict(seqs=70000)),
    ("amf_page_key_bounds", INV, "bounds", dict(bdt=0)),
    ("amf_page_key_bounds", INV, "bounds", dict(dtype=3, bdt=1)),
    ("amf_page_key_bounds", INV, "max_new_tokens", dict(new=-1)),
    ("amf_page_key_bounds", INV, "null", dict(bounds=None)),
    ("amf_page_key_bounds", INV, "alignment", dict(token=260)),
    ("amf_page_key_bounds", INV, "alignment", dict(k=FAKE + 8)),
    ("amf_select_pages", INV, "multiple", dict(hq=3)),
    ("amf_select_pages", INV, "first_pages", dict(first=2, last=1)),
    ("amf_select_pages", INV, "num_pages", dict(keep=0, first=0, last=0)),
    ("amf_select_pages", UNS, "dtype", dict(dtype=1)),
    ("amf_select_pages", UNS, "head_dim", dict(dim=264)),
    ("amf_select_pages", INV, "alignment", dict(q_head=100)),
    ("amf_select_pages", INV, "null", dict(counts=None)),
    ("amf_select_pages", WSP, "workspace", dict(ws=None)),
    ("amf_select_pages", WSP, "workspace", dict(wsb=63)),
    ("amf_build_slot_maps", INV, "num_tokens", dict(tokens=-1)),
    ("amf_build_slot_maps", INV, "num_seqs", dict(seqs=-1)),
    ("amf_build_slot_maps", INV, "n_free", dict(n_free=1 << 31)),
    ("amf_build_slot_maps", INV, "block_size", dict(block=0)),
    ("amf_build_slot_maps", INV, "bt_stride", dict(bt_stride=2)),
    ("amf_build_slot_maps", INV, "null", dict(start=None)),
    ("amf_build_slot_maps", INV, "null", dict(free=None)),
    ("amf_build_slot_maps", INV, "null", dict(slots=None)),
])
def test_refused(name, code, word, change):
    with pytest.raises(amf_hip.AmfHipError) as e:
        amf_hip.call(name, *(CALLS[name] | change).values())
    assert e.value.code == code and word in e.value.message


def test_nothing_to_do():
    amf_hip.call("amf_paged_decode_attn", *(ATTN | dict(seqs=0, q=None, ws=None)).values())
    amf_hip.call("amf_page_key_bounds", *(BOUNDS | dict(seqs=0)).values())
    amf_hip.call("amf_page_key_bounds", *(BOUNDS | dict(table=0)).values())
    amf_hip.call("amf_select_pages", *(SELECT | dict(seqs=0)).values())


def test_workspace_sizes():
    lib = amf_hip.load()
    f = lib.amf_paged_decode_workspace_bytes
    assert f(32, 8, 128) % 16 == 0 and f(32, 8, 128) > 0
    assert f(64, 8, 256) >= f(64, 8, 128) >= f(8, 8, 128) > 0
    assert f(7, 2, 128) == f(8, 0, 128) == f(8, 8, 300) == 0
    g = lib.amf_select_pages_workspace_bytes
    assert g(4, 2, 100, 16, 1600) == 4 * 2 * 100 * 8 == g(4, 2, 100, 16, 1 << 30)
    assert g(4, 2, 100, 16, 17) == 4 * 2 * 2 * 8
    assert g(0, 2, 100, 16, 17) == g(4, 2, 0, 16, 17) == g(4, 2, 100, 16, 0) == 0


def test_dispatch_takes_an_error_flag_with_a_cache_only():
    """Over an INT4 pool or dense K/V nothing would be written to it."""
    from korith_vllm_ext.kernels import hip_decode_attention

    q = torch.zeros(1, 4, 1, 64, dtype=torch.bfloat16)
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="err_flag"):
        hip_decode_attention(q, object(), block_tables=i[None], context_lens=i, err_flag=i)
    with pytest.raises(ValueError, match="err_flag"):
        hip_decode_attention(q, q, q, err_flag=i)


@pytest.fixture
def scratch(monkeypatch):
    """kernels.paged with an empty store of CPU scratch buffers, nothing captured."""
    from collections import OrderedDict

    from korith_vllm_ext.kernels import paged

    monkeypatch.setattr(paged, "_SCRATCH", OrderedDict())
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(paged, "_current_device", lambda: None)  # a CPU tensor's index
    return paged


def test_scratch_keeps_the_buffers_in_use(scratch):
    """More streams than buffers are kept for: the busy one's stays."""
    dev = torch.device("cpu")
    busy = scratch._scratch(dev, 0, 64)
    for stream in range(1, 3 * scratch._SCRATCH_MAX):
        scratch._scratch(dev, stream, 64)
        assert scratch._scratch(dev, 0, 64) is busy
        assert len(scratch._SCRATCH) <= scratch._SCRATCH_MAX
    assert scratch._scratch(dev, 0, 65) is not busy


@pytest.mark.parametrize("current,captured,kept", [(0, None, True), (0, 0, True), (0, 1, False),
                                                   (1, 0, True), (1, 1, False)])
def test_scratch_under_capture_is_of_the_tensors_device(scratch, monkeypatch, current, captured,
                                                        kept):
    """A buffer is kept between calls unless the stream of device 1, which
    holds the tensors, is captured, whichever device is current."""
    now = [current]

    class Guard:
        def __init__(self, idx):
            self.idx = idx

        def __enter__(self):
            self.before, now[0] = now[0], self.idx

        def __exit__(self, *_):
            now[0] = self.before

    class Device:
        index = 1

    empty = torch.empty
    monkeypatch.setattr(scratch, "_current_device", lambda: now[0])
    monkeypatch.setattr(torch.cuda, "device", Guard)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: now[0] == captured)
    monkeypatch.setattr(torch, "empty", lambda n, dtype, device: empty(n, dtype=dtype))
    bufs = [scratch._scratch(Device(), 5, 64) for _ in range(2)]
    assert (bufs[0] is bufs[1]) == kept and now[0] == current


def test_python_calls_need_the_gpu():
    """CPU tensors are turned away before anything is launched."""
    from korith_vllm_ext import kernels

    kv = torch.zeros(2, 4, 16, 2, 64, dtype=torch.bfloat16)
    bt = torch.zeros(1, 2, dtype=torch.int32)
    cl = torch.ones(1, dtype=torch.int32)
    q = torch.zeros(1, 4, 64, dtype=torch.bfloat16)
    for call in (
        lambda: kernels.paged_decode_attention(q, kv, block_tables=bt, context_lens=cl),
        lambda: kernels.page_key_bounds(kv, bt, cl),
        lambda: kernels.select_pages(q, torch.zeros(4, 2, 2, 64, dtype=torch.bfloat16), bt, cl,
                                     block_size=16, num_pages=2),
        lambda: kernels.build_slot_maps(cl, cl, bt, block_size=16, num_tokens=1),
    ):
        with pytest.raises(RuntimeError, match="GPU"):
            call()
