"""kernels/paged.py - a decode step over vLLM's own paged K/V cache.

The pages a restored prefix lands in are read where they are, in the cache's
element type (bf16, fp16, fp32, FP8 e4m3) and page order:

* build_slot_maps: block tables grown from a free list, and the slot, position
  and row of every new token, from lengths on the device (the host form, per
  request, is AMFReqMeta.make);
* paged_decode_attention: attention of one new token per sequence;
* page_key_bounds, select_pages: the smallest and largest key of each page, and
  the pages whose bounds allow a query the largest scores; with
  paged_decode_attention(pages=...) a long context is read in part.

Each is one or two launches on the current stream of its tensors' device, reads
nothing back and may be captured into a HIP graph.  Arguments are checked on
the host (ValueError, TypeError); what only the device knows (page ids, lengths
that a block table does not hold) is skipped there and reported in err_flag, an
int32 tensor of one element that the AMF_ERRFLAG_* bits are ORed into.

There is no CPU path: without a GPU or libamf_hip.so these raise
amf_hip.AmfHipUnavailable / RuntimeError.
"""

from __future__ import annotations

import math
import threading
from collections import OrderedDict
from typing import Any, NamedTuple, Optional, Tuple

import torch

import amf_hip

_TAGS = {torch.float16: amf_hip.DTYPE_F16, torch.float32: amf_hip.DTYPE_F32,
         torch.bfloat16: amf_hip.DTYPE_BF16}
_KV_TAGS = {**_TAGS, torch.float8_e4m3fn: amf_hip.DTYPE_E4M3}
_HALVES = (torch.bfloat16, torch.float16)
_I32 = torch.int32
_I32_MAX = 0x7FFFFFFF
_ATTN_WS, _SELECT_WS = "amf_paged_decode_workspace_bytes", "amf_select_pages_workspace_bytes"
_WS: dict = {_ATTN_WS: {}, _SELECT_WS: {}}  # entry point -> {sizes: workspace bytes}

# The checks below run on every call of a decode step, where the host's time is
# what a small batch waits for: they compare in place and leave the words of an
# error to a slow path.


_current_device = getattr(torch._C, "_cuda_getDevice", None)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _launch(idx: int, func: str, *args) -> None:
    """A status-returning entry point with device idx, which holds the tensors,
    as the current one (the null stream and the launch belong to it)."""
    fn = amf_hip.entry(func)
    if _current_device() == idx:
        rc = fn(*args)
    else:
        with torch.cuda.device(idx):
            rc = fn(*args)
    if rc:
        amf_hip.check(func, rc)


# Scratch kept between calls, one buffer per (device, stream, host thread): a call
# is two launches, and another thread's may come between them on the same stream.
# The least recently used is dropped, those of threads that ended among them.
# A stream under graph capture gets a buffer of its own per call instead.
_SCRATCH: "OrderedDict[Tuple[int, int, int], torch.Tensor]" = OrderedDict()
_SCRATCH_MAX = 16
_SCRATCH_LOCK = threading.Lock()


def _scratch(dev: torch.device, stream: int, nbytes: int) -> torch.Tensor:
    idx = dev.index
    if _current_device() == idx:
        capturing = torch.cuda.is_current_stream_capturing()
    else:  # torch answers for the current device's stream, not that of the launch
        with torch.cuda.device(idx):
            capturing = torch.cuda.is_current_stream_capturing()
    if capturing:
        return torch.empty(nbytes, dtype=torch.uint8, device=dev)
    key = (idx, stream, threading.get_ident())
    buf = _SCRATCH.get(key)
    if buf is not None and buf.numel() >= nbytes:
        try:
            _SCRATCH.move_to_end(key)  # one step under the interpreter's lock
        except KeyError:
            pass  # another thread's call has just dropped it
        return buf
    buf = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    with _SCRATCH_LOCK:
        _SCRATCH[key] = buf
        _SCRATCH.move_to_end(key)
        while len(_SCRATCH) > _SCRATCH_MAX:  # a call under way keeps its buffer itself
            _SCRATCH.popitem(last=False)
    return buf


def _workspace(name: str, sizes: tuple, given: Optional[torch.Tensor], dev: torch.device,
               stream: int) -> Tuple[Optional[torch.Tensor], int]:
    """(workspace, its bytes): the caller's, checked, or the scratch buffer of
    this device and stream (a new one under graph capture)."""
    known = _WS[name]
    need = known.get(sizes)
    if need is None:
        if len(known) > 4096:
            known.clear()
        need = known[sizes] = int(getattr(amf_hip.load(), name)(*sizes))
    if given is not None:
        _dispatch._check_buffer(given, "workspace", dev)
        have = given.numel() * given.element_size()
        if have < need:
            raise ValueError(f"workspace of {have} bytes, {need} needed")
        return given, have
    return (_scratch(dev, stream, need), need) if need else (None, 0)


def _cache(k: torch.Tensor, v: Optional[torch.Tensor], keys: bool = False) -> tuple:
    """(device index, K address, V address, strides of page, token and head,
    pages, block, heads, dim) of a layer [2, pages, block, heads, dim] (v
    None), or of K and V planes [pages, block, heads, dim] with the same
    strides; `keys`: a K plane alone will do.  The last dim is contiguous, the
    others may be strided."""
    if not isinstance(k, torch.Tensor):
        raise TypeError(f"a K/V cache is a tensor, got {type(k).__name__}")
    idx = k.get_device()
    if idx < 0:
        amf_hip.require_device_tensor(k, "paged cache")
    shape, st = k.shape, k.stride()
    kp = vp = k.data_ptr()
    if v is None and len(shape) == 5:
        planes, nb, bs, H, D = shape
        plane, ps, ts, hs, ds = st
        if planes != 2:
            raise ValueError(f"a layer's cache is [2, pages, block, heads, dim], got {tuple(shape)}")
        vp = kp + plane * k.element_size()
    elif len(shape) != 4:
        raise ValueError(f"K/V cache of shape {tuple(shape)}: expected [2, pages, block, heads, "
                         "dim], or planes [pages, block, heads, dim]")
    else:
        nb, bs, H, D = shape
        ps, ts, hs, ds = st
        if v is not None and v is not k:
            if (not isinstance(v, torch.Tensor) or v.shape != shape
                    or (v.stride() != st and any(a != b and n > 1 for a, b, n in
                                                 zip(v.stride(), st, shape)))):
                raise ValueError("K and V planes differ in shape or strides")
            if v.dtype != k.dtype or v.device != k.device:
                raise ValueError("K and V planes differ in type or device")
            vp = v.data_ptr()
        elif v is None and not keys:
            raise ValueError("a K plane comes with the V plane (v_cache=k_cache where it holds "
                             "both)")
    if k.dtype not in _KV_TAGS:
        raise TypeError(f"paged cache of {k.dtype}: bf16, fp16, fp32 or float8_e4m3fn")
    if ds != 1 and D != 1:
        raise ValueError("the cache's last dim must be contiguous")
    if not (nb and bs and H and D):
        raise ValueError(f"empty K/V cache {tuple(shape)}")
    if H == 1 or bs == 1 or nb == 1:  # strides that are never used, whatever their alignment
        ps, ts, hs = ps * (nb > 1), ts * (bs > 1), hs * (H > 1)
    return idx, kp, vp, ps, ts, hs, nb, bs, H, D


def _int32(t: Any, what: str, idx: int, shape: tuple) -> int:
    """The address of t, which has to be a contiguous int32 tensor of `shape` on
    device idx."""
    if (isinstance(t, torch.Tensor) and t.dtype is _I32 and t.get_device() == idx
            and t.shape == shape and t.is_contiguous()):
        return t.data_ptr()
    if not isinstance(t, torch.Tensor) or t.dtype != _I32:
        raise TypeError(f"{what} must be an int32 tensor, got "
                        f"{getattr(t, 'dtype', type(t).__name__)}")
    if t.get_device() != idx:
        raise ValueError(f"{what} is on {t.device}, the call's tensors on device {idx}")
    raise ValueError(f"{what} must be contiguous {tuple(shape)}, got {tuple(t.shape)}")


def _table(t: Any, idx: int, seqs: Optional[int]) -> Tuple[int, int, int, int]:
    """(address, row stride, sequences, pages of a row) of a block table: int32
    [seqs, pages] on device idx, rows contiguous and apart."""
    if not isinstance(t, torch.Tensor) or t.dtype is not _I32:
        raise TypeError(f"block_tables must be an int32 tensor, got "
                        f"{getattr(t, 'dtype', type(t).__name__)}")
    if t.get_device() != idx:
        raise ValueError(f"block_tables is on {t.device}, the call's tensors on device {idx}")
    shape = t.shape
    if len(shape) != 2 or (seqs is not None and shape[0] != seqs):
        raise ValueError(f"block_tables {tuple(shape)} does not match {seqs} sequences")
    S, n = shape
    row, one = t.stride()
    if (n > 1 and one != 1) or (S > 1 and row < n):
        raise ValueError("block_tables rows must be contiguous and apart")
    return t.data_ptr(), row if row > n else n, S, n


def _flag(err_flag: Optional[torch.Tensor], idx: int) -> Optional[int]:
    return None if err_flag is None else _int32(err_flag, "err_flag", idx, (1,))


def _query(q: Any, idx: int, dim: int) -> torch.Tensor:
    """q as [seqs, heads, dim] on device idx with contiguous, 16-byte aligned
    heads (a copy where they are not)."""
    if not isinstance(q, torch.Tensor):
        raise TypeError(f"q must be a tensor, got {type(q).__name__}")
    if q.dim() == 4:
        if q.shape[2] != 1:
            raise ValueError("paged decode takes one query token per sequence")
        q = q.select(2, 0)
    if q.dim() != 3 or q.shape[2] != dim:
        raise ValueError(f"q must be [seqs, heads, {dim}] or [seqs, heads, 1, {dim}], got "
                         f"{tuple(q.shape)}")
    if q.get_device() != idx:
        raise ValueError(f"q is on {q.device}, the call's tensors on device {idx}")
    if not q.is_contiguous():
        st, n = q.stride(), 16 // q.element_size()
        if st[2] != 1 or st[0] % n or st[1] % n or q.data_ptr() % 16:
            q = q.contiguous()
    if q.data_ptr() % 16:
        q = q.clone()
    return q


def paged_decode_attention(q: torch.Tensor, k_cache: torch.Tensor,
                           v_cache: Optional[torch.Tensor] = None, *,
                           block_tables: torch.Tensor, context_lens: torch.Tensor,
                           scale: Optional[float] = None, max_context_len: Optional[int] = None,
                           pages: Optional[torch.Tensor] = None,
                           page_counts: Optional[torch.Tensor] = None, k_scale: float = 1.0,
                           v_scale: float = 1.0, out: Optional[torch.Tensor] = None,
                           out_dtype: Optional[torch.dtype] = None,
                           workspace: Optional[torch.Tensor] = None,
                           err_flag: Optional[torch.Tensor] = None) -> torch.Tensor:
    """v_scale * softmax(q K^T * scale * k_scale) V over each sequence's pages.

    q [seqs, Hq, D] or [seqs, Hq, 1, D]; k_cache a layer [2, pages, block, Hkv,
    D], or the K plane [pages, block, Hkv, D] with v_cache the V plane of the
    same strides (any order of block and heads; k_cache itself, if one plane
    holds both); D at most 256, Hq a multiple of Hkv.  q has the cache's type,
    with an FP8 cache bf16 or fp16 (one kept as uint8 is given as
    k_cache.view(torch.float8_e4m3fn)).  16-byte aligned rows and out, and D a
    multiple of 16, take matrix tiles; other calls and fp32 a slower kernel.
    block_tables int32 [seqs, max_pages], context_lens int32 [seqs] (tokens in
    the cache, the new one among them); a sequence without tokens gives zeros.
    max_context_len, where the caller knows one, helps to cut the work.  pages
    int32 [seqs, Hkv, n] with page_counts int32 [seqs, Hkv] limits each KV head
    to the listed places of the block table (select_pages makes them).  out:
    contiguous, q's shape; otherwise one of out_dtype (q's type)."""
    idx, kp, vp, ps, ts, hs, nb, bs, H, D = _cache(k_cache, v_cache)
    q3 = _query(q, idx, D)
    S, Hq, _ = q3.shape
    kdt, qdt = k_cache.dtype, q3.dtype
    if qdt is not kdt and not (kdt is torch.float8_e4m3fn and qdt in _HALVES):
        raise TypeError(f"paged decode: q is {qdt}, the cache {kdt}")
    if Hq == 0 or Hq % H:
        raise ValueError(f"{Hq} query heads is not a multiple of {H} KV heads")
    bt, row, _, width = _table(block_tables, idx, S)
    cl = _int32(context_lens, "context_lens", idx, (S,))
    if scale is None:
        scale = 0.0
    elif not 1.2e-38 < scale < math.inf:
        raise ValueError(f"scale must be positive, finite and normal in fp32, got {scale}")
    pg = pc = None
    max_pages = 0
    if pages is not None:
        if page_counts is None:
            raise ValueError("pages and page_counts come together")
        if not isinstance(pages, torch.Tensor) or pages.dim() != 3:
            raise ValueError("pages must be an int32 tensor [seqs, KV heads, n]")
        max_pages = pages.shape[2]
        pg = _int32(pages, "pages", idx, (S, H, max_pages))
        pc = _int32(page_counts, "page_counts", idx, (S, H))
        pg = pg or pc  # lists without room hold nothing (an empty tensor has no address)
    elif page_counts is not None:
        raise ValueError("pages and page_counts come together")
    most = width * bs if max_context_len is None else int(max_context_len)
    dev = q.device
    if out is None:
        if out_dtype is None and q.is_contiguous():
            out = torch.empty_like(q)
        else:
            out = torch.empty(q.shape, dtype=out_dtype or qdt, device=dev)
    else:
        _dispatch._check_buffer(out, "out", dev)
        if out.shape != q.shape and tuple(out.shape) != (S, Hq, D):
            raise ValueError(f"paged decode: out has shape {tuple(out.shape)}, q {tuple(q.shape)}")
        if out_dtype is not None and out.dtype != out_dtype:
            raise ValueError(f"paged decode: out is {out.dtype}, out_dtype asks for {out_dtype}")
        if S > 0:  # q is read until the end
            st, at = q3.stride(), q3.data_ptr()
            end = at + ((S - 1) * st[0] + (Hq - 1) * st[1] + D) * q3.element_size()
            if at < out.data_ptr() + out.numel() * out.element_size() and out.data_ptr() < end:
                raise ValueError("paged decode: out must not lie in q")
    if out.dtype not in _TAGS:
        raise ValueError(f"paged decode: output dtype {out.dtype} is not bf16/fp16/fp32")
    stream = _raw_stream(idx)
    ws, wsb = _workspace(_ATTN_WS, (Hq, H, D), workspace, dev, stream)
    qs, qh, _ = q3.stride()
    _launch(
        idx, "amf_paged_decode_attn", q3.data_ptr(), _TAGS[qdt], qs, qh, out.data_ptr(),
        _TAGS[out.dtype], kp, vp, _KV_TAGS[kdt], ps, ts, hs, nb, bt, row, width, cl, pg, pc,
        max_pages, S, Hq, H, D, bs, most if most < _I32_MAX else _I32_MAX, scale, k_scale, v_scale,
        None if ws is None else ws.data_ptr(), wsb, _flag(err_flag, idx), stream)
    return out


def page_key_bounds(k_cache: torch.Tensor, block_tables: torch.Tensor,
                    context_lens: torch.Tensor, *, first_tokens: Optional[torch.Tensor] = None,
                    max_new_tokens: Optional[int] = None, bounds: Optional[torch.Tensor] = None,
                    dtype: Optional[torch.dtype] = None,
                    err_flag: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The smallest and largest key of each page, per KV head and channel.

    k_cache a layer's cache or its K plane (as paged_decode_attention; 16-bit
    or FP8, D a multiple of 8).  Written are the pages of each sequence, or
    only those from token first_tokens[s] (int32 [seqs]) on: after a step,
    first_tokens holds the lengths before it and max_new_tokens, if given, the
    most tokens that a sequence got (it sizes the grid: no sequence may have
    got more).  bounds [pages, Hkv, 2, D] of the cache's type (FP8: dtype, bf16
    by default) is updated in place, or made (zeros where nothing is written).
    Sequences that share a page have to use as many tokens of it, as those do
    that share a prefix in whole pages; else the bounds are either's.
    Returns bounds."""
    idx, kp, _, ps, ts, hs, nb, bs, H, D = _cache(k_cache, None, True)
    kdt = k_cache.dtype
    if kdt is torch.float32 or D % 8 or D > 256:
        raise ValueError(f"page bounds need a bf16, fp16 or FP8 cache with head_dim a multiple of "
                         f"8 up to 256, got {kdt}, {D}")
    bt, row, S, width = _table(block_tables, idx, None)
    cl = _int32(context_lens, "context_lens", idx, (S,))
    ft = None if first_tokens is None else _int32(first_tokens, "first_tokens", idx, (S,))
    if max_new_tokens is None:
        max_new_tokens = 0
    elif max_new_tokens <= 0 or ft is None:
        raise ValueError("max_new_tokens is positive and comes with first_tokens")
    if kdt is torch.float8_e4m3fn:
        bdt = dtype or (torch.bfloat16 if bounds is None else bounds.dtype)
    else:
        bdt = dtype or kdt
        if bdt != kdt:
            raise ValueError(f"bounds of a {kdt} cache have its type, not {bdt}")
    if bdt not in _HALVES:
        raise ValueError(f"page bounds are bf16 or fp16, not {bdt}")
    shape = (nb, H, 2, D)
    if bounds is None:
        bounds = torch.zeros(shape, dtype=bdt, device=k_cache.device)
    elif (not isinstance(bounds, torch.Tensor) or bounds.shape != shape or bounds.dtype != bdt
          or bounds.get_device() != idx or not bounds.is_contiguous()):
        raise ValueError(f"bounds must be contiguous {shape} of {bdt} on device {idx}")
    _launch(
        idx, "amf_page_key_bounds", kp, _KV_TAGS[kdt], ps, ts, hs, nb, bt, row, width, cl, ft,
        min(int(max_new_tokens), _I32_MAX), S, H, D, bs, bounds.data_ptr(), _TAGS[bdt],
        _flag(err_flag, idx), _raw_stream(idx))
    return bounds


def select_pages(q: torch.Tensor, bounds: torch.Tensor, block_tables: torch.Tensor,
                 context_lens: torch.Tensor, *, block_size: int, num_pages: int,
                 first_pages: int = 1, last_pages: int = 1,
                 max_context_len: Optional[int] = None,
                 out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None,
                 workspace: Optional[torch.Tensor] = None,
                 err_flag: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The num_pages pages of each (sequence, KV head) whose key bounds allow
    the largest score max_h sum_d max(q_d lo_d, q_d hi_d) over its query heads;
    the first first_pages and last last_pages always among them, the lower page
    first among equal scores (summed in 64 bits).

    q [seqs, Hq, D] of the bounds' type; bounds [pages, Hkv, 2, D] from
    page_key_bounds.  Returns (pages int32 [seqs, Hkv, num_pages], places in
    the block table in ascending order and -1 behind the last; counts int32
    [seqs, Hkv]), written into `out` if given.  max_context_len bounds the
    context lengths (default: what the block table holds) and sizes the
    workspace."""
    if not isinstance(bounds, torch.Tensor) or bounds.dim() != 4 or bounds.shape[2] != 2:
        raise ValueError("bounds must be [pages, KV heads, 2, head_dim]")
    idx = bounds.get_device()
    if idx < 0:
        amf_hip.require_device_tensor(bounds, "page bounds")
    dt = bounds.dtype
    if dt not in _HALVES or not bounds.is_contiguous():
        raise ValueError(f"bounds must be contiguous bf16 or fp16, got {dt}")
    nb, H, _, D = bounds.shape
    q3 = _query(q, idx, D)
    S, Hq, _ = q3.shape
    if q3.dtype is not dt:
        raise TypeError(f"select_pages: q is {q3.dtype}, the bounds {dt}")
    if Hq == 0 or Hq % H:
        raise ValueError(f"{Hq} query heads is not a multiple of {H} KV heads")
    bt, row, _, width = _table(block_tables, idx, S)
    cl = _int32(context_lens, "context_lens", idx, (S,))
    if num_pages <= 0 or first_pages < 0 or last_pages < 0 or first_pages + last_pages > num_pages:
        raise ValueError(f"num_pages {num_pages} has to hold first_pages {first_pages} and "
                         f"last_pages {last_pages}")
    if not 0 < block_size <= _I32_MAX:
        raise ValueError(f"block_size must be positive and an int32, got {block_size}")
    most = width * block_size if max_context_len is None else int(max_context_len)
    if most < 0:
        raise ValueError(f"max_context_len must not be negative, got {max_context_len}")
    most = min(most, _I32_MAX)
    dev = bounds.device
    if out is None:
        pages = context_lens.new_empty((S, H, num_pages))
        counts = pages.new_empty((S, H))
        pg, pc = pages.data_ptr(), counts.data_ptr()
    else:
        pages, counts = out
        pg = _int32(pages, "pages", idx, (S, H, num_pages))
        pc = _int32(counts, "page counts", idx, (S, H))
    stream = _raw_stream(idx)
    ws, wsb = _workspace(_SELECT_WS, (S, H, width, block_size, most), workspace, dev, stream)
    qs, qh, _ = q3.stride()
    _launch(
        idx, "amf_select_pages", q3.data_ptr(), _TAGS[dt], qs, qh, bounds.data_ptr(), nb, bt, row,
        width, cl, most, S, Hq, H, D, block_size, num_pages, first_pages, last_pages, pg, pc,
        None if ws is None else ws.data_ptr(), wsb, _flag(err_flag, idx), stream)
    return pages, counts


class SlotMaps(NamedTuple):
    """What build_slot_maps gives a step (device tensors)."""

    slot_mapping: torch.Tensor  # int64 [num_tokens]: page id * block_size + place, -1 = none
    positions: torch.Tensor     # int64 [num_tokens]: place in the sequence
    query_start: torch.Tensor   # int32 [seqs + 1]: first row of each sequence, then all rows
    context_lens: torch.Tensor  # int32 [seqs]: tokens after the step
    free_used: torch.Tensor     # int32 [1]: entries of the free list in use after the step


def build_slot_maps(context_lens: torch.Tensor, new_tokens: torch.Tensor,
                    block_tables: torch.Tensor, *, block_size: int, num_tokens: int,
                    free_pages: Optional[torch.Tensor] = None,
                    free_used: Optional[torch.Tensor] = None,
                    pool_pages: Optional[int] = None, out: Optional[SlotMaps] = None,
                    err_flag: Optional[torch.Tensor] = None) -> SlotMaps:
    """Block tables and slots of a step in which sequence s, with
    context_lens[s] tokens in the cache, gets new_tokens[s] more.

    context_lens, new_tokens int32 [seqs]; block_tables int32 [seqs,
    max_pages], extended in place with pages free_pages[free_used:] (int32
    [n], int32 [1]) in sequence order; out: buffers to write into, apart from
    each other and from what is read; num_tokens: rows of the step's buffers,
    at least the new tokens (rows behind the last one get slot -1, position
    0).  Without free_pages no sequence gets a page: new tokens have room only
    in the pages that context_lens reaches already.  The slots go to
    amf_kv_scatter_slots (or an engine's own cache write) as they are.

    A sequence whose pages the free list or its table row does not hold, or
    whose tokens the rows do not, keeps its length and gets slots of -1
    (AMF_ERRFLAG_FREE_LIST / _CONTEXT in err_flag); so do tokens of page ids
    outside [0, pool_pages) (_BLOCK_RANGE), whose sequence grows, with an entry
    of -1 where the free list held such an id."""
    if not isinstance(block_tables, torch.Tensor):
        raise TypeError("block_tables must be an int32 tensor")
    idx = block_tables.get_device()
    if idx < 0:
        amf_hip.require_device_tensor(block_tables, "block_tables")
    bt, row, S, width = _table(block_tables, idx, None)
    cl = _int32(context_lens, "context_lens", idx, (S,))
    nt = _int32(new_tokens, "new_tokens", idx, (S,))
    if not 0 < block_size <= _I32_MAX or num_tokens < 0:
        raise ValueError(f"bad block_size {block_size} or num_tokens {num_tokens}")
    if pool_pages is None:
        pool_pages = _I32_MAX
    elif pool_pages <= 0:
        raise ValueError(f"pool_pages must be positive, got {pool_pages}")
    n_free, fp = 0, None
    if free_pages is not None:
        if not isinstance(free_pages, torch.Tensor) or free_pages.dim() != 1:
            raise ValueError("free_pages must be an int32 tensor [n]")
        n_free = free_pages.shape[0]
        fp = _int32(free_pages, "free_pages", idx, (n_free,))
    fu = None if free_used is None else _int32(free_used, "free_used", idx, (1,))
    ef = _flag(err_flag, idx)
    if out is None:
        dev = block_tables.device
        slots = torch.empty(num_tokens, dtype=torch.int64, device=dev)
        pos = torch.empty_like(slots)
        start, lens, used = new_tokens.new_empty(2 * S + 2).split_with_sizes((S + 1, S, 1))
        out = SlotMaps(slots, pos, start, lens, used)
        ptrs = (slots.data_ptr(), pos.data_ptr(), start.data_ptr(), lens.data_ptr(),
                used.data_ptr())
    else:
        for t, name in ((out.slot_mapping, "slot_mapping"), (out.positions, "positions")):
            if (t.dtype != torch.int64 or t.get_device() != idx or t.shape != (num_tokens,)
                    or not t.is_contiguous()):
                raise ValueError(f"out.{name} must be contiguous int64 ({num_tokens},) on "
                                 f"device {idx}")
        ptrs = (out.slot_mapping.data_ptr(), out.positions.data_ptr(),
                _int32(out.query_start, "out.query_start", idx, (S + 1,)),
                _int32(out.context_lens, "out.context_lens", idx, (S,)),
                _int32(out.free_used, "out.free_used", idx, (1,)))
        given = [(p, p + 8 * num_tokens) for p in ptrs[:2]]
        given += [(p, p + 4 * n) for p, n in zip(ptrs[2:], (S + 1, S, 1))]
        taken = {"context_lens": (cl, 4 * S), "new_tokens": (nt, 4 * S),
                 "free_used": (fu or 0, 4), "free_pages": (fp or 0, 4 * n_free),
                 "block_tables": (bt, 4 * ((S - 1) * row + width)),
                 "err_flag": (ef or 0, 4)}
        for i, (lo, hi) in enumerate(given):  # the launch's workgroups have no order
            for name, (at, n) in taken.items():
                if at < hi and lo < at + n and n > 0:
                    raise ValueError(f"{name} must not overlap out.{SlotMaps._fields[i]}")
            if any(a < hi and lo < b for a, b in given[:i]):
                raise ValueError(f"out.{SlotMaps._fields[i]} must not overlap another output")
    _launch(
        idx, "amf_build_slot_maps", cl, nt, S, bt, row, width, block_size, pool_pages,
        fp if n_free else None, n_free, fu, num_tokens, *ptrs, ef, _raw_stream(idx))
    return out


__all__ = [
    "SlotMaps",
    "build_slot_maps",
    "page_key_bounds",
    "paged_decode_attention",
    "select_pages",
]

from . import dispatch as _dispatch  # noqa: E402  (it imports this module's attention)
