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

from typing import Any, NamedTuple, Optional, Tuple

import torch

import amf_hip

_KV_TAGS = {torch.float16: amf_hip.DTYPE_F16, torch.float32: amf_hip.DTYPE_F32,
            torch.bfloat16: amf_hip.DTYPE_BF16, torch.float8_e4m3fn: amf_hip.DTYPE_E4M3}
_HALVES = (torch.bfloat16, torch.float16)
_I32_MAX = 0x7FFFFFFF
_WS: dict = {}  # (entry point, sizes) -> workspace bytes


def _workspace(name: str, sizes: tuple, given: Optional[torch.Tensor], dev: torch.device,
               stream: int) -> Tuple[Optional[torch.Tensor], int]:
    """(workspace, its bytes): the caller's, checked, or the scratch buffer of
    this device and stream (a new one under graph capture)."""
    from .dispatch import _check_buffer, _scratch

    key = (name, sizes)
    need = _WS.get(key)
    if need is None:
        if len(_WS) > 4096:
            _WS.clear()
        need = _WS[key] = int(getattr(amf_hip.load(), name)(*sizes))
    if given is not None:
        _check_buffer(given, "workspace", dev)
        have = given.numel() * given.element_size()
        if have < need:
            raise ValueError(f"workspace of {have} bytes, {need} needed")
        return given, have
    return (_scratch(dev, stream, need), need) if need else (None, 0)


class _Cache(NamedTuple):
    """K and V of a layer as the C ABI takes them (strides in elements)."""

    k: int
    v: int
    strides: Tuple[int, int, int]
    pages: int
    block: int
    heads: int
    dim: int
    dtype: torch.dtype
    device: torch.device


def _cache(k: torch.Tensor, v: Optional[torch.Tensor]) -> _Cache:
    """A layer [2, pages, block, heads, dim] (v None), or K and V planes
    [pages, block, heads, dim] with the same strides; a plane alone holds both.
    The last dim is contiguous, the others may be strided."""
    if not isinstance(k, torch.Tensor):
        raise TypeError(f"a K/V cache is a tensor, got {type(k).__name__}")
    amf_hip.require_device_tensor(k, "paged cache")
    shape, st = k.shape, k.stride()
    kp = vp = k.data_ptr()
    if v is None and len(shape) == 5:
        if shape[0] != 2:
            raise ValueError(f"a layer's cache is [2, pages, block, heads, dim], got {tuple(shape)}")
        vp = kp + st[0] * k.element_size()
        shape, st = shape[1:], st[1:]
    elif len(shape) != 4:
        raise ValueError(f"K/V cache of shape {tuple(shape)}: expected [2, pages, block, heads, "
                         "dim], or planes [pages, block, heads, dim]")
    elif v is not None and v is not k:
        if not isinstance(v, torch.Tensor) or v.shape != shape or v.stride() != st:
            raise ValueError("K and V planes differ in shape or strides")
        if v.dtype != k.dtype or v.device != k.device:
            raise ValueError("K and V planes differ in type or device")
        vp = v.data_ptr()
    if k.dtype not in _KV_TAGS:
        raise TypeError(f"paged cache of {k.dtype}: bf16, fp16, fp32 or float8_e4m3fn")
    nb, bs, H, D = shape
    if st[3] != 1 and D != 1:
        raise ValueError("the cache's last dim must be contiguous")
    if nb == 0 or bs == 0 or H == 0 or D == 0:
        raise ValueError(f"empty K/V cache {tuple(shape)}")
    return _Cache(kp, vp, (st[0], st[1], st[2]), nb, bs, H, D, k.dtype, k.device)


def _int32(t: Any, what: str, dev: torch.device, shape: tuple) -> torch.Tensor:
    """t, checked to be a contiguous int32 tensor of `shape` on dev."""
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32:
        raise TypeError(f"{what} must be an int32 tensor, got "
                        f"{getattr(t, 'dtype', type(t).__name__)}")
    if t.device != dev:
        raise ValueError(f"{what} is on {t.device}, the call's tensors on {dev}")
    if tuple(t.shape) != shape or not t.is_contiguous():
        raise ValueError(f"{what} must be contiguous {shape}, got {tuple(t.shape)}")
    return t


def _table(t: Any, dev: torch.device, seqs: Optional[int]) -> torch.Tensor:
    """A block table: int32 [seqs, pages] on dev, rows contiguous."""
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32:
        raise TypeError(f"block_tables must be an int32 tensor, got "
                        f"{getattr(t, 'dtype', type(t).__name__)}")
    if t.device != dev:
        raise ValueError(f"block_tables is on {t.device}, the call's tensors on {dev}")
    if t.dim() != 2 or (seqs is not None and t.shape[0] != seqs):
        raise ValueError(f"block_tables {tuple(t.shape)} does not match {seqs} sequences")
    if (t.shape[1] > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < t.shape[1]):
        raise ValueError("block_tables rows must be contiguous and apart")
    return t


def _row_stride(t: torch.Tensor) -> int:
    return max(t.stride(0), t.shape[1])


def _flag(err_flag: Optional[torch.Tensor], dev: torch.device) -> Optional[int]:
    return None if err_flag is None else _int32(err_flag, "err_flag", dev, (1,)).data_ptr()


def _query(q: Any, dev: torch.device, dim: int) -> torch.Tensor:
    """q as [seqs, heads, dim] on dev with contiguous, 16-byte aligned heads (a
    copy where they are not)."""
    if not isinstance(q, torch.Tensor):
        raise TypeError(f"q must be a tensor, got {type(q).__name__}")
    if q.dim() == 4:
        if q.shape[2] != 1:
            raise ValueError("paged decode takes one query token per sequence")
        q = q.select(2, 0)
    if q.dim() != 3 or q.shape[2] != dim:
        raise ValueError(f"q must be [seqs, heads, {dim}] or [seqs, heads, 1, {dim}], got "
                         f"{tuple(q.shape)}")
    if q.device != dev:
        raise ValueError(f"q is on {q.device}, the cache on {dev}")
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
    same strides (any order of block and heads); D at most 256, Hq a multiple
    of Hkv.  q has the cache's type, with an FP8 cache bf16 or fp16.
    block_tables int32 [seqs, max_pages], context_lens int32 [seqs] (tokens in
    the cache, the new one among them); a sequence without tokens gives zeros.
    max_context_len, where the caller knows one, helps to cut the work.  pages
    int32 [seqs, Hkv, n] with page_counts int32 [seqs, Hkv] limits each KV head
    to the listed places of the block table (select_pages makes them).  out:
    contiguous, q's shape; otherwise one of out_dtype (q's type)."""
    c = _cache(k_cache, v_cache)
    dev = c.device
    q3 = _query(q, dev, c.dim)
    S, Hq, D = q3.shape
    if q3.dtype != c.dtype and not (c.dtype == torch.float8_e4m3fn and q3.dtype in _HALVES):
        raise TypeError(f"paged decode: q is {q3.dtype}, the cache {c.dtype}")
    if Hq == 0 or Hq % c.heads:
        raise ValueError(f"{Hq} query heads is not a multiple of {c.heads} KV heads")
    bt = _table(block_tables, dev, S)
    cl = _int32(context_lens, "context_lens", dev, (S,))
    if scale is not None and not scale > 0.0:
        raise ValueError(f"scale must be positive, got {scale}")
    if (pages is None) != (page_counts is None):
        raise ValueError("pages and page_counts come together")
    max_pages = 0
    if pages is not None:
        if not isinstance(pages, torch.Tensor) or pages.dim() != 3:
            raise ValueError("pages must be an int32 tensor [seqs, KV heads, n]")
        max_pages = pages.shape[2]
        _int32(pages, "pages", dev, (S, c.heads, max_pages))
        _int32(page_counts, "page_counts", dev, (S, c.heads))
    if max_context_len is None:
        max_context_len = bt.shape[1] * c.block
    if out is None:
        out = torch.empty(q.shape, dtype=out_dtype or q3.dtype, device=dev)
    else:
        from .dispatch import _check_buffer

        _check_buffer(out, "out", dev)
        if out.shape != q.shape and tuple(out.shape) != (S, Hq, D):
            raise ValueError(f"paged decode: out has shape {tuple(out.shape)}, q {tuple(q.shape)}")
        if out_dtype is not None and out.dtype != out_dtype:
            raise ValueError(f"paged decode: out is {out.dtype}, out_dtype asks for {out_dtype}")
    stream = amf_hip.stream_handle(dev)
    ws, wsb = _workspace("amf_paged_decode_workspace_bytes", (Hq, c.heads, D), workspace, dev,
                         stream)
    qs = q3.stride()
    amf_hip.call_on(
        dev, "amf_paged_decode_attn", q3.data_ptr(), amf_hip.dtype_tag(q3.dtype), qs[0], qs[1],
        out.data_ptr(), amf_hip.dtype_tag(out.dtype), c.k, c.v, _KV_TAGS[c.dtype], *c.strides,
        c.pages, bt.data_ptr(), _row_stride(bt), bt.shape[1], cl.data_ptr(),
        None if pages is None else pages.data_ptr(),
        None if pages is None else page_counts.data_ptr(), max_pages, S, Hq, c.heads, D, c.block,
        min(int(max_context_len), _I32_MAX), 0.0 if scale is None else float(scale),
        float(k_scale), float(v_scale), None if ws is None else ws.data_ptr(), wsb,
        _flag(err_flag, dev), stream)
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
    Returns bounds."""
    c = _cache(k_cache, None)
    dev = c.device
    if c.dtype not in _KV_TAGS or c.dtype == torch.float32 or c.dim % 8 or c.dim > 256:
        raise ValueError(f"page bounds need a bf16, fp16 or FP8 cache with head_dim a multiple of "
                         f"8 up to 256, got {c.dtype}, {c.dim}")
    bt = _table(block_tables, dev, None)
    S = bt.shape[0]
    cl = _int32(context_lens, "context_lens", dev, (S,))
    ft = None
    if first_tokens is not None:
        ft = _int32(first_tokens, "first_tokens", dev, (S,)).data_ptr()
    if max_new_tokens is not None and (max_new_tokens <= 0 or ft is None):
        raise ValueError("max_new_tokens is positive and comes with first_tokens")
    if c.dtype == torch.float8_e4m3fn:
        bdt = dtype or (torch.bfloat16 if bounds is None else bounds.dtype)
    else:
        bdt = dtype or c.dtype
        if bdt != c.dtype:
            raise ValueError(f"bounds of a {c.dtype} cache have its type, not {bdt}")
    if bdt not in _HALVES:
        raise ValueError(f"page bounds are bf16 or fp16, not {bdt}")
    shape = (c.pages, c.heads, 2, c.dim)
    if bounds is None:
        bounds = torch.zeros(shape, dtype=bdt, device=dev)
    elif (not isinstance(bounds, torch.Tensor) or tuple(bounds.shape) != shape
          or bounds.dtype != bdt or bounds.device != dev or not bounds.is_contiguous()):
        raise ValueError(f"bounds must be contiguous {shape} of {bdt} on {dev}")
    amf_hip.call_on(
        dev, "amf_page_key_bounds", c.k, _KV_TAGS[c.dtype], *c.strides, c.pages, bt.data_ptr(),
        _row_stride(bt), bt.shape[1], cl.data_ptr(), ft,
        min(int(max_new_tokens or 0), _I32_MAX), S, c.heads, c.dim, c.block, bounds.data_ptr(),
        amf_hip.dtype_tag(bdt), _flag(err_flag, dev), amf_hip.stream_handle(dev))
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
    amf_hip.require_device_tensor(bounds, "page bounds")
    if bounds.dtype not in _HALVES or not bounds.is_contiguous():
        raise ValueError(f"bounds must be contiguous bf16 or fp16, got {bounds.dtype}")
    dev = bounds.device
    nb, H, _, D = bounds.shape
    q3 = _query(q, dev, D)
    S, Hq, _ = q3.shape
    if q3.dtype != bounds.dtype:
        raise TypeError(f"select_pages: q is {q3.dtype}, the bounds {bounds.dtype}")
    if Hq == 0 or Hq % H:
        raise ValueError(f"{Hq} query heads is not a multiple of {H} KV heads")
    bt = _table(block_tables, dev, S)
    cl = _int32(context_lens, "context_lens", dev, (S,))
    if num_pages <= 0 or first_pages < 0 or last_pages < 0 or first_pages + last_pages > num_pages:
        raise ValueError(f"num_pages {num_pages} has to hold first_pages {first_pages} and "
                         f"last_pages {last_pages}")
    if block_size <= 0:
        raise ValueError(f"block_size must be positive, got {block_size}")
    if max_context_len is None:
        max_context_len = bt.shape[1] * block_size
    elif max_context_len < 0:
        raise ValueError(f"max_context_len must not be negative, got {max_context_len}")
    max_context_len = min(int(max_context_len), _I32_MAX)
    if out is None:
        pages = torch.empty((S, H, num_pages), dtype=torch.int32, device=dev)
        counts = torch.empty((S, H), dtype=torch.int32, device=dev)
    else:
        pages = _int32(out[0], "pages", dev, (S, H, num_pages))
        counts = _int32(out[1], "page counts", dev, (S, H))
    stream = amf_hip.stream_handle(dev)
    ws, wsb = _workspace("amf_select_pages_workspace_bytes",
                         (S, H, bt.shape[1], block_size, max_context_len), workspace, dev, stream)
    qs = q3.stride()
    amf_hip.call_on(
        dev, "amf_select_pages", q3.data_ptr(), amf_hip.dtype_tag(q3.dtype), qs[0], qs[1],
        bounds.data_ptr(), nb, bt.data_ptr(), _row_stride(bt), bt.shape[1], cl.data_ptr(),
        max_context_len, S, Hq, H, D, block_size, num_pages, first_pages, last_pages,
        pages.data_ptr(), counts.data_ptr(), None if ws is None else ws.data_ptr(), wsb,
        _flag(err_flag, dev), stream)
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
    [n], int32 [1]) in sequence order; num_tokens: rows of the step's buffers,
    at least the new tokens (rows behind the last one get slot -1, position
    0).  Without free_pages the tables must hold the new tokens' pages
    already.  The slots go to amf_kv_scatter_slots (or an engine's own cache
    write) as they are.

    A sequence whose pages the free list or its table row does not hold keeps
    its length and gets slots of -1 (AMF_ERRFLAG_FREE_LIST / _CONTEXT in
    err_flag), as do page ids outside [0, pool_pages)."""
    if not isinstance(block_tables, torch.Tensor):
        raise TypeError("block_tables must be an int32 tensor")
    amf_hip.require_device_tensor(block_tables, "block_tables")
    dev = block_tables.device
    bt = _table(block_tables, dev, None)
    S = bt.shape[0]
    cl = _int32(context_lens, "context_lens", dev, (S,))
    nt = _int32(new_tokens, "new_tokens", dev, (S,))
    if block_size <= 0 or num_tokens < 0:
        raise ValueError(f"bad block_size {block_size} or num_tokens {num_tokens}")
    if pool_pages is not None and pool_pages <= 0:
        raise ValueError(f"pool_pages must be positive, got {pool_pages}")
    n_free = 0
    if free_pages is not None:
        if not isinstance(free_pages, torch.Tensor) or free_pages.dim() != 1:
            raise ValueError("free_pages must be an int32 tensor [n]")
        n_free = free_pages.shape[0]
        _int32(free_pages, "free_pages", dev, (n_free,))
    if free_used is not None:
        _int32(free_used, "free_used", dev, (1,))
    if out is None:
        wide = torch.empty((2, num_tokens), dtype=torch.int64, device=dev)
        out = SlotMaps(wide[0], wide[1], torch.empty(S + 1, dtype=torch.int32, device=dev),
                       torch.empty(S, dtype=torch.int32, device=dev),
                       torch.empty(1, dtype=torch.int32, device=dev))
    else:
        for t, name in ((out.slot_mapping, "slot_mapping"), (out.positions, "positions")):
            if (t.dtype != torch.int64 or t.device != dev or tuple(t.shape) != (num_tokens,)
                    or not t.is_contiguous()):
                raise ValueError(f"out.{name} must be contiguous int64 ({num_tokens},) on {dev}")
        _int32(out.query_start, "out.query_start", dev, (S + 1,))
        _int32(out.context_lens, "out.context_lens", dev, (S,))
        _int32(out.free_used, "out.free_used", dev, (1,))
        for t, name in ((cl, "context_lens"), (nt, "new_tokens"), (free_used, "free_used")):
            if t is not None and any(t.numel() and t.data_ptr() == o.data_ptr() for o in out):
                raise ValueError(f"{name} must not be one of the outputs")
    amf_hip.call_on(
        dev, "amf_build_slot_maps", cl.data_ptr(), nt.data_ptr(), S, bt.data_ptr(),
        _row_stride(bt), bt.shape[1], block_size, _I32_MAX if pool_pages is None else pool_pages,
        free_pages.data_ptr() if n_free else None, n_free,
        None if free_used is None else free_used.data_ptr(), num_tokens,
        out.slot_mapping.data_ptr(), out.positions.data_ptr(), out.query_start.data_ptr(),
        out.context_lens.data_ptr(), out.free_used.data_ptr(), _flag(err_flag, dev),
        amf_hip.stream_handle(dev))
    return out


__all__ = [
    "SlotMaps",
    "build_slot_maps",
    "page_key_bounds",
    "paged_decode_attention",
    "select_pages",
]
