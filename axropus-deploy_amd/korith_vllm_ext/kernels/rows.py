"""kernels/rows.py - causal attention of several new rows per sequence over a
paged cache or an INT4 pool: prompt chunks, drafted tokens, and single rows of
decoding sequences among them in one call.

paged_attention takes the rows as build_slot_maps numbers them (query_start) and
the block tables and lengths that it leaves (context_lens counts the new rows).
It is two launches on the current stream of its tensors' device, reads nothing
back and may be captured into a HIP graph; checks, errors and err_flag as in
kernels/paged.py.
"""

from __future__ import annotations

from typing import Optional, Union

import torch

import amf_hip

from ..codecs import CompressedKV
from .paged import (_HALVES, _KV_TAGS, _ROWS_WS, _TAGS, _cache, _flag, _int32, _launch,
                    _raw_stream, _table, _workspace)
from .step import _apart, _extent, _planes_spans, _pool, _scales, _span

_TILE_DIMS = (64, 128, 256)  # of the matrix kernel


def paged_attention(q: torch.Tensor, k_cache: Union[torch.Tensor, CompressedKV],
                    v_cache: Optional[torch.Tensor] = None, *, query_start: torch.Tensor,
                    block_tables: torch.Tensor, context_lens: torch.Tensor,
                    scale: Optional[float] = None, k_scale: float = 1.0, v_scale: float = 1.0,
                    out: Optional[torch.Tensor] = None,
                    workspace: Optional[torch.Tensor] = None,
                    err_flag: Optional[torch.Tensor] = None) -> torch.Tensor:
    """v_scale * softmax(q K^T * scale * k_scale) V of every row over the tokens
    up to its own.

    q [rows, Hq, D]: rows query_start[s] .. query_start[s + 1] - 1 are the last
    tokens of sequence s, whose context_lens[s] tokens (int32 [seqs], the new
    ones among them) lie in the cache already (write_kv_cache); query_start
    int32 [seqs + 1].  Rows and heads strided as they come (a copy where dims
    are not contiguous); D at most 256, Hq a multiple of the KV heads.
    The cache: a layer [2, pages, block, Hkv, D] or K and V planes, as
    paged_decode_attention takes it, of q's type, or FP8 with q bf16 or fp16; or
    an INT4 pool (int4_page_pool, or the int4_asym_g32 CompressedKV of a page
    tensor), attended in the values that read_kv_cache gives in q's type.
    block_tables int32 [seqs, max_pages].  A row without tokens gives zeros.
    64, 128 or 256 dims take matrix tiles where the cache's rows and out are
    16-byte aligned (q is copied where it is not); other calls and fp32 a slower
    kernel.  out: contiguous, of q's shape and type, apart from what is read,
    otherwise a new one; rows that belong to no sequence are not written."""
    pool = isinstance(k_cache, CompressedKV)
    if pool:
        if v_cache is not None and v_cache is not k_cache:
            raise ValueError("K and V come from the one page pool given as k_cache")
        layout, idx, planes = _pool(k_cache, "paged_attention")
        if idx < 0:
            amf_hip.require_device_tensor(k_cache.meta["_blob"], "page pool")
        bs, H, D, kdt = 16, layout.num_heads, layout.head_dim, None
        _scales(k_scale, v_scale, False)
    else:
        idx, kp, vp, ps, ts, hs, nb, bs, H, D = _cache(k_cache, v_cache)
        kdt = k_cache.dtype
        _scales(k_scale, v_scale, True)  # of any cache, as the decode attention has them
    if not isinstance(q, torch.Tensor):
        raise TypeError(f"q must be a tensor, got {type(q).__name__}")
    if q.dim() != 3 or q.shape[2] != D:
        raise ValueError(f"q must be [rows, heads, {D}], got {tuple(q.shape)}")
    if q.get_device() != idx:
        raise ValueError(f"q is on {q.device}, the call's tensors on device {idx}")
    qdt = q.dtype
    if qdt is not kdt and not ((pool or kdt is torch.float8_e4m3fn) and qdt in _HALVES):
        raise TypeError(f"paged attention: q is {qdt}, the cache "
                        f"{'INT4 pages' if pool else kdt}")
    N, Hq, _ = q.shape
    if Hq == 0 or Hq % H:
        raise ValueError(f"{Hq} query heads is not a multiple of {H} KV heads")
    qs, qh, one = q.stride()
    if one != 1 and D > 1:
        q = q.contiguous()
    elif D in _TILE_DIMS and qdt in _HALVES and (
            q.data_ptr() % 16 or (N > 1 and qs % 8) or (Hq > 1 and qh % 8)):
        q = q.contiguous() if not q.is_contiguous() else q.clone()  # little beside the tiles' gain
    bt, row, S, width = _table(block_tables, idx, None)
    cl = _int32(context_lens, "context_lens", idx, (S,))
    start = _int32(query_start, "query_start", idx, (S + 1,))
    if scale is None:
        scale = 0.0
    elif not 1.2e-38 < scale < 3.4e38:
        raise ValueError(f"scale must be positive, finite and normal in fp32, got {scale}")
    given = out is not None
    if not given:
        out = torch.empty((N, Hq, D), dtype=qdt, device=q.device)
    elif (not isinstance(out, torch.Tensor) or out.shape != (N, Hq, D) or out.dtype != qdt
          or out.get_device() != idx or not out.is_contiguous()):
        raise ValueError(f"out must be contiguous {(N, Hq, D)} of {qdt} on device {idx}")
    elif N and (q.data_ptr() < out.data_ptr() + out.numel() * out.element_size()
                and out.data_ptr() < q.data_ptr() + _extent(q) * q.element_size()):
        raise ValueError("paged attention: out must not lie in q")  # q is read until the end
    stream = _raw_stream(idx)
    ws, wsb = _workspace(_ROWS_WS, (N, S, width, bs, Hq, H, D), workspace, q.device, stream)
    ef = _flag(err_flag, idx)
    if given or workspace is not None:
        at, n = out.data_ptr(), out.numel() * out.element_size()
        read = [("block_tables", bt, bt + 4 * ((S - 1) * row + width) if S else bt),
                ("context_lens", cl, cl + 4 * S), ("query_start", start, start + 4 * S + 4)]
        if ef is not None:
            read.append(("err_flag", ef, ef + 4))
        read += ((("the pool", planes[0], planes[0] + layout.total_bytes),) if pool else
                 _planes_spans(kp, vp, ps, ts, hs, nb, bs, H, D, kdt.itemsize))
        _apart((("out", at, at + n),), read)
        if workspace is not None:
            wp = ws.data_ptr()
            _apart((("workspace", wp, wp + wsb),), read + [_span(q, "q"), ("out", at, at + n)])
    qs, qh, _ = q.stride()
    rows = (q.data_ptr(), _TAGS[qdt], qs if N > 1 else 0, qh if Hq > 1 else 0, out.data_ptr(), N,
            start)
    seqs = (bt, row, width, cl, S, Hq, H, D)
    end = (None if ws is None else ws.data_ptr(), wsb, ef, stream)
    if pool:
        _launch(idx, "amf_int4_paged_attn_rows", *rows, *planes, layout.n_pages, *seqs, scale, *end)
    else:
        _launch(idx, "amf_paged_attn_rows", *rows, kp, vp, _KV_TAGS[kdt], ps, ts, hs, nb, *seqs,
                bs, scale, k_scale, v_scale, *end)
    return out


__all__ = ["paged_attention"]
