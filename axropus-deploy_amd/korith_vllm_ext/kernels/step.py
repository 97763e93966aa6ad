"""kernels/step.py - the rows of a step: rotary positions, and K and V written
into and read from a paged cache or an INT4 pool.

Between build_slot_maps, which gives every new token its slot and position, and
the attention over the pages:

* rotary_embedding: queries and keys turned by their positions (half or
  interleaved pairs, whole heads or part of them); rotary_frequencies makes the
  frequencies, scaled for long contexts or not;
* write_kv_cache: keys (rotated in the same launch, as the queries may be) and
  values at their slots, quantised as they are written into an FP8 cache or an
  int4_asym_g32 page pool;
* read_kv_cache: rows back by their slots, dequantised;
* int4_page_pool: a pool to write into, empty or over a blob.

Each is one launch on the current stream of its tensors' device, reads nothing
back and may be captured into a HIP graph.  Arguments are checked on the host
(ValueError, TypeError); slots outside the pool are left out and reported in
err_flag, an int32 tensor of one element (AMF_ERRFLAG_BLOCK_RANGE).

There is no CPU path: without a GPU or libamf_hip.so these raise
amf_hip.AmfHipUnavailable / RuntimeError.
"""

from __future__ import annotations

import math
from typing import Any, NamedTuple, Optional, Sequence, Tuple, Union

import torch

import amf_hip

from .. import _paged as _layouts
from ..codecs import FMT_INT4_ASYM_G32, CompressedKV, get_codec
from .paged import _KV_TAGS, _TAGS, _cache, _flag, _launch, _raw_stream


class Rotary(NamedTuple):
    """How heads are rotated: pair i by positions * frequencies[i]."""

    frequencies: torch.Tensor  # float64 [pairs] on the device: radians per position
    interleaved: bool = False  # pairs (2i, 2i + 1) instead of (i, i + pairs)
    factor: float = 1.0        # of the rotated dims


def rotary_frequencies(rotary_dim: int, *, base: float = 10000.0, scaling: Optional[str] = None,
                       factor: float = 1.0, original_context: int = 8192,
                       low_factor: float = 1.0, high_factor: float = 4.0,
                       beta_fast: float = 32.0, beta_slow: float = 1.0,
                       pair_factors: Optional[Sequence[float]] = None,
                       attention_factor: Optional[float] = None, interleaved: bool = False,
                       device: Union[str, torch.device, None] = None) -> Rotary:
    """Frequencies base^(-2i / rotary_dim) of the first rotary_dim dims of a head
    (rotary_dim even), computed in 64 bits, for a context `factor` times the
    original by `scaling`:

    None            as they are
    "linear"        all divided by factor (positions interpolated)
    "ntk"           base * factor^(rotary_dim / (rotary_dim - 2))
    "bands"         those of more than high_factor turns in original_context stay,
                    those of less than low_factor are divided by factor, linear
                    in the turns between
    "yarn"          the same by the pair's index, between the pairs that make
                    beta_fast and beta_slow turns (Peng et al. 2023); rotated dims
                    times attention_factor, by default 0.1 ln(factor) + 1
    "pairs"         pair i divided by pair_factors[i]

    attention_factor multiplies the rotated dims of the others too, if given."""
    if rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even and positive, got {rotary_dim}")
    if not (math.isfinite(base) and base > 1.0 and math.isfinite(factor) and factor > 0.0
            and original_context > 0):
        raise ValueError(f"bad base {base}, factor {factor} or original_context "
                         f"{original_context}")
    n = rotary_dim // 2
    if scaling == "ntk":
        if rotary_dim == 2:
            raise ValueError("ntk scaling needs more than one pair")
        base *= factor ** (rotary_dim / (rotary_dim - 2))
    i = torch.arange(n, dtype=torch.float64)
    f = float(base) ** (-2.0 * i / rotary_dim)
    if scaling == "linear":
        f = f / factor
    elif scaling == "bands":
        if not 0.0 < low_factor < high_factor:
            raise ValueError(f"low_factor {low_factor} must be below high_factor {high_factor}")
        turns = original_context * f / (2.0 * math.pi)
        keep = ((turns - low_factor) / (high_factor - low_factor)).clamp(0.0, 1.0)
        f = f * keep + f / factor * (1.0 - keep)
    elif scaling == "yarn":
        def place(turns: float) -> float:  # the pair that makes so many turns
            return (rotary_dim * math.log(original_context / (turns * 2.0 * math.pi))
                    / (2.0 * math.log(base)))

        if not 0.0 < beta_slow < beta_fast:
            raise ValueError(f"beta_slow {beta_slow} must be below beta_fast {beta_fast}")
        lo = max(math.floor(place(beta_fast)), 0)
        hi = min(math.ceil(place(beta_slow)), rotary_dim - 1)
        keep = 1.0 - ((i - lo) / max(hi - lo, 1e-3)).clamp(0.0, 1.0)
        f = f * keep + f / factor * (1.0 - keep)
        if attention_factor is None:
            attention_factor = 0.1 * math.log(factor) + 1.0 if factor > 1.0 else 1.0
    elif scaling == "pairs":
        if pair_factors is None or len(pair_factors) != n:
            raise ValueError(f"pairs scaling needs {n} pair_factors")
        f = f / torch.tensor(pair_factors, dtype=torch.float64)
    elif scaling not in (None, "ntk"):
        raise ValueError(f"unknown rotary scaling {scaling!r}")
    if not torch.isfinite(f).all():
        raise ValueError("rotary frequencies are not finite")
    return Rotary(f.to(device if device is not None else "cuda"), interleaved,
                  1.0 if attention_factor is None else float(attention_factor))


# ----------------------------------------------------------------- checks --


def _rows(t: Any, what: str, idx: int, n: int, dim: int, dtype: torch.dtype,
          heads: Optional[int] = None) -> torch.Tensor:
    """t as rows [n, heads, dim] of dtype on device idx, dims contiguous (a copy
    where they are not)."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what} must be a tensor, got {type(t).__name__}")
    if t.get_device() != idx:
        raise ValueError(f"{what} is on {t.device}, the call's tensors on device {idx}")
    if t.dtype is not dtype:
        raise TypeError(f"{what} is {t.dtype}, the call's rows {dtype}")
    shape = t.shape
    if (len(shape) != 3 or shape[0] != n or shape[2] != dim or shape[1] == 0
            or (heads is not None and shape[1] != heads)):
        raise ValueError(f"{what} must be [{n}, {heads or 'heads'}, {dim}], got {tuple(shape)}")
    return t if t.stride(2) == 1 or dim == 1 else t.contiguous()


def _extent(t: torch.Tensor) -> int:
    """Elements from t's first to behind its last."""
    (n, h, d), (row, head, _) = t.shape, t.stride()
    return (n - 1) * row + (h - 1) * head + d if n else 0


def _output(t: Any, what: str, like: torch.Tensor, others: Tuple[torch.Tensor, ...]) -> None:
    """Checks an output of like's shape: elements apart, and neither in `others`
    nor in `like`, unless it is `like`."""
    if (not isinstance(t, torch.Tensor) or t.shape != like.shape or t.dtype != like.dtype
            or t.get_device() != like.get_device()):
        raise ValueError(f"{what} must be {tuple(like.shape)} of {like.dtype} on {like.device}")
    n, h, d = t.shape
    row, head, one = t.stride()
    if (one != 1 and d > 1) or not (
            ((h == 1 or head >= d) and (n <= 1 or row >= (h - 1) * head + d))
            or ((n <= 1 or row >= d) and (h == 1 or head >= (n - 1) * row + d))):
        raise ValueError(f"{what}'s dims must be contiguous and its rows and heads apart")
    es = t.element_size()
    for i, x in enumerate((like,) + others):
        if i == 0 and x.data_ptr() == t.data_ptr() and (
                x.stride() == t.stride() or all(a == b or m == 1 for a, b, m in
                                                zip(x.stride(), t.stride(), x.shape))):
            continue  # in place
        lo, hi = t.data_ptr(), t.data_ptr() + _extent(t) * es
        a, b = x.data_ptr(), x.data_ptr() + _extent(x) * x.element_size()
        if a >= hi or lo >= b:
            continue
        # slices of the same wider rows lie beside each other in each of them
        pitch = row * es
        if pitch == x.stride(0) * x.element_size() and pitch > 0 and n > 1:
            mine, its = (h - 1) * head * es + d * es, ((x.shape[1] - 1) * x.stride(1)
                                                       + x.shape[2]) * x.element_size()
            at = (a - lo) % pitch
            if at >= mine and at + its <= pitch:
                continue
        raise ValueError(f"{what} must not overlap what the call reads or writes otherwise")


Span = Tuple[str, int, int]  # what, its first byte's address, the one behind its last


def _span(t: torch.Tensor, what: str) -> Span:
    """Of rows."""
    at = t.data_ptr()
    return what, at, at + _extent(t) * t.element_size()


def _planes_spans(kp: int, vp: int, ps: int, ts: int, hs: int, nb: int, bs: int, H: int, D: int,
                  es: int) -> Tuple[Span, Span]:
    """Of a cache's planes, from _cache's addresses and strides."""
    n = ((nb - 1) * ps + (bs - 1) * ts + (H - 1) * hs + D) * es
    return ("the cache", kp, kp + n), ("the cache", vp, vp + n)


def _apart(written: Sequence[Span], others: Sequence[Span]) -> None:
    """Refuses a call of which something written lies in what it reads, or
    writes otherwise: a launch's workgroups have no order."""
    for what, lo, hi in written:
        for name, a, b in others:
            if a < hi and lo < b:
                raise ValueError(f"{what} must not overlap {name}")


def _int64(t: Any, what: str, idx: int, n: int) -> int:
    """The address of t, a contiguous int64 tensor [n] on device idx."""
    if not isinstance(t, torch.Tensor) or t.dtype is not torch.int64:
        raise TypeError(f"{what} must be an int64 tensor, got "
                        f"{getattr(t, 'dtype', type(t).__name__)}")
    if t.get_device() != idx:
        raise ValueError(f"{what} is on {t.device}, the call's tensors on device {idx}")
    if t.shape != (n,) or not t.is_contiguous():
        raise ValueError(f"{what} must be contiguous ({n},), got {tuple(t.shape)}")
    return t.data_ptr()


def _rotary(rotary: Any, positions: Any, idx: int, n: int, dim: int) -> tuple:
    """(positions, frequencies, pairs, interleaved, factor) of a call."""
    if rotary is None:
        if positions is not None:
            raise ValueError("positions come with rotary")
        return None, None, 0, 0, 1.0
    if not isinstance(rotary, Rotary):
        raise TypeError(f"rotary must be a Rotary, got {type(rotary).__name__}")
    f, interleaved, factor = rotary
    if not isinstance(f, torch.Tensor) or f.dtype is not torch.float64:
        raise TypeError("rotary frequencies must be a float64 tensor")
    if f.get_device() != idx:
        raise ValueError(f"rotary frequencies are on {f.device}, the call's tensors on device "
                         f"{idx}")
    pairs = f.numel()
    if f.dim() != 1 or not f.is_contiguous() or pairs == 0 or 2 * pairs > dim:
        raise ValueError(f"rotary frequencies {tuple(f.shape)} must be contiguous [pairs], at most "
                         f"{dim // 2} for heads of {dim}")
    if not math.isfinite(factor):
        raise ValueError(f"rotary factor must be finite, got {factor}")
    return (_int64(positions, "positions", idx, n), f.data_ptr(), pairs, int(bool(interleaved)),
            float(factor))


def _step_rows(x: Any, what: str) -> Tuple[int, int, int, int, torch.dtype]:
    """(device index, rows, heads, dim, dtype) that a step's first tensor sets."""
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{what} must be a tensor, got {type(x).__name__}")
    idx = x.get_device()
    if idx < 0:
        amf_hip.require_device_tensor(x, what)
    if x.dim() != 3 or x.dtype not in _TAGS:
        raise ValueError(f"{what} must be bf16, fp16 or fp32 [rows, heads, head_dim], got "
                         f"{x.dtype} {tuple(x.shape)}")
    n, h, d = x.shape
    if not (1 <= h and 1 <= d <= 512):
        raise ValueError(f"{what} {tuple(x.shape)}: at least one head, of 1 to 512 dims")
    if n > 1 << 25:
        raise ValueError(f"{what} has {n} rows, at most {1 << 25} a call")
    return idx, n, h, d, x.dtype


def _scales(k_scale: float, v_scale: float, fp8: bool) -> None:
    # in fp32, in which the kernels take them
    if not (1.2e-38 < k_scale < 3.4e38 and 1.2e-38 < v_scale < 3.4e38):
        raise ValueError(f"scales must be positive, finite and normal in fp32, got {k_scale}, "
                         f"{v_scale}")
    if not fp8 and (k_scale != 1.0 or v_scale != 1.0):
        raise ValueError("k_scale and v_scale are for FP8 caches")


def _pool(kv: CompressedKV, what: str) -> tuple:
    """(layout, device index, addresses of K codes, K params, V codes, V params)."""
    layout = kv.meta.get("_layout")
    if layout is None or kv.format != FMT_INT4_ASYM_G32 or layout.n_planes != 2:
        raise ValueError(f"{what} needs the int4_asym_g32 CompressedKV of a layer page tensor [2, "
                         "pool_pages, 16, kv_heads, head_dim] (int4_page_pool makes one)")
    blob = kv.meta["_blob"]
    at = blob.data_ptr()
    return layout, blob.get_device(), (at + layout.code_offset(0), at + layout.param_offset(0),
                                       at + layout.code_offset(1), at + layout.param_offset(1))


def _outside(lo: int, hi: int, rows: tuple, qs: tuple, rot: tuple, ef: Optional[int],
             q_given: bool) -> None:
    """_apart of a write's cache, at lo .. hi, from the rest of its arguments, and of a
    q_out that the caller gave (every decode step waits for this: names come last)."""
    k, k_row, k_head, v, v_row, v_head, tag, n, H, dim, slots = rows
    q, q_row, q_head, o, o_row, o_head, Hq = qs
    if not n:
        return
    es = 4 if tag == amf_hip.DTYPE_F32 else 2
    k_end = k + ((n - 1) * k_row + (H - 1) * k_head + dim) * es
    v_end = v + ((n - 1) * v_row + (H - 1) * v_head + dim) * es
    q_end = o_end = 0
    if Hq:
        q_end = q + ((n - 1) * q_row + (Hq - 1) * q_head + dim) * es
        o_end = o + ((n - 1) * o_row + (Hq - 1) * o_head + dim) * es
    pos, freqs, pairs = rot[0] or 0, rot[1] or 0, rot[2]
    s_end, p_end, f_end = slots + 8 * n, pos + 8 * n, freqs + 8 * pairs
    if not (slots < hi and lo < s_end or pos < hi and lo < p_end or freqs < hi and lo < f_end
            or k < hi and lo < k_end or v < hi and lo < v_end or ef and lo <= ef < hi
            or q_end and (q < hi and lo < q_end or o < hi and lo < o_end)
            or q_given and (slots < o_end and o < s_end or pos < o_end and o < p_end
                            or freqs < o_end and o < f_end or ef and o <= ef < o_end)):
        return
    read = [("slot_mapping", slots, s_end), ("positions", pos, p_end),
            ("the frequencies", freqs, f_end), ("err_flag", ef or 0, (ef or -4) + 4)]
    if q_given:
        _apart((("q_out", o, o_end),), read)
    read += [("k", k, k_end), ("v", v, v_end)]
    if Hq:
        read += [("q", q, q_end), ("q_out", o, o_end)]
    _apart((("the cache", lo, hi),), read)


# -------------------------------------------------------------- operators --


def rotary_embedding(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor,
                     rotary: Rotary, *,
                     out: Optional[Tuple[torch.Tensor, Optional[torch.Tensor]]] = None
                     ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """(q, k) with the first 2 * pairs dims of each head rotated by its row's
    position: (a, b) -> factor * (a cos - b sin, b cos + a sin), computed in 64
    bits, rounded to fp32 and then to the type.

    q [rows, Hq, D], k [rows, Hkv, D] or None, of one type (bf16, fp16, fp32),
    rows and heads strided as they come (a copy where dims are not contiguous);
    D at most 512.  positions int64 [rows], of either sign: the negative ones
    turn back what the positive ones turned (for factor 1).  out: tensors to
    write into, q and k themselves among them, otherwise new contiguous ones."""
    idx, n, hq, dim, dt = _step_rows(q, "q")
    qi = _rows(q, "q", idx, n, dim, dt)
    ki = None if k is None else _rows(k, "k", idx, n, dim, dt)
    if rotary is None:
        raise TypeError("rotary_embedding needs a Rotary")
    rot = _rotary(rotary, positions, idx, n, dim)
    if out is None:
        qo = torch.empty((n, hq, dim), dtype=dt, device=q.device)
        ko = None if k is None else torch.empty(k.shape, dtype=dt, device=q.device)
    else:
        qo, ko = out
        if (ko is None) != (k is None):
            raise ValueError("out holds a tensor for k where there is one")
        _output(qo, "out[0]", q, () if k is None else (k, ko))
        if k is not None:
            _output(ko, "out[1]", k, (q, qo))
        read = (("positions", rot[0], rot[0] + 8 * n),
                ("the frequencies", rot[1], rot[1] + 8 * rot[2]))
        _apart([_span(t, what) for t, what in ((qo, "out[0]"), (ko, "out[1]")) if t is not None],
               read)
    qs, os = qi.stride(), qo.stride()
    ks = (None, 0, 0, None, 0, 0, 0)
    if ki is not None:
        a, b = ki.stride(), ko.stride()
        ks = (ki.data_ptr(), a[0], a[1], ko.data_ptr(), b[0], b[1], ki.shape[1])
    _launch(idx, "amf_rotary_embedding", qi.data_ptr(), qs[0], qs[1], qo.data_ptr(), os[0], os[1],
            hq, *ks, _TAGS[dt], n, dim, *rot, _raw_stream(idx))
    return qo, ko


def int4_page_pool(num_pages: int, num_heads: int, head_dim: int, *,
                   device: Union[str, torch.device, None] = None,
                   dtype: torch.dtype = torch.bfloat16,
                   blob: Optional[torch.Tensor] = None) -> CompressedKV:
    """The int4_asym_g32 pool of a layer: num_pages pages of 16 tokens, zeros, or
    over `blob`, a contiguous uint8 tensor [K codes][V codes][K params][V params]
    (what the codec makes of a page tensor, a CompressedVRAMPool's span among
    them).  dtype is what decompress_to takes for the type of its origin."""
    if num_pages <= 0 or num_heads <= 0:
        raise ValueError(f"a pool of {num_pages} pages of {num_heads} heads")
    layout = _layouts.BlobLayout(FMT_INT4_ASYM_G32, 2, num_pages, 16, num_heads, head_dim)
    layout.validate()
    n = layout.total_bytes
    if blob is None:
        blob = torch.zeros(n, dtype=torch.uint8, device=device if device is not None else "cuda")
    elif (not isinstance(blob, torch.Tensor) or blob.dtype != torch.uint8 or blob.dim() != 1
          or blob.numel() < n or not blob.is_contiguous() or blob.data_ptr() % 16):
        raise ValueError(f"a blob of {num_pages} pages is a contiguous uint8 tensor of {n} bytes, "
                         "16-byte aligned")
    return get_codec(FMT_INT4_ASYM_G32).wrap_blob(
        blob, 0, layout, (2, num_pages, 16, num_heads, head_dim), dtype, None, num_pages * 16)


def write_kv_cache(k: torch.Tensor, v: torch.Tensor,
                   k_cache: Union[torch.Tensor, CompressedKV],
                   v_cache: Optional[torch.Tensor] = None, *, slot_mapping: torch.Tensor,
                   positions: Optional[torch.Tensor] = None, rotary: Optional[Rotary] = None,
                   q: Optional[torch.Tensor] = None, q_out: Optional[torch.Tensor] = None,
                   k_scale: float = 1.0, v_scale: float = 1.0,
                   err_flag: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Row r of k (rotated by positions[r] if `rotary` is given) and of v written
    at slot_mapping[r] of the cache; returns q rotated (into q_out, if given),
    or None without q.

    k, v [rows, Hkv, D], q [rows, Hq, D] of one type (bf16, fp16, fp32), strided
    as they come.  The cache: a layer [2, pages, block, Hkv, D] or K and V planes,
    as paged_decode_attention takes it, of that type, or FP8 (codes of x /
    k_scale and x / v_scale, clamped to +-448); or an INT4 pool
    (int4_page_pool, or the int4_asym_g32 CompressedKV of a page tensor), whose
    other tokens stay.  A rotated key is rounded to its type before it is
    quantised: the codes are those of a page saved from an unquantised cache.
    slot_mapping int64 [rows] (build_slot_maps): negative ones are left out.
    Rows of the same slot leave it any of their values, in a pool a mixture.
    What is read, and q_out, lies outside the cache: rows from it are copied
    first."""
    idx, n, H, dim, dt = _step_rows(k, "k")
    ki = _rows(k, "k", idx, n, dim, dt)
    vi = _rows(v, "v", idx, n, dim, dt, H)
    slots = _int64(slot_mapping, "slot_mapping", idx, n)
    q_given = False
    if q is None:
        if q_out is not None:
            raise ValueError("q_out comes with q")
        qs = (None, 0, 0, None, 0, 0, 0)
    else:
        if rotary is None:
            raise ValueError("q comes with rotary")
        qi = _rows(q, "q", idx, n, dim, dt)
        q_given = q_out is not None
        if not q_given:
            q_out = torch.empty(q.shape, dtype=dt, device=q.device)
        else:
            _output(q_out, "q_out", q, (k, v))
        a, b = qi.stride(), q_out.stride()
        qs = (qi.data_ptr(), a[0], a[1], q_out.data_ptr(), b[0], b[1], qi.shape[1])
    rot = _rotary(rotary, positions, idx, n, dim)
    ks, vs = ki.stride(), vi.stride()
    rows = (ki.data_ptr(), ks[0], ks[1], vi.data_ptr(), vs[0], vs[1], _TAGS[dt], n, H, dim, slots)
    ef, stream = _flag(err_flag, idx), _raw_stream(idx)
    if isinstance(k_cache, CompressedKV):
        if v_cache is not None and v_cache is not k_cache:
            raise ValueError("K and V go into the one page pool given as k_cache")
        _scales(k_scale, v_scale, False)
        layout, pidx, planes = _pool(k_cache, "write_kv_cache")
        if pidx != idx or layout.num_heads != H or layout.head_dim != dim:
            raise ValueError(f"rows of {H} heads of {dim} on device {idx} do not fit the pool: "
                             f"{layout.num_heads} of {layout.head_dim} on device {pidx}")
        _outside(planes[0], planes[0] + layout.total_bytes, rows, qs, rot, ef, q_given)
        _launch(idx, "amf_int4_kv_write", *rows, *planes, layout.n_pages, *rot, *qs, ef, stream)
        return q_out
    cidx, kp, vp, ps, ts, hs, nb, bs, ch, cd = _cache(k_cache, v_cache)
    if kp == vp:
        raise ValueError("write_kv_cache needs a V plane of its own")
    kdt = k_cache.dtype
    if cidx != idx or ch != H or cd != dim:
        raise ValueError(f"rows of {H} heads of {dim} on device {idx} do not fit the cache: {ch} "
                         f"of {cd} on device {cidx}")
    if kdt is not dt and kdt is not torch.float8_e4m3fn:
        raise TypeError(f"write_kv_cache: rows are {dt}, the cache {kdt}")
    _scales(k_scale, v_scale, kdt is torch.float8_e4m3fn)
    size = ((nb - 1) * ps + (bs - 1) * ts + (ch - 1) * hs + cd) * kdt.itemsize
    if kp <= vp <= kp + size or vp <= kp <= vp + size:
        _outside(min(kp, vp), max(kp, vp) + size, rows, qs, rot, ef, q_given)
    else:
        _outside(kp, kp + size, rows, qs, rot, ef, q_given)
        _outside(vp, vp + size, rows, qs, rot, ef, False)
    _launch(idx, "amf_kv_write", *rows, kp, vp, _KV_TAGS[kdt], ps, ts, hs, nb, bs, k_scale,
            v_scale, *rot, *qs, ef, stream)
    return q_out


def read_kv_cache(k_cache: Union[torch.Tensor, CompressedKV],
                  v_cache: Optional[torch.Tensor] = None, *, slot_mapping: torch.Tensor,
                  dtype: Optional[torch.dtype] = None, k_scale: float = 1.0,
                  v_scale: float = 1.0,
                  out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None,
                  err_flag: Optional[torch.Tensor] = None
                  ) -> Tuple[torch.Tensor, torch.Tensor]:
    """(K, V) rows [rows, Hkv, D] of the slots of a cache or an INT4 pool (as
    write_kv_cache takes them): as they are, or of an FP8 cache code * scale, of a
    pool u * s + z, in fp32 and rounded to dtype (bf16, fp16, fp32; by default bf16,
    a cache's own type where it is not FP8).  Rows of negative slots, and of
    slots outside the pool, become zeros.  out: tensors to write into, outside
    the cache."""
    pool = isinstance(k_cache, CompressedKV)
    if pool:
        if v_cache is not None and v_cache is not k_cache:
            raise ValueError("K and V come from the one page pool given as k_cache")
        layout, idx, planes = _pool(k_cache, "read_kv_cache")
        if idx < 0:
            amf_hip.require_device_tensor(k_cache.meta["_blob"], "page pool")
        H, dim, own = layout.num_heads, layout.head_dim, None
        _scales(k_scale, v_scale, False)
    else:
        idx, kp, vp, ps, ts, hs, nb, bs, H, dim = _cache(k_cache, v_cache)
        own = None if k_cache.dtype is torch.float8_e4m3fn else k_cache.dtype
        _scales(k_scale, v_scale, own is None)
        if dim > 512:
            raise ValueError(f"heads of {dim} dims: at most 512")
    if not isinstance(slot_mapping, torch.Tensor) or slot_mapping.dim() != 1:
        raise ValueError("slot_mapping must be an int64 tensor [rows]")
    n = slot_mapping.shape[0]
    slots = _int64(slot_mapping, "slot_mapping", idx, n)
    if n > 1 << 25:
        raise ValueError(f"{n} rows, at most {1 << 25} a call")
    dt = dtype or (out[0].dtype if out is not None else own or torch.bfloat16)
    if dt not in _TAGS or (own is not None and dt is not own):
        raise TypeError(f"read_kv_cache: rows of {dt} from a cache of "
                        f"{'INT4 pages' if pool else k_cache.dtype}")
    ef = _flag(err_flag, idx)
    if out is None:
        ko = torch.empty((n, H, dim), dtype=dt, device=slot_mapping.device)
        vo = torch.empty_like(ko)
    else:
        ko, vo = out
        for t, what in ((ko, "out[0]"), (vo, "out[1]")):
            if (not isinstance(t, torch.Tensor) or t.shape != (n, H, dim) or t.dtype != dt
                    or t.get_device() != idx):
                raise ValueError(f"{what} must be {(n, H, dim)} of {dt} on device {idx}")
        _output(ko, "out[0]", ko, (vo,))
        _output(vo, "out[1]", vo, ())
        read = [("slot_mapping", slots, slots + 8 * n)]
        if ef is not None:
            read.append(("err_flag", ef, ef + 4))
        read += ((("the pool", planes[0], planes[0] + layout.total_bytes),) if pool else
                 _planes_spans(kp, vp, ps, ts, hs, nb, bs, H, dim, k_cache.dtype.itemsize))
        _apart((_span(ko, "out[0]"), _span(vo, "out[1]")), read)
    a, b = ko.stride(), vo.stride()
    rows = (slots, ko.data_ptr(), a[0], a[1], vo.data_ptr(), b[0], b[1], _TAGS[dt], n, H, dim, ef,
            _raw_stream(idx))
    if pool:
        _launch(idx, "amf_int4_kv_read", *planes, layout.n_pages, *rows)
    else:
        _launch(idx, "amf_kv_read", kp, vp, _KV_TAGS[k_cache.dtype], ps, ts, hs, nb, bs, k_scale,
                v_scale, *rows)
    return ko, vo


__all__ = [
    "Rotary",
    "int4_page_pool",
    "read_kv_cache",
    "rotary_embedding",
    "rotary_frequencies",
    "write_kv_cache",
]
