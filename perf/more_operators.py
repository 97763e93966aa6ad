"""A serving step's own K and V in a quantised paged cache, as cases to be timed.

  rotate  rotary positions of queries and keys (rotary_embedding): half and
          interleaved pairs, whole heads or part of them, scaled frequencies
  store   keys rotated and, with the values, written at their slots into an FP8
          cache (write_kv_cache, which rotates the queries in the same call)
  store4  the same into an INT4 page pool, and the rows read back from it
          (write_kv_cache, read_kv_cache)
  load    rows of whole contexts read back by their slots (read_kv_cache), of
          FP8 caches and INT4 pools
  attend  several new rows per sequence, causal, over the pages of its block
          table (paged_attention): 16-bit and FP8 caches and INT4 pools

`own` chooses between the package's operators and their plain form.  An INT4
pool is the int4_asym_g32 blob of a layer: K codes, V codes, K params, V params.
"""

import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32,
          "fp8": torch.float8_e4m3fn}
# query heads, KV heads, head_dim of one attention layer
HEADS = [(32, 8, 128), (64, 8, 128), (8, 1, 128), (8, 8, 128), (14, 2, 64), (8, 2, 64),
         (16, 2, 256)]
# FP8 scales of K and V: fp32 values that are no powers of two
K_SCALE, V_SCALE = 0.017578125, 0.0234375


def listed():
    return [
        # a decode step of a few sequences with long contexts: nothing but latency
        {"name": "rotate_24_step", "kind": "rotate", "seqs": 24, "rows_lo": 1, "rows_hi": 1,
         "ctx_lo": 900, "ctx_hi": 131072, "q_heads": 32, "kv_heads": 8, "dim": 128, "rot": 128,
         "pairs": "half", "scaling": "bands", "dtype": "bf16"},
        # prompts of a model that rotates a quarter of its heads, neighbours paired
        {"name": "rotate_7_part_fp16", "kind": "rotate", "seqs": 7, "rows_lo": 1001,
         "rows_hi": 2003, "ctx_lo": 1001, "ctx_hi": 9000, "q_heads": 16, "kv_heads": 2,
         "dim": 256, "rot": 64, "pairs": "interleaved", "scaling": "none", "dtype": "fp16"},
        # a decode step of a busy server into its FP8 cache
        {"name": "store_64_step_fp8", "kind": "store", "seqs": 64, "rows_lo": 1, "rows_hi": 1,
         "ctx_lo": 3, "ctx_hi": 900, "q_heads": 32, "kv_heads": 8, "dim": 128, "rot": 128,
         "pairs": "half", "scaling": "bands", "dtype": "bf16", "block": 16},
        # prompts of a long-context model, 8 query heads a KV head
        {"name": "store_8_prompts_fp8", "kind": "store", "seqs": 8, "rows_lo": 700,
         "rows_hi": 2049, "ctx_lo": 700, "ctx_hi": 4100, "q_heads": 64, "kv_heads": 8,
         "dim": 128, "rot": 128, "pairs": "half", "scaling": "yarn", "dtype": "bf16",
         "block": 16},
        # a decode step into an INT4 pool, pages partly filled
        {"name": "store4_40_step", "kind": "store4", "seqs": 40, "rows_lo": 1, "rows_hi": 1,
         "ctx_lo": 1, "ctx_hi": 3001, "q_heads": 32, "kv_heads": 8, "dim": 128, "rot": 128,
         "pairs": "half", "scaling": "bands", "dtype": "bf16", "block": 16},
        # prompt chunks into an INT4 pool, which begin and end inside pages
        {"name": "store4_3_chunks", "kind": "store4", "seqs": 3, "rows_lo": 1500,
         "rows_hi": 3001, "ctx_lo": 1777, "ctx_hi": 6003, "q_heads": 32, "kv_heads": 8,
         "dim": 128, "rot": 128, "pairs": "half", "scaling": "none", "dtype": "bf16",
         "block": 16},
        # FP8 contexts back in 16 bits, 32-token head-major pages
        {"name": "load_5_fp8", "kind": "load", "seqs": 5, "ctx_lo": 501, "ctx_hi": 9001,
         "kv_heads": 8, "dim": 128, "dtype": "fp16", "cache": "fp8", "block": 32,
         "order": "htd"},
        # two long contexts of an INT4 pool back in 16 bits
        {"name": "load_2_int4", "kind": "load", "seqs": 2, "ctx_lo": 20000, "ctx_hi": 32768,
         "kv_heads": 8, "dim": 128, "dtype": "bf16", "cache": "int4", "block": 16},
        # four drafted tokens and the last one checked over INT4 contexts
        {"name": "attend_32_drafts_int4", "kind": "attend", "seqs": 32, "rows_lo": 5,
         "rows_hi": 5, "ctx_lo": 1024, "ctx_hi": 16384, "singles": 0, "q_heads": 32,
         "kv_heads": 8, "dim": 128, "dtype": "bf16", "cache": "int4", "block": 16},
        # decoding sequences beside one prompt chunk, in one launch
        {"name": "attend_48_and_chunk", "kind": "attend", "seqs": 1, "rows_lo": 2048,
         "rows_hi": 2048, "ctx_lo": 8192, "ctx_hi": 8192, "singles": 48, "q_heads": 32,
         "kv_heads": 8, "dim": 128, "dtype": "bf16", "cache": "bf16", "block": 16},
        # a small model's prompts, odd lengths, FP8 cache in head-major pages
        {"name": "attend_6_small_fp8", "kind": "attend", "seqs": 6, "rows_lo": 33,
         "rows_hi": 1201, "ctx_lo": 400, "ctx_hi": 2999, "singles": 0, "q_heads": 14,
         "kv_heads": 2, "dim": 64, "dtype": "fp16", "cache": "fp8", "block": 16,
         "order": "htd"},
        # a whole long prompt
        {"name": "attend_1_prompt", "kind": "attend", "seqs": 1, "rows_lo": 12000,
         "rows_hi": 12000, "ctx_lo": 12000, "ctx_hi": 12000, "singles": 0, "q_heads": 32,
         "kv_heads": 8, "dim": 128, "dtype": "bf16", "cache": "bf16", "block": 16},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["rotate", "store", "store4", "load", "attend", "attend", "attend"])
    hq, hkv, dim = rng.choice(HEADS)
    c = {"kind": kind, "q_heads": hq, "kv_heads": hkv, "dim": dim}
    if kind in ("rotate", "store", "store4"):
        seqs = _log(rng, 1, 200)
        rows = 1 if rng.random() < 0.4 else _log(rng, 1, max(1, 20000 // seqs))
        hi = _log(rng, rows, max(rows, 40000 // seqs, 600))
        c |= {"seqs": seqs, "rows_lo": rng.randint((rows + 1) // 2, rows), "rows_hi": rows,
              "ctx_lo": rng.randint(1, hi), "ctx_hi": hi,
              "rot": rng.choice([dim, dim, dim // 2, dim // 4]),
              "pairs": rng.choice(["half", "half", "interleaved"]),
              "scaling": rng.choice(["none", "bands", "yarn"]),
              "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]), "block": 16}
        if kind == "store":
            c["block"] = rng.choice([16, 16, 32, 64])
        return c
    c["cache"] = rng.choice(["fp8", "int4"] if kind == "load" else ["bf16", "fp16", "fp8", "int4"])
    c["dtype"] = c["cache"] if c["cache"] in ("bf16", "fp16") else rng.choice(["bf16", "fp16"])
    c["block"] = 16 if c["cache"] == "int4" else rng.choice([16, 16, 32])
    c["order"] = "thd" if c["cache"] == "int4" else rng.choice(["thd", "htd"])
    if kind == "load":
        seqs = _log(rng, 1, 64)
        hi = _log(rng, 1, max(1, (1 << 26) // (seqs * hkv * dim)))
        return c | {"seqs": seqs, "ctx_lo": rng.randint(1, hi), "ctx_hi": hi}
    # the plain form's padded scores and the attention's products stay below the largest listed
    rows = rng.choice([_log(rng, 1, 16), _log(rng, 16, 4000)])
    seqs = _log(rng, 1, max(1, min(64, 4000 // rows)))
    hi = _log(rng, rows, max(rows, min(32768, (1 << 38) // (seqs * rows * hq * dim),
                                      (1 << 28) // (seqs * hkv * dim))))
    return c | {"seqs": seqs, "rows_lo": rng.randint((rows + 1) // 2, rows), "rows_hi": rows,
                "ctx_lo": rng.randint(max(1, hi // 8), hi), "ctx_hi": hi,
                "singles": rng.choice([0, 0, rng.randint(1, 40)]) if hi < 8192 else 0}


# ---------------------------------------------------------------- inputs --


def _even(n, lo, hi):
    """n lengths spread evenly over lo .. hi."""
    x = torch.linspace(lo, hi, n, dtype=torch.float64).round().long()
    if n == 1:
        x[0] = hi
    return x


def _lengths(case):
    """(rows, contexts) of a case's sequences, single rows first."""
    rows = _even(case["seqs"], case["rows_lo"], case["rows_hi"])
    ctx = torch.maximum(_even(case["seqs"], case["ctx_lo"], case["ctx_hi"]), rows)
    n = case.get("singles", 0)
    if n:
        rows = torch.cat((torch.ones(n, dtype=torch.long), rows))
        ctx = torch.cat((_even(n, min(case["ctx_lo"], 64), case["ctx_hi"]), ctx))
    return rows, ctx


def _tables(ctx, block, c):
    """(block table, pool pages): each sequence's pages at random places of a
    pool with a quarter more pages than are used."""
    n = -(-ctx // block)
    pool = int(n.sum()) + int(n.sum()) // 4 + 4
    ids = torch.randperm(pool, generator=c)
    table = torch.zeros(len(n), max(int(n.max()), 1), dtype=torch.int32)
    at = 0
    for s, k in enumerate(n.tolist()):
        table[s, :k] = ids[at:at + k]
        at += k
    return table, pool


def _rows_of(rows, ctx, table, block):
    """(sequence, position, slot) of every new row."""
    seq = torch.repeat_interleave(torch.arange(len(rows)), rows)
    first = torch.cumsum(rows, 0) - rows
    pos = (ctx - rows)[seq] + torch.arange(int(rows.sum())) - first[seq]
    return seq, pos, table[seq, pos // block].long() * block + pos % block


def _frequencies(rot, scaling):
    """(radians per position of each pair, factor of the rotated pairs) at base
    500000; `bands`: waves longer than an original context of 8192 stretched 8
    times, those between a quarter of it and it in part; `yarn`: 4 times, by the
    turns that a pair makes in 4096 positions."""
    f = 500000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    if scaling == "bands":
        part = ((8192 * f / (2 * math.pi) - 1.0) / 3.0).clamp(0, 1)
        f = f / 8 * (1 - part) + f * part
    elif scaling == "yarn":
        turns = 4096 * f / (2 * math.pi)
        part = ((turns - 1.0) / 31.0).clamp(0, 1)
        f = f / 4 * (1 - part) + f * part
    return f, 0.1 * math.log(4.0) + 1.0 if scaling == "yarn" else 1.0


def _normal(shape, dtype, g, scale=1.0):
    """Normal values of a 16-bit or 32-bit type, or of FP8 codes."""
    x = torch.empty(shape, dtype=dtype, device="cuda")
    made = torch.float16 if dtype == torch.float8_e4m3fn else dtype
    for part in x.split(max(1, (1 << 28) // max(1, math.prod(shape[1:])))):
        part.copy_(torch.randn(part.shape, generator=g, dtype=made, device="cuda").mul_(scale))
    return x


def _blob(pool, H, D, g):
    """An INT4 pool: codes, scales about 0.2 and zeros about -1.5 (what normal
    values in groups of 32 give, 4.1 wide)."""
    n = pool * 16 * H * D // 2
    blob = torch.empty(2 * n + 2 * pool * H * 16 * (D // 32) * 4, dtype=torch.uint8, device="cuda")
    blob[:2 * n].random_(0, 256, generator=g)
    p = blob[2 * n:].view(torch.float16).view(-1, 2)
    p[:, 0] = torch.rand(p.shape[0], generator=g, device="cuda") * 0.1 + 0.22
    p[:, 1] = torch.rand(p.shape[0], generator=g, device="cuda") - 2.5
    return blob


def _planes(blob, H, D):
    """Views (K codes, V codes, K params, V params) of a pool's blob."""
    pool = blob.numel() // (H * (16 * D + 4 * D))
    n, m = pool * H * 8 * D, pool * H * 2 * D
    at = 2 * n
    return (blob[:n].view(pool, H, 16, D // 2), blob[n:at].view(pool, H, D // 8, 2, 8, 4),
            blob[at:at + m].view(torch.float16).view(pool, H, 16, D // 32, 2),
            blob[at + m:].view(torch.float16).view(pool, H, D // 32, 16, 2))


def prepare(case, seed):
    c = torch.Generator().manual_seed(seed)
    g = torch.Generator("cuda").manual_seed(seed)
    kind, H, D, bs = case["kind"], case["kv_heads"], case["dim"], case.get("block", 16)
    dt = DTYPES[case["dtype"]]
    if kind == "load":
        ctx = _even(case["seqs"], case["ctx_lo"], case["ctx_hi"])
        rows = ctx
    else:
        rows, ctx = _lengths(case)
    mix = torch.randperm(len(rows), generator=c)
    if case.get("singles", 0) == 0:
        rows, ctx = rows[mix], ctx[mix]
    table, pool = _tables(ctx, bs, c)
    seq, pos, slots = _rows_of(rows, ctx, table, bs)
    N = len(seq)
    s = {"kind": kind, "heads": H, "dim": D, "block": bs}
    if kind in ("rotate", "store", "store4"):
        Hq = case["q_heads"]
        # one projection's output, cut into queries, keys and values
        qkv = _normal((N, Hq + 2 * H, D), dt, g)
        f, s["factor"] = _frequencies(case["rot"], case["scaling"])
        s |= {"q": qkv[:, :Hq], "k": qkv[:, Hq:Hq + H], "v": qkv[:, Hq + H:],
              "positions": pos.cuda(), "frequencies": f.cuda(),
              "interleaved": case["pairs"] == "interleaved"}
        if kind == "store":
            s["kv"] = _normal((2, pool, bs, H, D), torch.float8_e4m3fn, g, 50.0)
        elif kind == "store4":
            s["blob"] = _blob(pool, H, D, g)
        s["slots"] = slots.cuda()
        return s
    if case["cache"] == "int4":
        s["blob"] = _blob(pool, H, D, g)
    else:
        fp8 = case["cache"] == "fp8"
        shape = (2, pool, bs, H, D) if case.get("order", "thd") == "thd" else (2, pool, H, bs, D)
        s["kv"] = _normal(shape, DTYPES[case["cache"]], g, 50.0 if fp8 else 1.0)
        if case.get("order", "thd") == "htd":
            s["kv"] = s["kv"].transpose(2, 3)
        s["k_scale"], s["v_scale"] = (K_SCALE, V_SCALE) if fp8 else (1.0, 1.0)
    s["dtype"] = dt
    if kind == "load":
        s["slots"] = slots.cuda()
        return s
    s["q"] = _normal((N, case["q_heads"], D), dt, g)
    s["start"] = torch.cat((torch.zeros(1, dtype=torch.long), torch.cumsum(rows, 0))).int().cuda()
    s["table"], s["lens"] = table.cuda(), ctx.int().cuda()
    s["singles"], s["rows"] = case.get("singles", 0), int(rows.max())
    return s


# ------------------------------------------------------------ plain forms --


def _plain_rotate(s, x):
    """x [rows, heads, dim] by the angles of its rows, in 64 bits."""
    angle = (s["positions"].double()[:, None] * s["frequencies"])[:, None]
    cos, sin = torch.cos(angle) * s["factor"], torch.sin(angle) * s["factor"]
    R = 2 * s["frequencies"].numel()
    y = x[..., :R].double()
    if s["interleaved"]:
        a, b = y[..., 0::2], y[..., 1::2]
        y = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = y[..., :R // 2], y[..., R // 2:]
        y = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((y.to(x.dtype), x[..., R:]), -1)


def _plain_fp8(x, scale):
    """Codes, from correctly rounded quotients."""
    return (x.double() / scale).float().clamp(-448, 448).to(torch.float8_e4m3fn)


def _plain_store(s):
    k = _plain_rotate(s, s["k"])
    page, at = s["slots"] // s["block"], s["slots"] % s["block"]
    bytes_ = s["kv"].view(torch.uint8)
    bytes_[0, page, at] = _plain_fp8(k, K_SCALE).view(torch.uint8)
    bytes_[1, page, at] = _plain_fp8(s["v"], V_SCALE).view(torch.uint8)
    return {"q": _plain_rotate(s, s["q"]), "cache": s["kv"]}


def _plain_int4(x):
    """(codes, scale, zero) of each group of 32, divisions correctly rounded."""
    x = x.float().unflatten(-1, (-1, 32))
    lo = x.amin(-1, keepdim=True)
    scale = ((x.amax(-1, keepdim=True) - lo).clamp_min(1e-8).double() / 15.0).float()
    u = torch.round(((x - lo).double() / scale.double()).float()).clamp(0, 15).to(torch.uint8)
    return u.flatten(-2), scale[..., 0].half(), lo[..., 0].half()


def _plain_read4(s, slots, dtype):
    """(K, V) rows [..., heads, dim] of the pool, rounded to dtype."""
    H, D = s["heads"], s["dim"]
    kc, vc, kp, vp = _planes(s["blob"], H, D)
    page, at = slots // 16, slots % 16
    k = kc[page, :, at]
    k = torch.stack((k & 15, k >> 4), -1).flatten(-2).float().unflatten(-1, (-1, 32))
    p = kp[page, :, at].float()
    k = (k * p[..., :1] + p[..., 1:]).flatten(-2).to(dtype)
    v = vc[page, :, :, at // 8, :, at % 8 // 2]
    v = (v >> (at % 2 * 4).to(torch.uint8)[..., None, None, None]) & 15
    p = vp[page, :, :, at].float()
    v = (v.flatten(-2).float().unflatten(-1, (-1, 32)) * p[..., :1] + p[..., 1:]).flatten(-2)
    return k, v.to(dtype)


def _plain_store4(s):
    H, D, page, at = s["heads"], s["dim"], s["slots"] // 16, s["slots"] % 16
    kc, vc, kp, vp = _planes(s["blob"], H, D)
    u, scale, zero = _plain_int4(_plain_rotate(s, s["k"]))
    kc[page, :, at] = u[..., 0::2] | u[..., 1::2] << 4
    kp[page, :, at] = torch.stack((scale, zero), -1)
    u, scale, zero = _plain_int4(s["v"])
    vp[page, :, :, at] = torch.stack((scale, zero), -1)
    # a byte holds two tokens: each adds what its half changes by
    i = (page[:, None, None, None], torch.arange(H, device="cuda")[:, None, None],
         torch.arange(D // 8, device="cuda")[:, None], (at // 8)[:, None, None, None],
         torch.arange(8, device="cuda"), (at % 8 // 2)[:, None, None, None])
    shift = (at % 2 * 4).to(torch.uint8)[:, None, None, None]
    was = (vc[i] >> shift) & 15
    vc.index_put_(i, (u.unflatten(-1, (-1, 8)) - was) << shift, accumulate=True)
    k, v = _plain_read4(s, s["slots"], s["k"].dtype)
    return {"q": _plain_rotate(s, s["q"]), "k": k, "v": v}


def _plain_rows(s, slots, dtype):
    """(K, V) rows [..., heads, dim] of a cache or pool, rounded to dtype."""
    if "blob" in s:
        return _plain_read4(s, slots, dtype)
    page, at = slots // s["block"], slots % s["block"]
    if s["kv"].dtype != torch.float8_e4m3fn:
        return s["kv"][0, page, at], s["kv"][1, page, at]
    k, v = (s["kv"].view(torch.uint8)[i, page, at].view(torch.float8_e4m3fn).float()
            for i in range(2))
    return (k * s["k_scale"]).to(dtype), (v * s["v_scale"]).to(dtype)


def _plain_load(s):
    k, v = _plain_rows(s, s["slots"], s["dtype"])
    return {"k": k, "v": v}


def _plain_padded(s, lo, hi, rows, out):
    """Attention of sequences lo .. hi, padded to `rows` rows each, into out."""
    q, table, lens = s["q"], s["table"][lo:hi].long(), s["lens"][lo:hi].long()
    start = s["start"].long()
    first, n = start[lo:hi, None], (start[lo + 1:hi + 1] - start[lo:hi])[:, None]
    Hq, D = q.shape[1:]
    H, S = s["heads"], hi - lo
    j = torch.arange(rows, device="cuda")
    row = torch.where(j < n, first + j, q.shape[0])  # the padding goes behind the last row
    qg = q[row.clamp_max(q.shape[0] - 1)].float().view(S, rows, H, Hq // H, D)
    qg = qg.permute(0, 2, 3, 1, 4).reshape(S, H, -1, D)
    t = torch.arange(table.shape[1] * s["block"], device="cuda")
    slots = table[:, t // s["block"]] * s["block"] + t % s["block"]
    if "blob" in s or s["kv"].dtype != torch.float8_e4m3fn:
        k, v = _plain_rows(s, slots, s["dtype"])
    else:
        k, v = _plain_rows(s, slots, torch.float32)
    k, v = (x.float().permute(0, 2, 1, 3).contiguous() for x in (k, v))
    score = torch.matmul(qg, k.transpose(2, 3).contiguous()).mul_(1.0 / math.sqrt(D))
    seen = t <= (lens[:, None] - n + j)[..., None]
    score.view(S, H, Hq // H, rows, -1).masked_fill_(~seen[:, None, None], -math.inf)
    score.sub_(score.amax(3, keepdim=True)).exp_()
    o = torch.matmul(score, v) / score.sum(3, keepdim=True)
    out[row] = o.view(S, H, Hq // H, rows, D).permute(0, 3, 1, 2, 4).reshape(S, rows, Hq,
                                                                          D).to(out.dtype)


def _plain_attend(s):
    q = s["q"]
    out = torch.empty(q.shape[0] + 1, *q.shape[1:], dtype=q.dtype, device="cuda")
    if s["singles"]:
        _plain_padded(s, 0, s["singles"], 1, out)
    _plain_padded(s, s["singles"], s["lens"].shape[0], s["rows"], out)
    return out[:-1]


# ------------------------------------------------------ the package's calls --


def _operators():
    pkg = os.path.join(os.getcwd(), "axropus-deploy_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from korith_vllm_ext import kernels

    return kernels


_kernels = None


def _pool(s):
    """The handle of an INT4 pool, made once."""
    if "pool" not in s:
        H, D = s["heads"], s["dim"]
        s["pool"] = _kernels.int4_page_pool(s["blob"].numel() // (H * 20 * D), H, D,
                                            blob=s["blob"])
    return s["pool"]


def _own(s):
    global _kernels
    if _kernels is None:
        _kernels = _operators()
    kind = s["kind"]
    if kind == "rotate":
        r = _kernels.Rotary(s["frequencies"], s["interleaved"], s["factor"])
        q, k = _kernels.rotary_embedding(s["q"], s["k"], s["positions"], r)
        return {"q": q, "k": k}
    if kind == "store":
        r = _kernels.Rotary(s["frequencies"], s["interleaved"], s["factor"])
        q = _kernels.write_kv_cache(s["k"], s["v"], s["kv"], slot_mapping=s["slots"], rotary=r,
                                    positions=s["positions"], q=s["q"], k_scale=K_SCALE,
                                    v_scale=V_SCALE)
        return {"q": q, "cache": s["kv"]}
    if kind == "store4":
        r = _kernels.Rotary(s["frequencies"], s["interleaved"], s["factor"])
        q = _kernels.write_kv_cache(s["k"], s["v"], _pool(s), slot_mapping=s["slots"], rotary=r,
                                    positions=s["positions"], q=s["q"])
        k, v = _kernels.read_kv_cache(_pool(s), slot_mapping=s["slots"], dtype=s["k"].dtype)
        return {"q": q, "k": k, "v": v}
    scales = {} if "blob" in s else {"k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    cache = _pool(s) if "blob" in s else s["kv"]
    if kind == "load":
        k, v = _kernels.read_kv_cache(cache, slot_mapping=s["slots"], dtype=s["dtype"], **scales)
        return {"k": k, "v": v}
    return _kernels.paged_attention(s["q"], cache, query_start=s["start"],
                                    block_tables=s["table"], context_lens=s["lens"], **scales)


def _plain_rotated(s):
    return {"q": _plain_rotate(s, s["q"]), "k": _plain_rotate(s, s["k"])}


_PLAIN = {"rotate": _plain_rotated, "store": _plain_store, "store4": _plain_store4,
          "load": _plain_load, "attend": _plain_attend}


def run(state):
    return _own(state) if own else _PLAIN[state["kind"]](state)


# ----------------------------------------------------------------- work --


def work(case):
    kind, H, D = case["kind"], case["kv_heads"], case["dim"]
    es = DTYPES[case["dtype"]].itemsize
    bits = {"fp8": 8, "int4": 5, "bf16": 16, "fp16": 16}.get(case.get("cache"))
    if kind == "load":
        n = int(_even(case["seqs"], case["ctx_lo"], case["ctx_hi"]).sum())
        return {"bytes": n * (2 * H * D * (bits / 8 + es) + 8), "flops": 2 * n * 2 * H * D}
    rows, ctx = _lengths(case)
    n, Hq = int(rows.sum()), case["q_heads"]
    if kind == "attend":
        tokens = int(ctx.sum())
        pairs = int((rows * (ctx - rows) + rows * (rows + 1) // 2).sum())
        return {"bytes": tokens * 2 * H * D * bits / 8 + 2 * n * Hq * D * es
                + 4 * tokens / case["block"], "flops": 4 * pairs * Hq * D}
    b = 2 * n * Hq * D * es + 8 * n + 4 * case["rot"]
    fl = 3 * n * (Hq + H) * case["rot"] + 20 * n * case["rot"]
    if kind == "rotate":
        return {"bytes": b + 2 * n * H * D * es, "flops": fl}
    b += 2 * n * H * D * es + 8 * n
    if kind == "store":
        return {"bytes": b + 2 * n * H * D, "flops": fl + 4 * n * H * D}
    # written in 5 bits a value, read back, and written in k's type
    return {"bytes": b + 2 * n * H * D * (2 * 5 / 8 + es) + 8 * n, "flops": fl + 16 * n * H * D}


# --------------------------------------------------------------- 64 bits --


def _rotated64(s, x):
    """x by complex multiplication, in 64 bits."""
    f, n = s["frequencies"], 2 * s["frequencies"].numel()
    turn = torch.polar(torch.full_like(f, s["factor"]).expand(len(s["positions"]), -1),
                       s["positions"].double()[:, None] * f)[:, None]
    head = x[..., :n].double()
    if s["interleaved"]:
        z = torch.view_as_complex(head.unflatten(-1, (-1, 2)).contiguous()) * turn
        z = torch.view_as_real(z).flatten(-2)
    else:
        z = torch.complex(head[..., :n // 2].contiguous(), head[..., n // 2:].contiguous()) * turn
        z = torch.cat((z.real, z.imag), -1)
    return torch.cat((z, x[..., n:].double()), -1)


def _e4m3_64(x):
    """The nearest e4m3 values, in 64 bits: steps of 2^-3 of the leading bit, at least 2^-9."""
    x = x.clamp(-448, 448)
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def _int4_64(x, dtype):
    """What the codec keeps of each group of 32 values, rounded to dtype."""
    x = x.unflatten(-1, (-1, 32))
    lo, hi = torch.aminmax(x, dim=-1, keepdim=True)
    scale = (hi - lo).clamp_min(1e-8) / 15
    u = torch.round((x - lo) / scale).clamp(0, 15)
    return (u * scale.half().double() + lo.half().double()).flatten(-2).to(dtype).double()


def _pool64(s, slots, dtype):
    """Rows of the pool from whole pages taken apart, in 64 bits."""
    H, D = s["heads"], s["dim"]
    kc, vc, kp, vp = _planes(s["blob"], H, D)
    page, at = slots // 16, slots % 16
    k, v = kc[page], vc[page]
    k = torch.stack((k % 16, k // 16), -1).reshape(-1, H, 16, D // 32, 32)
    v = torch.stack((v % 16, v // 16), -1).reshape(-1, H, D // 8, 2, 8, 8)
    v = v.permute(0, 1, 3, 5, 2, 4).reshape(-1, H, 16, D // 32, 32)
    kq, vq = kp[page].double(), vp[page].transpose(2, 3).double()
    i = torch.arange(len(page), device="cuda")
    return tuple((x[i, :, at].double() * p[i, :, at, :, :1] + p[i, :, at, :, 1:]).to(dtype)
                 .double().flatten(-2) for x, p in ((k, kq), (v, vq)))


def _cache64(s, slots, dtype):
    if "blob" in s:
        parts = [_pool64(s, x, dtype) for x in slots.split(4096)]
        return tuple(torch.cat(x) for x in zip(*parts))
    page, at, kv = slots // s["block"], slots % s["block"], s["kv"]
    out = []
    for i, scale in ((0, s["k_scale"]), (1, s["v_scale"])):
        rows = kv[i].view(torch.uint8)[page, at].view(kv.dtype) if kv.dtype.itemsize == 1 else \
            kv[i][page, at]
        out.append(rows.double() * scale)
    return tuple(out)


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind == "rotate":
        return {"q": _rotated64(s, s["q"]), "k": _rotated64(s, s["k"])}
    if kind == "load":
        k, v = _cache64(s, s["slots"], s["dtype"])
        return {"k": k, "v": v}
    if kind in ("store", "store4"):
        # the key that a cache of k's type would hold is what is quantised
        k, v = _rotated64(s, s["k"]).to(s["k"].dtype).double(), s["v"].double()
        out = {"q": _rotated64(s, s["q"])}
        if kind == "store4":
            return out | {"k": _int4_64(k, s["k"].dtype), "v": _int4_64(v, s["k"].dtype)}
        cache = s["kv"].double()
        page, at = s["slots"] // s["block"], s["slots"] % s["block"]
        cache[0, page, at], cache[1, page, at] = _e4m3_64(k / K_SCALE), _e4m3_64(v / V_SCALE)
        return out | {"cache": cache}
    q, H = s["q"], s["heads"]
    Hq, D = q.shape[1:]
    out = torch.empty(q.shape, dtype=torch.float64, device="cuda")
    start, lens, bs = s["start"].tolist(), s["lens"].tolist(), s["block"]
    for i, c in enumerate(lens):
        lo, hi = start[i], start[i + 1]
        t = torch.arange(c, device="cuda")
        slots = s["table"][i].long()[t // bs] * bs + t % bs
        k, v = _cache64(s, slots, s["dtype"])
        hidden = t[None] > torch.arange(c - (hi - lo), c, device="cuda")[:, None]
        for h in range(Hq):
            g = h // (Hq // H)
            w = (q[lo:hi, h].double() @ k[:, g].t().contiguous()) / math.sqrt(D)
            w = torch.softmax(w.masked_fill_(hidden, -math.inf), 1)
            out[lo:hi, h] = w @ v[:, g].contiguous()
    return out
