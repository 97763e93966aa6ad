"""float64 restatements of the paged operators and the inputs of their tests
(not collected)."""

from __future__ import annotations

import math

import torch

DEV = torch.device("cuda")


def make_cache(pool, block, H, D, dtype, g, order="thd", scale=1.0):
    """A layer [2, pool, block, H, D] on the GPU, in either page order."""
    shape = (2, pool, H, block, D) if order == "htd" else (2, pool, block, H, D)
    kv = (torch.randn(shape, generator=g) * scale).to(dtype).to(DEV)
    return kv.transpose(2, 3) if order == "htd" else kv


def make_tables(lens, block, g, spare=3, fill=-7, extra=0):
    """(int32 table with `fill` behind each sequence's pages, pool pages)."""
    n = [-(-max(c, 0) // block) for c in lens]
    pool = sum(n) + spare
    ids = torch.randperm(pool, generator=g).to(torch.int32)
    table = torch.full((len(n), max(max(n, default=0), 1) + extra), fill, dtype=torch.int32)
    at = 0
    for s, k in enumerate(n):
        table[s, :k] = ids[at:at + k]
        at += k
    return table, pool


def token_places(s, h, lens, block, pages, counts, width):
    """Positions that (sequence, KV head) attends to, in order, repeats kept."""
    c = min(lens[s], width * block)
    if pages is None:
        return list(range(max(c, 0)))
    out = []
    for p in pages[s, h, :counts[s, h]].tolist():
        if 0 <= p < width:
            out += [t for t in range(p * block, p * block + block) if t < c]
    return out


def attend64(q, kv, table, lens, scale, k_scale=1.0, v_scale=1.0, pages=None, counts=None):
    """float64 attention on the CPU over each (sequence, KV head)'s tokens;
    tokens of pages outside the pool are left out."""
    S, Hq, D = q.shape
    _, pool, block, H, _ = kv.shape
    q, kv = q.cpu().double(), kv.cpu()
    G = Hq // H
    out = torch.zeros(S, Hq, D, dtype=torch.float64)
    for s in range(S):
        for h in range(H):
            at = token_places(s, h, lens, block, pages, counts, table.shape[1])
            at = [t for t in at if 0 <= int(table[s, t // block]) < pool]
            if not at:
                continue
            at = torch.tensor(at)
            ids = table[s, at // block].long()
            k, v = (kv[i][ids, at % block, h].double() for i in range(2))
            x = q[s, h * G:(h + 1) * G] @ k.t() * (scale * k_scale)
            out[s, h * G:(h + 1) * G] = torch.softmax(x, -1) @ v * v_scale
    return out


def attend_tolerance(q, kv, lens, scale, k_scale=1.0, v_scale=1.0):
    """Largest error of an fp32 result.  A score is a sum of D exact products
    in fp32: off by at most (D + 4) 2^-24 of sum |q_d k_d|, which |q| |k|
    bounds; a weight by twice that, for its own and the row's sum, and by what
    summing up to T / 32 + 64 terms in fp32 and the 2^x add."""
    D = q.shape[-1]
    k, v = kv[0].float(), kv[1].float()
    k, v = k[torch.isfinite(k).all(-1)], v[torch.isfinite(v).all(-1)]
    top = float(q.float().norm(dim=-1).max()) * float(k.norm(dim=-1).max()) * abs(scale * k_scale)
    score = (D + 4) * 2.0 ** -24 * top
    terms = 2 * (max(lens) / 32 + 64) * 2.0 ** -24
    return float(v.abs().max()) * abs(v_scale) * (2 * score + terms + 2.0 ** -21)


def bounds64(k, table, lens, block, first=None):
    """{page id: [H, 2, D]} of the pages that page_key_bounds writes."""
    out = {}
    pool = k.shape[0]
    for s, c in enumerate(lens):
        c = min(c, table.shape[1] * block)
        for p in range(0 if first is None else max(first[s], 0) // block, -(-max(c, 0) // block)):
            i = int(table[s, p])
            if 0 <= i < pool:
                x = k[i, :min(block, c - p * block)].double()
                out[i] = torch.stack((x.amin(0), x.amax(0)), 1)
    return out


def select64(q, bounds, table, lens, block, keep, first, last):
    """(pages, counts) by sorting float64 scores."""
    S, Hq, D = q.shape
    pool, H = bounds.shape[:2]
    q, b = q.cpu().double(), bounds.cpu().double()
    G = Hq // H
    pages = torch.full((S, H, keep), -1, dtype=torch.int32)
    counts = torch.zeros(S, H, dtype=torch.int32)
    for s, c in enumerate(lens):
        n = min(-(-max(c, 0) // block), table.shape[1])
        for h in range(H):
            rank = []
            for p in range(n):
                i = int(table[s, p])
                if p < first or p >= n - last:
                    u = (2, 0.0)
                elif not 0 <= i < pool:
                    u = (-1, 0.0)
                else:
                    lo, hi = b[i, h]
                    x = torch.maximum(q[s, h * G:(h + 1) * G] * lo,
                                      q[s, h * G:(h + 1) * G] * hi).sum(-1)
                    good = bool(torch.isfinite(lo).all() and torch.isfinite(hi).all()
                                and torch.isfinite(x).all())
                    u = (0, float(x.max())) if good else (1, math.inf)
                rank.append(u)
            took = sorted(sorted(range(n), key=lambda p: (-rank[p][0], -rank[p][1], p))[:keep])
            pages[s, h, :len(took)] = torch.tensor(took, dtype=torch.int32)
            counts[s, h] = len(took)
    return pages, counts


def slot_maps_ref(lens, new, table, block, rows, free=(), used=0, pool=1 << 31):
    """Plain Python step: (slots, positions, starts, lens, used, table, flags)."""
    table = table.clone()
    width = table.shape[1]
    slots, pos, starts, out = [], [], [0], []
    flags, place, end = 0, 0, 0
    for s, (c, n) in enumerate(zip(lens, new)):
        c, n = max(c, 0), max(n, 0)
        have, need = -(-c // block), -(-(c + n) // block)
        ok = need <= width and (n == 0 or len(slots) + n <= rows)
        if not ok:
            flags |= 2
        elif need > have:
            place += need - have
            ok = place <= max(len(free) - used, 0)
            if not ok:
                flags |= 8
            else:
                end = place
        for j in range(n):
            p, at = divmod(c + j, block)
            pos.append(c + j)
            slot = -1
            if ok:
                i = int(table[s, p]) if p < have else free[used + place - (need - have) + p - have]
                if 0 <= i < pool:
                    slot = i * block + at
                    if len(slots) < rows and at == 0 and p >= have:
                        table[s, p] = i
                else:
                    flags |= 1 if len(slots) < rows else 0
            slots.append(slot)
        starts.append(len(slots))
        out.append(c + n if ok else c)
    pad = max(0, rows - len(slots))
    return (slots[:rows] + [-1] * pad, pos[:rows] + [0] * pad, starts, out, used + end, table,
            flags)
