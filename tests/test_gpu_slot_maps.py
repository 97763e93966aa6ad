"""build_slot_maps against a plain Python step."""

from __future__ import annotations

import pytest
import torch

from paged_ref import DEV, slot_maps_ref

pytestmark = pytest.mark.gpu


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _start(lens, block, g, extra):
    """(table with the sequences' pages, the ids left over)."""
    n = [-(-max(c, 0) // block) for c in lens]
    ids = torch.randperm(sum(n) + 4000, generator=g).int()
    table = torch.full((len(n), max(n, default=0) + extra), -1, dtype=torch.int32)
    at = 0
    for s, k in enumerate(n):
        table[s, :k] = ids[at:at + k]
        at += k
    return table, ids[at:].tolist()


def _compare(lens, new, block, rows, table, free, used=0, pool=None, cut=None):
    from korith_vllm_ext.kernels import build_slot_maps

    free = free if cut is None else free[:cut]
    bt = table.to(DEV)
    flag = torch.zeros(1, dtype=torch.int32, device=DEV)
    m = build_slot_maps(_i32(lens), _i32(new), bt, block_size=block, num_tokens=rows,
                        free_pages=_i32(free) if free else None, free_used=_i32([used]),
                        pool_pages=pool, err_flag=flag)
    want = slot_maps_ref(lens, new, table, block, rows, free, used, pool or 1 << 31)
    for got, ref in zip(m, want):
        assert got.tolist() == (ref if isinstance(ref, list) else [ref])
    assert torch.equal(bt.cpu(), want[5])
    assert int(flag) == want[6], (int(flag), want[6])
    return m


@pytest.mark.parametrize("seqs,hi,most,block,pad", [
    (1, 0, 1, 16, 0), (1, 100, 5000, 16, 7), (32, 500, 1, 16, 0), (255, 90, 9, 16, 3),
    (256, 90, 30, 16, 1), (257, 40, 3, 1, 0), (1000, 33, 20, 5, 2000), (2100, 64, 2, 32, 0),
    (5, 300, 1024, 16, 0)])
def test_matches_a_plain_step(seqs, hi, most, block, pad):
    g = torch.Generator().manual_seed(seqs + most)
    lens = torch.randint(0, hi + 1, (seqs,), generator=g).tolist()
    new = torch.randint(0, most + 1, (seqs,), generator=g).tolist()
    table, free = _start(lens, block, g, -(-most // block) + 1)
    free = (free * 6)[:sum(new) // block + seqs + 60]
    _compare(lens, new, block, sum(new) + pad, table, free, used=5)


def test_edges():
    g = torch.Generator().manual_seed(0)
    for lens, new in (([0], [16]), ([16], [1]), ([15], [1]), ([15], [2]), ([0, 0], [0, 0]),
                      ([-4, 7], [3, -2]), ([31, 32, 33], [1, 1, 1])):
        table, free = _start(lens, 16, g, 3)
        _compare(lens, new, 16, 24, table, free)
    _compare([], [], 16, 5, torch.zeros(0, 4, dtype=torch.int32), [3])
    _compare([5], [1], 16, 0, torch.tensor([[2, -1]], dtype=torch.int32), [3])  # no rows at all


def test_free_list_runs_out():
    """Sequences are served in order while the pages last; those that need none
    always are."""
    g = torch.Generator().manual_seed(3)
    lens, new = [16, 5, 32, 10, 16, 3], [1, 2, 40, 1, 1, 1]
    table, free = _start(lens, 16, g, 4)
    for cut in (0, 1, 2, 3, 4, 5):
        _compare(lens, new, 16, 50, table, free, used=0, cut=cut)
    _compare(lens, new, 16, 50, table, free, used=9, cut=3)  # more in use than there are


def test_table_row_too_short():
    g = torch.Generator().manual_seed(4)
    lens, new = [30, 31, 30], [2, 3, 1]
    table, free = _start(lens, 16, g, 0)
    _compare(lens, new, 16, 6, table, free)


def test_tables_without_a_free_list():
    """The tables hold every page already: only slots are made."""
    table = torch.tensor([[4, 9, 2], [7, 1, 0]], dtype=torch.int32)
    _compare([48, 20], [0, 4], 16, 8, table, [])
    from korith_vllm_ext.kernels import build_slot_maps

    m = build_slot_maps(_i32([33, 20]), _i32([3, 5]), table.to(DEV), block_size=16, num_tokens=8)
    assert m.slot_mapping.tolist() == [33, 34, 35, 20, 21, 22, 23, 24]
    assert m.free_used.tolist() == [0]


def test_bad_pages_and_too_few_rows():
    g = torch.Generator().manual_seed(5)
    lens, new = [20, 16, 40], [3, 20, 2]
    table, free = _start(lens, 16, g, 3)
    table[0, 1] = -1
    free[1] = 100000
    _compare(lens, new, 16, 30, table, free, pool=5000)
    table, free = _start(lens, 16, g, 3)
    _compare(lens, new, 16, 10, table, free)


@pytest.mark.parametrize("bad_id", [1000, -5, (1 << 31) - 1])
def test_bad_page_of_the_free_list_stays_bad(bad_id):
    """A reused row still holds old page ids behind its last page; a page id
    outside the pool must not leave them in place for the next step."""
    from korith_vllm_ext.kernels import build_slot_maps

    bt = torch.tensor([[4, 7, 9], [5, 6, 8]], dtype=torch.int32, device=DEV)
    free, used, flag = _i32([bad_id, 3, 11]), _i32([0]), _i32([0])
    m = build_slot_maps(_i32([16, 15]), _i32([2, 3]), bt, block_size=16, num_tokens=5,
                        free_pages=free, free_used=used, pool_pages=20, err_flag=flag)
    assert m.slot_mapping.tolist() == [-1, -1, 95, 48, 49] and int(flag) == 1
    assert m.context_lens.tolist() == [18, 18] and m.free_used.tolist() == [2]
    assert bt.tolist() == [[4, -1, 9], [5, 3, 8]]
    flag.zero_()
    m = build_slot_maps(m.context_lens, _i32([1, 1]), bt, block_size=16, num_tokens=2,
                        free_pages=free, free_used=m.free_used, pool_pages=20, err_flag=flag)
    assert m.slot_mapping.tolist() == [-1, 50] and int(flag) == 1


def test_sequences_behind_the_rows_do_not_grow():
    """Their new pages have no rows that would write them into the table."""
    table, free = _start([16, 16, 16], 16, torch.Generator().manual_seed(6), 2)
    m = _compare([16, 16, 16], [2, 2, 2], 16, 5, table, free)
    assert m.context_lens.tolist() == [18, 18, 16] and m.slot_mapping[4] == -1
    g = torch.Generator().manual_seed(7)
    lens = torch.randint(0, 40, (700,), generator=g).tolist()
    new = torch.randint(0, 9, (700,), generator=g).tolist()
    for rows in (0, 1, sum(new) // 2, sum(new) - 1):
        table, free = _start(lens, 16, g, 2)
        _compare(lens, new, 16, rows, table, free, used=2)


def test_outputs_that_overlap_are_refused():
    from korith_vllm_ext.kernels import SlotMaps, build_slot_maps

    buf = torch.zeros(64, dtype=torch.int32, device=DEV)
    wide = torch.zeros(8, dtype=torch.int64, device=DEV)
    table = torch.tensor([[4, -1], [7, 1]], dtype=torch.int32, device=DEV)
    good = dict(context_lens=buf[0:2], new_tokens=buf[2:4], block_tables=table, block_size=16,
                num_tokens=3, free_pages=buf[4:7], free_used=buf[7:8], err_flag=buf[8:9])
    out = SlotMaps(wide[:3], wide[3:6], buf[9:12], buf[12:14], buf[14:15])
    buf[:8] = _i32([16, 20, 1, 1, 6, 5, 3, 0])
    want = build_slot_maps(**{k: v.clone() if isinstance(v, torch.Tensor) else v
                              for k, v in good.items()})
    for o in (
        out._replace(context_lens=buf[1:3]),   # half of context_lens, half of new_tokens
        out._replace(query_start=buf[1:4]), out._replace(free_used=buf[3:4]),
        out._replace(query_start=buf[6:9]), out._replace(context_lens=buf[5:7]),
        out._replace(free_used=buf[7:8]), out._replace(free_used=buf[8:9]),
        out._replace(context_lens=table[1]), out._replace(slot_mapping=buf[:6].view(torch.int64)),
        out._replace(positions=wide[2:5]), out._replace(context_lens=buf[11:13]),
        out._replace(free_used=buf[13:14]), out._replace(free_used=buf[9:10]),
    ):
        with pytest.raises(ValueError, match="overlap"):
            build_slot_maps(out=o, **good)
    got = build_slot_maps(out=out, **good)  # side by side
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and int(buf[8]) == 0
    # no rows, no sequences: nothing that could overlap
    none = SlotMaps(wide[:0], wide[:0], buf[9:10], buf[9:9], buf[14:15])
    build_slot_maps(buf[0:0], buf[0:0], table[:0], block_size=16, num_tokens=0, out=none)
    assert none.query_start.tolist() == [0] and none.free_used.tolist() == [0]


def test_outputs_given_and_refusals():
    from korith_vllm_ext.kernels import SlotMaps, build_slot_maps

    table = torch.tensor([[4, -1], [7, 1]], dtype=torch.int32)
    cl, nt, bt, free = _i32([16, 20]), _i32([1, 1]), table.to(DEV), _i32([6, 5])
    want = build_slot_maps(cl, nt, bt.clone(), block_size=16, num_tokens=3, free_pages=free)
    out = SlotMaps(*(torch.full_like(t, 99) for t in want))
    got = build_slot_maps(cl, nt, bt, block_size=16, num_tokens=3, free_pages=free, out=out)
    assert got is out and all(torch.equal(a, b) for a, b in zip(out, want))
    bad = [
        dict(context_lens=cl.long()), dict(new_tokens=nt[:1]), dict(context_lens=cl.cpu()),
        dict(block_tables=bt.long()), dict(block_tables=bt.cpu()), dict(block_tables=bt[0]),
        dict(block_tables=bt.t().contiguous().t()), dict(block_tables=bt[:1].expand(2, 2)),
        dict(block_size=0), dict(num_tokens=-1), dict(pool_pages=0), dict(free_pages=free.long()),
        dict(free_pages=free[:, None]), dict(free_used=free),
        dict(out=out._replace(slot_mapping=out.slot_mapping[:2])),
        dict(out=out._replace(positions=out.positions.int())),
        dict(out=out._replace(query_start=out.query_start[:2])),
        dict(out=out._replace(context_lens=cl)),
        dict(err_flag=torch.zeros(2, dtype=torch.int32, device=DEV)),
    ]
    for kw in bad:
        args = dict(context_lens=cl, new_tokens=nt, block_tables=bt, block_size=16, num_tokens=3,
                    free_pages=free) | kw
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            build_slot_maps(**args)
