"""A step's operators over caches whose pages lie more than 4 GiB apart: the bits of a small
cache that holds the same rows."""

from __future__ import annotations

import pytest
import torch

from paged_ref import DEV
from test_gpu_paged_rows import _i32

pytestmark = pytest.mark.gpu

BF16, F16, F32, FP8 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn
GIB = 1 << 30


@pytest.fixture(autouse=True)
def _give_back():
    yield
    torch.cuda.empty_cache()


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _room(n):
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < n + 8 * GIB:
        pytest.skip(f"needs {n / GIB:.0f} GiB of GPU memory")


def _step(cache, table, slots, rows, D, dtype, scales):
    """Writes, reads and attends; (K, V) rows and the attention's."""
    from korith_vllm_ext.kernels import (paged_attention, read_kv_cache, rotary_frequencies,
                                         write_kv_cache)

    k, v, q = rows
    flag = torch.zeros(1, dtype=torch.int32, device=DEV)
    at = dict(slot_mapping=slots, err_flag=flag, **scales)
    write_kv_cache(k, v, cache, rotary=rotary_frequencies(D),
                   positions=torch.arange(len(k), device=DEV), **at)
    back = read_kv_cache(cache, dtype=dtype, **at)
    n = len(k)
    out = [paged_attention(q[:m], cache, query_start=_i32([0, m]), block_tables=_i32([table]),
                           context_lens=_i32([n]), err_flag=flag, **scales) for m in (1, 37)]
    assert int(flag) == 0
    return *back, *out


def _slots(table, block, n):
    t = torch.arange(n)
    return (torch.tensor(table)[t // block] * block + t % block).to(DEV)


@pytest.mark.parametrize("dtype,cache", [(BF16, BF16), (F16, FP8), (F32, F32)])
@pytest.mark.parametrize("D,block", [(128, 16), (64, 32), (80, 16), (256, 16)])
@pytest.mark.parametrize("page", [3 * GIB, 33 * GIB])
def test_far_pages_of_a_cache(dtype, cache, D, block, page):
    """3 GiB: offsets of 32 bits in whole vectors; 33 GiB: beyond those too."""
    n, H = 3 * block - 5, 2
    _room(3 * page)
    buf = torch.empty(2 * page + page // 2 + GIB, dtype=torch.uint8, device=DEV).view(cache)
    es = buf.element_size()
    far = buf.as_strided((2, 3, block, H, D), (page // 2 // es, page // es, H * D, D, 1))
    near = torch.zeros(2, 3, block, H, D, dtype=cache, device=DEV)
    g = _gen(D)
    rows = tuple(torch.randn(n, h, D, generator=g).to(dtype).to(DEV) for h in (H, H, 4 * H))
    scales = dict(k_scale=0.02, v_scale=0.03) if cache is FP8 else {}
    table = [2, 0, 1]
    got = _step(far, table, _slots(table, block, n), rows, D, dtype, scales)
    want = _step(near, table, _slots(table, block, n), rows, D, dtype, scales)
    # (the attention too: where pages are looked up row by row, the same products in the same order)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_far_pages_of_a_pool():
    from korith_vllm_ext.kernels import int4_page_pool

    H, D, pages, n = 8, 128, 600000, 90  # 4.9 GB of codes and 1.2 of parameters a plane
    _room(14 * GIB)
    far, near = int4_page_pool(pages, H, D), int4_page_pool(6, H, D)
    g = _gen(9)
    rows = tuple(torch.randn(n, h, D, generator=g).to(BF16).to(DEV) for h in (H, H, 4 * H))
    table, small = [pages - 1, 3, 524288, 262144, pages - 2, 524289], [5, 0, 3, 1, 2, 4]
    got = _step(far, table, _slots(table, 16, n), rows, D, BF16, {})
    want = _step(near, small, _slots(small, 16, n), rows, D, BF16, {})
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert got[0].any() and got[1].any()
