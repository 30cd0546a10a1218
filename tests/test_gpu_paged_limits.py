"""Calls at the ends of what the operators over a KV cache in pages take."""
import numpy as np
import pytest
from test_gpu_paged import _cache, attend64, check
from test_gpu_paged_budget import _attend, _check_evict, _evict_case, _i32, given64

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("type_,page,missing,new", [("bfloat16", 1024, 16382, [2]), ("float16", 8192, 16382, [1, 1, 1])])
def test_weights_of_hundreds_of_millions_of_keys(agpu, dev, type_, page, missing, new):
    """32 K/V heads over more keys than 2^29 / 32 (scores formed again) or 2^32 / 32 (added up from scratch), more than are numbered at a time, nearly all of them on pages that are not in the cache: those behind are given
    their weights too, and new ones begin at zero."""
    import torch
    H, lens, n = 32, [2 * page + missing * page + 2 * page + page // 3] + [5] * (len(new) - 1), sum(new)
    g = torch.Generator(device=dev).manual_seed(page)
    kc, vc = (torch.randn((7, H, page, 64), generator=g, device=dev).to(getattr(torch, type_)) for _ in range(2))
    w, q = torch.rand(kc.shape[:3], generator=g, device=dev), torch.randn((n, H, 64), generator=g, device=dev)
    tables = np.full((len(new), missing + 5), -1)
    tables[0, [0, 1, -3, -2, -1]], tables[1:, 0] = [3, 0, 6, 1, 4], [5, 2][:len(new) - 1]
    start = np.concatenate([[0], np.cumsum(new)]).tolist()
    # without the missing pages the rows see the same keys
    short = [[3, 0, 6, 1, 4]] + [[p] * 5 for p in (5, 2)][:len(new) - 1]
    want, tol = given64(q, kc, w, short, [lens[0] - missing * page] + lens[1:], start)
    assert (tol[4, :, :page // 3] > 0).all()
    _attend(dev, q, kc, vc, w, tables, lens, start)
    check(w, want, tol)


@pytest.mark.parametrize("n,limit,keep,recent,sinks", [(100000, 40000, 40000, 40000, 0), (200000, 100000, 100000, 100000, 0), (200000, 150000, 99990, 99980, 4), (140000, 70000, 65536, 0, 65536)])
def test_evict_where_all_of_a_range_moves(agpu, dev, n, limit, keep, recent, sinks):
    """2^15 positions in a row of which all are evicted, all move or all stay: the last ones are nearly all that is kept, or the first ones."""
    kc, vc, w, tables = _evict_case(dev, [n, 3], 1, 100, "bfloat16", keep)
    _check_evict(dev, kc, vc, w, tables, [n, 3], limit, keep, recent, sinks)


def test_trim_gives_back_what_the_tables_have(agpu, dev):
    """Ids outside the cache behind `keep` go onto the stack like any others; a request that gets them has nowhere to keep what it appends there, and nobody sees it or is touched by it."""
    import torch
    from async_gpu_amd import ops
    i, page, pages, H = _i32(dev), 4, 9, 2
    tables, stack = i([[0, 1, pages, -1, 2**31 - 1], [2, 3, 4, 5, 6]]), i([7, 8, -5, -5, -5, -5])
    kv, gone, n = ops.paged_trim(i([20, 0]), tables, stack, i([2]), page, 10, 8)
    assert kv.tolist() == [8, 0] and gone.tolist() == [12, 0] and n.tolist() == [5] and stack.tolist() == [7, 8, pages, -1, 2**31 - 1, -5]
    kv, start, slots, pos, n = ops.paged_plan(kv, i([0, 18]), tables, stack, n, page, 18)
    assert kv.tolist() == [8, 18] and n.tolist() == [0] and tables.tolist()[1] == [2**31 - 1, -1, pages, 8, 7]
    g = torch.Generator(device=dev).manual_seed(1)
    kc, vc = _cache(torch, g, dev, pages, H, page, "float32")
    k, v, q = (torch.randn((18, H, 64), generator=g, device=dev) for _ in range(3))
    want = [x.clone() for x in (kc, vc)]
    for x, rows in zip(want, (k, v)):
        x[8], x[7, :, :2] = rows[12:16].transpose(0, 1), rows[16:].transpose(0, 1)
    ops.paged_kv_append(k, v, kc, vc, slots)
    assert torch.equal(kc, want[0]) and torch.equal(vc, want[1])
    check(ops.paged_attention(q, kc, vc, tables, kv, start), *attend64(q, kc, vc, tables.tolist(), kv.tolist(), start.tolist()))
