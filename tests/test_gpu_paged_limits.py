"""Calls at the ends of what the operators over a KV cache in pages take."""
import numpy as np
import pytest
from test_gpu_paged import check
from test_gpu_paged_budget import _attend, _check_evict, _evict_case, given64

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
