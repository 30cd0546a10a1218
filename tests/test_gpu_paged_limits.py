"""Calls at the ends of what the operators over a KV cache in pages take."""
import numpy as np
import pytest
from test_gpu_paged import _cache, attend64, check
from test_gpu_paged_budget import _attend, _check_evict, _evict_case, _i32, _state, given64

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


@pytest.mark.parametrize("type_", ["float32", "bfloat16"])
def test_one_arena(agpu, dev, type_):
    """K, V and weights page by page in one allocation, rows and results behind them: the same bits as in allocations of their own."""
    import torch
    from async_gpu_amd import ops
    lens, new, page, H, i = [100, 50, 300, 33], [1, 50, 140, 1], 16, 3, _i32(dev)
    kc, vc, w, tables, start, q = _state(dev, lens, new, 2 * H, H, page, type_, 3)
    n, each, ints = kc.shape[0], H * page * 64 * kc.element_size(), i(tables)
    room = 2 * each + H * page * 4
    arena = torch.zeros(n * room + 2 * q.numel() * 4, dtype=torch.uint8, device=dev)
    by_page = arena[:n * room].view(n, room)
    k, v = (by_page[:, a:a + each].view(kc.dtype).unflatten(1, (H, page, 64)) for a in (0, each))
    own = by_page[:, 2 * each:].view(torch.float32).unflatten(1, (H, page))
    rows, out = arena[n * room:].view(torch.float32).view(2, *q.shape)
    for to, x in ((k, kc), (v, vc), (own, w), (rows, q)):
        to.copy_(x)
    want, _ = ops.paged_attention_weights(q, kc, vc, w, ints, i(lens), i(start))
    ops.paged_attention_weights(rows, k, v, own, ints, i(lens), i(start), out=out)
    assert torch.equal(out, want) and torch.equal(own, w)
    ops.paged_evict(kc, vc, w, ints, i(lens), 40, 30, 5, 2)
    ops.paged_evict(k, v, own, ints, i(lens), 40, 30, 5, 2)
    assert torch.equal(k, kc) and torch.equal(v, vc) and torch.equal(own, w) and torch.equal(rows, q) and torch.equal(out, want)


def test_evict_where_keys_are_the_values(agpu, dev):
    import torch
    from async_gpu_amd import ops
    i = _i32(dev)
    kc, vc, w, tables = _evict_case(dev, [300, 200, 90], 2, 16, "float16", 3)
    same, weights = kc.clone(), w.clone()
    ops.paged_evict(kc, vc, w, i(tables), i([300, 200, 90]), 80, 64, 10, 4)
    ops.paged_evict(same, same, weights, i(tables), i([300, 200, 90]), 80, 64, 10, 4)
    assert torch.equal(same, kc) and torch.equal(weights, w)


def test_memory_that_overlaps_is_refused(agpu, dev):
    """By the entry points themselves, whoever calls them, before anything is launched."""
    import torch
    from async_gpu_amd import ops
    i, c = _i32(dev), ops.context(0)
    kc, vc, w, tables = _evict_case(dev, [60, 40], 2, 16, "float32", 3)
    n, page, stride = kc.shape[0], 16, kc.stride(0)
    t, lens, q, o = i(tables), i([60, 40]), torch.zeros((2, 2, 64), device=dev), torch.zeros((2, 2, 64), device=dev)
    at = lambda x, more=0: x.data_ptr() + 4 * more  # noqa: E731
    before = [x.clone() for x in (kc, vc, w, t, lens, q, o)]

    def refuses(name, *args):
        with pytest.raises(agpu.AgpuError) as e:
            c.call(name, *args)
        assert e.value.code == -5 and ("share memory" in str(e.value) or "overlap" in str(e.value))

    attend = lambda weights, q_at=at(q), o_at=at(o): ("agpu_paged_attention_weights", q_at, 128, 64, at(kc), at(vc), stride, stride, weights, 2 * page, at(t), at(lens), None, o_at, 2, 2, 2, 2, n, page,  # noqa: E731
                                                      t.shape[1], 0, 0, 64, 0)
    refuses(*attend(at(kc)))
    refuses(*attend(at(vc, stride * n - 1)))
    refuses(*attend(at(w), q_at=at(w, 2 * page * n - 4)))
    refuses(*attend(at(w), o_at=at(w, 2 * page * n - 4)))
    evict = lambda k, v, weights: ("agpu_paged_evict", k, v, stride, stride, weights, 2 * page, at(t), at(lens), 2, 2, n, page, t.shape[1], 30, 20, 4, 2, 64, 0)  # noqa: E731
    refuses(*evict(at(kc), at(vc), at(vc, 5 * stride)))
    refuses(*evict(at(kc), at(kc, 64), at(w)))
    ints = torch.zeros(64, dtype=torch.int32, device=dev)
    stack, out = ints[:20], ints[40:]

    def trim(lens_at=at(lens), tables_at=at(t), free=at(stack), count=at(ints, 30), kv=at(out), gone=at(out, 2), left=at(out, 4)):
        return "agpu_paged_trim", lens_at, tables_at, free, count, kv, gone, left, 2, t.shape[1], 20, page, 30, 20

    for bad in (dict(lens_at=at(out, 1)), dict(lens_at=at(out, 3)), dict(lens_at=at(out, 4)), dict(tables_at=at(out, 1 - t.numel())), dict(tables_at=at(stack, 19)), dict(count=at(stack, 19)), dict(count=at(out, 4)),
                dict(kv=at(out, 1)), dict(gone=at(out, 4)), dict(left=at(stack, 7)), dict(kv=at(stack, 19)), dict(lens_at=at(stack, 3))):
        refuses(*trim(**bad))
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip((kc, vc, w, t, lens, q, o), before)) and not ints.any()
    c.call(*trim(lens_at=at(lens), count=at(ints, 20), kv=at(out, 2), gone=at(out), left=at(out, 4)))
    torch.cuda.synchronize()
    assert out[:5].tolist() == [40, 20, 20, 20, 3] and stack[:4].tolist() == [*tables[0, 2:4], tables[1, 2], 0]
