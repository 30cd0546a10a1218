"""Several requests over a KV cache in pages: paged_plan, paged_kv_append and paged_attention against plain forms in 64 bits, and together."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

TYPES = ["float32", "float16", "bfloat16"]


def _cache(torch, g, dev, pages, heads, page, type_):
    return tuple(torch.randn((pages, heads, page, 64), generator=g, device=dev).to(getattr(torch, type_)) for _ in range(2))


def _tables(rng, lens, page, pages, width=None):
    """Pages of a shuffled pool for requests of these lengths; entries that nobody needs hold nonsense."""
    order, at = rng.permutation(pages), 0
    held = [-(-n // page) for n in lens]
    width = max(held, default=0) if width is None else width
    t = rng.choice(np.array([-1, -2**31, 2**31 - 1, pages, 0]), (len(lens), width))
    for b, h in enumerate(held):
        t[b, :h] = order[at:at + h]
        at += h
    assert at <= pages
    return t.astype(np.int32)


def attend64(q, k_cache, v_cache, tables, kv_lens, start, window=0, sinks=0):
    """The definition in 64 bits, row by row of the requests, on the CPU; rows of nobody NaN.  Also, per element, a bound of what fp32 may be off by."""
    import torch
    q, kc, vc = (x.detach().cpu().double() for x in (q, k_cache, v_cache))
    pages, heads, page, _ = kc.shape
    group = q.shape[1] // heads
    out, tol = torch.full(q.shape, float("nan"), dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    for b, kv in enumerate(kv_lens):
        n = start[b + 1] - start[b]
        if n == 0:
            continue
        ids = torch.as_tensor(np.asarray(tables[b][:-(-max(kv, 0) // page)], dtype=np.int64))
        real = (ids >= 0) & (ids < pages)
        there = real.repeat_interleave(page)[:kv]
        k, v = (c[torch.where(real, ids, 0)].transpose(0, 1).reshape(heads, -1, 64)[:, :max(kv, 0)] for c in (kc, vc))
        pos, j = torch.arange(kv - n, kv)[:, None], torch.arange(max(kv, 0))[None]
        seen = (j <= pos) & there
        if window:
            seen = seen & ((pos - j < window) | (j < sinks))
        for h in range(q.shape[1]):
            rows, kh, vh = q[start[b]:start[b + 1], h], k[h // group], v[h // group]
            # what nobody sees is nothing, whatever it is
            kh, vh = torch.where(seen.any(0)[:, None], kh, 0.0), torch.where(seen.any(0)[:, None], vh, 0.0)
            s = torch.where(seen, rows @ kh.T / 8, -torch.inf)
            top = s.amax(1, keepdim=True) if kv > 0 else torch.zeros(n, 1)
            w = torch.where(seen, torch.exp(s - torch.where(top == -torch.inf, 0.0, top)), 0.0)
            total = w.sum(1, keepdim=True)
            if torch.isfinite(vh).all():
                o = w @ vh
            else:  # 0 times infinity is not part of a sum over what is seen
                o = torch.stack([(w[i][seen[i]][:, None] * vh[seen[i]]).sum(0) for i in range(n)])
            out[start[b]:start[b + 1], h] = torch.where(total > 0, o / total, 0.0)
            # A score of 64 products in fp32 (one more rounding for q, one for the maximum's subtraction): 67 half steps of its sum of magnitudes; the exponential 2^-22 and a
            # half step of its argument; a weight counts in numerator and denominator, whose sums of n terms go through n / 16 + 100 additions.
            size = torch.where(seen, rows.abs() @ kh.abs().T / 8, 0.0).amax(1, keepdim=True) if kv > 0 else torch.zeros(n, 1)
            off = 2 * (size * (67 + 2) * 2.0**-24 + 2.0**-21) + 2 * (seen.sum(1, keepdim=True) / 16 + 100) * 2.0**-24
            tol[start[b]:start[b + 1], h] = off * ((w @ vh.abs().nan_to_num(0, 0, 0)) / torch.where(total > 0, total, 1.0)) + 1e-37
    return out, tol


def check(got, want, tol):
    import torch
    got = got.detach().cpu().double()
    of_someone = ~want.isnan()
    bad = of_someone & ~((got - want).abs() <= tol) & (got != want)
    assert not bad.any(), f"{int(bad.sum())} of {int(of_someone.sum())} off, the worst by {float(torch.where(bad, (got - want).abs() / tol, 0).max()):.3g} of the bound, " \
                          f"first at {bad.nonzero()[0].tolist()}"


# (kv, new) of the requests
BATCHES = {
    "one token": [(1, 1)],
    "one of many": [(777, 1)],
    "tokens": [(1, 1), (2, 1), (15, 1), (16, 1), (17, 1), (300, 1), (1030, 1), (64, 1)],
    "with idle ones": [(0, 0), (40, 1), (7, 0), (0, 0), (129, 1), (33, 0)],
    "chunks": [(5, 5), (33, 33), (100, 60), (257, 128), (300, 129), (64, 64)],
    "mixed": [(400, 1), (200, 150), (31, 1), (260, 9), (700, 3), (90, 90), (1, 1)],
    "one long": [(3000, 1)],
    "long chunk": [(1100, 300)],
}


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("heads,kv_heads,page", [(3, 3, 16), (4, 2, 7), (8, 2, 64), (5, 1, 1), (8, 1, 100), (11, 1, 32)])
@pytest.mark.parametrize("batch", list(BATCHES))
def test_attention(agpu, dev, type_, heads, kv_heads, page, batch):
    import torch
    from async_gpu_amd import ops
    lens, new = zip(*BATCHES[batch])
    rng, g = np.random.default_rng(heads * page + len(batch)), torch.Generator(device=dev).manual_seed(page)
    pages = sum(-(-n // page) for n in lens) + 2
    kc, vc = _cache(torch, g, dev, pages, kv_heads, page, type_)
    tables, start = _tables(rng, lens, page, pages), np.concatenate([[0], np.cumsum(new)]).tolist()
    q = torch.randn((start[-1], heads, 64), generator=g, device=dev) * 1.5
    i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=dev)  # noqa: E731
    for window, sinks in ((0, 0), (50, 3)) if page in (7, 16, 64) else ((0, 0),):
        got = ops.paged_attention(q, kc, vc, i32(tables), i32(lens), i32(start), window, sinks)
        again = ops.paged_attention(q, kc, vc, i32(tables), i32(lens), i32(start), window, sinks)
        check(got, *attend64(q, kc, vc, tables, lens, start, window, sinks))
        assert torch.equal(got, again)
        if all(n == 1 for n in new):
            assert torch.equal(got, ops.paged_attention(q, kc, vc, i32(tables), i32(lens), window=window, sinks=sinks))


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (17, 0), (64, 64), (200, 5), (0, 9), (5000, 4), (250, 400)])
@pytest.mark.parametrize("type_", ["float32", "bfloat16"])
def test_windows(agpu, dev, window, sinks, type_):
    import torch
    from async_gpu_amd import ops
    lens, new = [900, 1, 350, 700, 60], [1, 1, 200, 140, 60]
    rng, g = np.random.default_rng(window), torch.Generator(device=dev).manual_seed(sinks)
    kc, vc = _cache(torch, g, dev, 140, 2, 16, type_)
    tables, start = _tables(rng, lens, 16, 140), np.concatenate([[0], np.cumsum(new)]).tolist()
    q = torch.randn((start[-1], 4, 64), generator=g, device=dev)
    i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=dev)  # noqa: E731
    check(ops.paged_attention(q, kc, vc, i32(tables), i32(lens), i32(start), window, sinks), *attend64(q, kc, vc, tables, lens, start, window, sinks))
    # with no more than the pages that somebody sees
    dead = tables.copy()
    for b, (kv, n) in enumerate(zip(lens, new)):
        for j in range(0, kv, 16):
            if window and all(not (p - x < window or x < sinks) for x in range(j, min(j + 16, kv)) for p in (max(kv - n, x),)):
                dead[b, j // 16] = -1
    got = ops.paged_attention(q, kc, vc, i32(dead), i32(lens), i32(start), window, sinks)
    assert torch.equal(got, ops.paged_attention(q, kc, vc, i32(tables), i32(lens), i32(start), window, sinks))


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("filler", [float("nan"), float("inf"), "lowest"])
def test_what_is_not_seen_does_not_count(agpu, dev, type_, filler):
    """Places of pages behind the last position, pages of nobody, and positions after a row's own: NaN, infinities and the type's lowest value there change no bit."""
    import torch
    from async_gpu_amd import ops
    lens, new, page = [70, 37, 200, 130], [1, 37, 77, 1], 16
    rng, g = np.random.default_rng(3), torch.Generator(device=dev).manual_seed(4)
    kc, vc = _cache(torch, g, dev, 40, 2, page, type_)
    x = torch.finfo(kc.dtype).min if filler == "lowest" else filler
    tables, start = _tables(rng, lens, page, 40), np.concatenate([[0], np.cumsum(new)]).tolist()
    q = torch.randn((start[-1], 4, 64), generator=g, device=dev)
    i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=dev)  # noqa: E731
    want = ops.paged_attention(q, kc, vc, i32(tables), i32(lens), i32(start))
    held = torch.zeros(40, page, dtype=torch.bool)
    for b, n in enumerate(lens):
        for p in range(n):
            held[tables[b, p // page], p % page] = True
    held = held.to(dev)[:, None, :, None]
    kb, vb = (torch.where(held, c.float(), x).to(c.dtype) for c in (kc, vc))
    assert torch.equal(want, ops.paged_attention(q, kb, vb, i32(tables), i32(lens), i32(start)))
    if filler == "lowest":
        return
    # the last five positions of request 2: rows before them are as they were, rows from there on are what the formula says
    for p in range(195, 200):
        kb[tables[2, p // page], :, p % page] = 0.5
        vb[tables[2, p // page], :, p % page, ::3] = x
    got = ops.paged_attention(q, kb, vb, i32(tables), i32(lens), i32(start))
    first = start[2] + 195 - (200 - 77)
    others = torch.ones(start[-1], dtype=torch.bool)
    others[first:start[3]] = False
    assert torch.equal(got[others], want[others])
    ref, tol = attend64(q, kb, vb, tables, lens, start)
    rows = got[first:start[3]].cpu().double()
    assert not torch.isfinite(rows[:, :, ::3]).any() and torch.isfinite(rows[:, :, 1::3]).all()
    if filler == float("inf"):
        assert (rows[:, :, ::3] == float("inf")).all()


def test_rows_that_see_nothing_and_rows_of_nobody(agpu, dev):
    import torch
    from async_gpu_amd import ops
    g = torch.Generator(device=dev).manual_seed(1)
    kc, vc = _cache(torch, g, dev, 12, 3, 8, "float32")
    i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=dev)  # noqa: E731
    # 0 positions; 3 of which 5 rows are said to be the last: the first two lie before position 0; a table of two pages for 20 positions
    lens, new = [0, 3, 20, -4], [2, 5, 3, 1]
    start = np.concatenate([[0], np.cumsum(new)]).tolist()
    tables = np.array([[0, 1], [2, 3], [4, 5], [6, 7]], np.int32)
    q = torch.randn((start[-1] + 4, 3, 64), generator=g, device=dev)
    out = torch.full_like(q, 7.0)
    got = ops.paged_attention(q, kc, vc, i32(tables), i32(lens), i32(start), out=out)
    assert got is out and (out[start[-1]:] == 7.0).all()
    assert (out[:4] == 0).all() and (out[start[3]:start[4]] == 0).all() and (out[4:7] != 0).all()
    check(out[:start[2]], *attend64(q[:start[2]], kc, vc, tables, lens[:2], start[:3]))
    # positions 17, 18, 19 of the third: they see the 16 keys that the table has pages for
    ref, tol = attend64(q[start[2]:start[3]], kc, vc, tables[2:3], [16], [0, 1])
    check(out[start[2]:start[2] + 1], ref[:1], tol[:1])
    # pages outside the cache are not seen
    bad = np.array([[3, -1, 5, 99], [12, 12, -7, 2**31 - 1], [1, 2, 3, 4]], np.int32)
    lens, start = [32, 32, 32], [0, 4, 5, 6]
    q = q[:6].contiguous()
    got = ops.paged_attention(q, kc, vc, i32(bad), i32(lens), i32(start))
    check(got, *attend64(q, kc, vc, bad, lens, start))
    assert (got[4] == 0).all()
    # no rows, no requests
    assert ops.paged_attention(q[:0], kc, vc, i32(bad), i32(lens), i32([0, 0, 0, 0])).shape == (0, 3, 64)
    assert ops.paged_attention(q[:0], kc, vc, i32(bad[:0]), i32([]), i32([0])).shape == (0, 3, 64)
    keep = torch.full_like(q, 3.0)
    assert (ops.paged_attention(q, kc, vc, i32(bad[:0]), i32([]), i32([0]), out=keep) == 3.0).all()
    assert (ops.paged_attention(q, kc, vc, i32(np.zeros((3, 0))), i32(lens), i32(start)) == 0).all()


@pytest.mark.parametrize("type_", ["float32", "float16"])
def test_strides(agpu, dev, type_):
    """q and K, V as slices of QKV rows, at an odd float, and head by head; K and V interleaved by pages, and one layer of several."""
    import torch
    from async_gpu_amd import ops
    lens, new, page, H = [100, 50, 300, 33], [1, 50, 140, 1], 16, 5
    rng, g = np.random.default_rng(5), torch.Generator(device=dev).manual_seed(6)
    pages = 40
    tables, start = _tables(rng, lens, page, pages), np.concatenate([[0], np.cumsum(new)]).tolist()
    T = start[-1]
    i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=dev)  # noqa: E731
    pool = torch.randn((pages, 3, 2, H, page, 64), generator=g, device=dev).to(getattr(torch, type_))  # [page, layer, K or V]
    kc, vc = pool[:, 1, 0], pool[:, 1, 1]
    before = pool.clone()
    qkv = torch.randn(T * (3 * H * 64 + 3) + 1, generator=g, device=dev)[1:].view(T, 3 * H * 64 + 3)[:, :3 * H * 64].unflatten(1, (3, H, 64))
    q, k, v = qkv[:, 0], qkv[:, 1], qkv[:, 2]
    slots = np.concatenate([[tables[b, p // page] * page + p % page for p in range(kv - n, kv)] for b, (kv, n) in enumerate(zip(lens, new))])
    got_k, got_v = ops.paged_kv_append(k, v, kc, vc, i32(slots))
    assert got_k is kc and got_v is vc
    for s, p in enumerate(slots):
        before[p // page, 1, 0, :, p % page] = k[s].to(pool.dtype)
        before[p // page, 1, 1, :, p % page] = v[s].to(pool.dtype)
    assert torch.equal(pool, before)
    want = ops.paged_attention(q.contiguous(), kc.contiguous(), vc.contiguous(), i32(tables), i32(lens), i32(start))
    check(want, *attend64(q, kc, vc, tables, lens, start))
    assert torch.equal(want, ops.paged_attention(q, kc, vc, i32(tables), i32(lens), i32(start)))
    by_head = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(want, ops.paged_attention(by_head, kc, vc, i32(tables), i32(lens), i32(start)))
    one = q[:, :1].expand(T, H, 64)
    assert torch.equal(ops.paged_attention(one, kc, vc, i32(tables), i32(lens), i32(start)), ops.paged_attention(one.contiguous(), kc, vc, i32(tables), i32(lens), i32(start)))
    pool.zero_()
    by_head = k.transpose(0, 1).contiguous().transpose(0, 1)
    ops.paged_kv_append(by_head, v, kc, vc, i32(slots))
    assert torch.equal(pool[:, 1, 0].float(), before[:, 1, 0].float() * torch.isin(torch.arange(pages * page, device=dev).view(pages, 1, page, 1), i32(slots)))
    with pytest.raises(agpu.AgpuError):  # pages at 16 bytes
        odd = torch.zeros(pages * (H * page * 64 + 1), dtype=pool.dtype, device=dev).view(pages, -1)[:, :H * page * 64].unflatten(1, (H, page, 64))
        ops.paged_attention(q, odd, odd, i32(tables), i32(lens), i32(start))
    with pytest.raises(agpu.AgpuError):
        ops.paged_kv_append(k, v, kc[:1].expand(pages, H, page, 64), vc, i32(slots))


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("heads,page,tokens", [(1, 16, 1), (12, 16, 16), (3, 7, 50), (25, 64, 333), (2, 1, 40)])
def test_append_rounds_to_nearest(agpu, dev, type_, heads, page, tokens):
    import torch
    from async_gpu_amd import ops
    g, rng = torch.Generator(device=dev).manual_seed(tokens), np.random.default_rng(tokens)
    pages = -(-tokens // page) + 2
    kc, vc = _cache(torch, g, dev, pages, heads, page, type_)
    k, v = (torch.randn((tokens, heads, 64), generator=g, device=dev) * 10.0 ** torch.randint(-12, 6, (tokens, heads, 64), generator=g, device=dev) for _ in range(2))
    special = torch.tensor([0.0, -0.0, float("inf"), -float("inf"), float("nan"), 65504.0, 65519.9, 65520.0, 1e-45, 5.9e-8, 2.98e-8, 2.9e-8, 3.4e38, 1.00390625, 1.01171875, 1.00048828125,
                            1.00146484375, -3.39e38], device=dev)
    k[0, 0, :len(special)] = special
    v[-1, -1, -len(special):] = special
    slots = rng.permutation(pages * page)[:tokens].astype(np.int64)
    slots[rng.random(tokens) < 0.2] = -1
    slots[-1] = max(slots[-1], 0)
    if tokens > 20:
        slots[3:8] = [pages * page, 2**31 - 1, -2**31, -2, pages * page + 5]
    want_k, want_v = kc.clone(), vc.clone()
    for t, p in enumerate(slots):
        if 0 <= p < pages * page:
            want_k[p // page, :, p % page] = k[t].to(kc.dtype)
            want_v[p // page, :, p % page] = v[t].to(kc.dtype)
    ops.paged_kv_append(k, v, kc, vc, torch.tensor(slots, device=dev).int())
    for got, want in ((kc, want_k), (vc, want_v)):
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(1.0), want.nan_to_num(1.0))
    ops.paged_kv_append(k[:0], v[:0], kc, vc, torch.zeros(0, dtype=torch.int32, device=dev))


def plan64(cached, new, tables, stack, n_free, page, max_tokens):
    """paged_plan request by request, on lists."""
    tables, stack, rest = [list(r) for r in tables], list(stack[:n_free]), list(stack)
    for b, n in enumerate(new):
        if n < 0:
            stack += tables[b][:-(-cached[b] // page)]
    kv, start, slots, positions, full = [], [0], [], [], False
    for b, n in enumerate(new):
        have, want = -(-cached[b] // page), -(-(cached[b] + max(n, 0)) // page)
        too_long = want > len(tables[b])
        if n >= 0 and not too_long:
            full = full or want - have > len(stack) or len(slots) + n > max_tokens
        if n < 0 or too_long or full:
            kv.append(0 if n < 0 else cached[b])
            start.append(len(slots))
            continue
        for i in range(have, want):
            tables[b][i] = stack.pop()
        for p in range(cached[b], cached[b] + n):
            slots.append(tables[b][p // page] * page + p % page)
            positions.append(p)
        kv.append(cached[b] + n)
        start.append(len(slots))
    pad = max_tokens - len(slots)
    return kv, start, slots + [-1] * pad, positions + [0] * pad, [len(stack)], tables, stack + rest[len(stack):]


@pytest.mark.parametrize("batch,page,longest,spare,max_tokens", [(1, 16, 5, 3, 8), (1, 1, 1, 0, 0), (7, 16, 40, 100, 400), (7, 16, 40, 3, 400), (7, 16, 40, 100, 50), (64, 7, 100, 40, 1000),
                                                                 (257, 16, 1, 300, 257), (300, 33, 64, 1000, 20000), (1000, 16, 30, 200, 9000), (4096, 16, 20, 9000, 50000)])
def test_plan(agpu, dev, batch, page, longest, spare, max_tokens):
    import torch
    from async_gpu_amd import ops
    rng = np.random.default_rng(batch + spare)
    for trial in range(3):
        cached = rng.integers(0, 3 * longest + 1, batch)
        new = rng.integers(0, longest + 1, batch)
        new[rng.random(batch) < 0.1 * trial] = -rng.integers(1, 5)
        width = -(-(3 * longest + longest * (2 if trial < 2 else 1) // 2) // page)  # too narrow for some
        held = -(-cached // page)
        cached = np.where(held > width, width * page, cached)
        held = -(-cached // page)
        order = rng.permutation(int(held.sum()) + spare)
        tables = np.full((batch, width), -1)
        at = 0
        for b in range(batch):
            tables[b, :held[b]] = order[at:at + held[b]]
            at += held[b]
        stack = np.concatenate([order[at:], np.full(at, -9)])
        want = plan64(cached.tolist(), new.tolist(), tables.tolist(), stack.tolist(), spare, page, max_tokens)
        i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=dev)  # noqa: E731
        t, s, args = i32(tables), i32(stack), (i32(cached), i32(new))
        for _ in range(2):  # the same step once more finds what it needs where it was
            got = ops.paged_plan(*args, t, s, i32([spare]), page, max_tokens)
            for name, x, y in zip(("kv_lens", "query_start", "slots", "positions", "n_free", "block_tables", "free_pages"), (*got, t, s), want):
                assert np.array_equal(x.cpu().numpy(), np.asarray(y).reshape(x.shape)), (name, trial)


def test_plan_of_nobody_and_of_nonsense(agpu, dev):
    import torch
    from async_gpu_amd import ops
    i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=dev)  # noqa: E731
    kv, start, slots, pos, n = ops.paged_plan(i32([]), i32([]), i32(np.zeros((0, 4))), i32([5, 6]), i32([2]), 16, 3)
    assert kv.numel() == 0 and start.tolist() == [0] and slots.tolist() == [-1] * 3 and pos.tolist() == [0] * 3 and n.tolist() == [2]
    # lengths and counts out of range: nothing is read or written outside of what is there
    big = 2**31 - 1
    kv, start, slots, pos, n = ops.paged_plan(i32([-5, big, 3, 0]), i32([2, big, big, 2]), i32([[0, 1], [2, 3], [4, 5], [6, 7]]), i32([8, 9, 10]), i32([big]), 4, 6)
    assert kv.tolist() == [2, 8, 3, 2] and start.tolist() == [0, 2, 2, 2, 4] and n.tolist() == [1]
    assert slots.tolist() == [40, 41, 36, 37, -1, -1] and pos.tolist() == [0, 1, 0, 1, 0, 0]
    with pytest.raises(agpu.AgpuError):
        ops.paged_plan(i32(np.zeros(4097)), i32(np.zeros(4097)), i32(np.zeros((4097, 1))), i32([1]), i32([1]), 16, 3)


def test_a_cache_beyond_32_bits(agpu, dev):
    """Elements of a cache beyond number 2^32."""
    import torch
    from async_gpu_amd import ops
    page, H = 64, 4
    pages = (1 << 32) // (page * H * 64) + 40
    kc, vc = (torch.empty((pages, H, page, 64), dtype=torch.bfloat16, device=dev) for _ in range(2))
    lens, new = [200, 150, 90], [1, 140, 3]
    g = torch.Generator(device=dev).manual_seed(2)
    ids = [pages - 1, 3, pages - 2, 4, pages - 7, 0, pages - 9, 8, pages - 11]
    kc[ids], vc[ids] = (torch.randn((len(ids), H, page, 64), generator=g, device=dev).bfloat16() for _ in range(2))
    tables = np.full((3, 4), -1)
    tables[0, :4], tables[1, :3], tables[2, :2] = ids[:4], ids[4:7], ids[7:]
    start = np.concatenate([[0], np.cumsum(new)]).tolist()
    i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=dev)  # noqa: E731
    slots = np.concatenate([[tables[b, p // page] * page + p % page for p in range(kv - n, kv)] for b, (kv, n) in enumerate(zip(lens, new))])
    k, v, q = (torch.randn((start[-1], h, 64), generator=g, device=dev) for h in (H, H, 2 * H))
    ops.paged_kv_append(k, v, kc, vc, i32(slots))
    for t in (0, 5, start[-1] - 1):
        assert torch.equal(kc[slots[t] // page, :, slots[t] % page], k[t].bfloat16()) and torch.equal(vc[slots[t] // page, :, slots[t] % page], v[t].bfloat16())
    got = ops.paged_attention(q, kc, vc, i32(tables), i32(lens), i32(start))
    small = {p: i for i, p in enumerate(ids)}
    check(got, *attend64(q, kc[ids], vc[ids], np.vectorize(lambda p: small.get(p, -1))(tables), lens, start))


@pytest.mark.parametrize("type_", ["float32", "bfloat16"])
@pytest.mark.parametrize("heads,kv_heads", [(2, 2), (6, 1)])
@pytest.mark.parametrize("kind", ["tokens", "tokens of a few requests", "mixed"])
def test_more_requests_than_are_numbered(agpu, dev, type_, heads, kv_heads, kind):
    """Hundreds of requests, whose work a workgroup no longer counts before it begins."""
    import torch
    from async_gpu_amd import ops
    rng, g = np.random.default_rng(heads), torch.Generator(device=dev).manual_seed(1)
    B, page = 311, 16
    lens = rng.integers(0, 90, B)
    lens[[5, 200]] = 2500, 1300
    if kind == "tokens":
        new = np.ones(B, int)
    elif kind == "tokens of a few requests":
        new = (rng.random(B) < 0.9).astype(int)
    else:
        new = np.minimum(rng.choice([0, 1, 1, 3, 9, 60, 140], B), lens)
        new[5] = 290
    lens = np.maximum(lens, new)
    pages = int((-(-lens // page)).sum()) + 1
    kc, vc = _cache(torch, g, dev, pages, kv_heads, page, type_)
    tables, start = _tables(rng, lens.tolist(), page, pages), np.concatenate([[0], np.cumsum(new)]).tolist()
    i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=dev)  # noqa: E731
    q = torch.randn((start[-1] + 3, heads, 64), generator=g, device=dev)
    for window, sinks in ((0, 0), (30, 2)):
        out = torch.full_like(q, 7.0)
        ops.paged_attention(q, kc, vc, i32(tables), i32(lens), i32(start), window, sinks, out=out)
        check(out[:start[-1]], *attend64(q[:start[-1]], kc, vc, tables, lens.tolist(), start, window, sinks))
        assert (out[start[-1]:] == 7.0).all()


@pytest.mark.parametrize("type_", ["float32", "float16"])
@pytest.mark.parametrize("window,sinks", [(0, 0), (260, 3)])
def test_more_tiles_than_find_a_place_at_once(agpu, dev, type_, window, sinks):
    """Prompts of so many rows that a workgroup takes several tiles, the second time in the opposite order."""
    import torch
    from async_gpu_amd import ops
    rng, g = np.random.default_rng(21), torch.Generator(device=dev).manual_seed(21)
    lens, new, heads, page = [1100, 1400, 30, 900, 1], [1100, 900, 2, 300, 1], 24, 16
    kc, vc = _cache(torch, g, dev, 230, heads, page, type_)
    tables, start = _tables(rng, lens, page, 230), np.concatenate([[0], np.cumsum(new)]).tolist()
    q = torch.randn((start[-1], heads, 64), generator=g, device=dev)
    i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=dev)  # noqa: E731
    args = (q, kc, vc, i32(tables), i32(lens), i32(start), window, sinks)
    got = ops.paged_attention(*args)
    check(got, *attend64(q, kc, vc, tables, lens, start, window, sinks))
    assert all(torch.equal(got, ops.paged_attention(*args)) for _ in range(3))


@pytest.mark.parametrize("type_", TYPES)
def test_little_scratch(agpu, dev, type_):
    """With a scratch of 1 MiB rows are cut into fewer runs; the results are as good."""
    import torch
    from async_gpu_amd import ops
    rng, g = np.random.default_rng(5), torch.Generator(device=dev).manual_seed(2)
    lens, new = [3000, 2100, 1700, 40, 1200], [1, 300, 5, 40, 140]
    kc, vc = _cache(torch, g, dev, 600, 4, 16, type_)
    tables, start = _tables(rng, lens, 16, 600), np.concatenate([[0], np.cumsum(new)]).tolist()
    q = torch.randn((start[-1], 8, 64), generator=g, device=dev)
    i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=dev)  # noqa: E731
    args = (kc, vc, i32(tables), i32(lens))
    small = torch.empty(1 << 20, dtype=torch.uint8, device=dev)
    c = ops.context(0)
    c.call("agpu_ctx_set_workspace", small.data_ptr(), small.numel())
    try:
        rows, tokens = ops.paged_attention(q, *args, i32(start)), ops.paged_attention(q[:5], *args)
        torch.cuda.synchronize()
    finally:
        c.call("agpu_ctx_set_workspace", None, 0)
    check(rows, *attend64(q, kc, vc, tables, lens, start))
    check(tokens, *attend64(q[:5], kc, vc, tables, lens, [0, 1, 2, 3, 4, 5]))


def test_hand_over_of_runs_under_the_memory_model(agpu, dev):
    """With fences around the tickets the results are the same bits, and tickets are left as they were found."""
    import torch
    from async_gpu_amd import ops
    lens, new = [3000, 2100, 700, 40], [1, 100, 5, 40]
    rng, g = np.random.default_rng(8), torch.Generator(device=dev).manual_seed(9)
    kc, vc = _cache(torch, g, dev, 400, 2, 16, "float32")
    tables, start = _tables(rng, lens, 16, 400), np.concatenate([[0], np.cumsum(new)]).tolist()
    q = torch.randn((start[-1], 2, 64), generator=g, device=dev)
    i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=dev)  # noqa: E731
    args = (kc, vc, i32(tables), i32(lens))
    c = ops.context(0)
    plain = ops.paged_attention(q, *args, i32(start)), ops.paged_attention(q[:4], *args)
    try:
        c.call("agpu_ctx_set_strict_sync", 1)
        strict = ops.paged_attention(q, *args, i32(start)), ops.paged_attention(q[:4], *args)
    finally:
        c.call("agpu_ctx_set_strict_sync", 0)
    for a, b in zip(plain, strict):
        assert torch.equal(a, b)
    check(plain[0], *attend64(q, kc, vc, tables, lens, start))


def test_captured_step(agpu, dev):
    """A step in a graph: replayed with other lengths, tables and rows, between eager work of the program's own."""
    import torch
    from async_gpu_amd import ops
    B, H, page, width, T = 5, 3, 16, 20, 40
    g, rng = torch.Generator(device=dev).manual_seed(3), np.random.default_rng(4)
    pages = B * width
    i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=dev)  # noqa: E731
    state = dict(cached=i32(np.zeros(B)), new=i32(np.zeros(B)), tables=i32(np.full((B, width), -1)), stack=i32(rng.permutation(pages)), n=i32([pages]))
    kc, vc = _cache(torch, g, dev, pages, H, page, "float32")
    qkv, u = torch.zeros((T, 3, H, 64), device=dev), torch.zeros(B, device=dev)
    head = torch.randn((H * 64, 500), generator=g, device=dev)

    def step(s, kc, vc):
        kv, start, slots, pos, n = ops.paged_plan(s["cached"], s["new"], s["tables"], s["stack"], s["n"], page, T)
        ops.paged_kv_append(qkv[:, 1], qkv[:, 2], kc, vc, slots)
        out = torch.zeros((T, H, 64), device=dev)
        ops.paged_attention(qkv[:, 0], kc, vc, s["tables"], kv, start, 100, 2, out=out)
        last = out[(start[1:] - 1).clamp(min=0).long()].reshape(B, -1)
        return kv, start, slots, pos, n, out, ops.sample(ops.gemm_f32(last, head), u, 0.9, 50, 0.9)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step({k: v.clone() for k, v in state.items()}, kc.clone(), vc.clone())
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):  # the stream that has its context already
        made = step(state, kc, vc)
    eager, ek, ev = {k: v.clone() for k, v in state.items()}, kc.clone(), vc.clone()
    for i in range(8):
        new = rng.integers(0, 9, B) if i else np.array([8, 8, 8, 8, 8])
        new[rng.random(B) < (0.2 if i > 3 else 0)] = -1
        for s in (state, eager):
            s["new"].copy_(i32(new))
        qkv.copy_(torch.randn(qkv.shape, generator=g, device=dev))
        u.copy_(torch.rand(B, generator=g, device=dev))
        want = step(eager, ek, ev)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(made, want):
            assert torch.equal(x, y), i
        assert torch.equal(kc, ek) and torch.equal(state["tables"], eager["tables"]) and torch.equal(state["stack"], eager["stack"])
        for s, out in ((state, made), (eager, want)):
            s["cached"].copy_(out[0])
            s["n"].copy_(out[4])


def test_streams(agpu, dev):
    """Two streams at once, each with its own scratch, against the default one."""
    import torch
    from async_gpu_amd import ops
    lens, new = [2500, 1800, 300], [1, 120, 300]
    rng, g = np.random.default_rng(8), torch.Generator(device=dev).manual_seed(9)
    kc, vc = _cache(torch, g, dev, 300, 4, 16, "float16")
    tables, start = _tables(rng, lens, 16, 300), np.concatenate([[0], np.cumsum(new)]).tolist()
    i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=dev)  # noqa: E731
    args = (kc, vc, i32(tables), i32(lens), i32(start))
    q = [torch.randn((start[-1], 4, 64), generator=g, device=dev) for _ in range(2)]
    want = [ops.paged_attention(x, *args) for x in q]
    streams = [torch.cuda.Stream() for _ in q]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ops.paged_attention(q[i], *args))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(want[i], x) for x in got[i])


@pytest.mark.parametrize("type_", ["float32", "bfloat16"])
def test_a_server(agpu, dev, type_):
    """Requests that come in chunks of their prompts, decode, end and make room for others, over one layer: what each of them gets is what attention over its
    own K and V gives, pages belong to one request at a time, and draws are those of the definition."""
    import torch
    from async_gpu_amd import ops
    from test_gpu_sample import draw64
    H, page, width, B, T, vocab = 4, 16, 12, 6, 96, 700
    pages = 40
    g, rng = torch.Generator(device=dev).manual_seed(12), np.random.default_rng(13)
    i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=dev)  # noqa: E731
    kc, vc = _cache(torch, g, dev, pages, H, page, type_)
    kc.fill_(float("nan")), vc.fill_(float("nan"))
    tables, stack, n_free, kv = i32(np.full((B, width), -1)), i32(rng.permutation(pages)), i32([pages]), i32(np.zeros(B))
    head = torch.randn((H * 64, vocab), generator=g, device=dev)
    mine = [([], []) for _ in range(B)]  # K and V rows of each request
    left = [int(x) for x in rng.integers(20, 120, B)]  # of its prompt
    life = [int(x) for x in rng.integers(2, 12, B)]
    served_total = 0
    for step in range(25):
        new = []
        for b in range(B):
            if left[b] == 0 and life[b] == 0:  # ended: another one in the next step
                new.append(-1)
            elif left[b] > 0:
                new.append(min(left[b], int(rng.integers(1, 60))))
            else:
                new.append(1)
        qkv = torch.randn((T, 3, H, 64), generator=g, device=dev)
        u = torch.rand(B, generator=g, device=dev)
        was = kv.tolist()
        kv, start, slots, positions, n_free = ops.paged_plan(kv, i32(new), tables, stack, n_free, page, T)
        ops.paged_kv_append(qkv[:, 1], qkv[:, 2], kc, vc, slots)
        out = ops.paged_attention(qkv[:, 0], kc, vc, tables, kv, start)
        st, now = start.tolist(), kv.tolist()
        owned = [p for b in range(B) for p in tables[b, :-(-now[b] // page)].tolist()]
        assert len(set(owned)) == len(owned) and len(owned) + int(n_free) == pages
        assert sorted(owned + stack[:int(n_free)].tolist()) == list(range(pages))
        for b in range(B):
            n = st[b + 1] - st[b]
            assert positions[st[b]:st[b + 1]].tolist() == list(range(now[b] - n, now[b])) and n in (0, max(new[b], 0))
            if new[b] < 0:
                mine[b], left[b], life[b] = ([], []), int(rng.integers(20, 120)), int(rng.integers(2, 12))
                assert now[b] == 0
                continue
            assert now[b] == was[b] + n
            if n == 0:
                continue
            served_total += n
            left[b], life[b] = max(left[b] - n, 0), life[b] - (1 if left[b] == 0 else 0)
            for rows, i in zip(mine[b], (1, 2)):
                rows.append(qkv[st[b]:st[b + 1], i].to(kc.dtype).float())
            k, v = (torch.cat(rows).transpose(0, 1).contiguous() for rows in mine[b])
            one = ops.attention(qkv[st[b]:st[b + 1], 0].transpose(0, 1).contiguous(), k, v, kv_len=now[b], q_offset=now[b] - n)
            ref, tol = attend64(qkv[st[b]:st[b + 1], 0], k.transpose(0, 1).reshape(1, now[b], H, 64).transpose(1, 2), v.transpose(0, 1).reshape(1, now[b], H, 64).transpose(1, 2),
                                [[0]], [now[b]], [0, n])
            check(out[st[b]:st[b + 1]], ref, tol)
            check(one.transpose(0, 1), ref, 4 * tol)  # (the contiguous operator's own arithmetic)
        last = out[(start[1:] - 1).clamp(min=0).long()].reshape(B, -1)
        logits = ops.gemm_f32(last.nan_to_num(0.0), head)
        tokens = ops.sample(logits, u, 0.8, 30, 0.95)
        assert tokens.tolist() == draw64(logits.cpu().numpy(), u.cpu().numpy(), 0.8, 30, 0.95, 0.0)
    assert served_total > 500
