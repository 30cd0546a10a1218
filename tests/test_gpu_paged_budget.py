"""A cache with a budget: paged_attention_weights against sums of softmax weights in 64 bits, paged_evict and paged_trim against their definitions, and all of them together."""
import numpy as np
import pytest
from test_gpu_paged import BATCHES, TYPES, _cache, _tables, attend64, check

pytestmark = pytest.mark.gpu


def _i32(dev):
    import torch
    return lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=dev)


def given64(q, k_cache, weights, tables, kv_lens, start, window=0, sinks=0):
    """The weights after a call, in 64 bits on the CPU, and a bound of what fp32 may be off by."""
    import torch
    q, kc, w = (x.detach().cpu().double() for x in (q, k_cache, weights))
    pages, heads, page, _ = kc.shape
    group, tol, there_all = q.shape[1] // heads, torch.zeros_like(w), q.shape[0]
    for b, kv in enumerate(kv_lens):
        n = start[b + 1] - start[b]
        have = min(start[b + 1], there_all) - start[b]
        m = min(max(kv, 0), len(tables[b]) * page)
        if have <= 0 or m == 0:
            continue
        j = torch.arange(m)
        ids = torch.as_tensor(np.asarray(tables[b], dtype=np.int64))[j // page]
        real = (ids >= 0) & (ids < pages)
        at, place = ids[real], (j % page)[real]
        k = torch.zeros(heads, m, 64, dtype=torch.float64)
        k[:, real] = kc[at, :, place].transpose(0, 1)
        pos = torch.arange(kv - n, kv - n + have)[:, None]
        seen = (j <= pos) & real
        if window:
            seen = seen & ((pos - j < window) | (j < sinks))
        for h in range(heads):
            given, off = torch.zeros(m, dtype=torch.float64), torch.zeros(m, dtype=torch.float64)
            for hq in range(h * group, (h + 1) * group):
                rows = q[start[b]:start[b] + have, hq]
                s = torch.where(seen, rows @ k[h].T / 8, -torch.inf)
                top = s.amax(1, keepdim=True)
                p = torch.where(seen, torch.exp(s - torch.where(top == -torch.inf, 0.0, top)), 0.0)
                p = p / p.sum(1, keepdim=True).clamp(min=1e-300)
                # As the rows' results: a score twice (in the weight and in the sum it is divided by), 67 half steps of its sum of magnitudes and two of its units, the
                # exponential 2^-22 and a half step of its argument; the sum over the keys n / 16 + 100 additions.
                size = torch.where(seen, rows.abs() @ k[h].abs().T / 8, 0.0).amax(1, keepdim=True)
                e = 2 * (size * (67 + 2) * 2.0**-24 + 2.0**-21) + (seen.sum(1, keepdim=True) / 16 + 100) * 2.0**-24
                given += p.sum(0)
                off += (p * e).sum(0)
            old = torch.where(j < kv - n, w[ids.clamp(0, pages - 1), h, j % page], 0.0)
            new = old + given
            # the sum over rows and heads: each of its terms goes through as many additions as there are steps of 32 rows, and 8 more
            off += given * (have * group / 32 + 8) * 2.0**-24 + new.abs() * 2.0**-24 + 1e-37 * have * group
            w[at, h, place], tol[at, h, place] = new[real], off[real]
    return w, tol


def _weights(torch, g, dev, cache):
    return torch.rand(cache.shape[:3], generator=g, device=dev) * 3


def _state(dev, lens, new, heads, kv_heads, page, type_, seed, spare=2):
    import torch
    rng, g = np.random.default_rng(seed), torch.Generator(device=dev).manual_seed(seed)
    pages = sum(-(-max(n, 0) // page) for n in lens) + spare
    kc, vc = _cache(torch, g, dev, pages, kv_heads, page, type_)
    tables, start = _tables(rng, [max(n, 0) for n in lens], page, pages), np.concatenate([[0], np.cumsum(new)]).tolist()
    q = torch.randn((start[-1], heads, 64), generator=g, device=dev) * 1.5
    return kc, vc, _weights(torch, g, dev, kc), tables, start, q


def _attend(dev, q, kc, vc, w, tables, lens, start, window=0, sinks=0, **kw):
    from async_gpu_amd import ops
    i = _i32(dev)
    return ops.paged_attention_weights(q, kc, vc, w, i(tables), i(lens), None if start is None else i(start), window, sinks, **kw)


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("heads,kv_heads,page", [(3, 3, 16), (4, 2, 7), (8, 2, 64), (5, 1, 1), (8, 1, 100), (11, 1, 32)])
@pytest.mark.parametrize("batch", list(BATCHES))
def test_weights(agpu, dev, type_, heads, kv_heads, page, batch):
    import torch
    from async_gpu_amd import ops
    lens, new = zip(*BATCHES[batch])
    kc, vc, w, tables, start, q = _state(dev, lens, new, heads, kv_heads, page, type_, heads * page + len(batch))
    for window, sinks in ((0, 0), (50, 3)) if page in (7, 16, 64) else ((0, 0),):
        own = w.clone()
        out, same = _attend(dev, q, kc, vc, own, tables, lens, start, window, sinks)
        assert same is own
        check(own, *given64(q, kc, w, tables, lens, start, window, sinks))
        check(out, *attend64(q, kc, vc, tables, lens, start, window, sinks))
        i = _i32(dev)
        assert torch.equal(out, ops.paged_attention(q, kc, vc, i(tables), i(lens), i(start), window, sinks)) or q.shape[0] > len(lens)  # (runs may be cut otherwise)
        again = w.clone()
        _attend(dev, q, kc, vc, again, tables, lens, start, window, sinks)
        assert torch.equal(own, again)
        if all(n == 1 for n in new):
            again = w.clone()
            _attend(dev, q, kc, vc, again, tables, lens, None, window, sinks)
            assert torch.equal(own, again)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (17, 0), (64, 64), (200, 5), (0, 9), (5000, 4), (250, 400), (2**31 - 1, 2**31 - 1)])
@pytest.mark.parametrize("type_", ["float32", "bfloat16"])
def test_windows(agpu, dev, window, sinks, type_):
    lens, new = [900, 1, 350, 700, 60, 420], [1, 1, 200, 140, 60, 3]
    kc, vc, w, tables, start, q = _state(dev, lens, new, 4, 2, 16, type_, window % 1000)
    own = w.clone()
    _attend(dev, q, kc, vc, own, tables, lens, start, window, sinks)
    check(own, *given64(q, kc, w, tables, lens, start, window, sinks))


def test_weights_add_up(agpu, dev):
    """Over the keys of a request each row gives one a head: after a prompt in chunks and some tokens there is that much more."""
    import torch
    kc, vc, w, tables, _, _ = _state(dev, [400, 90], [0, 0], 4, 2, 16, "float32", 1)
    g, w = torch.Generator(device=dev).manual_seed(1), torch.full_like(w, float("nan"))  # (keys begin at zero whatever a page held)
    lens, total = [0, 0], np.zeros(2)
    for step in [(100, 30), (60, 1), (0, 1), (1, 1), (130, 40), (1, 0), (1, 1)]:
        lens = [a + b for a, b in zip(lens, step)]
        start = np.concatenate([[0], np.cumsum(step)]).tolist()
        _attend(dev, torch.randn((start[-1], 4, 64), generator=g, device=dev), kc, vc, w, tables, lens, start)
        total += np.array(step) * 2.0
        for b in range(2):
            have = w[torch.tensor(tables[b, :-(-lens[b] // 16)].astype(np.int64), device=dev)].transpose(0, 1).reshape(2, -1)[:, :lens[b]].double().sum(1).cpu().numpy()
            assert np.abs(have - total[b]).max() <= total[b] * 400 * 2.0**-24  # (each sum of weights is one to within the additions of fp32)


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("filler", [float("nan"), float("inf"), "lowest"])
def test_what_is_not_seen_does_not_count(agpu, dev, type_, filler):
    """NaN, infinities and the type's lowest value behind the last position and on pages of nobody: no bit of the weights changes, and weights there stay what they are.  Seen
    by some rows, they reach the weights of what these rows see."""
    import torch
    lens, new, page = [70, 37, 200, 130], [1, 37, 77, 1], 16
    kc, vc, w, tables, start, q = _state(dev, lens, new, 4, 2, page, type_, 3)
    held = torch.zeros(kc.shape[0], page, dtype=torch.bool)
    for b, n in enumerate(lens):
        for p in range(n):
            held[tables[b, p // page], p % page] = True
    held = held.to(dev)[:, None]
    w = torch.where(held, w, float("nan"))
    want = w.clone()
    _attend(dev, q, kc, vc, want, tables, lens, start)
    assert want[held.expand_as(want)].isfinite().all() and want[~held.expand_as(want)].isnan().all()
    x = torch.finfo(kc.dtype).min if filler == "lowest" else filler
    kb, vb = (torch.where(held[..., None], c.float(), x).to(c.dtype) for c in (kc, vc))
    got = w.clone()
    _attend(dev, q, kb, vb, got, tables, lens, start)
    assert torch.equal(got[held.expand_as(got)], want[held.expand_as(got)])
    if filler == "lowest":
        return
    # the key at 197 of request 2 is seen by its last three rows, which have no weights then; V has none in it
    vb[held.expand(-1, 2, -1)] = x
    kb[tables[2, 197 // page], :, 197 % page] = x
    got = w.clone()
    _attend(dev, q, kb, vb, got, tables, lens, start)
    mine = torch.zeros_like(held)
    for p in range(200):
        mine[tables[2, p // page], 0, p % page] = True
    # (an infinite V has the rows that see it take a new unit with every new maximum, which rounds their sums otherwise: the bound holds for any units)
    assert got[mine.expand_as(got)].isnan().all() and got[(held & ~mine).expand_as(got)].isfinite().all()
    check(got, *given64(q, kb, w, tables, lens, start))


@pytest.mark.parametrize("heads,kv_heads", [(3, 3), (16, 1)])
def test_rows_of_nobody_and_pages_outside(agpu, dev, heads, kv_heads):
    import torch
    lens, new = [0, 3, 20, 7, 64, 30], [2, 5, 3, 0, 1, 12]
    kc, vc, w, tables, start, q = _state(dev, lens, new, heads, kv_heads, 8, "float32", 2)
    tables[4, 2], tables[4, 5], tables[5, 0] = -1, 2**31 - 1, -7
    own = w.clone()
    _attend(dev, q, kc, vc, own, tables, lens, start)
    check(own, *given64(q, kc, w, tables, lens, start))
    # a table too narrow for its request, and fewer rows than query_start says
    narrow, own = tables[:, :5].copy(), w.clone()
    out, _ = _attend(dev, q[:start[-1] - 9], kc, vc, own, narrow, lens, start)
    check(own, *given64(q[:start[-1] - 9], kc, w, narrow, lens, start))
    # rows before the first request's and behind the last one's
    more, out, own = torch.cat([q[:2], q, q[:3]]), torch.full((q.shape[0] + 5, heads, 64), 7.0, device=dev), w.clone()
    got, _ = _attend(dev, more, kc, vc, own, tables, lens, [x + 2 for x in start], out=out)
    assert got is out and (out[:2] == 7.0).all() and (out[-3:] == 7.0).all()
    check(own, *given64(q, kc, w, tables, lens, start))


@pytest.mark.parametrize("type_", ["float32", "float16"])
def test_strides(agpu, dev, type_):
    """q as slices of QKV rows at an odd float; K, V and weights one layer of several."""
    import torch
    lens, new = [100, 50, 300, 33], [1, 50, 140, 1]
    kc, vc, w, tables, start, q = _state(dev, lens, new, 10, 5, 16, type_, 5)
    want = w.clone()
    out, _ = _attend(dev, q, kc, vc, want, tables, lens, start)
    pool, all_w = torch.zeros((kc.shape[0], 3, 2, 5, 16, 64), device=dev, dtype=kc.dtype), torch.full((kc.shape[0], 3, 5, 16), 5.0, device=dev)
    pool[:, 1, 0], pool[:, 1, 1], all_w[:, 1] = kc, vc, w
    rows = torch.zeros(start[-1] * 1283 + 1, device=dev)[1:].view(-1, 1283)[:, :1280].unflatten(1, (2, 10, 64))
    rows[:, 1] = q
    got, _ = _attend(dev, rows[:, 1], pool[:, 1, 0], pool[:, 1, 1], all_w[:, 1], tables, lens, start)
    assert torch.equal(got, out) and torch.equal(all_w[:, 1], want) and (all_w[:, ::2] == 5.0).all()


@pytest.mark.parametrize("heads,kv_heads,type_", [(2, 2, "float32"), (6, 1, "bfloat16"), (4, 2, "float16")])
@pytest.mark.parametrize("kind", ["tokens", "mixed"])
def test_hundreds_of_requests(agpu, dev, heads, kv_heads, type_, kind):
    rng, B = np.random.default_rng(heads), 311
    lens = rng.integers(0, 90, B)
    lens[[5, 200]] = 2500, 1300
    new = np.ones(B, int) if kind == "tokens" else np.minimum(rng.choice([0, 1, 1, 3, 9, 60, 140], B), lens)
    lens = np.maximum(lens, new).tolist()
    kc, vc, w, tables, start, q = _state(dev, lens, new.tolist(), heads, kv_heads, 16, type_, 7)
    own = w.clone()
    _attend(dev, q, kc, vc, own, tables, lens, start)
    check(own, *given64(q, kc, w, tables, lens, start))


@pytest.mark.parametrize("type_", TYPES)
def test_little_scratch(agpu, dev, type_):
    """With a scratch of 1 MiB there is no room for scores: they are formed again, and the weights are as good."""
    import torch
    from async_gpu_amd import ops
    lens, new = [3000, 2100, 700, 40, 1200, 1], [1, 300, 5, 40, 1, 1]
    kc, vc, w, tables, start, q = _state(dev, lens, new, 32, 4, 16, type_, 5)
    c, small, own, tokens = ops.context(0), torch.empty(1 << 20, dtype=torch.uint8, device=dev), w.clone(), w.clone()
    c.call("agpu_ctx_set_workspace", small.data_ptr(), small.numel())
    try:
        _attend(dev, q, kc, vc, own, tables, lens, start)
        _attend(dev, q[:6], kc, vc, tokens, tables, lens, None)
        torch.cuda.synchronize()
        with pytest.raises(agpu.AgpuError) as e:
            _attend(dev, torch.zeros((4000, 32, 64), device=dev), kc, vc, own, tables, lens, [0, 1, 2, 3, 4, 5, 4000])
        assert e.value.code == -6
    finally:
        c.call("agpu_ctx_set_workspace", None, 0)
    check(own, *given64(q, kc, w, tables, lens, start))
    check(tokens, *given64(q[:6], kc, w, tables, lens, list(range(7))))


def test_hand_over_of_runs_under_the_memory_model(agpu, dev):
    import torch
    from async_gpu_amd import ops
    lens, new = [3000, 2100, 700, 40], [1, 100, 5, 1]
    kc, vc, w, tables, start, q = _state(dev, lens, new, 4, 2, 16, "float32", 5)
    c, plain, strict = ops.context(0), w.clone(), w.clone()
    out, _ = _attend(dev, q, kc, vc, plain, tables, lens, start)
    try:
        c.call("agpu_ctx_set_strict_sync", 1)
        again, _ = _attend(dev, q, kc, vc, strict, tables, lens, start)
    finally:
        c.call("agpu_ctx_set_strict_sync", 0)
    assert torch.equal(plain, strict) and torch.equal(out, again)


# ---- eviction ----------------------------------------------------------------------------


def evict_by_hand(caches, tables, kv_lens, limit, keep, recent, sinks):
    """The definition, place by place, on numpy arrays [pages, heads, page, ...] with the weights last; in place."""
    w = caches[-1]
    pages, heads, page = w.shape[:3]
    for b, n in enumerate(kv_lens):
        n = min(n, len(tables[b]) * page)
        if n <= limit:
            continue
        place = [(int(tables[b][j // page]), j % page) for j in range(n)]
        real = [0 <= p < pages for p, _ in place]
        for h in range(heads):
            worth = [(-2, 0.0) if not real[j] else (-1, 0.0) if np.isnan(w[place[j][0], h, place[j][1]]) else (0, float(w[place[j][0], h, place[j][1]])) for j in range(n)]
            rest = sorted(range(sinks, n - recent), key=lambda j: (-worth[j][0], -worth[j][1], j))[:keep - sinks - recent]
            kept = {*rest, *range(sinks), *range(n - recent, n)}
            assert len(kept) == keep
            holes, moves = [j for j in range(keep) if j not in kept], [j for j in range(keep, n) if j in kept]
            assert len(holes) == len(moves)
            for to, source in zip(holes, moves):
                if real[to] and real[source]:
                    for c in caches:
                        c[place[to][0], h, place[to][1]] = c[place[source][0], h, place[source][1]]


def _evict_case(dev, lens, heads, page, type_, seed, weights="heavy", narrow=0):
    import torch
    rng, g = np.random.default_rng(seed), torch.Generator(device=dev).manual_seed(seed)
    pages = sum(-(-n // page) for n in lens) + 3
    kc, vc = _cache(torch, g, dev, pages, heads, page, type_)
    tables = _tables(rng, lens, page, pages)
    u = torch.rand((pages, heads, page), generator=g, device=dev)
    w = {"heavy": lambda: 0.01 * (-torch.log(u)) ** 4, "ties": lambda: torch.floor(u * 4) - 1, "equal": lambda: torch.zeros_like(u),
         "odd": lambda: torch.where(u < 0.2, float("nan"), torch.where(u < 0.4, 0.0, torch.where(u < 0.6, -0.0, torch.where(u < 0.7, float("inf"), torch.where(u < 0.8, -float("inf"), u - 1)))))
         }[weights]()
    return kc, vc, w, tables[:, :tables.shape[1] - narrow]


def _check_evict(dev, kc, vc, w, tables, lens, limit, keep, recent, sinks):
    import torch
    from async_gpu_amd import ops
    i = _i32(dev)
    bits = [x.view(torch.int32 if x.element_size() == 4 else torch.int16) for x in (kc, vc)]
    want = [x.cpu().numpy().copy() for x in bits] + [w.cpu().numpy().copy()]
    evict_by_hand(want, tables, lens, limit, keep, recent, sinks)
    got = ops.paged_evict(kc, vc, w, i(tables), i(lens), limit, keep, recent, sinks)
    assert got[0] is kc and got[1] is vc and got[2] is w
    for x, y in zip(bits, want):
        assert np.array_equal(x.cpu().numpy(), y)
    assert np.array_equal(w.cpu().numpy().view(np.int32), want[2].view(np.int32))


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("weights", ["heavy", "ties", "equal", "odd"])
@pytest.mark.parametrize("lens,limit,keep,recent,sinks,page", [
    ([40, 3, 17, 0, 64, 33], 16, 16, 4, 2, 16), ([40, 3, 17, 0, 64, 33], 20, 10, 0, 0, 7), ([2, 1, 5], 1, 1, 0, 0, 1), ([2, 1, 5], 1, 1, 1, 0, 4), ([9, 8], 1, 0, 0, 0, 4),
    ([300, 200, 1100], 150, 140, 140, 0, 16), ([300, 200, 1100], 150, 140, 0, 140, 16), ([300, 200, 1100], 150, 150, 30, 4, 33), ([700], 500, 500, 499, 1, 64), ([5000, 4096, 4097, 9000], 4000, 3000, 200, 4, 64),
    ([5000, 130], 100, 64, 10, 3, 128)])
def test_evict(agpu, dev, type_, weights, lens, limit, keep, recent, sinks, page):
    if weights != "heavy" and type_ == "float16":
        pytest.skip("the weights' order does not depend on the cache's type")
    kc, vc, w, tables = _evict_case(dev, lens, 3, page, type_, limit + keep, weights)
    _check_evict(dev, kc, vc, w, tables, lens, limit, keep, recent, sinks)


def test_evict_long(agpu, dev):
    """More positions than are in registers at a time, and more moves than are listed at a time."""
    for lens, limit, keep, weights in (([20000, 40000], 10000, 9000, "heavy"), ([40000], 30000, 20000, "ties"), ([70001], 50, 33000, "heavy")):
        kc, vc, w, tables = _evict_case(dev, lens, 2, 100, "bfloat16", keep, weights)
        _check_evict(dev, kc, vc, w, tables, lens, max(limit, keep), keep, 300, 4)


def test_evict_where_pages_are_missing(agpu, dev):
    """Pages outside the cache in a table: they are the first to go, and nothing is moved from or to them; tables too narrow for their requests."""
    kc, vc, w, tables = _evict_case(dev, [300, 200, 90], 2, 16, "float32", 3)
    tables[0, 2], tables[0, 10], tables[1, 0], tables[1, 12], tables[2, :] = -1, 2**31 - 1, -2**31, kc.shape[0], -1
    _check_evict(dev, kc, vc, w, tables, [300, 200, 90], 80, 64, 10, 4)
    kc, vc, w, tables = _evict_case(dev, [300, 200, 90], 2, 16, "float32", 3, narrow=8)
    _check_evict(dev, kc, vc, w, tables, [300, 2**31 - 1, 90], 80, 64, 10, 4)


def test_evict_leaves_others_alone(agpu, dev):
    """At or below the limit, negative, empty: nothing is touched; layers beside the one that is cut down neither."""
    import torch
    from async_gpu_amd import ops
    i = _i32(dev)
    kc, vc, w, tables = _evict_case(dev, [100, 64, 10], 2, 16, "float16", 3)
    before = [x.clone() for x in (kc, vc, w)]
    for lens, limit in (([100, 64, 10], 100), ([-5, 0, 10], 10), ([100, 64, 10], 2**31 - 1)):
        ops.paged_evict(kc, vc, w, i(tables), i(lens), limit, 10)
        assert all(torch.equal(x, y) for x, y in zip((kc, vc, w), before))
    ops.paged_evict(kc, vc, w, i(tables[:0]), i([]), 10, 10)
    pool, all_w = torch.zeros((kc.shape[0], 3, 2, 2, 16, 64), device=dev, dtype=kc.dtype), torch.full((kc.shape[0], 3, 2, 16), 5.0, device=dev)
    pool[:, 1, 0], pool[:, 1, 1], all_w[:, 1] = kc, vc, w
    _check_evict(dev, kc, vc, w, tables, [100, 64, 10], 50, 40, 8, 2)
    ops.paged_evict(pool[:, 1, 0], pool[:, 1, 1], all_w[:, 1], i(tables), i([100, 64, 10]), 50, 40, 8, 2)
    assert torch.equal(pool[:, 1, 0], kc) and torch.equal(pool[:, 1, 1], vc) and torch.equal(all_w[:, 1], w)
    assert (pool[:, ::2] == 0).all() and (all_w[:, ::2] == 5.0).all()


def trim_by_hand(kv, tables, stack, n_free, page, limit, keep):
    stack, rest, lens, gone = list(stack[:n_free]), list(stack), [], []
    for b, n in enumerate(kv):
        n = max(0, min(n, len(tables[b]) * page))
        left = keep if n > limit else n
        stack += [int(x) for x in tables[b][-(-left // page):-(-n // page)]]
        lens.append(left), gone.append(n - left)
    stack = stack[:len(rest)]
    return lens, gone, [len(stack)], stack + rest[len(stack):]


@pytest.mark.parametrize("batch,page,longest,limit,keep", [(1, 16, 5, 3, 2), (7, 16, 400, 100, 90), (7, 1, 40, 20, 20), (64, 7, 100, 40, 0), (257, 16, 900, 300, 290), (1000, 33, 640, 100, 99), (4096, 16, 200, 64, 50)])
def test_trim(agpu, dev, batch, page, longest, limit, keep):
    import torch
    from async_gpu_amd import ops
    rng, i = np.random.default_rng(batch), _i32(dev)
    kv = rng.integers(0, longest + 1, batch)
    width = -(-longest // page)
    tables = rng.permutation(batch * width).reshape(batch, width)
    n_free = 5
    for size in (n_free + batch * width, n_free + batch * width // 4):  # the second: what has no place is lost
        stack, t = i(np.arange(size) - 2 * size), i(tables)
        want = trim_by_hand(kv.tolist(), tables.tolist(), stack.tolist(), n_free, page, limit, keep)
        for _ in range(2):
            got = ops.paged_trim(i(kv), t, stack, i([n_free]), page, limit, keep)
            for name, x, y in zip(("kv_lens", "evicted", "n_free", "free_pages"), (*got, stack), want):
                assert np.array_equal(x.cpu().numpy(), np.asarray(y)), name
        assert torch.equal(t, i(tables))


def test_trim_of_nobody_and_of_nonsense(agpu, dev):
    from async_gpu_amd import ops
    i = _i32(dev)
    kv, gone, n = ops.paged_trim(i([]), i(np.zeros((0, 4))), i([5, 6]), i([2]), 16, 3, 3)
    assert kv.numel() == 0 and gone.numel() == 0 and n.tolist() == [2]
    stack = i([8, 9, 10, -1, -1, -1])
    kv, gone, n = ops.paged_trim(i([-5, 2**31 - 1, 3, 8]), i([[0, 1], [2, 3], [4, 5], [6, 7]]), stack, i([3]), 4, 3, 3)
    assert kv.tolist() == [0, 3, 3, 3] and gone.tolist() == [0, 5, 0, 5] and n.tolist() == [5] and stack.tolist() == [8, 9, 10, 3, 7, -1]
    for bad in (-4, 2**31 - 1):
        kv, gone, n = ops.paged_trim(i([8]), i([[0, 1]]), i([7]), i([bad]), 4, 4, 4)
        assert n.tolist() == [1]


def test_a_cache_beyond_32_bits(agpu, dev):
    """Elements of a cache beyond number 2^32, weighed and evicted."""
    import torch
    from async_gpu_amd import ops
    page, H = 64, 4
    pages = (1 << 32) // (page * H * 64) + 40
    kc, vc = (torch.empty((pages, H, page, 64), dtype=torch.bfloat16, device=dev) for _ in range(2))
    w = torch.zeros((pages, H, page), device=dev)
    ids, lens, new = [pages - 1, 3, pages - 2, 4, pages - 7, 0, pages - 9, 8, pages - 11], [200, 150, 90], [1, 140, 3]
    g, i = torch.Generator(device=dev).manual_seed(2), _i32(dev)
    kc[ids], vc[ids] = (torch.randn((len(ids), H, page, 64), generator=g, device=dev).bfloat16() for _ in range(2))
    w[ids] = torch.rand((len(ids), H, page), generator=g, device=dev)
    tables = np.full((3, 4), -1)
    tables[0, :4], tables[1, :3], tables[2, :2] = ids[:4], ids[4:7], ids[7:]
    start = np.concatenate([[0], np.cumsum(new)]).tolist()
    q = torch.randn((start[-1], 2 * H, 64), generator=g, device=dev)
    small = {p: n for n, p in enumerate(ids)}
    local = np.vectorize(lambda p: small.get(p, -1))(tables)
    want, tol = given64(q, kc[ids], w[ids], local, lens, start)
    _attend(dev, q, kc, vc, w, tables, lens, start)
    check(w[ids], want, tol)
    by_hand = [kc[ids].view(torch.int16).cpu().numpy(), vc[ids].view(torch.int16).cpu().numpy(), w[ids].cpu().numpy()]
    evict_by_hand(by_hand, local, lens, 80, 70, 10, 2)
    ops.paged_evict(kc, vc, w, i(tables), i(lens), 80, 70, 10, 2)
    for x, y in zip((kc[ids].view(torch.int16), vc[ids].view(torch.int16), w[ids]), by_hand):
        assert np.array_equal(x.cpu().numpy(), y)


@pytest.mark.parametrize("type_", ["float32", "bfloat16"])
def test_a_server_with_a_budget(agpu, dev, type_):
    """Requests that come in chunks, decode and end, over two layers whose caches are cut down when they pass the limit, in a graph that is replayed between eager work: each step's
    attention and weights against 64 bits, what is evicted and where pages go against the definitions, and positions of embeddings from places and what was evicted."""
    import torch
    from async_gpu_amd import ops
    H, page, width, B, T, layers = 3, 16, 12, 5, 100, 2
    limit, keep, recent, sinks, pages = 96, 64, 20, 4, 45
    g, rng, i32 = torch.Generator(device=dev).manual_seed(12), np.random.default_rng(13), _i32(dev)
    state = dict(cached=i32(np.zeros(B)), new=i32(np.zeros(B)), tables=i32(np.full((B, width), -1)), stack=i32(rng.permutation(pages)), n=i32([pages]))
    for layer in range(layers):
        state[f"k{layer}"], state[f"v{layer}"] = _cache(torch, g, dev, pages, H, page, type_)
        state[f"w{layer}"] = torch.full((pages, H, page), float("nan"), device=dev)
    qkv = torch.zeros((layers, T, 3, 2 * H, 64), device=dev)

    def attend(s):
        kv, start, slots, pos, n = ops.paged_plan(s["cached"], s["new"], s["tables"], s["stack"], s["n"], page, T)
        outs = []
        for i in range(layers):
            ops.paged_kv_append(qkv[i, :, 1, :H], qkv[i, :, 2, :H], s[f"k{i}"], s[f"v{i}"], slots)
            out = torch.zeros((T, 2 * H, 64), device=dev)
            ops.paged_attention_weights(qkv[i, :, 0], s[f"k{i}"], s[f"v{i}"], s[f"w{i}"], s["tables"], kv, start, out=out)
            outs.append(out)
        return kv, start, n, outs

    def cut(s, kv, n):
        for i in range(layers):
            ops.paged_evict(s[f"k{i}"], s[f"v{i}"], s[f"w{i}"], s["tables"], kv, limit, keep, recent, sinks)
        return ops.paged_trim(kv, s["tables"], s["stack"], n, page, limit, keep)

    def step(s):
        kv, start, n, outs = attend(s)
        return (kv, start, *outs, *cut(s, kv, n))

    copy = lambda s: {k: v.clone() for k, v in s.items()}  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(copy(state))
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        made = step(state)
    eager, cuts = copy(state), 0
    for n in range(30):  # (a step has 100 rows at most: it serves the requests that fit)
        new = rng.integers(0, 21, B) if n % 3 else np.ones(B, int)
        if n > 14 and n % 4 == 0:
            new[n % B] = -1
        for s in (state, eager):
            s["new"].copy_(i32(new))
        qkv.copy_(torch.randn(qkv.shape, generator=g, device=dev))
        before = copy(eager)
        kv, start, left, outs = attend(eager)
        lens, at, tables = kv.tolist(), start.tolist(), eager["tables"].tolist()
        for i in range(layers):
            check(outs[i], *attend64(qkv[i, :, 0], eager[f"k{i}"], eager[f"v{i}"], tables, lens, at))
            ref, tol = given64(qkv[i, :, 0], eager[f"k{i}"], before[f"w{i}"].nan_to_num(0.0), tables, lens, at)
            check(torch.where((tol > 0).to(dev), eager[f"w{i}"], 0.0), torch.where(tol > 0, ref, 0.0), tol)
        by_hand = [[eager[f"{x}{i}"].float().cpu().numpy() for x in "kvw"] for i in range(layers)]
        for c in by_hand:
            evict_by_hand(c, tables, lens, limit, keep, recent, sinks)
        want = trim_by_hand(lens, tables, eager["stack"].tolist(), int(left), page, limit, keep)
        made_eager = cut(eager, kv, left)
        for x, y in zip((*made_eager, eager["stack"]), want):
            assert np.array_equal(x.cpu().numpy(), np.asarray(y))
        for i in range(layers):
            for x, y in zip("kvw", by_hand[i]):
                assert np.array_equal(eager[f"{x}{i}"].float().cpu().numpy(), y, equal_nan=True)
        cuts += sum(x > 0 for x in want[1])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(made, (kv, start, *outs, *made_eager)):
            assert torch.equal(x, y), n
        for name in state:
            assert np.array_equal(state[name].float().cpu().numpy(), eager[name].float().cpu().numpy(), equal_nan=True), (n, name)
        owned = [p for b in range(B) for p in tables[b][:-(-want[0][b] // page)]]
        assert sorted(owned + want[3][:want[2][0]]) == list(range(pages))
        for s, out in ((state, made[-3:]), (eager, made_eager)):
            s["cached"].copy_(out[0]), s["n"].copy_(out[2])
    assert cuts > 5


@pytest.mark.parametrize("type_", ["float32", "float16"])
@pytest.mark.parametrize("heads,kv_heads", [(3, 3), (9, 1), (8, 2)])
def test_chunks_beside_idle_requests(agpu, dev, type_, heads, kv_heads):
    """No more rows than requests, but not one each."""
    new = [0, 9, 0, 0, 40, 0, 1, 0, 2, 0] + [0, 1] * 30
    lens = [20 + 3 * i for i in range(len(new))]
    kc, vc, w, tables, start, q = _state(dev, lens, new, heads, kv_heads, 16, type_, 7)
    for window, sinks in ((0, 0), (30, 4)):
        own = w.clone()
        _attend(dev, q, kc, vc, own, tables, lens, start, window, sinks)
        check(own, *given64(q, kc, w, tables, lens, start, window, sinks))


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("lens", [[3000], [5000] * 20, [70, 1, 9000, 2048, 1024, 1025]])
def test_tokens_of_long_requests(agpu, dev, type_, lens):
    """Weights from scores, by the last workgroup at a token or by a launch of their own; with and without query_start the same bits."""
    import torch
    kc, vc, w, tables, start, q = _state(dev, lens, [1] * len(lens), 12, 6, 16, type_, 7)
    own, plain = w.clone(), w.clone()
    _attend(dev, q, kc, vc, own, tables, lens, start)
    check(own, *given64(q, kc, w, tables, lens, start))
    _attend(dev, q, kc, vc, plain, tables, lens, None)
    assert torch.equal(own, plain)


def test_evict_twice_and_in_a_graph(agpu, dev):
    """What is cut down stays as it is cut down again with the lengths it has now; a graph of both calls gives what eager calls give, replay by replay."""
    import torch
    from async_gpu_amd import ops
    i = _i32(dev)
    kc, vc, w, tables = _evict_case(dev, [300, 200, 90, 1000], 3, 16, "float16", 3)
    t, lens, stack, n = i(tables), i([300, 200, 90, 1000]), i(np.full(200, -1)), i([0])
    first = [x.clone() for x in (kc, vc, w)]

    def both(kc, vc, w, lens, stack):
        ops.paged_evict(kc, vc, w, t, lens, 120, 100, 10, 2)
        return ops.paged_trim(lens, t, stack, n, 16, 120, 100)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both(*[x.clone() for x in first], lens, stack.clone())
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    gl, gs = lens.clone(), stack.clone()
    with torch.cuda.graph(graph, stream=side):
        made = both(kc, vc, w, gl, gs)
    for x, y in zip((kc, vc, w), first):
        x.copy_(y)
    for step in ([300, 200, 90, 1000], [120, 121, 90, 700], [100, 100, 90, 100]):
        gl.copy_(i(step)), lens.copy_(i(step))
        eager = [x.clone() for x in (kc, vc, w)]
        es = gs.clone()
        want = both(*eager, lens, es)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip((*made, kc, vc, w, gs), (*want, *eager, es)))


def test_evict_under_a_wide_table(agpu, dev):
    """Tables that stand for 2^20 positions, whose bits take most of a workgroup's LDS."""
    import torch
    kc, vc, w, tables = _evict_case(dev, [300, 5000, 20], 2, 16, "float16", 3)
    wide = np.full((3, 65536), -1, np.int32)
    wide[:, :tables.shape[1]] = tables
    _check_evict(dev, kc, vc, w, wide, [300, 5000, 20], 200, 150, 10, 2)
    from async_gpu_amd import ops
    i = _i32(dev)
    with pytest.raises(agpu.AgpuError) as e:
        ops.paged_evict(kc, vc, w, i(np.zeros((1, 65537))), i([5]), 4, 4)
    assert e.value.code == -5
    with pytest.raises(agpu.AgpuError) as e:
        ops.paged_evict(kc, vc, w, i(tables), i([300, 5000, 20]), 4, 5)
    assert e.value.code == -1
    with pytest.raises(agpu.AgpuError) as e:
        ops.paged_trim(i([300, 5000, 20]), i(tables), i([1]), i([1]), 16, 4, 5)
    assert e.value.code == -1


def test_evict_of_pages_that_two_requests_have(agpu, dev):
    """A page belongs to one request only; where one does not, what becomes of it is left open, but of nothing else."""
    import torch
    from async_gpu_amd import ops
    i = _i32(dev)
    lens = [9000, 9000, 6000]
    kc, vc, w, tables = _evict_case(dev, lens, 2, 64, "bfloat16", 3)
    tables[1] = tables[0]
    others = torch.as_tensor(np.setdiff1d(np.arange(kc.shape[0]), tables[0]), device=dev)
    alone = [x.clone() for x in (kc, vc, w)]
    ops.paged_evict(*alone, i(tables[2:]), i(lens[2:]), 4500, 4000, 100, 4)
    ops.paged_evict(kc, vc, w, i(tables), i(lens), 4500, 4000, 100, 4)
    assert all(torch.equal(x[others], y[others]) for x, y in zip((kc, vc, w), alone))


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("heads,kv_heads,window,sinks", [(3, 3, 0, 0), (8, 2, 0, 0), (5, 1, 300, 7), (16, 2, 0, 0)])
@pytest.mark.parametrize("new", [[1] * 6, [1, 1, 30, 1, 0, 1]])
def test_tokens_of_a_large_cache(agpu, dev, type_, heads, kv_heads, window, sinks, new):
    """Where scores wait depends on which are fewer, places of the cache or keys of the requests; what comes out does not."""
    import torch
    lens = [3000, 2100, 700, 40, 1200, 1]
    kc, vc, w, tables, start, q = _state(dev, lens, new, heads, kv_heads, 16, type_, heads)
    large = [torch.cat([x, torch.full((2000, *x.shape[1:]), float("nan"), device=dev, dtype=x.dtype)]) for x in (kc, vc, w)]
    wide = np.full((6, 2000), -1, np.int32)
    wide[:, :tables.shape[1]] = tables
    got = []
    for cache, table in (((kc, vc, w.clone()), wide), (large, np.where(tables >= kc.shape[0], -1, tables))):
        out, weights = _attend(dev, q, *cache, table, lens, start, window, sinks)
        got.append((out, weights[:kc.shape[0]]))
        assert torch.isnan(weights[kc.shape[0]:]).all()
    check(got[0][1], *given64(q, kc, w, tables, lens, start, window, sinks))
    assert torch.equal(got[0][1], got[1][1]) and torch.equal(got[0][0], got[1][0])
