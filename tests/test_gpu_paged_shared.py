"""paged_attention_shared: requests behind prefixes that the cache holds once, against the same attention in 64 bits over prefix and own keys together."""
import numpy as np
import pytest
from test_gpu_paged import TYPES, _cache, _tables, attend64, check

pytestmark = pytest.mark.gpu


def _i32(dev):
    import torch
    return lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=dev)


class Batch:
    """Prefixes of the lengths `prefixes`, requests (kv, new, prefix), their pages in one shuffled pool."""

    def __init__(self, dev, prefixes, requests, heads, kv_heads, page, type_, seed=0, spare=2, scale=1.5):
        import torch
        self.dev, self.page = dev, page
        rng, g = np.random.default_rng(seed), torch.Generator(device=dev).manual_seed(seed)
        self.lens, self.new, self.of = ([r[i] for r in requests] for i in range(3))
        self.prefixes = list(prefixes)
        pages = sum(-(-n // page) for n in self.lens + self.prefixes) + spare
        self.kc, self.vc = _cache(torch, g, dev, pages, kv_heads, page, type_)
        every = _tables(rng, self.prefixes + self.lens, page, pages)
        k = len(self.prefixes)
        self.ptables, self.tables = every[:k, :max((-(-n // page) for n in self.prefixes), default=0)], every[k:, :max(-(-n // page) for n in self.lens)]
        self.start = np.concatenate([[0], np.cumsum(self.new)]).tolist()
        self.q = torch.randn((self.start[-1], heads, 64), generator=g, device=dev) * scale

    def run(self, window=0, sinks=0, start=True, **kw):
        from async_gpu_amd import ops
        i = _i32(self.dev)
        return ops.paged_attention_shared(self.q, self.kc, self.vc, i(self.ptables), i(self.prefixes), i(self.of), i(self.tables), i(self.lens), i(self.start) if start else None,
                                          window, sinks, **kw)

    def joint(self):
        """K, V and tables with a slot a page, and lengths, of prefixes and requests together."""
        pages, heads, page, _ = self.kc.shape
        k, v = (c.transpose(1, 2).reshape(pages * page, heads, 1, 64) for c in (self.kc, self.vc))

        def slots(table, n):
            ids = np.array([int(x) for x in table] + [-1], np.int64)
            at = np.minimum(np.arange(max(n, 0)) // page, len(ids) - 1)
            return [int(ids[a]) * page + j % page if 0 <= ids[a] < pages else -1 for j, a in enumerate(at)]

        rows = []
        for b, g in enumerate(self.of):
            before = slots(self.ptables[g], min(self.prefixes[g], self.ptables.shape[1] * page)) if 0 <= g < len(self.prefixes) else []
            rows.append(before + slots(self.tables[b], self.lens[b]))
        wide = max(map(len, rows), default=0)
        return k, v, [r + [-1] * (wide - len(r)) for r in rows], [len(r) for r in rows]

    def check(self, got, window=0, sinks=0):
        k, v, tables, lens = self.joint()
        check(got, *attend64(self.q, k, v, tables, lens, self.start, window, sinks))


# prefixes, (kv, new, prefix) of the requests
BATCHES = {
    "one": ([500], [(3, 1, 0)]),
    "one key each": ([1], [(1, 1, 0), (1, 1, 0)]),
    "tokens": ([700], [(1, 1, 0), (2, 1, 0), (15, 1, 0), (16, 1, 0), (17, 1, 0), (300, 1, 0), (64, 1, 0), (33, 1, 0), (5, 1, 0)]),
    "tokens behind several": ([300, 1, 65, 0, 130], [(10, 1, 2), (20, 1, -1), (1, 1, 0), (40, 1, 4), (7, 1, 3), (9, 1, 0), (5, 1, 1), (3, 1, 5), (31, 1, 4), (2, 1, -2**31), (77, 1, 0)]),
    "with idle ones": ([200], [(0, 0, 0), (40, 1, 0), (7, 0, 0), (129, 1, -1), (33, 0, 0)]),
    "chunks": ([257, 100], [(5, 5, 0), (33, 33, 1), (100, 60, 0), (257, 128, -1), (140, 129, 0), (64, 64, 1)]),
    "mixed": ([600, 31], [(400, 1, 0), (200, 150, 1), (31, 1, 0), (60, 9, 0), (70, 3, 1), (90, 90, 0), (1, 1, 0), (8, 8, -1)]),
    "long": ([3000], [(30, 1, 0), (20, 4, 0), (300, 290, 0)]),
    "hundreds of rows": ([333], [(3 + i % 40, 1 + i % 3, 0) for i in range(150)]),
}


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("heads,kv_heads,page", [(3, 3, 16), (4, 2, 7), (8, 2, 64), (5, 1, 1), (11, 1, 32)])
@pytest.mark.parametrize("batch", list(BATCHES))
def test_shared(agpu, dev, type_, heads, kv_heads, page, batch):
    import torch
    s = Batch(dev, *BATCHES[batch], heads, kv_heads, page, type_, seed=heads * page + len(batch))
    for window, sinks in ((0, 0), (150, 3)) if page in (7, 16, 64) else ((0, 0),):
        got = s.run(window, sinks)
        s.check(got, window, sinks)
        assert torch.equal(got, s.run(window, sinks))
        if all(n == 1 for n in s.new):
            assert torch.equal(got, s.run(window, sinks, start=False))


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (40, 0), (64, 700), (200, 5), (0, 9), (5000, 4), (350, 400), (2**31 - 1, 3), (30, 2**31 - 1)])
@pytest.mark.parametrize("type_", ["float32", "float16"])
def test_windows(agpu, dev, window, sinks, type_):
    """Windows that end in the prefix, among own keys and before both; sinks that reach over the prefix's end."""
    s = Batch(dev, [310, 40], [(900, 1, 0), (1, 1, 0), (50, 50, 1), (100, 60, 0), (60, 60, 1), (200, 150, 0), (10, 1, -1)], 4, 2, 16, type_, seed=window % 1000)
    s.check(s.run(window, sinks), window, sinks)


def test_as_one_request(agpu, dev):
    """A prefix of whole pages in front of the block tables: what paged_attention gives for the requests one by one, with the same accuracy."""
    from async_gpu_amd import ops
    s = Batch(dev, [320], [(40, 1, 0), (100, 1, 0), (7, 1, 0), (64, 1, 0)], 4, 4, 16, "float32")
    i = _i32(dev)
    wide = np.concatenate([np.repeat(s.ptables[:, :20], 4, 0), s.tables], 1)
    one = ops.paged_attention(s.q, s.kc, s.vc, i(wide), i([n + 320 for n in s.lens]), i(s.start))
    k, v, tables, lens = s.joint()
    ref, tol = attend64(s.q, k, v, tables, lens, s.start)
    check(one, ref, tol), check(s.run(), ref, tol)


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("filler", [float("nan"), float("inf"), "lowest"])
def test_what_is_not_seen_does_not_count(agpu, dev, type_, filler):
    """NaN, infinities and the type's lowest value behind a prefix's end, on pages of nobody, and in a prefix of others change no bit; seen ones reach who sees them."""
    import torch
    s = Batch(dev, [70, 90], [(20, 1, 0), (37, 37, 0), (50, 1, 1), (30, 10, 1), (9, 1, -1)], 4, 2, 16, type_)
    x = torch.finfo(s.kc.dtype).min if filler == "lowest" else filler
    want, held = s.run(), torch.zeros(s.kc.shape[0], 16, dtype=torch.bool)
    for table, n in [*zip(s.ptables, s.prefixes), *zip(s.tables, s.lens)]:
        for p in range(n):
            held[table[p // 16], p % 16] = True
    held = held.to(dev)[:, None, :, None]
    s.kc, s.vc = (torch.where(held, c.float(), x).to(c.dtype) for c in (s.kc, s.vc))
    assert torch.equal(want, s.run())
    if filler == "lowest":
        return
    for p in (60, 75, 89):  # of prefix 1
        s.vc[s.ptables[1, p // 16], :, p % 16, ::3] = x
    got = s.run()
    behind = torch.zeros(s.start[-1], dtype=torch.bool)
    behind[s.start[2]:s.start[4]] = True
    assert torch.equal(got[~behind], want[~behind])
    seen = got[behind].cpu()
    assert torch.isfinite(seen[:, :, 1::3]).all() and not torch.isfinite(seen[:, :, ::3]).any()
    if filler == float("inf"):
        assert (seen[:, :, ::3] == float("inf")).all()
    # ... and not who has a window that ends behind them
    assert torch.isfinite(s.run(window=5)[behind]).all()


def test_pages_outside_the_cache_and_rows_of_nobody(agpu, dev):
    import torch
    s = Batch(dev, [100], [(20, 1, 0), (30, 12, 0), (9, 1, -1)], 3, 3, 16, "float32")
    s.ptables[0, 1], s.ptables[0, 4] = -1, 2**31 - 1
    s.check(s.run())
    # more positions than the tables have pages for
    s.prefixes[0], s.lens[0] = 5000, 600
    s.check(s.run())
    s.prefixes[0], s.lens[0] = 100, 20
    # rows behind the last request's, and before the first one's
    out = torch.full((s.start[-1] + 4, 3, 64), 7.0, device=dev)
    s.q = torch.cat([s.q, s.q[:4]])
    s.run(out=out)
    assert (out[s.start[-1]:] == 7.0).all()
    k, v, tables, lens = s.joint()
    ref, tol = attend64(s.q[:s.start[-1]], k, v, tables, lens, s.start)
    check(out[:s.start[-1]], ref, tol)
    s.start = [x + 3 for x in s.start]
    s.q = s.q[torch.tensor([0, 0, 0, *range(s.start[-1] - 3)], device=dev)]
    out = torch.full((s.start[-1], 3, 64), 7.0, device=dev)
    s.run(out=out)
    assert (out[:3] == 7.0).all()
    check(out[3:], ref, tol)
    # fewer rows than query_start says: the first ones
    s.start, s.q = [x - 3 for x in s.start], s.q[3:10]
    got = s.run()
    check(got, ref[:7], tol[:7])
    # nobody
    from async_gpu_amd import ops
    i = _i32(dev)
    assert ops.paged_attention_shared(s.q[:0], s.kc, s.vc, i(s.ptables), i(s.prefixes), i([]), i(np.zeros((0, 2))), i([]), i([0])).shape == (0, 3, 64)


def test_no_prefix(agpu, dev):
    """No prefixes at all, or none with a key: paged_attention."""
    import torch
    from async_gpu_amd import ops
    s = Batch(dev, [0, 0], [(20, 1, 0), (200, 140, 1), (9, 1, -1)], 4, 2, 16, "bfloat16")
    i = _i32(dev)
    want = ops.paged_attention(s.q, s.kc, s.vc, i(s.tables), i(s.lens), i(s.start))
    own = (i(s.of), i(s.tables), i(s.lens), i(s.start))
    assert torch.equal(want, ops.paged_attention_shared(s.q, s.kc, s.vc, i(np.zeros((0, 5))), i([]), *own))
    assert torch.equal(want, ops.paged_attention_shared(s.q, s.kc, s.vc, i(np.zeros((2, 0))), i([40, 50]), *own))
    s.check(ops.paged_attention_shared(s.q, s.kc, s.vc, i(np.zeros((2, 3))), i([0, -4]), *own))


def test_only_the_prefix(agpu, dev):
    """Requests whose rows have no keys of their own in the cache: tables of no width, and rows before place 0."""
    s = Batch(dev, [77], [(0, 1, 0), (3, 9, 0), (0, 40, 0)], 2, 2, 8, "float32")
    s.check(s.run())


@pytest.mark.parametrize("type_", ["float32", "float16"])
def test_strides(agpu, dev, type_):
    """q as slices of QKV rows at an odd float; K and V one layer of several, interleaved by pages; an out of the caller's."""
    import torch
    s = Batch(dev, [130], [(100, 1, 0), (50, 50, 0), (60, 20, -1), (33, 1, 0)], 4, 4, 16, type_)
    want = s.run()
    s.check(want)
    pool = torch.randn((s.kc.shape[0], 3, 2, 4, 16, 64), device=dev).to(s.kc.dtype)
    pool[:, 1, 0], pool[:, 1, 1] = s.kc, s.vc
    s.kc, s.vc = pool[:, 1, 0], pool[:, 1, 1]
    T = s.start[-1]
    qkv = torch.randn(T * (3 * 256 + 3) + 1, device=dev)[1:].view(T, 3 * 256 + 3)[:, :768].unflatten(1, (3, 4, 64))
    qkv[:, 0] = s.q
    s.q = qkv[:, 0]
    out = torch.empty((T, 4, 64), device=dev)
    assert s.run(out=out) is out and torch.equal(out, want)


@pytest.mark.parametrize("heads,kv_heads", [(2, 2), (6, 1)])
def test_many_requests_and_prefixes(agpu, dev, heads, kv_heads):
    rng = np.random.default_rng(heads)
    prefixes = rng.integers(0, 60, 256).tolist()
    prefixes[7] = 1500
    requests = [(int(n), int(n > 0), int(g)) for n, g in zip(rng.integers(0, 60, 700), rng.choice([7, *range(-1, 256)], 700))]
    s = Batch(dev, prefixes, requests, heads, kv_heads, 16, "bfloat16", seed=1)
    s.check(s.run())
    requests = [(int(n) + 40, int(m), int(g)) for n, m, g in zip(rng.integers(0, 60, 311), rng.choice([0, 1, 3, 9, 30], 311), rng.choice([7, 7, *range(-1, 256)], 311))]
    s = Batch(dev, prefixes, requests, heads, kv_heads, 16, "float32", seed=2)
    s.check(s.run())


@pytest.mark.parametrize("type_", TYPES)
def test_little_scratch(agpu, dev, type_):
    import torch
    from async_gpu_amd import ops
    s = Batch(dev, [2100], [(500, 1, 0), (400, 300, 0), (60, 5, 0), (40, 40, 0)], 8, 4, 16, type_)
    c, small = ops.context(0), torch.empty(1 << 20, dtype=torch.uint8, device=dev)
    c.call("agpu_ctx_set_workspace", small.data_ptr(), small.numel())
    try:
        got = s.run()
        torch.cuda.synchronize()
        many = torch.zeros((13000, 8, 64), device=dev)  # 8 bytes for each of their rows of heads is more than there is
        with pytest.raises(agpu.AgpuError) as e:
            i = _i32(dev)
            ops.paged_attention_shared(many, s.kc, s.vc, i(s.ptables), i(s.prefixes), i(s.of), i(s.tables), i(s.lens), i([0, 5, 6, 7, 13000]))
        assert e.value.code == -6
    finally:
        c.call("agpu_ctx_set_workspace", None, 0)
    s.check(got)


def test_hand_over_of_runs_under_the_memory_model(agpu, dev):
    import torch
    from async_gpu_amd import ops
    s = Batch(dev, [3000], [(2100, 1, 0), (700, 100, 0), (40, 5, 0)], 2, 2, 16, "float32")
    plain, c = s.run(), ops.context(0)
    try:
        c.call("agpu_ctx_set_strict_sync", 1)
        assert torch.equal(plain, s.run())
    finally:
        c.call("agpu_ctx_set_strict_sync", 0)
    s.check(plain)


def test_streams(agpu, dev):
    """Two streams at once, each with its own scratch, against the default one."""
    import torch
    batches = [Batch(dev, [2000], [(300, 1, 0), (200, 120, 0), (30, 1, 0)], 4, 4, 16, "float16", seed=i) for i in range(2)]
    want, streams, got = [s.run() for s in batches], [torch.cuda.Stream() for _ in batches], [[], []]
    torch.cuda.synchronize()
    for _ in range(10):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(batches[i].run())
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(want[i], x) for x in got[i])


def test_captured_server(agpu, dev):
    """Request 0 is the prefix, which comes in chunks like any prompt; the others then begin behind it.  One graph of a step, replayed with other lengths and rows between eager
    work, against eager steps bit by bit and against attention in 64 bits over what each request has seen."""
    import torch
    from async_gpu_amd import ops
    B, H, page, width, T = 6, 3, 16, 20, 60
    g, rng, i32 = torch.Generator(device=dev).manual_seed(3), np.random.default_rng(4), _i32(dev)
    pages = 100
    state = dict(cached=i32(np.zeros(B)), new=i32(np.zeros(B)), tables=i32(np.full((B, width), -1)), stack=i32(rng.permutation(pages)), n=i32([pages]), of=i32([-1] * B))
    kc, vc = _cache(torch, g, dev, pages, H, page, "bfloat16")
    qkv = torch.zeros((T, 3, H, 64), device=dev)

    def step(s, kc, vc):
        kv, start, slots, pos, n = ops.paged_plan(s["cached"], s["new"], s["tables"], s["stack"], s["n"], page, T)
        ops.paged_kv_append(qkv[:, 1], qkv[:, 2], kc, vc, slots)
        out = torch.zeros((T, H, 64), device=dev)
        ops.paged_attention_shared(qkv[:, 0], kc, vc, s["tables"][:1], kv[:1], s["of"], s["tables"], kv, start, out=out)
        return kv, start, slots, pos, n, out

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step({k: v.clone() for k, v in state.items()}, kc.clone(), vc.clone())
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        made = step(state, kc, vc)
    eager, ek, ev = {k: v.clone() for k, v in state.items()}, kc.clone(), vc.clone()
    seen = [([], []) for _ in range(B)]
    for n in range(12):
        new = np.array([50, 0, 0, 0, 0, 0]) if n < 3 else np.concatenate([[0], rng.integers(0, 10, B - 1)])
        of = [-1] * B if n < 3 else [-1, 0, 0, 0, -1, 0]
        if n > 7:
            new[1 + n % 5] = -1
        for s in (state, eager):
            s["new"].copy_(i32(new)), s["of"].copy_(i32(of))
        qkv.copy_(torch.randn(qkv.shape, generator=g, device=dev))
        want = step(eager, ek, ev)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(made, want):
            assert torch.equal(x, y), n
        start, kv = want[1].tolist(), want[0].tolist()
        for b in range(B):
            rows = slice(start[b], start[b + 1])
            if new[b] < 0:
                seen[b] = ([], [])
            for have, i in zip(seen[b], (1, 2)):
                have.append(qkv[rows, i].to(kc.dtype).float())
            m = start[b + 1] - start[b]
            if m == 0:
                continue
            k, v = (torch.cat((seen[0][i] if of[b] == 0 else []) + seen[b][i]) for i in range(2))
            check(want[5][rows], *attend64(qkv[rows, 0], k.transpose(0, 1)[None], v.transpose(0, 1)[None], [[0]], [k.shape[0]], [0, m]))
        for s, out in ((state, made), (eager, want)):
            s["cached"].copy_(out[0]), s["n"].copy_(out[4])


@pytest.mark.parametrize("type_", TYPES)
def test_out_at_any_float(agpu, dev, type_):
    """Results to memory that begins at any float, behind a prefix of several runs: the same bits."""
    import torch
    s = Batch(dev, [900], [(100, 1, 0), (150, 140, 0), (60, 20, -1), (33, 2, 0)], 6, 3, 16, type_)
    want, buf = s.run(), torch.full((s.q.numel() + 5,), 7.0, device=dev)
    s.check(want)
    for odd in (1, 2, 3):
        buf.fill_(7.0)
        out = buf[odd:odd + s.q.numel()].view(s.q.shape)
        assert s.run(out=out) is out and torch.equal(out, want) and (buf[:odd] == 7.0).all() and (buf[odd + s.q.numel():] == 7.0).all()


@pytest.mark.parametrize("type_", ["float32", "bfloat16"])
@pytest.mark.parametrize("heads,kv_heads", [(3, 3), (9, 1)])
def test_chunks_beside_idle_requests(agpu, dev, type_, heads, kv_heads):
    """No more rows than requests, but not one each: rows of chunks go one by one over their own pages, and in tiles over the prefix."""
    new = [0, 9, 0, 0, 40, 0, 1, 0, 0, 0] + [0] * 50
    s = Batch(dev, [250, 33], [(20 + 3 * i, n, (0, 1, -1)[i % 3]) for i, n in enumerate(new)], heads, kv_heads, 16, type_)
    s.check(s.run())
    s.check(s.run(30, 4), 30, 4)


@pytest.mark.parametrize("type_", ["float32", "float16"])
def test_far_apart_magnitudes(agpu, dev, type_):
    """Runs and waves whose maxima lie far apart, and rows of which one key has all the weight."""
    import torch
    s = Batch(dev, [1500], [(20, 1, 0), (40, 30, 0), (70, 1, 0)], 4, 2, 16, type_, scale=8.0)
    for p in (3, 700, 1499):
        s.kc[s.ptables[0, p // 16], :, p % 16] *= 6.0
    s.check(s.run())
    s.kc *= 0.0
    got = s.run()  # equal scores: the mean
    k, v, tables, lens = s.joint()
    check(got, *attend64(s.q, k, v, tables, lens, s.start))


def test_a_cache_beyond_32_bits(agpu, dev):
    """Elements of a cache beyond number 2^32, of the prefix and of own pages."""
    import torch
    page, H = 64, 4
    pages = (1 << 32) // (page * H * 64) + 40
    s = Batch(dev, [400], [(200, 1, 0), (150, 140, 0), (90, 3, 0)], 2 * H, H, page, "bfloat16")
    ids = np.array([pages - 1 - 2 * i if i % 2 else i for i in range(s.kc.shape[0])])
    big = [torch.empty((pages, H, page, 64), dtype=torch.bfloat16, device=dev) for _ in range(2)]
    for b, small in zip(big, (s.kc, s.vc)):
        b[torch.tensor(ids, device=dev)] = small
    want, small = s.run(), (s.kc, s.vc, s.ptables, s.tables)
    s.check(want)
    move = lambda t: np.where((t >= 0) & (t < len(ids)), ids[np.clip(t, 0, len(ids) - 1)], -1)  # noqa: E731
    s.kc, s.vc, s.ptables, s.tables = *big, move(small[2]), move(small[3])
    assert torch.equal(s.run(), want)
