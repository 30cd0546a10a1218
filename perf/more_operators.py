"""Performance cases of the operators that make long contexts cheaper on a server over a KV cache in pages.

Requests that begin alike hold what they share once: paged_attention_shared attends over a prefix of many requests and over the pages of each
one's own.  Requests that grow beyond a budget give places up: paged_attention_weights attends and adds up how much weight each key was given,
paged_evict keeps the places with the most of it (and the first and the last ones), layer by layer, and paged_trim gives the pages behind back,
once a step.  Each case is one call of one of them.

run() is the plain form, elementary torch operations in 32 bits, or with `own` set the framework's operator.  exact() is the same in 64 bits,
request by request.
"""
import math
import random

import torch

own = False
DH = 64  # the framework's head size
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # A handful of chats behind one short instruction: the smallest call, the small model's heads over an fp32 cache.
        dict(name="shared_tokens_8", kind="shared", batch=8, heads=12, kv_heads=12, page=16, type="f32", new=1, cached=60, chunks=0, prefix=500, groups=1, window=0, sinks=0, mix=3),
        # A full decode batch behind one long instruction, the widest model.
        dict(name="shared_tokens_64", kind="shared", batch=64, heads=25, kv_heads=25, page=64, type="bf16", new=1, cached=500, chunks=0, prefix=4000, groups=1, window=0, sinks=0, mix=5),
        # Several instructions of their own lengths, some requests behind none, four query heads to a K/V head.
        dict(name="shared_groups_48", kind="shared", batch=48, heads=32, kv_heads=8, page=32, type="f16", new=1, cached=1000, chunks=0, prefix=2500, groups=3, window=0, sinks=0, mix=7),
        # The questions of six users about one document arrive together.
        dict(name="shared_chunks_6", kind="shared", batch=6, heads=16, kv_heads=16, page=16, type="f32", new=150, cached=1, chunks=6, prefix=1800, groups=1, window=0, sinks=0, mix=2),
        # One user, one new token in the middle of a context.
        dict(name="weights_token_kv777", kind="weights", batch=1, heads=12, kv_heads=12, page=16, type="f32", new=1, cached=776, chunks=0, window=0, sinks=0, mix=0),
        # A full decode batch, contexts of very different lengths.
        dict(name="weights_tokens_64", kind="weights", batch=64, heads=32, kv_heads=8, page=32, type="f16", new=1, cached=4096, chunks=0, window=0, sinks=0, mix=11),
        # Prompts that come in chunks, four at a time, each behind three earlier chunks.
        dict(name="weights_chunks_4x512", kind="weights", batch=4, heads=16, kv_heads=16, page=16, type="f32", new=512, cached=1536, chunks=4, window=0, sinks=0, mix=0),
        # The usual step of a busy server: two prompts of no round length among requests that decode.
        dict(name="weights_mixed_24", kind="weights", batch=24, heads=25, kv_heads=25, page=64, type="bf16", new=300, cached=1000, chunks=2, window=0, sinks=0, mix=5),
        # A few requests, most a little above their budget: what an ordinary step of a small server evicts.
        dict(name="evict_8", kind="evict", batch=8, heads=12, kv_heads=12, page=16, type="f32", cached=1200, limit=1100, keep=1000, recent=64, sinks=4, mix=1),
        # Long prompts of a full batch are cut down to their budget.
        dict(name="evict_64", kind="evict", batch=64, heads=25, kv_heads=25, page=64, type="bf16", cached=4096, limit=2200, keep=2000, recent=200, sinks=4, mix=9),
        # Bookkeeping of a small step.
        dict(name="trim_8", kind="trim", batch=8, page=16, cached=1200, limit=1100, keep=1000, mix=1),
        # Bookkeeping of a large step: half of the requests give pages back.
        dict(name="trim_512", kind="trim", batch=512, page=16, cached=4000, limit=2000, keep=1500, mix=4),
    ]


def _log(rng, lo, hi):
    """An integer of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["shared"] * 4 + ["weights"] * 4 + ["evict"] * 2 + ["trim"])
    page = rng.choice([8, 16, 16, 16, 32, 64, 128, rng.randint(1, 100)])
    type_ = rng.choice(["f32", "f32", "f16", "bf16"])
    mix = rng.randint(1, 1000)
    while kind in ("evict", "trim"):
        c = dict(kind=kind, batch=_log(rng, 1, 64 if kind == "evict" else 512), page=page, cached=_log(rng, 16, 8000 if kind == "evict" else 4000), mix=mix)
        c["limit"] = rng.randint(c["cached"] // 4, c["cached"])
        c["keep"] = rng.randint(c["limit"] // 2, c["limit"])
        if kind == "trim":
            return c
        c["kv_heads"] = c["heads"] = _log(rng, 1, 25)
        c["type"], c["sinks"] = type_, rng.choice([0, 1, 4, min(16, c["keep"])])
        c["sinks"] = min(c["sinks"], c["keep"])
        c["recent"] = rng.randint(0, min(c["keep"] - c["sinks"], max(c["keep"] // 4, 1)))
        if c["batch"] * c["kv_heads"] * c["cached"] * TYPES[type_].itemsize <= 64 * 25 * 4096 * 2:
            return c
    while True:
        kv_heads = _log(rng, 1, 25)
        c = dict(kind=kind, batch=_log(rng, 1, 64), heads=kv_heads * rng.choice([1, 1, 1, 2, 4, 5, 8]), kv_heads=kv_heads, page=page, type=type_, new=1,
                 cached=_log(rng, 1, 1000 if kind == "shared" else 8000), chunks=0, window=0, sinks=0, mix=mix)
        if kind == "shared":
            c["prefix"], c["groups"] = _log(rng, 1, 8000), rng.choice([1, 1, rng.randint(1, 6)])
        if rng.random() < 0.45:
            c["new"], c["chunks"] = _log(rng, 2, 512), rng.randint(1, c["batch"])
        if rng.random() < 0.25:
            c["window"], c["sinks"] = _log(rng, 1, 2000), rng.choice([0, 1, 4, 16])
        keys = c["cached"] + c["new"] + c.get("prefix", 0)
        # no dearer than the largest listed ones in K and V, rows and scores of the plain form
        if (c["heads"] <= 64 and c["batch"] * c["kv_heads"] * keys <= 64 * 25 * 4501 and c["batch"] * c["heads"] * c["new"] * keys <= 24 * 25 * 300 * 1300
                and work(c)["flops"] <= 15e9):
            return c


# ---- inputs ------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, std=1.0):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * std


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _pages(n, page):
    return -(-n // page)


def _lengths(case):
    """(cached, new) of every request, as plain lists: they belong to the case, so that work() knows them."""
    rng, batch = random.Random(case["mix"]), case["batch"]
    if case["kind"] in ("evict", "trim"):  # lengths around the limit: some requests have grown beyond it
        return [rng.randint(min(case["keep"], case["cached"]), case["cached"]) for _ in range(batch)], [0] * batch
    cached = [case["cached"] if case["mix"] == 0 else _log(rng, 1, case["cached"]) for _ in range(batch)]
    new = [1] * batch
    for b in rng.sample(range(batch), case["chunks"]):
        new[b] = case["new"] if case["mix"] == 0 else rng.randint((case["new"] + 1) // 2, case["new"])
    return cached, new


def _prefixes(case):
    """Lengths of the prefixes, and which one each request is behind (-1: none, where there are several)."""
    rng, groups = random.Random(case["mix"] + 1000), case["groups"]
    lens = [case["prefix"]] + [_log(rng, max(1, case["prefix"] // 8), case["prefix"]) for _ in range(groups - 1)]
    return lens, [0 if groups == 1 else rng.randrange(-1, groups) for _ in range(case["batch"])]


def _tables(g, held, width, order, at):
    """Block tables of the given width with held[b] pages of `order` a row, from place `at` on, and -1 behind them; the next place."""
    held = _ints(held)
    j = torch.arange(width, device="cuda")
    where = at + (torch.cumsum(held, 0) - held)[:, None] + j
    return torch.where(j < held[:, None], order[where.clamp(max=order.shape[0] - 1)], -1).int().contiguous(), at + int(held.sum())


def prepare(case, seed):
    g, kind, page, s = _gen(seed), case["kind"], case["page"], dict(case=case)
    cached, new = _lengths(case)
    kv = [c + n for c, n in zip(cached, new)]
    held = [_pages(n, page) for n in kv]
    prefixes, prefix_of = _prefixes(case) if kind == "shared" else ([], [])
    prefix_held = [_pages(n, page) for n in prefixes]
    pool = sum(held) + sum(prefix_held) + 3
    order = torch.randperm(pool, generator=g, device="cuda").int()
    s["block_tables"], at = _tables(g, held, max(held), order, 0)
    s["kv_lens"] = _ints(kv)
    if kind == "trim":
        s["n_free"], s["free_pages"] = _ints([3]), torch.cat([order[at:], order.new_full((at,), -1)])
        return s
    s["k_cache"], s["v_cache"] = (_randn(g, pool, case["kv_heads"], page, DH).to(TYPES[case["type"]]) for _ in range(2))
    if kind in ("evict", "weights"):
        # sums of attention weights: most keys have little, a few much, and some none at all
        w = torch.rand((pool, case["kv_heads"], page), generator=g, device="cuda")
        s["weights"] = torch.where(w < 0.05, 0.0, 0.01 * (-torch.log(w)) ** 4)
    if kind == "evict":
        return s
    s["query_start"] = _ints([sum(new[:b]) for b in range(len(new) + 1)])
    s["q"] = _randn(g, sum(new), case["heads"], DH, std=1.5)
    if kind == "shared":
        s["prefix_tables"], _ = _tables(g, prefix_held, max(prefix_held), order, at)
        s["prefix_lens"], s["prefix_of"] = _ints(prefixes), _ints(prefix_of)
    return s


# ---- the plain forms ---------------------------------------------------------------------

def _slots(table, keys, page):
    """The slot of each of the first `keys` positions of a table's rows (whatever, where there is no page)."""
    j = torch.arange(keys, device="cuda")
    return table.clamp(min=0).long()[:, (j // page).clamp(max=table.shape[1] - 1)] * page + j % page


def _attend(s, slots, kv, pos, weights=False):
    """Requests side by side, padded to the longest chunk and the most keys: slots [batch, keys], kv [batch] positions, pos [batch] of the first row.
    -> rows of o, and the weights that each key was given [batch, kv_heads, keys]."""
    c, q, start = s["case"], s["q"], s["query_start"].long()
    batch, kv_heads, longest, keys = c["batch"], c["kv_heads"], c["new"], slots.shape[1]
    group = c["heads"] // kv_heads
    i, j = torch.arange(longest, device="cuda"), torch.arange(keys, device="cuda")
    n_new = start[1:] - start[:-1]
    rows = q[(start[:-1, None] + i).clamp(max=q.shape[0] - 1)]
    rows = rows.view(batch, longest, kv_heads, group, DH).permute(0, 2, 3, 1, 4).reshape(batch, kv_heads, group * longest, DH)
    held = (j < kv[:, None])[:, None, :, None]

    def gather(cache):
        x = cache[slots // c["page"], :, slots % c["page"]].float().permute(0, 2, 1, 3)
        return torch.where(held, x, 0.0)

    scores = torch.matmul(rows, gather(s["k_cache"]).transpose(-1, -2).contiguous()) * DH ** -0.5
    at = pos[:, None, None] + i[:, None]
    seen = (j <= at) & (j < kv[:, None, None])
    if c["window"]:
        seen = seen & ((at - j < c["window"]) | (j < c["sinks"]))
    scores = scores.view(batch, kv_heads, group, longest, keys).masked_fill(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    w = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = w.sum(-1, keepdim=True)
    w = torch.where(total > 0, w / total, 0.0)
    out = torch.matmul(w.view(batch, kv_heads, group * longest, keys), gather(s["v_cache"]).contiguous())
    out = out.view(batch, kv_heads, group, longest, DH).permute(0, 3, 1, 2, 4).reshape(batch, longest, c["heads"], DH)
    t = torch.arange(q.shape[0], device="cuda")
    b = torch.searchsorted(start[1:].contiguous(), t, right=True)
    given = torch.where((i < n_new[:, None])[:, None, None, :, None], w, 0.0).sum((2, 3)) if weights else None
    return out[b, t - start[b]], given


def _plain_shared(s):
    page, kv, start = s["case"]["page"], s["kv_lens"].long(), s["query_start"].long()
    group = s["prefix_of"].long()
    real = (group >= 0) & (group < s["prefix_lens"].shape[0])
    before = torch.where(real, s["prefix_lens"].long()[group.clamp(min=0, max=s["prefix_lens"].shape[0] - 1)], 0)
    j = torch.arange(s["block_tables"].shape[1] * page + s["prefix_tables"].shape[1] * page, device="cuda")
    first = _slots(s["prefix_tables"], s["prefix_tables"].shape[1] * page, page)[group.clamp(min=0)]
    rest = _slots(s["block_tables"], s["block_tables"].shape[1] * page, page)
    slots = torch.where(j < before[:, None], first[:, j.clamp(max=first.shape[1] - 1)], rest.gather(1, (j - before[:, None]).clamp(min=0, max=rest.shape[1] - 1)))
    return _attend(s, slots, before + kv, before + kv - (start[1:] - start[:-1]))[0]


def _plain_weights(s):
    page, kv, start, table = s["case"]["page"], s["kv_lens"].long(), s["query_start"].long(), s["block_tables"]
    slots, n_new = _slots(table, table.shape[1] * page, page), start[1:] - start[:-1]
    out, given = _attend(s, slots, kv, kv - n_new, True)
    j = torch.arange(slots.shape[1], device="cuda")
    b, at = torch.nonzero((j < kv[:, None]) & (n_new > 0)[:, None], as_tuple=True)
    place = slots[b, at]
    old = torch.where((at < (kv - n_new)[b])[:, None], s["weights"][place // page, :, place % page], 0.0)
    s["weights"][place // page, :, place % page] = old + given[b, :, at]
    return out, s["weights"]


def _plain_evict(s):
    c, page, table, kv = s["case"], s["case"]["page"], s["block_tables"], s["kv_lens"].long()
    heads, keep = c["kv_heads"], c["keep"]
    slots = _slots(table, table.shape[1] * page, page)
    j = torch.arange(slots.shape[1], device="cuda")
    over = kv > c["limit"]
    n = kv[:, None, None]
    w = s["weights"][slots // page, :, slots % page].permute(0, 2, 1)
    # the first and the last ones before all others, then by weight
    w = torch.where((j < c["sinks"]) | (j >= n - c["recent"]), math.inf, w).masked_fill(j >= n, -math.inf)
    order = torch.sort(w, dim=-1, descending=True, stable=True)[1]
    kept = torch.zeros_like(w, dtype=torch.bool).scatter_(2, order[:, :, :keep], True) & (j < n) & over[:, None, None]
    hole = (j < keep) & ~kept & over[:, None, None]
    moves = kept & (j >= keep)
    # the i-th hole gets the i-th of those that move: both in order of requests, heads and places
    b, h, to = torch.nonzero(hole, as_tuple=True)
    b2, _, source = torch.nonzero(moves, as_tuple=True)
    to, source = slots[b, to], slots[b2, source]
    for cache in (s["k_cache"], s["v_cache"], s["weights"]):
        cache[to // page, h, to % page] = cache[source // page, h, source % page]
    return s["k_cache"], s["v_cache"], s["weights"]


def _plain_trim(s):
    c, page, table, kv, pages = s["case"], s["case"]["page"], s["block_tables"], s["kv_lens"].long(), s["free_pages"]
    n_free, capacity = s["n_free"].long(), pages.shape[0]
    over = kv > c["limit"]
    left = torch.where(over, c["keep"], kv)
    have, first = (kv + page - 1) // page, (left + page - 1) // page
    given = have - first
    j = torch.arange(table.shape[1], device="cuda")
    at = n_free + (torch.cumsum(given, 0) - given)[:, None] + j - first[:, None]
    at = torch.where((j >= first[:, None]) & (j < have[:, None]), at, capacity).clamp(max=capacity)
    pages.copy_(torch.cat([pages, pages.new_zeros(1)]).scatter(0, at.reshape(-1), table.reshape(-1))[:-1])
    return left.int(), (kv - left).int(), (n_free + given.sum()).int(), pages


PLAIN = {"shared": _plain_shared, "weights": _plain_weights, "evict": _plain_evict, "trim": _plain_trim}


# ---- the framework's operators -----------------------------------------------------------

_ops = None


def _framework():
    global _ops
    if _ops is None:
        import __graft_entry__ as entry
        entry.load_package()
        from async_gpu_amd import ops
        _ops = ops
    return _ops


def _own(s):
    ops, c = _ops or _framework(), s["case"]
    if c["kind"] == "shared":
        return ops.paged_attention_shared(s["q"], s["k_cache"], s["v_cache"], s["prefix_tables"], s["prefix_lens"], s["prefix_of"], s["block_tables"], s["kv_lens"],
                                          s["query_start"], c["window"], c["sinks"])
    if c["kind"] == "weights":
        return ops.paged_attention_weights(s["q"], s["k_cache"], s["v_cache"], s["weights"], s["block_tables"], s["kv_lens"], s["query_start"], c["window"], c["sinks"])
    if c["kind"] == "evict":
        return ops.paged_evict(s["k_cache"], s["v_cache"], s["weights"], s["block_tables"], s["kv_lens"], c["limit"], c["keep"], c["recent"], c["sinks"])
    return (*ops.paged_trim(s["kv_lens"], s["block_tables"], s["free_pages"], s["n_free"], c["page"], c["limit"], c["keep"]), s["free_pages"])


def run(state):
    if own:
        return _own(state)
    return PLAIN[state["case"]["kind"]](state)


# ---- what a pass cannot do without -------------------------------------------------------

def _visible(case, i):
    """How many keys the row at position i sees."""
    return i + 1 if not case["window"] or i < case["window"] else case["window"] + min(case["sinks"], i + 1 - case["window"])


def work(case):
    kind, page = case["kind"], case["page"]
    cached, new = _lengths(case)
    if kind == "trim":
        given = sum(_pages(n, page) - _pages(case["keep"], page) for n in cached if n > case["limit"])
        return {"bytes": 12 * case["batch"] + 8 * given, "flops": 0}
    size = TYPES[case["type"]].itemsize
    if kind == "evict":
        read, moved = 0, 0.0
        for n in cached:
            if n <= case["limit"]:
                continue
            read += n
            # of the places from `keep` on the last ones stay, and of the others as many as of all that are neither first nor last
            last, rest = min(case["recent"], n - case["keep"]), n - case["sinks"] - case["recent"]
            moved += last + (n - case["keep"] - last) * (case["keep"] - case["sinks"] - case["recent"]) / max(rest, 1)
        return {"bytes": int(case["kv_heads"] * (4 * read + moved * 2 * (2 * DH * size + 4))), "flops": 0}
    prefixes, prefix_of = _prefixes(case) if kind == "shared" else ([], [-1] * case["batch"])
    pairs, read, shared = 0, 0, {}
    for c, n, g in zip(cached, new, prefix_of):
        before = prefixes[g] if g >= 0 else 0
        seen = [_visible(case, before + i) for i in (c, c + n - 1)]  # of the chunk's first and last row
        pairs += sum(seen) * n // 2
        union = seen[0] + n - 1  # each later row brings a key more
        own_keys = min(union, c + n)
        read += own_keys
        if g >= 0:
            shared[g] = max(shared.get(g, 0), min(union - own_keys, before))
    read += sum(shared.values())
    rows = sum(new)
    moved = 2 * read * case["kv_heads"] * DH * size + 8 * rows * case["heads"] * DH
    if kind == "weights":
        moved += 8 * read * case["kv_heads"]
    return {"bytes": moved, "flops": 4 * DH * case["heads"] * pairs}


# ---- the definitions in 64 bits ----------------------------------------------------------

def _rows64(case, q, k, v, first):
    """Rows [n, heads, 64] at positions first .. over keys [kv_heads, m, 64]: o, and the weight that each key was given [kv_heads, m]."""
    n, m, group = q.shape[0], k.shape[1], case["heads"] // case["kv_heads"]
    at, j = torch.arange(first, first + n, device="cuda")[:, None], torch.arange(m, device="cuda")[None]
    bias = torch.zeros((n, m), dtype=torch.float64, device="cuda")
    bias[j > at] = -math.inf
    if case["window"]:
        bias[(j <= at - case["window"]) & (j >= case["sinks"])] = -math.inf
    out, given = torch.empty_like(q), torch.zeros((case["kv_heads"], m), dtype=torch.float64, device="cuda")
    for h in range(case["heads"]):
        p = torch.softmax(torch.mm(q[:, h], k[h // group].t().contiguous()) / 8.0 + bias, -1)
        out[:, h] = torch.mm(p, v[h // group])
        given[h // group] += p.sum(0)
    return out, given


def _held64(cache, table, n, page):
    """The first n positions that a row of a table stands for: [kv_heads, n, ...] in 64 bits."""
    x = cache[table[:_pages(n, page)].long()].double()
    return x.transpose(0, 1).flatten(1, 2)[:, :n]


def _exact_shared(s):
    c, page = s["case"], s["case"]["page"]
    start, kv, lens, of = (s[k].tolist() for k in ("query_start", "kv_lens", "prefix_lens", "prefix_of"))
    out = torch.zeros_like(s["q"], dtype=torch.float64)
    for b in range(c["batch"]):
        parts = [(s["block_tables"][b], kv[b])]
        if of[b] >= 0:
            parts.insert(0, (s["prefix_tables"][of[b]], lens[of[b]]))
        k, v = (torch.cat([_held64(s[name], table, n, page) for table, n in parts], 1) for name in ("k_cache", "v_cache"))
        rows = slice(start[b], start[b + 1])
        out[rows] = _rows64(c, s["q"][rows].double(), k, v, k.shape[1] - (start[b + 1] - start[b]))[0]
    return out


def _exact_weights(s):
    c, page = s["case"], s["case"]["page"]
    start, kv = s["query_start"].tolist(), s["kv_lens"].tolist()
    out, weights = torch.zeros_like(s["q"], dtype=torch.float64), s["weights"].double()
    for b in range(c["batch"]):
        n = start[b + 1] - start[b]
        k, v, before = (_held64(s[name], s["block_tables"][b], kv[b], page) for name in ("k_cache", "v_cache", "weights"))
        rows = slice(start[b], start[b + 1])
        out[rows], given = _rows64(c, s["q"][rows].double(), k, v, kv[b] - n)
        before[:, kv[b] - n:] = 0.0
        ids = s["block_tables"][b, :_pages(kv[b], page)].long()
        flat = weights[ids].transpose(0, 1).flatten(1, 2)
        flat[:, :kv[b]] = before + given
        weights[ids] = flat.unflatten(1, (-1, page)).transpose(0, 1)
    return out, weights


def _exact_evict(s):
    c, page = s["case"], s["case"]["page"]
    caches = {name: s[name].double() for name in ("k_cache", "v_cache", "weights")}
    weights, tables = s["weights"].cpu(), s["block_tables"].cpu()
    for b, n in enumerate(s["kv_lens"].tolist()):
        if n <= c["limit"]:
            continue
        ids = tables[b, :_pages(n, page)].long()
        for h in range(c["kv_heads"]):
            w = weights[ids, h].reshape(-1)[:n].tolist()
            rest = sorted(range(c["sinks"], n - c["recent"]), key=lambda j: (-w[j], j))[:c["keep"] - c["sinks"] - c["recent"]]
            kept = set(rest) | set(range(c["sinks"])) | set(range(n - c["recent"], n))
            holes, moves = [j for j in range(c["keep"]) if j not in kept], [j for j in range(c["keep"], n) if j in kept]
            to, source = torch.tensor(holes, dtype=torch.long), torch.tensor(moves, dtype=torch.long)
            at, source = (ids[to // page].cuda(), (to % page).cuda()), (ids[source // page].cuda(), (source % page).cuda())
            for x in caches.values():
                x[at[0], h, at[1]] = x[source[0], h, source[1]]
    return caches["k_cache"], caches["v_cache"], caches["weights"]


def _exact_trim(s):
    c, page = s["case"], s["case"]["page"]
    tables, pages, n_free = s["block_tables"].tolist(), s["free_pages"].tolist(), int(s["n_free"])
    kv, evicted = [], []
    for b, n in enumerate(s["kv_lens"].tolist()):
        left = c["keep"] if n > c["limit"] else n
        for j in range(_pages(left, page), _pages(n, page)):
            pages[n_free] = tables[b][j]
            n_free += 1
        kv.append(left)
        evicted.append(n - left)
    return _ints(kv), _ints(evicted), _ints([n_free]), _ints(pages)


def exact(case, seed):
    s = prepare(case, seed)
    return {"shared": _exact_shared, "weights": _exact_weights, "evict": _exact_evict, "trim": _exact_trim}[case["kind"]](s)
