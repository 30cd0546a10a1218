"""Performance cases of the operators that serve several requests over a KV cache in pages.

A server step is: paged_plan turns the requests' lengths into block tables, slots and positions; paged_kv_append puts the new K and V
rows into their pages; paged_attention attends ragged chunks and single tokens over them, with or without a sliding window; sample draws
the next tokens.  Each case is one call of one of them.

run() is the plain form, elementary torch operations in 32 bits (64 for the draw, whose result hangs on sums next to a border), or with
`own` set the framework's operator.  exact() is the same in 64 bits, request by request.
"""
import math
import random

import torch

own = False
DH = 64  # the framework's head size
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # One user, one new token in the middle of a context: the smallest call, the small model's heads over an fp32 cache.
        dict(name="attend_token_kv777", kind="attention", batch=1, heads=12, kv_heads=12, page=16, type="f32", new=1, cached=776, chunks=0, window=0, sinks=0, mix=0),
        # A full decode batch, contexts of very different lengths, four query heads to a K/V head, a cache of half the bytes.
        dict(name="attend_tokens_64_shared", kind="attention", batch=64, heads=32, kv_heads=8, page=32, type="f16", new=1, cached=4096, chunks=0, window=0, sinks=0, mix=11),
        # Prompts that come in chunks, four at a time, each behind three earlier chunks.
        dict(name="attend_chunks_4x512", kind="attention", batch=4, heads=16, kv_heads=16, page=16, type="f32", new=512, cached=1536, chunks=4, window=0, sinks=0, mix=0),
        # The usual step of a busy server: two prompts of no round length among requests that decode, the widest model.
        dict(name="attend_mixed_24", kind="attention", batch=24, heads=25, kv_heads=25, page=64, type="bf16", new=300, cached=1000, chunks=2, window=0, sinks=0, mix=5),
        # Long streams under a sliding window, whose first tokens stay visible.
        dict(name="attend_window_8x256", kind="attention", batch=8, heads=16, kv_heads=16, page=16, type="bf16", new=256, cached=8000, chunks=8, window=1024, sinks=4, mix=0),
        # The K and V rows of a decode step of sixteen, three of them padding.
        dict(name="append_16", kind="append", rows=16, pad=3, kv_heads=12, page=16, type="f32"),
        # The rows of a large prefill step go to a 16-bit cache.
        dict(name="append_4096_bf16", kind="append", rows=4096, pad=0, kv_heads=25, page=64, type="bf16"),
        # Bookkeeping of a small decode step.
        dict(name="plan_8", kind="plan", batch=8, page=16, new=1, cached=1000, ended=0, mix=3),
        # Bookkeeping of a large step: many requests, prompts of all lengths, some requests that have ended.
        dict(name="plan_512_prompts", kind="plan", batch=512, page=16, new=200, cached=2000, ended=20, mix=4),
        # One user's draw as the example programs make it: temperature 0.8, top 40 of the full vocabulary.
        dict(name="sample_1_top40", kind="sample", rows=1, vocab=50257, temperature=0.8, top_k=40, top_p=1.0, min_p=0.0),
        # A batch whose requests each bring their own settings.
        dict(name="sample_32_mixed", kind="sample", rows=32, vocab=50257, temperature=-1.0, top_k=0, top_p=1.0, min_p=0.0),
        # A large batch of nucleus sampling.
        dict(name="sample_256_nucleus", kind="sample", rows=256, vocab=50257, temperature=1.0, top_k=0, top_p=0.95, min_p=0.0),
    ]


def _log(rng, lo, hi):
    """An integer of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["attention"] * 5 + ["sample"] * 3 + ["append"] * 2 + ["plan"] * 2)
    page = rng.choice([8, 16, 16, 16, 32, 64, 128, rng.randint(1, 100)])
    type_ = rng.choice(["f32", "f32", "f16", "bf16"])
    if kind == "append":
        rows = _log(rng, 1, 4096)
        return dict(kind=kind, rows=rows, pad=rng.choice([0, 0, rng.randint(0, rows)]), kv_heads=_log(rng, 1, 25), page=page, type=type_)
    if kind == "plan":
        batch = _log(rng, 1, 512)
        return dict(kind=kind, batch=batch, page=page, new=_log(rng, 1, 200), cached=_log(rng, 1, 2000), ended=rng.choice([0, rng.randint(0, batch // 4)]),
                    mix=rng.randint(1, 1000))
    if kind == "sample":
        vocab = 50257 if rng.random() < 0.5 else _log(rng, 2, 60000)
        if rng.random() < 0.4:
            return dict(kind=kind, rows=_log(rng, 1, 200), vocab=vocab, temperature=-1.0, top_k=0, top_p=1.0, min_p=0.0)
        return dict(kind=kind, rows=_log(rng, 1, 200), vocab=vocab, temperature=rng.choice([0.0, 0.7, 1.0, 1.3]), top_k=rng.choice([0, 0, 1, 40, _log(rng, 1, 2000)]),
                    top_p=rng.choice([1.0, 1.0, 0.9, round(rng.uniform(0.05, 0.99), 3)]), min_p=rng.choice([0.0, 0.0, 0.05, 0.2]))
    while True:
        kv_heads = _log(rng, 1, 25)
        c = dict(kind=kind, batch=_log(rng, 1, 64), heads=kv_heads * rng.choice([1, 1, 1, 2, 4, 5, 8]), kv_heads=kv_heads, page=page, type=type_, new=1,
                 cached=_log(rng, 1, 8000), chunks=0, window=0, sinks=0, mix=rng.choice([0, rng.randint(1, 1000), rng.randint(1, 1000)]))
        if rng.random() < 0.55:
            c["new"], c["chunks"] = _log(rng, 2, 512), rng.randint(1, c["batch"])
        if rng.random() < 0.3:
            c["window"], c["sinks"] = _log(rng, 1, 2000), rng.choice([0, 1, 4, 16])
        # no dearer than the largest listed ones in K and V, rows and scores of the plain form
        if (c["heads"] <= 64 and c["batch"] * c["kv_heads"] * (c["cached"] + c["new"]) <= 64 * 8 * 4097
                and c["batch"] * c["heads"] * c["new"] * (c["cached"] + c["new"]) <= 24 * 25 * 300 * 1300 and work(c)["flops"] <= 15e9):
            return c


# ---- inputs ------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, std=1.0, mean=0.0):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * std + mean


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _lengths(case):
    """(cached, new) of every request, as plain lists: they belong to the case, so that work() knows them."""
    rng, batch = random.Random(case["mix"]), case["batch"]
    cached = [case["cached"] if case["mix"] == 0 else _log(rng, 1, case["cached"]) for _ in range(batch)]
    if case["kind"] == "plan":
        new = [_log(rng, 1, case["new"]) for _ in range(batch)]
        for b in rng.sample(range(batch), case["ended"]):
            new[b] = -1
    else:
        new = [1] * batch
        for b in rng.sample(range(batch), case["chunks"]):
            new[b] = case["new"] if case["mix"] == 0 else rng.randint((case["new"] + 1) // 2, case["new"])
    return cached, new


def _pages(n, page):
    return -(-n // page)


def _table(g, held, width, pool):
    """Block tables [batch, width] with `held` pages of a shuffled pool a row, -1 behind them, and the shuffled pool."""
    order = torch.randperm(pool, generator=g, device="cuda").to(torch.int32)
    j = torch.arange(width, device="cuda")
    at = (torch.cumsum(held, 0) - held)[:, None] + j
    return torch.where(j < held[:, None], order[at.clamp(max=pool - 1)], -1).contiguous(), order


def prepare(case, seed):
    g, kind, s = _gen(seed), case["kind"], dict(case=case)
    if kind == "sample":
        rows, n = case["rows"], case["vocab"]
        # a language model's logits: a broad mass, and a few tokens well above it
        s["logits"] = _randn(g, rows, n, std=2.5, mean=-35.0)
        likely = torch.randint(0, n, (rows, 24), generator=g, device="cuda")
        s["logits"].scatter_add_(1, likely, 10.0 * torch.rand((rows, 24), generator=g, device="cuda"))
        s["u"] = torch.rand(rows, generator=g, device="cuda")
        s["settings"] = {k: case[k] for k in ("temperature", "top_k", "top_p", "min_p")}
        if case["temperature"] < 0:  # each request its own
            pick = lambda values, dtype: torch.tensor(values, dtype=dtype, device="cuda")[torch.randint(0, len(values), (rows,), generator=g, device="cuda")]  # noqa: E731
            s["settings"] = dict(temperature=pick([0.0, 0.6, 0.8, 1.0, 1.2], torch.float32), top_k=pick([0, 0, 1, 40, 200], torch.int32),
                                 top_p=pick([1.0, 0.9, 0.95], torch.float32), min_p=pick([0.0, 0.0, 0.05], torch.float32))
        return s
    if kind == "append":
        rows, page, heads = case["rows"], case["page"], case["kv_heads"]
        pool = _pages(rows, page) + 3
        # K and V as they lie in the rows of a QKV projection
        qkv = _randn(g, rows, 3 * heads, DH)
        s["k"], s["v"] = qkv[:, heads:2 * heads], qkv[:, 2 * heads:]
        s["slots"] = torch.randperm(pool * page, generator=g, device="cuda")[:rows].to(torch.int32)
        s["slots"][rows - case["pad"]:] = -1
        s["k_cache"], s["v_cache"] = (_randn(g, pool, heads, page, DH).to(TYPES[case["type"]]) for _ in range(2))
        return s
    cached, new = _lengths(case)
    page = case["page"]
    if kind == "plan":
        held = _ints([_pages(c, page) for c in cached])
        total = sum(_pages(c + max(n, 0), page) for c, n in zip(cached, new))
        pool, width = total + 5, _pages(case["cached"] + case["new"], page)
        s["block_tables"], order = _table(g, held, width, pool)
        n_held = sum(_pages(c, page) for c in cached)
        s["n_free"] = _ints([pool - n_held])
        s["free_pages"] = torch.cat([order[n_held:], order.new_full((n_held,), -1)])
        s["cached_lens"], s["new_lens"] = _ints(cached), _ints(new)
        s["max_tokens"] = sum(max(n, 0) for n in new) + 7  # padded, as for a fixed launch shape
        return s
    kv = [c + n for c, n in zip(cached, new)]
    held, width = _ints([_pages(n, page) for n in kv]), _pages(case["cached"] + case["new"], page)
    pool = sum(_pages(n, page) for n in kv) + 3
    s["block_tables"], _ = _table(g, held, width, pool)
    s["kv_lens"] = _ints(kv)
    s["query_start"] = _ints([sum(new[:b]) for b in range(len(new) + 1)])
    s["q"] = _randn(g, sum(new), case["heads"], DH, std=1.5)
    s["k_cache"], s["v_cache"] = (_randn(g, pool, case["kv_heads"], page, DH).to(TYPES[case["type"]]) for _ in range(2))
    return s


# ---- the plain forms ---------------------------------------------------------------------

def _plain_plan(s):
    page, max_tokens, width = s["case"]["page"], s["max_tokens"], s["block_tables"].shape[1]
    cached, new, table, pages = s["cached_lens"].long(), s["new_lens"].long(), s["block_tables"], s["free_pages"]
    n_free, capacity = s["n_free"].long(), pages.shape[0]
    ended, have = new < 0, (cached + page - 1) // page
    rel = torch.where(ended, have, 0)
    new = new.clamp(min=0)
    need = (cached + new + page - 1) // page - have
    fits = ~ended & (have + need <= width)
    new, need = torch.where(fits, new, 0), torch.where(fits, need, 0)
    top = n_free + rel.sum()
    ok = (torch.cumsum(need, 0) <= top) & (torch.cumsum(new, 0) <= max_tokens)
    new, need = torch.where(ok, new, 0), torch.where(ok, need, 0)
    kv = torch.where(ended, 0, cached + new)
    start = torch.cat([new.new_zeros(1), torch.cumsum(new, 0)])
    # the stack with the released pages on it; one place more takes what is none
    j = torch.arange(width, device="cuda")
    at = torch.where(j < rel[:, None], n_free + (torch.cumsum(rel, 0) - rel)[:, None] + j, capacity).clamp(max=capacity)
    stack = torch.cat([pages, pages.new_zeros(1)]).scatter(0, at.reshape(-1), table.reshape(-1))
    # new pages, from the top of the stack down
    nth = (torch.cumsum(need, 0) - need)[:, None] + j - have[:, None]
    fresh = (j >= have[:, None]) & (j < (have + need)[:, None])
    table.copy_(torch.where(fresh, stack[torch.where(fresh, top - 1 - nth, 0)], table))
    left = top - need.sum()
    pages.copy_(torch.where(torch.arange(capacity, device="cuda") < left, stack[:-1], pages))
    t = torch.arange(max_tokens, device="cuda")
    b = torch.searchsorted(start[1:].contiguous(), t, right=True).clamp(max=new.shape[0] - 1)
    real = t < start[-1]
    pos = torch.where(real, cached[b] + t - start[b], 0)
    slots = torch.where(real, table[b, pos // page].long() * page + pos % page, -1)
    return kv.int(), start.int(), slots.int(), pos.int(), left.int(), table, pages


def _plain_append(s):
    k_cache, v_cache, slots, page = s["k_cache"], s["v_cache"], s["slots"].long(), s["case"]["page"]
    pool = k_cache.shape[0] * page
    real = torch.nonzero((slots >= 0) & (slots < pool))[:, 0]
    slots = slots[real]
    k_cache[slots // page, :, slots % page] = s["k"][real].to(k_cache.dtype)
    v_cache[slots // page, :, slots % page] = s["v"][real].to(v_cache.dtype)
    return k_cache, v_cache


def _plain_attention(s):
    c, q, start, kv, table = s["case"], s["q"], s["query_start"].long(), s["kv_lens"].long(), s["block_tables"]
    batch, kv_heads, longest = c["batch"], c["kv_heads"], c["new"]
    group, keys = c["heads"] // kv_heads, table.shape[1] * c["page"]
    # requests side by side, padded to the longest chunk and the widest table
    i, j = torch.arange(longest, device="cuda"), torch.arange(keys, device="cuda")
    n_new = start[1:] - start[:-1]
    rows = q[(start[:-1, None] + i).clamp(max=q.shape[0] - 1)]
    rows = rows.view(batch, longest, kv_heads, group, DH).permute(0, 2, 3, 1, 4).reshape(batch, kv_heads, group * longest, DH)
    held = (j < kv[:, None])[:, None, :, None]

    def gather(cache):
        x = cache[table.clamp(min=0).long()].float().permute(0, 2, 1, 3, 4).reshape(batch, kv_heads, keys, DH)
        return torch.where(held, x, 0.0)

    scores = torch.matmul(rows, gather(s["k_cache"]).transpose(-1, -2).contiguous()) * DH ** -0.5
    pos = (kv - n_new)[:, None, None] + i[:, None]
    seen = (j <= pos) & (j < kv[:, None, None])
    if c["window"]:
        seen = seen & ((pos - j < c["window"]) | (j < c["sinks"]))
    scores = scores.view(batch, kv_heads, group, longest, keys).masked_fill(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    w = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = w.sum(-1, keepdim=True)
    out = torch.matmul(w.view(batch, kv_heads, group * longest, keys), gather(s["v_cache"])).view(batch, kv_heads, group, longest, DH)
    out = torch.where(total > 0, out / total, 0.0).permute(0, 3, 1, 2, 4).reshape(batch, longest, c["heads"], DH)
    t = torch.arange(q.shape[0], device="cuda")
    b = torch.searchsorted(start[1:].contiguous(), t, right=True)
    return out[b, t - start[b]]


def _plain_sample(s):
    x, u, settings = s["logits"], s["u"].double(), s["settings"]
    rows, n = x.shape
    # settings are numbers of 32 bits, whether they come as one for all rows or as one a row
    temperature, top_k, top_p, min_p = (torch.as_tensor(settings[k], dtype=torch.float32, device="cuda").double().expand(rows)[:, None]
                                        for k in ("temperature", "top_k", "top_p", "min_p"))
    x, order = torch.sort(torch.where(x.isnan(), -math.inf, x).double(), dim=-1, descending=True, stable=True)
    top = x[:, :1]
    w = torch.exp(torch.where(x == top, 0.0, x - top) / temperature.clamp(min=1e-8))
    rank = torch.arange(n, device="cuda")
    w = torch.where((rank < top_k) | (top_k <= 0), w, 0.0)
    before = torch.cumsum(w, -1) - w
    w = torch.where(((before < top_p * w.sum(-1, keepdim=True)) & (w >= min_p)) | (rank == 0), w, 0.0)
    run_ = torch.cumsum(w, -1)
    past = (run_ > u[:, None] * run_[:, -1:]) & (w > 0)
    last = (w > 0).sum(-1) - 1  # what is kept comes first
    at = torch.where(past.any(-1), past.int().argmax(-1), last)
    token = order.gather(1, at[:, None])[:, 0]
    return torch.where(top[:, 0] == -math.inf, -1, token).int()


PLAIN = {"plan": _plain_plan, "append": _plain_append, "attention": _plain_attention, "sample": _plain_sample}


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
    if c["kind"] == "plan":
        made = ops.paged_plan(s["cached_lens"], s["new_lens"], s["block_tables"], s["free_pages"], s["n_free"], c["page"], s["max_tokens"])
        return (*made, s["block_tables"], s["free_pages"])
    if c["kind"] == "append":
        return ops.paged_kv_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"])
    if c["kind"] == "attention":
        return ops.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["block_tables"], s["kv_lens"], s["query_start"], c["window"], c["sinks"])
    return ops.sample(s["logits"], s["u"], **s["settings"])


def run(state):
    if own:
        return _own(state)
    return PLAIN[state["case"]["kind"]](state)


# ---- what a pass cannot do without -------------------------------------------------------

def _visible(case, kv, i):
    """How many keys query i (of the last ones of kv) sees."""
    return i + 1 if not case["window"] or i < case["window"] else case["window"] + min(case["sinks"], i + 1 - case["window"])


def work(case):
    kind = case["kind"]
    if kind == "sample":
        return {"bytes": 4 * case["rows"] * (case["vocab"] + 6), "flops": 2 * case["rows"] * case["vocab"]}
    if kind == "append":
        real = case["rows"] - case["pad"]
        return {"bytes": 2 * real * case["kv_heads"] * DH * (4 + TYPES[case["type"]].itemsize) + 4 * case["rows"], "flops": 0}
    cached, new = _lengths(case)
    page = case["page"]
    if kind == "plan":
        made = sum(_pages(c + n, page) - _pages(c, page) for c, n in zip(cached, new) if n > 0)
        given = sum(_pages(c, page) for c, n in zip(cached, new) if n < 0)
        return {"bytes": 20 * case["batch"] + 8 * sum(max(n, 0) for n in new) + 8 * (made + given), "flops": 0}
    pairs, read = 0, 0
    for c, n in zip(cached, new):
        first = _visible(case, c + n, c)  # of the chunk's first query; each later one brings a key more
        pairs += sum(_visible(case, c + n, i) for i in (c, c + n - 1)) * n // 2
        read += first + n - 1
    rows = sum(new)
    return {"bytes": 2 * read * case["kv_heads"] * DH * TYPES[case["type"]].itemsize + 8 * rows * case["heads"] * DH, "flops": 4 * DH * case["heads"] * pairs}


# ---- the definitions in 64 bits ----------------------------------------------------------

def _exact_plan(s):
    page, max_tokens = s["case"]["page"], s["max_tokens"]
    cached, new, table, pages = (s[k].tolist() for k in ("cached_lens", "new_lens", "block_tables", "free_pages"))
    stack = pages[:int(s["n_free"])]
    for b, n in enumerate(new):
        if n < 0:
            stack += table[b][:_pages(cached[b], page)]
    kv, start, slots, positions, full = [], [0], [], [], False
    for b, n in enumerate(new):
        have, want = _pages(cached[b], page), _pages(cached[b] + max(n, 0), page)
        if n >= 0 and want <= len(table[b]):
            full = full or want - have > len(stack) or len(slots) + n > max_tokens
        if n < 0 or want > len(table[b]) or full:
            kv.append(0 if n < 0 else cached[b])
            start.append(len(slots))
            continue
        for k in range(have, want):
            table[b][k] = stack.pop()
        for p in range(cached[b], cached[b] + n):
            slots.append(table[b][p // page] * page + p % page)
            positions.append(p)
        kv.append(cached[b] + n)
        start.append(len(slots))
    pad = max_tokens - len(slots)
    pages[:len(stack)] = stack
    return _ints(kv), _ints(start), _ints(slots + [-1] * pad), _ints(positions + [0] * pad), _ints([len(stack)]), _ints(table), _ints(pages)


def _exact_append(s):
    page, slots, made = s["case"]["page"], s["slots"].tolist(), []
    for rows, cache in ((s["k"], s["k_cache"]), (s["v"], s["v_cache"])):
        flat = cache.double().transpose(1, 2).reshape(-1, cache.shape[1], DH)  # [slot, head, dh]
        for t, slot in enumerate(slots):
            if 0 <= slot < flat.shape[0]:
                flat[slot] = rows[t].double()
        made.append(flat.view(-1, page, cache.shape[1], DH).transpose(1, 2).contiguous())
    return tuple(made)


def _exact_attention(s):
    c, q = s["case"], s["q"].double()
    group, out = c["heads"] // c["kv_heads"], torch.zeros_like(s["q"], dtype=torch.float64)
    start, kv = s["query_start"].tolist(), s["kv_lens"].tolist()
    for b in range(c["batch"]):
        n = start[b + 1] - start[b]
        if n == 0 or kv[b] == 0:
            continue
        ids = s["block_tables"][b, :_pages(kv[b], c["page"])].long()
        k, v = (t[ids].double().transpose(0, 1).reshape(c["kv_heads"], -1, DH)[:, :kv[b]] for t in (s["k_cache"], s["v_cache"]))
        at, j = torch.arange(kv[b] - n, kv[b], device="cuda")[:, None], torch.arange(kv[b], device="cuda")[None]
        bias = torch.zeros((n, kv[b]), dtype=torch.float64, device="cuda")
        bias[j > at] = -math.inf
        if c["window"]:
            bias[(j <= at - c["window"]) & (j >= c["sinks"])] = -math.inf
        for h in range(c["heads"]):
            p = torch.softmax(torch.mm(q[start[b]:start[b + 1], h], k[h // group].t().contiguous()) / 8.0 + bias, -1)
            out[start[b]:start[b + 1], h] = torch.mm(p, v[h // group])
    return out


def _exact_sample(s):
    settings, tokens = s["settings"], []
    rows = s["logits"].shape[0]
    value = lambda k, r: float(settings[k][r] if torch.is_tensor(settings[k]) else torch.tensor(settings[k], dtype=torch.float32))  # noqa: E731
    for r in range(rows):
        x = s["logits"][r].double()
        temperature, top_k, top_p, min_p = (value(k, r) for k in ("temperature", "top_k", "top_p", "min_p"))
        x, order = torch.sort(x, descending=True, stable=True)
        w = torch.exp((x - x[0]) / max(temperature, 1e-8))
        if top_k > 0:
            w = w[:int(top_k)]
        share = torch.cumsum(w / w.sum(), 0)
        kept = 1 + int((share[:-1] < top_p).sum())
        kept = max(1, min(kept, int((w >= min_p).sum())))
        share = torch.cumsum(w[:kept] / w[:kept].sum(), 0)
        tokens.append(int(order[min(kept - 1, int((share <= float(s["u"][r])).sum()))]))
    return _ints(tokens)


def exact(case, seed):
    s = prepare(case, seed)
    return {"plan": _exact_plan, "append": _exact_append, "attention": _exact_attention, "sample": _exact_sample}[case["kind"]](s)
