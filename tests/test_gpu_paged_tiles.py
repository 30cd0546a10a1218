"""paged_attention where tiles of rows and single rows could differ: windows at the end of 32 bits, magnitudes far from one, rows of nobody at either end of the
calls, and many heads a K/V head in many requests."""
import numpy as np
import pytest
from test_gpu_paged import TYPES, _cache, _tables, attend64, check

pytestmark = pytest.mark.gpu


def _i32(dev):
    import torch
    return lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=dev)


def _call(dev, q, kc, vc, tables, lens, start, window=0, sinks=0, **kw):
    from async_gpu_amd import ops
    i32 = _i32(dev)
    return ops.paged_attention(q, kc, vc, i32(tables), i32(lens), i32(start), window, sinks, **kw)


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("window", [2**31 - 1, 2**31 - 12, 2**31 - 30, 2**30])
@pytest.mark.parametrize("sinks", [0, 3, 2**31 - 1])
def test_windows_as_large_as_numbers_go(agpu, dev, type_, window, sinks):
    """Requests with fewer positions than rows, whose first rows lie before position 0 and see nothing, under a window that hides nothing."""
    import torch
    lens, new = [5, 33, 1, 0, 200], [12, 40, 30, 20, 200]
    rng, g = np.random.default_rng(2), torch.Generator(device=dev).manual_seed(3)
    kc, vc = _cache(torch, g, dev, 40, 2, 16, type_)
    tables, start = _tables(rng, lens, 16, 40), np.concatenate([[0], np.cumsum(new)]).tolist()
    q = torch.randn((start[-1], 4, 64), generator=g, device=dev)
    got = _call(dev, q, kc, vc, tables, lens, start, window, sinks)
    check(got, *attend64(q, kc, vc, tables, lens, start, window, sinks))
    assert torch.equal(got, _call(dev, q, kc, vc, tables, lens, start))
    # the same rows one by one
    for b in (0, 1):
        one = _call(dev, q[start[b]:start[b] + 2], kc, vc, tables[[b, b]], [lens[b] - new[b] + 1, 0], [0, 1, 1], window, sinks)
        check(one[:1], *(x[:1] for x in attend64(q[start[b]:start[b] + 2], kc, vc, tables[[b, b]], [lens[b] - new[b] + 1, 0], [0, 1, 1], window, sinks)))


@pytest.mark.parametrize("type_", ["float32", "bfloat16"])
@pytest.mark.parametrize("large", [1e36, 1e37, 3e37])
@pytest.mark.parametrize("step", [5.9, 3.0, -5.9])
def test_large_values_behind_rising_scores(agpu, dev, type_, large, step):
    """Scores that rise by a little less than 6 octaves from tile to tile of 32 keys, and values whose sums with weights of one stay finite."""
    import torch
    kv, rows, page = 192 + 40, 40, 16
    kc, vc = (torch.zeros((15, 1, page, 64), dtype=getattr(torch, type_), device=dev) for _ in range(2))
    tables = np.arange(15, dtype=np.int32)[None]
    flat_k, flat_v = kc.view(-1, 64), vc.view(-1, 64)
    for t in range(6):
        flat_k[32 * t:32 * t + 32, 0] = step * t / 1.4426950408889634
        flat_v[32 * t:32 * t + 32, 1] = 0.5
        flat_v[32 * t + 3:32 * t + 6, 0] = large
        flat_v[32 * t + 7, 2:4] = -large
    q = torch.zeros((rows, 2, 64), device=dev)
    q[:, :, 0] = 8.0
    want, tol = attend64(q, kc, vc, tables, [kv], [0, rows])
    assert torch.isfinite(want).all() and want.abs().max() > large / 50
    check(_call(dev, q, kc, vc, tables, [kv], [0, rows]), want, tol)
    check(_call(dev, q[:1], kc, vc, tables, [kv - rows + 1], [0, 1]), want[:1], tol[:1])


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("what", ["scores", "infinite scores", "nan", "values", "infinite values"])
def test_keys_of_later_rows_change_no_bits(agpu, dev, type_, what):
    """Rows of a tile share the keys that are fetched for them; what only later ones see leaves the bits of the earlier ones as they are."""
    import torch
    lens, new, heads, page = [500, 130], [200, 130], 2, 16
    rng, g = np.random.default_rng(3), torch.Generator(device=dev).manual_seed(11)
    kc, vc = _cache(torch, g, dev, 42, heads, page, type_)
    tables, start = _tables(rng, lens, page, 42), np.concatenate([[0], np.cumsum(new)]).tolist()
    q = torch.randn((start[-1], heads, 64), generator=g, device=dev).abs()
    want = _call(dev, q, kc, vc, tables, lens, start)
    for b, from_ in ((0, 340), (0, 417), (1, 77)):
        k, v = kc.clone(), vc.clone()
        for p in range(from_, lens[b]):
            at = (tables[b, p // page], slice(None), p % page)
            if what == "values":
                v[at] = 60000.0 if type_ == "float16" else 1e36
            elif what == "infinite values":
                v[at] = float("inf")
            else:
                k[at] = {"scores": 4.0, "infinite scores": float("inf"), "nan": float("nan")}[what]
        got = _call(dev, q, k, v, tables, lens, start)
        first = start[b] + from_ - (lens[b] - new[b])
        others = torch.ones(start[-1], dtype=torch.bool)
        others[first:start[b + 1]] = False
        assert torch.equal(got[others], want[others])
        assert not (got[first:start[b + 1]] == want[first:start[b + 1]]).all()
        if what in ("scores", "values"):
            check(got, *attend64(q, k, v, tables, lens, start))


@pytest.mark.parametrize("type_", ["float32", "float16"])
@pytest.mark.parametrize("batch", [3, 300])
@pytest.mark.parametrize("kind", ["tokens", "chunks"])
def test_rows_before_the_first_request(agpu, dev, type_, batch, kind):
    """query_start may begin behind row 0: the rows before it are nobody's and stay as they were, like those behind the last request's."""
    import torch
    rng, g = np.random.default_rng(batch), torch.Generator(device=dev).manual_seed(7)
    new = np.ones(batch, int) if kind == "tokens" else np.where(np.arange(batch) % 7 == 2, 40, 1)
    if kind == "tokens":
        new[batch // 2:] = 0  # room for rows of nobody in a call of as many rows as requests
    lens = rng.integers(40, 90, batch)
    first, behind = 1, 0 if kind == "tokens" else 2
    start = (first + np.concatenate([[0], np.cumsum(new)])).tolist()
    pages = int((-(-lens // 16)).sum())
    kc, vc = _cache(torch, g, dev, pages, 2, 16, type_)
    tables = _tables(rng, lens.tolist(), 16, pages)
    q = torch.randn((start[-1] + behind, 2, 64), generator=g, device=dev)
    assert (len(q) <= batch) == (kind == "tokens")
    out = torch.full_like(q, 7.0)
    _call(dev, q, kc, vc, tables, lens, start, out=out)
    want, tol = attend64(q, kc, vc, tables, lens.tolist(), start)
    check(out, want, tol)
    assert (out[:first] == 7.0).all() and (out[start[-1]:] == 7.0).all()


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("batch", [4, 260])
def test_fewer_rows_than_the_requests_have(agpu, dev, type_, batch):
    """A call with the first rows only: each is at the position that query_start gives it, whichever way it is worked out."""
    import torch
    rng, g = np.random.default_rng(9), torch.Generator(device=dev).manual_seed(8)
    new = np.full(batch, 1 if batch > 100 else 3)
    new[-1] = 150
    lens = new + rng.integers(0, 60, batch)
    start = np.concatenate([[0], np.cumsum(new)]).tolist()
    pages = int((-(-lens // 16)).sum())
    kc, vc = _cache(torch, g, dev, pages, 2, 16, type_)
    tables = _tables(rng, lens.tolist(), 16, pages)
    q = torch.randn((start[-1], 4, 64), generator=g, device=dev)
    want, tol = attend64(q, kc, vc, tables, lens.tolist(), start)
    for rows in (start[-1] - 20, start[-2] + 3, start[-2], 2):
        got = _call(dev, q[:rows], kc, vc, tables, lens, start)
        check(got, want[:rows], tol[:rows])


@pytest.mark.parametrize("type_", TYPES)
def test_magnitudes_far_apart(agpu, dev, type_):
    """Elements of q and K over 2^24 with scores of ordinary size, rows of q over 2^60, and values over as much as the type has."""
    import torch
    lens, new, heads = [300, 40, 1, 90], [140, 40, 1, 3], 3
    rng, g = np.random.default_rng(4), torch.Generator(device=dev).manual_seed(5)
    kc, vc = _cache(torch, g, dev, 40, heads, 16, type_)
    tables, start = _tables(rng, lens, 16, 40), np.concatenate([[0], np.cumsum(new)]).tolist()
    q = torch.randn((start[-1], heads, 64), generator=g, device=dev)
    by = 2.0 ** torch.randint(-12, 13, (64,), generator=g, device=dev)
    far = 2.0 ** torch.randint(-14, 13, vc.shape, generator=g, device=dev) if type_ == "float16" else 10.0 ** torch.randint(-30, 31, vc.shape, generator=g, device=dev).float()
    args = kc, (vc.float() * far).to(vc.dtype), tables, lens, start
    check(_call(dev, q, *args), *attend64(q, *args))
    wide = (kc.float() / by).to(kc.dtype), *args[1:]
    check(_call(dev, q * by, *wide), *attend64(q * by, *wide))
    tiny = q * 2.0 ** torch.randint(-60, 1, (start[-1], heads, 1), generator=g, device=dev)
    check(_call(dev, tiny, *args), *attend64(tiny, *args))


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("octaves", [10, 24, 32, 40])
def test_many_small_weights_beside_a_large_one(agpu, dev, type_, octaves):
    """A key with nearly all of the weight and a small value, and a thousand keys of weights 2^-octaves with large ones."""
    import torch
    kv, rows, page = 1000, 60, 16
    g = torch.Generator(device=dev).manual_seed(6)
    kc = torch.zeros((63, 1, page, 64), dtype=getattr(torch, type_), device=dev)
    vc = (torch.rand((63, 1, page, 64), generator=g, device=dev) * 3e4 + 3e4).to(kc.dtype)
    kc.view(-1, 64)[500, 0] = octaves / 1.4426950408889634
    vc.view(-1, 64)[500] *= 2.0**-20
    tables = np.arange(63, dtype=np.int32)[None]
    q = torch.zeros((rows, 1, 64), device=dev)
    q[:, :, 0] = 8.0
    want, tol = attend64(q, kc, vc, tables, [kv], [0, rows])
    if type_ == "float16":
        # weights times 512 are two f16 numbers there, which no smaller steps than 2^-24 have: half a step is 2^-34 of a weight of one, and the sum of weights at least one
        tol = tol + 2.0**-34 * vc.double().abs().sum((0, 1, 2)).cpu()
    check(_call(dev, q, kc, vc, tables, [kv], [0, rows]), want, tol)
    check(_call(dev, q[:1], kc, vc, tables, [kv - rows + 1], [0, 1]), want[:1], tol[:1])


def test_pieces_at_their_worst(agpu, dev):
    """fp32 caches go to the matrix cores in three pieces, cut off one after the other, and of nine products the three smallest are left out: 2^-7 times 2^-15, twice, and
    2^-15 squared, 2^-21 of a product of numbers whose last 16 bits are ones.  Scores and outputs of such numbers."""
    import torch
    kv, rows, page = 96, 96, 16
    worst = float(np.uint32(0x3f80ffff).view(np.float32))
    kc, vc = (torch.zeros((6, 1, page, 64), device=dev) for _ in range(2))
    kc.view(-1, 64)[::3] = worst
    kc.view(-1, 64)[1::3] = -worst / 2
    vc.view(-1, 64)[:, 0] = worst
    vc.view(-1, 64)[::2, 1] = worst
    vc.view(-1, 64)[1::2, 2] = worst * 4
    q = torch.full((rows, 1, 64), worst, device=dev)
    tables = np.arange(6, dtype=np.int32)[None]
    want, tol = attend64(q, kc, vc, tables, [kv], [0, rows])
    got = _call(dev, q, kc, vc, tables, [kv], [0, rows])
    check(got, want, tol)
    # what is left out by itself: scores of up to 8.1 octaves' 2^-21 each way, and 2^-21 of the output; and the sums' roundings as above
    s = 8.0 * worst * worst
    bound = 2 * s * (2.0**-21 + 64 * 2.0**-24) + 2.0**-21 + 2.0**-20 + 2 * (kv / 16 + 100) * 2.0**-24
    assert ((got.cpu().double() - want).abs() <= bound * want.abs().amax()).all()


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("heads,kv_heads", [(11, 1), (24, 2), (130, 1)])
def test_many_heads_in_many_requests(agpu, dev, type_, heads, kv_heads):
    """More than eight heads a K/V head in more requests than are numbered, rows of every number."""
    import torch
    rng, g = np.random.default_rng(heads), torch.Generator(device=dev).manual_seed(1)
    batch, page = 290, 16
    new = rng.choice([0, 1, 1, 1, 2, 9], batch)
    new[[7, 123]] = 40, 17
    lens = new + rng.integers(0, 40, batch)
    lens[200] = 900
    start = np.concatenate([[0], np.cumsum(new)]).tolist()
    pages = int((-(-lens // page)).sum())
    kc, vc = _cache(torch, g, dev, pages, kv_heads, page, type_)
    tables = _tables(rng, lens.tolist(), page, pages)
    q = torch.randn((start[-1], heads, 64), generator=g, device=dev)
    assert start[-1] > batch
    for window, sinks in ((0, 0), (20, 3)):
        check(_call(dev, q, kc, vc, tables, lens, start, window, sinks), *attend64(q, kc, vc, tables, lens.tolist(), start, window, sinks))
