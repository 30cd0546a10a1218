"""The draw of the next tokens (ops.sample) against its definition in 64 bits: the same token.  (Both sides decide by sums next to borders; the operator's weights are
off by 2^-43 of the largest one at most, and a draw that close to a border is a matter of one row in many millions.)"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def draw64(x, u, temperature, top_k, top_p, min_p):
    """Row by row; settings are numbers or one a row."""
    tokens = []
    at = lambda v, r: np.float64(np.float32(np.asarray(v).reshape(-1)[r if np.ndim(v) else 0]))  # noqa: E731
    for r in range(x.shape[0]):
        row = np.where(np.isnan(x[r]), -np.inf, x[r]).astype(np.float64)
        order = np.argsort(-row, kind="stable")
        s = row[order]
        if s[0] == -np.inf:
            tokens.append(-1)
            continue
        with np.errstate(invalid="ignore"):
            w = np.exp(np.where(s == s[0], 0.0, s - s[0]) / max(at(temperature, r), 1e-8))
        k = int(at(top_k, r))
        if k > 0:
            w = w[:k]
        run = np.cumsum(w)
        p, m = at(top_p, r), at(min_p, r)
        if p < 1:
            inside = run - w < p * run[-1]
            w = w[:max(1, int(inside.sum()))]
        if m > 0:
            w = w[:max(1, int((w >= m).sum()))]
        run = np.cumsum(w)
        past = np.nonzero(run > np.float64(u[r]) * run[-1])[0]
        tokens.append(int(order[past[0] if len(past) else int((w > 0).sum()) - 1]))
    return tokens


def _logits(rng, rows, n):
    x = rng.standard_normal((rows, n)).astype(np.float32) * 2.5 - 35
    likely = rng.integers(0, n, (rows, min(n, 24)))
    x[np.arange(rows)[:, None], likely] += 12 * rng.random(likely.shape).astype(np.float32)
    return x


def _draw(dev, x, u, *settings):
    import torch
    from async_gpu_amd import ops
    on = lambda v, d: torch.tensor(np.asarray(v, d), device=dev) if np.ndim(v) else v  # noqa: E731
    t, k, p, m = settings
    return ops.sample(torch.tensor(x, device=dev), torch.tensor(np.asarray(u, np.float32), device=dev), on(t, np.float32), on(k, np.int32), on(p, np.float32), on(m, np.float32)).tolist()


SETTINGS = [(1.0, 0, 1.0, 0.0), (0.8, 40, 1.0, 0.0), (1.0, 0, 0.95, 0.0), (1.3, 0, 1.0, 0.05), (0.7, 50, 0.9, 0.02), (1.0, 1, 1.0, 0.0), (0.0, 0, 1.0, 0.0), (1.0, 0, 0.0, 0.0), (1.0, 700, 0.999, 0.0),
            (5.0, 5000, 1.0, 0.0), (1.0, 0, 1.0, 1.0), (1.0, 0, 1.0, 2.0), (100.0, 0, 0.5, 0.0), (1.0, 1 << 30, 2.0, -1.0), (2.0, 0, 0.5, 0.5)]


@pytest.mark.parametrize("n,rows", [(1, 3), (2, 5), (63, 4), (4096, 3), (4099, 3), (50257, 4), (65537, 2), (300001, 1)])
@pytest.mark.parametrize("settings", SETTINGS)
def test_draw(agpu, dev, n, rows, settings):
    rng = np.random.default_rng(n + rows)
    x = _logits(rng, rows, n)
    for u in (rng.random(rows).astype(np.float32), np.zeros(rows, np.float32), np.full(rows, 1 - 2.0**-24, np.float32), rng.random(rows).astype(np.float32)):
        assert _draw(dev, x, u, *settings) == draw64(x, u, *settings)


@pytest.mark.parametrize("rows", [1, 2, 7, 64, 300])
def test_settings_of_each_row(agpu, dev, rows):
    rng = np.random.default_rng(rows)
    n = 5003
    x, u = _logits(rng, rows, n), rng.random(rows).astype(np.float32)
    t, k = rng.choice([0.0, 0.5, 1.0, 1.7, -3.0], rows), rng.choice([0, 1, 2, 40, 600, 5002, 5003, 9999, -5], rows)
    p, m = rng.choice([1.0, 0.9, 0.3, 0.0, 7.0], rows), rng.choice([0.0, 0.1, 0.9, 0.0], rows)
    p[p == 1.0] = 1.0
    assert _draw(dev, x, u, t, k, p, m) == draw64(x, u, t, k, p, m)
    assert _draw(dev, x, u, 0.9, k, 0.8, m) == draw64(x, u, 0.9, k, 0.8, m)


@pytest.mark.parametrize("case", ["all equal", "few values", "masked", "lowest", "one left", "nothing left", "nan", "infinite", "zeros", "close", "wide", "subnormal"])
@pytest.mark.parametrize("n", [700, 50257])
def test_values(agpu, dev, case, n):
    """Equals by the thousand, masks, infinities, NaN, zeros of both signs, differences of a last bit, and rows whose mask leaves nothing."""
    rng = np.random.default_rng(n)
    rows = 6
    x = _logits(rng, rows, n)
    if case == "all equal":
        x[:] = -3.5
    elif case == "few values":
        x = rng.integers(-3, 1, (rows, n)).astype(np.float32)
    elif case == "masked":
        x[rng.random((rows, n)) < 0.9] = -np.inf
    elif case == "lowest":
        x[rng.random((rows, n)) < 0.9] = np.finfo(np.float32).min
        x[0] = np.finfo(np.float32).min
    elif case == "one left":
        x[:] = -np.inf
        x[np.arange(rows), rng.integers(0, n, rows)] = -7e30
    elif case == "nothing left":
        x[:] = -np.inf
        x[1, ::2] = np.nan
        x[2] = np.nan
    elif case == "nan":
        x[rng.random((rows, n)) < 0.5] = np.nan
        x[3, :] = np.nan
        x[3, 5] = 1.0
    elif case == "infinite":
        x[:, 7] = np.inf
        x[::2, 11::100] = np.inf
    elif case == "zeros":
        x = np.minimum(x + 40, 0) * rng.integers(0, 2, (rows, n)).astype(np.float32)
    elif case == "close":
        x = np.nextafter(np.float32(-35), np.float32(-36), dtype=np.float32) + rng.integers(0, 3, (rows, n)).astype(np.float32) * np.float32(2.0**-18)
    elif case == "wide":
        x = (rng.standard_normal((rows, n)) * 1e30).astype(np.float32)
    elif case == "subnormal":
        x = (rng.standard_normal((rows, n)) * 1e-42).astype(np.float32)
    for settings in [(1.0, 0, 1.0, 0.0), (0.8, 40, 1.0, 0.0), (1.0, 600, 0.9, 0.0), (1.0, 0, 0.37, 0.0), (0.0, 0, 1.0, 0.0), (1.1, 0, 1.0, 0.3), (3e30, 0, 1.0, 0.0)]:
        u = rng.random(rows).astype(np.float32)
        assert _draw(dev, x, u, *settings) == draw64(x, u, *settings), settings


def test_numbers_outside_of_the_range(agpu, dev):
    """u of 1 and above: the last candidate; below 0: the first."""
    rng = np.random.default_rng(1)
    x = _logits(rng, 4, 1000)
    order = np.argsort(-x, axis=1, kind="stable")
    got = _draw(dev, x, [1.0, 5.0, -1.0, 0.0], 1.0, 30, 1.0, 0.0)
    assert got == [order[0, 29], order[1, 29], order[2, 0], order[3, 0]]


def test_shapes_and_the_top_k_draw(agpu, dev):
    """One row without a row dimension, several of them; the same number draws what top_k_sample draws."""
    import torch
    from async_gpu_amd import ops
    rng = np.random.default_rng(2)
    x = torch.tensor(_logits(rng, 24, 50257), device=dev)
    u = torch.tensor(rng.random(24).astype(np.float32), device=dev)
    flat = ops.sample(x, u, 0.8, 40)
    assert flat.shape == (24,) and flat.dtype == torch.int32
    assert torch.equal(ops.sample(x.view(2, 3, 4, -1), u.view(2, 3, 4), 0.8, 40), flat.view(2, 3, 4))
    one = ops.sample(x[3], u[3], 0.8, 40)
    assert one.shape == () and int(one) == int(flat[3])
    assert ops.sample(x[:0], u[:0]).shape == (0,)
    a, b = ops.SimpleRng(77), ops.SimpleRng(77)
    for r in range(24):
        t = torch.tensor([a.next_f32()], device=dev)
        assert int(ops.sample(x[r:r + 1], t, 0.8, 40)) == ops.top_k_sample(x[r], 40, 0.8, b)
    with pytest.raises(agpu.AgpuError):
        ops.sample(torch.zeros((1, (1 << 20) + 1), device=dev), u[:1])


def test_odd_addresses(agpu, dev):
    import torch
    from async_gpu_amd import ops
    rng = np.random.default_rng(3)
    x = _logits(rng, 3, 9001)
    u = rng.random(3).astype(np.float32)
    for off in (0, 1, 2, 3):
        t = torch.empty(3 * 9001 + off, device=dev)[off:].view(3, 9001)
        t.copy_(torch.tensor(x))
        assert ops.sample(t, torch.tensor(u, device=dev), 1.0, 0, 0.9).tolist() == draw64(x, u, 1.0, 0, 0.9, 0.0)


@pytest.mark.parametrize("case", ["a little later", "much later", "masked first", "nan first", "infinite later", "lowest first", "steps", "16 bits"])
@pytest.mark.parametrize("n", [9001, 70001])
def test_where_the_largest_lies(agpu, dev, case, n):
    """Largest logits far behind the row's first few thousand, by less and by more than the sums of weights have room for, and steps of many octaves."""
    rng = np.random.default_rng(n)
    rows = 5
    x = _logits(rng, rows, n)
    if case == "a little later":
        x[:, n - 700:] += 6
    elif case == "much later":
        x[:, 8000] += 300
        x[::2, n - 5:] += 301
    elif case == "masked first":
        x[:, :8500] = -np.inf
    elif case == "nan first":
        x[:, :8500] = np.nan
        x[0, 8700:] = np.nan
    elif case == "infinite later":
        x[:, 8600] = np.inf
        x[1, 8700] = np.inf
        x[2, :8192] = -np.inf
    elif case == "lowest first":
        x[:, :8500] = np.finfo(np.float32).min
    elif case == "steps":
        x = (-rng.integers(0, 60, (rows, n)) * 0.5 * np.log(2)).astype(np.float32)
    elif case == "16 bits":
        x = (x.view(np.uint32) & 0xffff0000).view(np.float32)
    for settings in SETTINGS + [(0.01, 0, 1.0, 0.0), (1.0, 300, 0.9, 0.01)]:
        for u in (rng.random(rows).astype(np.float32), np.full(rows, 1 - 2.0**-24, np.float32)):
            assert _draw(dev, x, u, *settings) == draw64(x, u, *settings), settings


@pytest.mark.parametrize("ties", [False, True])
@pytest.mark.parametrize("k", [2, 63, 64, 255, 256, 257, 511, 512, 513, 1023])
def test_top_k_at_the_ends_of_its_ways(agpu, dev, k, ties):
    rng = np.random.default_rng(k)
    for n in (k, k + 1, 1024, 5000):
        if n < k:
            continue
        x = _logits(rng, 3, n)
        if ties:
            x = np.round(x)
        u = np.array([0.0, 0.5, 1 - 2.0**-24], np.float32)
        for p, m in ((1.0, 0.0), (0.9, 0.0), (1.0, 0.01)):
            assert _draw(dev, x, u, 1.2, k, p, m) == draw64(x, u, 1.2, k, p, m), (n, p, m)


def test_draws_of_a_graph_and_of_two_streams(agpu, dev):
    import torch
    from async_gpu_amd import ops
    rng = np.random.default_rng(12)
    rows, n = 40, 30011
    settings = [(0.8, 40, 1.0, 0.0), (1.0, 0, 0.9, 0.01)]
    x, u = torch.zeros((rows, n), device=dev), torch.zeros(rows, device=dev)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for s in settings:
            ops.sample(x, u, *s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        made = [ops.sample(x, u, *s) for s in settings]
    for _ in range(4):
        x.copy_(torch.tensor(_logits(rng, rows, n)))
        u.copy_(torch.tensor(rng.random(rows).astype(np.float32)))
        torch.cuda.synchronize()
        graph.replay()
        here = [ops.sample(x, u, *s) for s in settings]
        torch.cuda.synchronize()
        want = [draw64(x.cpu().numpy(), u.cpu().numpy(), *s) for s in settings]
        assert [m.tolist() for m in made] == want and [m.tolist() for m in here] == want


@pytest.mark.parametrize("n", [5000, 50257, 60001])
@pytest.mark.parametrize("temperature", [2.0, 5.0, 20.0])
def test_borders_among_many(agpu, dev, n, temperature):
    """Borders in bins of hundreds to thousands of candidates, some of them equal, more than one list holds."""
    rng = np.random.default_rng(n)
    x = _logits(rng, 4, n)
    x[2:] = (x[2:].view(np.uint32) & 0xfff00000).view(np.float32)
    for k, p, m in ((0, 0.9, 0.0), (0, 1.0, 0.0), (n // 2, 0.8, 0.0), (n // 3, 1.0, 0.02), (0, 0.97, 0.1)):
        u = rng.random(4).astype(np.float32)
        assert _draw(dev, x, u, temperature, k, p, m) == draw64(x, u, temperature, k, p, m), (k, p, m)
