"""The rules of the cache in pages (async-gpu_amd/csrc/paged.h) compiled by themselves, and what the operators over torch tensors refuse before they reach
a GPU: no GPU here."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    """A program that answers a line of numbers with a line of numbers: `div size n`, `vis pos kv held window sinks` (keys that are seen),
    `most items longest least item_bytes space tickets`, `run count run most`, `for work fill least longest most`, and the refusals."""
    d = tmp_path_factory.mktemp("paged")
    src, exe = d / "rules.cpp", d / "rules"
    src.write_text('''
#include <cstdio>
#include <cstring>
#include "paged.h"
int main() {
    char what[16];
    long long a[9];
    while (std::scanf("%15s", what) == 1) {
        int n = 0;
        char c;
        while (std::scanf("%c", &c) == 1 && c != '\\n')
            if (std::scanf("%lld", &a[n]) == 1) ++n;
        if (!std::strcmp(what, "div")) {
            const paged::PageDiv div = paged::PageDiv::of((int)a[0]);
            std::printf("%d\\n", div.page((int)a[1]));
        } else if (!std::strcmp(what, "vis")) {
            const paged::Visible v = paged::visible((int)a[0], (int)a[1], (int)a[2], (int)a[3], (int)a[4]);
            for (int i = 0; i < v.count; ++i) std::printf("%d ", v.key(i));
            std::printf("\\n");
        } else if (!std::strcmp(what, "run")) {
            const paged::RunsOf r = paged::runs_of((int)a[0], (int)a[1], (int)a[2]);
            std::printf("%d %d\\n", r.runs, r.keys);
        } else if (!std::strcmp(what, "for")) {
            std::printf("%d\\n", paged::run_for((float)a[0], (float)a[1], (int)a[2], (int)a[3], (int)a[4]));
        } else if (!std::strcmp(what, "most")) {
            std::printf("%d\\n", paged::most_runs(a[0], a[1], a[2], (size_t)a[3], (size_t)a[4], a[5]));
        } else if (!std::strcmp(what, "cache")) {
            std::printf("%d\\n", paged::refuse_cache(a[0], a[1], a[2], a[3], (int)a[4], (int)a[5], (int)a[6], (int)a[7], (int)a[8]).code);
        } else if (!std::strcmp(what, "attention")) {
            std::printf("%d\\n", paged::refuse_attention((int)a[0], (int)a[1], (int)a[2], (int)a[3], (int)a[4], (int)a[5], (int)a[6], (int)a[7], a[8] != 0).code);
        } else if (!std::strcmp(what, "plan")) {
            std::printf("%d\\n", paged::refuse_plan((int)a[0], (int)a[1], (int)a[2], (int)a[3], (int)a[4]).code);
        } else if (!std::strcmp(what, "append")) {
            std::printf("%d\\n", paged::refuse_append((int)a[0], (int)a[1]).code);
        }
    }
    return 0;
}
''')
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-I", os.path.join(ROOT, "async-gpu_amd", "csrc"), str(src), "-o", str(exe)], check=True)

    def ask(lines):
        r = subprocess.run([str(exe)], input="\n".join(lines) + "\n", capture_output=True, text=True, timeout=60, check=True)
        got = [[int(x) for x in line.split()] for line in r.stdout.splitlines()]
        assert len(got) == len(lines)
        return got

    return ask


def test_pages_of_positions(rules):
    """Every page size up to 300 and some large ones, at quotients' borders up to the largest position."""
    sizes = list(range(1, 301)) + [511, 512, 513, 4095, 4097, 65535, 65537, 999983, (1 << 20) - 1, 1 << 20]
    asked = [(p, n) for p in sizes for q in (0, 1, 2, 1000, (2**31 - 1) // p - 1, (2**31 - 1) // p) for n in (q * p - 1, q * p, q * p + p - 1) if 0 <= n < 2**31]
    got = rules([f"div {p} {n}" for p, n in asked])
    assert all(g == [n // p] for g, (p, n) in zip(got, asked))


def test_what_a_query_sees(rules):
    asked = [(pos, kv, held, window, sinks) for pos in (-2, -1, 0, 1, 5, 9, 12) for kv in (0, 1, 6, 10, 13) for held in (0, 4, 8, 16) for window in (0, 1, 3, 6, 20)
             for sinks in (0, 1, 4, 30)]
    got = rules(["vis " + " ".join(map(str, a)) for a in asked])
    for g, (pos, kv, held, window, sinks) in zip(got, asked):
        want = [j for j in range(max(0, min(kv, held))) if j <= pos and (window == 0 or pos - j < window or j < sinks)]
        assert g == want, (pos, kv, held, window, sinks)
    far = rules([f"vis {2**30 - 1} {2**30} {2**30} 3 2"])[0]
    assert far == [0, 1, 2**30 - 3, 2**30 - 2, 2**30 - 1]


def test_runs_cover_all_keys(rules):
    """However a call is cut, its runs hold every key that a row sees, and more keys never make fewer runs: a request's runs are counted with the most that a
    row of it sees, and every row's own have to be among them."""
    asked = [(n, run, most) for run in (128, 160, 256, 1024, 4096) for most in (1, 2, 5, 7, 64) for n in [*range(0, 3000, 7), *range(3000, 70000, 999), 2**30 - 1, 2**30]]
    got = rules([f"run {n} {run} {most}" for n, run, most in asked])
    before = None
    for (n, run, most), (runs, keys) in zip(asked, got):
        assert 1 <= runs <= most and keys % 32 == 0 and runs * keys >= n
        if before and before[:2] == (run, most):
            assert runs >= before[2]
        before = (run, most, runs)


def test_runs_keep_to_scratch_and_tickets(rules):
    calls = [(items, longest, least, bytes_, space, tickets) for items in (1, 12, 200, 1536, 70000) for longest in (1, 31, 777, 4128, 32768, 2**30) for least in (128, 1024)
             for bytes_ in (264, 2112, 33792) for space in (1 << 18, 24 << 20) for tickets in (8191, 65534)]
    for (items, longest, least, bytes_, space, tickets), (most,) in zip(calls, rules(["most " + " ".join(map(str, c)) for c in calls])):
        assert 1 <= most <= 64 and (most == 1 or (items <= tickets and items * most * bytes_ <= space and (most - 1) * least < longest))
    asked = [(work, fill, 128, longest, most) for work in (0, 1, 1000, 10**6, 10**9, 10**15) for fill in (1, 512, 1024) for longest in (1, 129, 4000, 2**30) for most in (1, 3, 64)]
    for (work, fill, least, longest, most), (run,) in zip(asked, rules(["for " + " ".join(map(str, a)) for a in asked])):
        assert run % 32 == 0 and least <= run and run * most >= longest and run <= max(least, work / fill, longest / most + 1, 1) + 32


SHAPE, UNSUPPORTED = -1, -5


def test_refusals(rules):
    #        k_cache v_cache  k_page v_page heads pages size dh type
    fine = [4096, 8192, 1024, 1024, 1, 4, 16, 64, 0]

    def cache(**other):
        names = ("k", "v", "kp", "vp", "heads", "pages", "size", "dh", "type")
        return "cache " + " ".join(str(other.get(n, x)) for n, x in zip(names, fine))

    asked = {cache(): 0, cache(dh=128): SHAPE, cache(type=3): UNSUPPORTED, cache(type=-1): UNSUPPORTED, cache(heads=0): SHAPE, cache(pages=0): SHAPE, cache(size=0): SHAPE,
             cache(size=-4): SHAPE, cache(kp=1020): SHAPE, cache(vp=0): SHAPE, cache(kp=1025): UNSUPPORTED, cache(kp=1026, type=1): UNSUPPORTED, cache(k=4104): UNSUPPORTED,
             cache(v=8196): UNSUPPORTED, cache(pages=1, kp=0, vp=7): 0, cache(size=2**20 + 1, kp=2**40, vp=2**40): UNSUPPORTED,
             cache(pages=2**27, kp=1024, vp=1024): UNSUPPORTED, cache(heads=2**25, kp=2**40, vp=2**40): UNSUPPORTED,
             "attention 5 2 12 4 9 16 0 0 1": 0, "attention 5 2 12 5 9 16 0 0 1": SHAPE, "attention 5 2 0 5 9 16 0 0 1": SHAPE, "attention -1 2 12 4 9 16 0 0 1": SHAPE,
             "attention 5 2 12 4 9 16 -1 0 1": SHAPE, "attention 5 2 12 4 9 16 0 -1 1": SHAPE, "attention 5 2 12 4 -9 16 0 0 1": SHAPE, "attention 5 2 12 4 9 16 0 0 0": SHAPE,
             "attention 2 2 12 4 9 16 0 0 0": 0, "attention 700000 2 12 4 9 16 0 0 1": UNSUPPORTED, "attention 5 2 12 4 65537 16384 0 0 1": UNSUPPORTED, "attention 5 2 12 4 65536 16384 0 0 1": 0,
             "plan 4 8 100 16 50": 0, "plan 0 0 0 1 0": 0, "plan -1 8 100 16 50": SHAPE, "plan 4 8 100 0 50": SHAPE, "plan 4 8 -1 16 50": SHAPE, "plan 4 8 100 16 -1": SHAPE,
             "plan 4097 8 100 16 50": UNSUPPORTED, "plan 4 8 100 1048577 50": UNSUPPORTED, "plan 4 1025 100 1048576 50": UNSUPPORTED, "plan 4 1024 100 1048576 50": 0,
             "append 10 12": 0, "append -1 12": SHAPE, "append 2796203 25": UNSUPPORTED}
    got = rules(list(asked))
    for line, g in zip(asked, got):
        assert g == [asked[line]], line


def test_operators_refuse_what_does_not_fit(agpu):
    """Sizes, types and layouts are looked at before the device is."""
    import torch
    from async_gpu_amd import ops
    E = agpu.AgpuError
    i32, f32 = torch.int32, torch.float32
    k, v = torch.zeros(4, 3, 16, 64), torch.zeros(4, 3, 16, 64)
    q, tables, lens, start = torch.zeros(5, 6, 64), torch.zeros(2, 4, dtype=i32), torch.zeros(2, dtype=i32), torch.zeros(3, dtype=i32)

    def refuses(f, *args, **kw):
        with pytest.raises(E) as e:
            f(*args, **kw)
        assert e.value.code == SHAPE

    A = ops.paged_attention
    refuses(A, q, k, v[:, :, :8], tables, lens, start)
    refuses(A, q, k, v.half(), tables, lens, start)
    refuses(A, q, k.double(), v.double(), tables, lens, start)
    refuses(A, q[0], k, v, tables, lens, start)
    refuses(A, q[:, :, :32], k, v, tables, lens, start)
    refuses(A, q.half(), k, v, tables, lens, start)
    refuses(A, q.transpose(1, 2).contiguous().transpose(1, 2), k, v, tables, lens, start)
    refuses(A, q, k.transpose(1, 2), v.transpose(1, 2), tables, lens, start)
    refuses(A, q, k, v, tables.long(), lens, start)
    refuses(A, q, k, v, tables.t(), lens, start)
    refuses(A, q, k, v, tables, lens[:1], start)
    refuses(A, q, k, v, tables, lens, start[:2])
    refuses(A, q, k, v, tables, lens)  # without query_start: five rows for two requests
    refuses(A, q, k, v, tables, lens, start, out=torch.zeros(5, 6, 32))
    refuses(A, q, k, v, tables, lens, start, out=q)
    refuses(A, q, k, v, tables, lens, start, out=torch.zeros(6, 5, 64).transpose(0, 1))
    K = ops.paged_kv_append
    rows, slots = torch.zeros(5, 3, 64), torch.zeros(5, dtype=i32)
    refuses(K, rows[:4], rows, k, v, slots)
    refuses(K, rows, rows.half(), k, v, slots)
    refuses(K, rows[:, :2], rows, k, v, slots)
    refuses(K, rows, rows, k, v, slots.long())
    refuses(K, rows, rows, k[0], v[0], slots)
    P = ops.paged_plan
    stack, n_free = torch.zeros(9, dtype=i32), torch.zeros(1, dtype=i32)
    refuses(P, lens, lens[:1], tables, stack, n_free, 16, 8)
    refuses(P, lens, lens, tables.float(), stack, n_free, 16, 8)
    refuses(P, lens, lens, tables, stack[::2], n_free, 16, 8)
    refuses(P, lens, lens, tables, stack, stack, 16, 8)
    refuses(P, lens, lens, tables, stack, n_free, 16, -1)
    S = ops.sample
    x, u = torch.zeros(5, 100), torch.zeros(5)
    refuses(S, x.half(), u)
    refuses(S, x, u.double())
    refuses(S, x, u[:4])
    refuses(S, x[:, :0], u)
    refuses(S, x[:, ::2], u)
    refuses(S, x, u, temperature=torch.ones(4))
    refuses(S, x, u, top_k=torch.ones(5))
    refuses(S, x, u, top_k=torch.ones(5, dtype=torch.int64))
    refuses(S, x, u, top_p=torch.ones(10)[::2])
    refuses(S, x, u, min_p=torch.ones(5, 1))
    for call in (lambda: A(q, k, v, tables, lens, start), lambda: K(rows, rows, k, v, slots), lambda: P(lens, lens, tables, stack, n_free, 16, 8), lambda: S(x, u)):
        with pytest.raises(AssertionError):  # nothing of it is on a GPU
            call()
    with pytest.raises(OverflowError):
        S(x, u, top_k=1 << 40)
    with pytest.raises(TypeError):
        S(x, u, temperature="warm")
