"""Rules at the ends of the operators over a KV cache in pages (async-gpu_amd/csrc/paged.h), compiled by themselves with overflow trapped, and which memory their arguments may have in
common: no GPU here."""
import os
import random
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    """A program that answers a line of numbers with a line of numbers: `tiles n_kv`, and `both holes moves times` (holes and movers of that many parts, added up), `share` with
    the address, number, stride and bytes of two times some pieces of memory, and `rows tokens heads row head` (the pieces that rows of q are in, from address 4096 on)."""
    d = tmp_path_factory.mktemp("paged_limits")
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
        if (!std::strcmp(what, "tiles")) std::printf("%d\\n", paged::weight_tiles((int)a[0]));
        if (!std::strcmp(what, "share")) std::printf("%d\\n", paged::share({(uintptr_t)a[0], a[1], a[2], a[3]}, {(uintptr_t)a[4], a[5], a[6], a[7]}));
        if (!std::strcmp(what, "rows")) {
            const paged::Pieces p = paged::Pieces::rows((const float *)4096, a[0], a[1], a[2], a[3]);
            std::printf("%lld %lld %lld %lld\\n", (long long)p.at, (long long)p.n, (long long)p.stride, (long long)p.bytes);
        }
        if (!std::strcmp(what, "both")) {
            paged::HolesMoves all = {0};
            for (long long i = 0; i < a[2]; ++i) all.both += paged::HolesMoves::of((int)a[0], (int)a[1]).both;
            std::printf("%d %d\\n", all.holes(), all.moves());
        }
    }
    return 0;
}
''')
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-fsanitize=signed-integer-overflow", "-fno-sanitize-recover=all", "-I", os.path.join(ROOT, "async-gpu_amd", "csrc"),
                    str(src), "-o", str(exe)], check=True)

    def ask(lines):
        r = subprocess.run([str(exe)], input="\n".join(lines) + "\n", capture_output=True, text=True, timeout=60, check=True)
        got = [[int(x) for x in line.split()] for line in r.stdout.splitlines()]
        assert len(got) == len(lines)
        return got

    return ask


def test_numbers_of_tiles_fit(rules):
    """256 requests' numbers stay below 2^31 whatever the heads, and there are as many of them at a time as that allows within a factor of two."""
    heads = (1, 3, 32, 33, 4096, 2**22 - 1, 2**22, 2**23 - 1)
    for n_kv, (most,) in zip(heads, rules([f"tiles {n}" for n in heads])):
        assert most >= 1 and 256 * most * n_kv < 2**31 and (most == 1 or most * n_kv > 2**21)


def test_holes_and_movers_add_up(rules):
    """512 parts of 64 positions, of which all are holes, all move, or any mixture."""
    asked = [(64, 0), (0, 64), (63, 1), (1, 63), (32, 32), (0, 0), (7, 50)]
    assert rules([f"both {h} {m} 512" for h, m in asked]) == [[512 * h, 512 * m] for h, m in asked]


def test_pieces_of_memory_that_meet(rules):
    """Against all bytes one by one: of one stride, of two, of none, one within the gaps of the other and not."""
    rng = random.Random(1)
    asked = []
    for _ in range(6000):
        strides = [rng.choice([0, 1, 5, 8, 12, 16, 24, 30])] * 2 if rng.random() < 0.4 else [rng.choice([0, 1, 4, 5, 6, 8, 10, 12, 16, 24, 30]) for _ in range(2)]
        asked.append([x for s in strides for x in (100 + rng.randrange(40), rng.choice([0, 1, 1, 2, 3, 7]), s, rng.choice([0, 1, 2, 3, 4, 7, 12]))])
    met = 0
    for a, (got,) in zip(asked, rules(["share " + " ".join(map(str, a)) for a in asked])):
        one, two = ({at + i * stride + b for i in range(n) for b in range(size)} for at, n, stride, size in (a[:4], a[4:]))
        assert got == bool(one & two), a
        met += got
    assert 1000 < met < 5000
    # caches of 2^31 pages, in one arena and in two
    page, n = 1 << 20, 2**31 - 1
    far = [([0, n, page, 4096], [4096, n, page, 4096], 0), ([0, n, page, 4097], [4096, n, page, 4096], 1), ([0, n, page, page], [n * page, n, page, page], 0), ([0, n, page, page], [n * page - 1, 1, 0, 1], 1),
           ([0, n, page, 4096], [8192, n // 2, 2 * page, 4096], 0), ([0, n, page, 4096], [(n - 1) * page - 2 * page, 5, 3 * page // 2, 4096], 1)]
    assert rules(["share " + " ".join(map(str, a + b)) for a, b, _ in far]) == [[x] for _, _, x in far]


def test_rows_in_pieces(rules):
    """Rows of 64 floats at any two strides are within their pieces, and nothing else is where the strides leave no gaps that are not the pieces'."""
    asked = [(t, h, row, head) for t in (1, 3) for h in (1, 4) for row, head in ((h * 64, 64), (900, 64), (64, t * 64), (64, 1000), (700, 70), (0, 64), (64, 0), (-300, 64), (64, -500))]
    for (t, h, row, head), (at, n, stride, size) in zip(asked, rules([f"rows {t} {h} {row} {head}" for t, h, row, head in asked])):
        rows = {4096 + 4 * (i * row + j * head) + b for i in range(t) for j in range(h) for b in range(256)}
        pieces = {at + i * stride + b for i in range(n) for b in range(size)}
        assert rows <= pieces and min(rows) == min(pieces) and max(rows) == max(pieces)
        if head == 64 and row > 0 or row == 64 and head > 0:
            assert rows == pieces
    assert rules(["rows 0 4 256 64", "rows 4 0 0 64"]) == [[4096, 1, 0, 0]] * 2


def test_arguments_of_one_arena(agpu):
    """Caches, weights, rows and results may be parts of one allocation, page by page too; what overlaps is refused."""
    import torch
    from async_gpu_amd import ops
    i32 = torch.int32
    tables, lens, start = torch.zeros(2, 4, dtype=i32), torch.zeros(2, dtype=i32), torch.zeros(3, dtype=i32)
    H, page, n = 3, 16, 4
    each = H * page * 64
    arena = torch.zeros(n * (2 * each + H * page) + 2 * 5 * 6 * 64)
    by_page = arena[:n * (2 * each + H * page)].view(n, -1)
    k, v, w = by_page[:, :each].view(n, H, page, 64), by_page[:, each:2 * each].view(n, H, page, 64), by_page[:, 2 * each:].view(n, H, page)
    q, o = arena[-2 * 5 * 6 * 64:].view(2, 5, 6, 64)
    fine = [lambda: ops.paged_attention(q, k, v, tables, lens, start, out=o), lambda: ops.paged_attention_weights(q, k, v, w, tables, lens, start, out=o), lambda: ops.paged_evict(k, v, w, tables, lens, 10, 8),
            lambda: ops.paged_attention_shared(q, k, v, tables, lens, lens, tables, lens, start, out=o), lambda: ops.paged_evict(k, k, w, tables, lens, 10, 8)]
    for call in fine:
        with pytest.raises(AssertionError):  # all of it fits, but is not on a GPU
            call()
    late = arena.as_strided((n, H, page), (by_page.stride(0), page, 1), 2 * each - page)  # begins in V
    shifted = arena.as_strided((n, H, page, 64), k.stride(), 64)
    whole = by_page.flatten()
    bad = [lambda: ops.paged_attention_weights(q, k, v, late, tables, lens, start), lambda: ops.paged_evict(k, v, late, tables, lens, 10, 8), lambda: ops.paged_evict(k, shifted, w, tables, lens, 10, 8),
           lambda: ops.paged_attention_weights(q, k, v, w, tables, lens, start, out=whole[each - 64:each - 64 + 5 * 6 * 64].view(5, 6, 64)),
           lambda: ops.paged_attention_weights(q, k, v, o.flatten()[:n * H * page].view(n, H, page), tables, lens, start, out=o),
           lambda: ops.paged_attention_weights(q, k, v, q.flatten()[-n * H * page:].view(n, H, page), tables, lens, start),
           lambda: ops.paged_attention(q, k, v, tables, lens, start, out=whole[2 * each - 64:2 * each - 64 + 5 * 6 * 64].view(5, 6, 64))]
    for call in bad:
        with pytest.raises(agpu.AgpuError) as e:
            call()
        assert e.value.code == -1
