"""Rules of shared prefixes and of caches with a budget (async-gpu_amd/csrc/paged.h) compiled by themselves, and what the operators over torch tensors refuse before they
reach a GPU: no GPU here."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SHAPE, UNSUPPORTED = -1, -5
BIG = 2**31 - 1


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    """A program that answers a line of numbers with a line of numbers: `runs batch rows held apart scratch` and `room rows places group scratch` (how scratch is shared out), and the refusals."""
    d = tmp_path_factory.mktemp("paged_more")
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
        if (!std::strcmp(what, "runs")) {
            const paged::PrefixRuns r = paged::prefix_runs(a[0], a[1], a[2], a[3] != 0, (size_t)a[4]);
            std::printf("%d %zu %zu %zu\\n", r.most, r.ml, r.rest, r.bytes);
        } else if (!std::strcmp(what, "room")) {
            const paged::WeightsRoom r = paged::weights_room(a[0], a[1], (int)a[2], (size_t)a[3]);
            std::printf("%zu %zu\\n", r.scores, r.bytes);
        } else if (!std::strcmp(what, "shared")) {
            std::printf("%d\\n", paged::refuse_shared((int)a[0], (int)a[1], (int)a[2], (int)a[3]).code);
        } else if (!std::strcmp(what, "weights")) {
            std::printf("%d\\n", paged::refuse_weights((uintptr_t)a[0], a[1], (int)a[2], (int)a[3], (int)a[4]).code);
        } else if (!std::strcmp(what, "budget")) {
            std::printf("%d\\n", paged::refuse_budget((int)a[0], (int)a[1], (int)a[2], (int)a[3], (int)a[4], (int)a[5], (int)a[6]).code);
        } else if (!std::strcmp(what, "evict")) {
            std::printf("%d\\n", paged::refuse_evict((int)a[0], (int)a[1], (int)a[2], (int)a[3]).code);
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


def test_runs_of_a_prefix_keep_to_scratch(rules):
    """Whatever is asked for, (m, l) and o of all runs lie one after the other within the scratch, and leave room for partial results; one run has to be possible for 2^23 rows."""
    asked = [(batch, rows, held, apart, scratch) for apart in (0, 1) for batch in (1, 300, 5000) for rows in (1, 12, 1600, 14400, 131072, 1 << 20, (1 << 23) - 1) for held in (1, 128, 129, 5000, 2**30) for scratch in (1 << 20, 10 << 20, 96 << 20, 1 << 30)]
    for (batch, rows, held, apart, scratch), (most, ml, rest, size) in zip(asked, rules(["runs " + " ".join(map(str, a)) for a in asked])):
        if most == 0:
            assert 4 * batch + (264 if apart else 8) * rows + 512 > scratch // 4 * 3
            continue
        assert 4 * batch <= ml and ml % 256 == 0
        assert 1 <= most <= 64 and (most - 1) * 128 < held
        assert ml + 8 * rows * most <= rest and rest + 256 * rows * (most - 1 + apart) <= size <= scratch - (scratch // 4 - 256) and rest % 256 == 0 and size % 256 == 0
        assert most == 1 or size <= scratch // 2 + 512 + 256 * rows * apart
    assert rules([f"runs 4096 {(1 << 23) - 1} 1000 0 {96 << 20}"])[0][0] == 1


def test_scores_keep_to_scratch(rules):
    asked = [(rows, places, group, scratch) for rows in (1, 1600, 131072, 1 << 20, (1 << 23) - 1) for places in (16, 10**6, 10**8, 2**31 * 64) for group in (1, 8, 9) for scratch in (1 << 20, 96 << 20, 8 << 30)]
    for (rows, places, group, scratch), (scores, size) in zip(asked, rules(["room " + " ".join(map(str, a)) for a in asked])):
        if size == 0:
            assert 8 * rows + 256 > scratch // 4 * 3
            continue
        assert 8 * rows <= size <= scratch // 4 * 3 + 256 and size % 256 == 0
        if scores:
            assert group <= 8 and 8 * rows <= scores and scores + 4 * places <= size <= scratch // 2 + 256 and scores % 256 == 0
        else:
            assert group > 8 or 8 * rows + 256 + 4 * places > scratch // 2


def test_refusals(rules):
    asked = {"shared 1 8 4 16": 0, "shared 0 0 0 16": 0, "shared -1 8 4 16": SHAPE, "shared 1 -8 4 16": SHAPE, "shared 257 8 4 16": UNSUPPORTED, "shared 256 8 4 16": 0,
             "shared 1 32768 32768 16384": 0, "shared 1 32769 32768 16384": UNSUPPORTED, "shared 1 67108865 0 16": UNSUPPORTED,
             "weights 4096 48 3 10 16": 0, "weights 4096 47 3 10 16": SHAPE, "weights 4096 0 3 1 16": 0, "weights 4098 48 3 10 16": UNSUPPORTED,
             "budget 2 8 16 100 90 10 4": 0, "budget 0 0 1 0 0 0 0": 0, "budget 2 8 16 100 100 96 4": 0, "budget 2 8 16 100 101 10 4": SHAPE, "budget 2 8 16 100 90 87 4": SHAPE,
             f"budget 2 8 16 {BIG} {BIG} {BIG} {BIG}": SHAPE, "budget 2 8 16 -1 0 0 0": SHAPE, "budget 2 8 16 5 -1 0 0": SHAPE, "budget 2 8 16 5 4 -1 0": SHAPE, "budget 2 8 16 5 4 0 -1": SHAPE,
             "budget -1 8 16 5 4 0 0": SHAPE, "budget 2 -8 16 5 4 0 0": SHAPE, "budget 2 8 0 5 4 0 0": SHAPE, "budget 2 8 1048577 5 4 0 0": UNSUPPORTED, "budget 2 1025 1048576 5 4 0 0": UNSUPPORTED,
             "evict 2 25 65536 16": 0, "evict 2 25 65537 16": UNSUPPORTED, "evict 400000 25 8 16": UNSUPPORTED}
    for line, got in zip(asked, rules(list(asked))):
        assert got == [asked[line]], line


def test_operators_refuse_what_does_not_fit(agpu):
    """Sizes, types and layouts are looked at before the device is."""
    import torch
    from async_gpu_amd import ops
    i32 = torch.int32
    k, v, w = torch.zeros(4, 3, 16, 64), torch.zeros(4, 3, 16, 64), torch.zeros(4, 3, 16)
    q, tables, lens, start = torch.zeros(5, 6, 64), torch.zeros(2, 4, dtype=i32), torch.zeros(2, dtype=i32), torch.zeros(3, dtype=i32)
    pt, pl, of = torch.zeros(3, 7, dtype=i32), torch.zeros(3, dtype=i32), torch.zeros(2, dtype=i32)
    stack, n_free = torch.zeros(9, dtype=i32), torch.zeros(1, dtype=i32)

    def refuses(f, *args, **kw):
        with pytest.raises(agpu.AgpuError) as e:
            f(*args, **kw)
        assert e.value.code == SHAPE

    S = ops.paged_attention_shared
    refuses(S, q, k, v[:, :, :8], pt, pl, of, tables, lens, start)
    refuses(S, q, k.double(), v.double(), pt, pl, of, tables, lens, start)
    refuses(S, q.half(), k, v, pt, pl, of, tables, lens, start)
    refuses(S, q, k, v, pt[0], pl, of, tables, lens, start)
    refuses(S, q, k, v, pt.long(), pl, of, tables, lens, start)
    refuses(S, q, k, v, pt, pl[:2], of, tables, lens, start)
    refuses(S, q, k, v, pt, pl, of[:1], tables, lens, start)
    refuses(S, q, k, v, pt, pl, of.long(), tables, lens, start)
    refuses(S, q, k, v, pt, pl, of, tables, lens, start[:2])
    refuses(S, q, k, v, pt, pl, of, tables, lens)  # without query_start: five rows for two requests
    refuses(S, q, k, v, pt, pl, of, tables, lens, start, out=q)
    refuses(S, q, k, v, pt, pl, of, tables, lens, start, out=torch.zeros(6, 5, 64).transpose(0, 1))
    W = ops.paged_attention_weights
    refuses(W, q, k, v, w[:, :2], tables, lens, start)
    refuses(W, q, k, v, w.half(), tables, lens, start)
    refuses(W, q, k, v, w.transpose(1, 2).contiguous().transpose(1, 2), tables, lens, start)
    refuses(W, q, k, v, w.permute(1, 0, 2).contiguous().permute(1, 0, 2), tables.long(), lens, start)
    refuses(W, q, k, v, w, tables, lens, start, out=q)
    refuses(W, q, k, v, q.view(-1)[:192].view(4, 3, 16), tables, lens, start)
    o = torch.zeros(5, 6, 64)
    refuses(W, q, k, v, o.view(-1)[:192].view(4, 3, 16), tables, lens, start, out=o)
    E = ops.paged_evict
    refuses(E, k, v.half(), w, tables, lens, 10, 8)
    refuses(E, k, v, w[:3], tables, lens, 10, 8)
    refuses(E, k, v, w, tables, lens[:1], 10, 8)
    refuses(E, k.transpose(1, 2), v.transpose(1, 2), w, tables, lens, 10, 8)
    T = ops.paged_trim
    refuses(T, lens[:1], tables, stack, n_free, 16, 10, 8)
    refuses(T, lens, tables, stack[::2], n_free, 16, 10, 8)
    refuses(T, lens, tables, stack, stack, 16, 10, 8)
    refuses(T, lens, tables.float(), stack, n_free, 16, 10, 8)
    for call in (lambda: S(q, k, v, pt, pl, of, tables, lens, start), lambda: W(q, k, v, w, tables, lens, start), lambda: E(k, v, w, tables, lens, 10, 8),
                 lambda: T(lens, tables, stack, n_free, 16, 10, 8)):
        with pytest.raises(AssertionError):  # nothing of it is on a GPU
            call()
