"""Rules at the ends of the operators over a KV cache in pages (async-gpu_amd/csrc/paged.h), compiled by themselves with overflow trapped: no GPU here."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    """A program that answers a line of numbers with a line of numbers: `tiles n_kv`, and `both holes moves times` (holes and movers of that many parts, added up)."""
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
