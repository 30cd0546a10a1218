"""Rules at the ends of the operators over a KV cache in pages (async-gpu_amd/csrc/paged.h), compiled by themselves with overflow trapped: no GPU here."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    """A program that answers a line of numbers with a line of numbers: `tiles n_kv`."""
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
