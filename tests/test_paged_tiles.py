"""What a tile of rows sees of a cache in pages (async-gpu_amd/csrc/paged.h, tile_keys and row_keys), against what its rows see one by one: no GPU here."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BIG = 2**31 - 1


@pytest.fixture(scope="module")
def tiles(tmp_path_factory):
    """A program that answers `kv rows held window sinks first last` with what rows first .. last (of `rows`, the last of kv positions) see of the tile's keys: the first
    of them that differs from paged::visible, or -1; then how many keys the tile has, and how many of them no row sees.  Signed overflow ends it."""
    d = tmp_path_factory.mktemp("tiles")
    src, exe = d / "tiles.cpp", d / "tiles"
    src.write_text('''
#include <cstdio>
#include <vector>
#include "paged.h"
int main() {
    int kv, rows, held, window, sinks, first, last;
    while (std::scanf("%d %d %d %d %d %d %d", &kv, &rows, &held, &window, &sinks, &first, &last) == 7) {
        const paged::TileKeys t = paged::tile_keys(kv - rows + first, kv - rows + last, held, window, sinks);
        std::vector<char> used(t.count > 0 ? t.count : 0, 0);
        int wrong = -1;
        for (int r = last; r >= first; --r) {
            const int pos = kv - rows + r;
            const paged::RowKeys row = paged::row_keys(t, pos, window, sinks);
            const paged::Visible vis = paged::visible(pos, kv, held, window, sinks);
            int n = 0;
            for (int v = 0; v < t.count; ++v)
                if (row.sees(v)) {
                    used[v] = 1;
                    if (n >= vis.count || vis.key(n) != t.key(v)) wrong = r;
                    ++n;
                }
            if (n != vis.count) wrong = r;
        }
        int idle = 0;
        for (char u : used) idle += !u;
        std::printf("%d %d %d\\n", wrong, t.count, idle);
    }
}
''')
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-fsanitize=signed-integer-overflow", "-fno-sanitize-recover=all", "-I", os.path.join(ROOT, "async-gpu_amd", "csrc"),
                    str(src), "-o", str(exe)], check=True)

    def ask(lines):
        r = subprocess.run([str(exe)], input="\n".join(" ".join(map(str, x)) for x in lines) + "\n", capture_output=True, text=True, timeout=60, check=True)
        got = [[int(x) for x in line.split()] for line in r.stdout.splitlines()]
        assert len(got) == len(lines)
        return got

    return ask


def test_a_tile_sees_what_its_rows_see(tiles):
    """With windows and sinks from none to the largest numbers, rows before position 0, and tables that end before the request does."""
    asked = [(kv, rows, held, window, sinks, first, last)
             for kv, rows in ((0, 3), (5, 12), (1, 1), (12, 12), (40, 9), (200, 130), (90, 200)) for held in (0, 7, 64, 4096)
             for window in (0, 1, 2, 17, 64, 500, BIG - 1, BIG) for sinks in (0, 1, 4, 30, 300, BIG)
             for first, last in ((0, rows - 1), (0, 0), (rows - 1, rows - 1), (rows // 3, min(rows // 3 + 127, rows - 1)))]
    for a, (wrong, count, idle) in zip(asked, tiles(asked)):
        assert wrong == -1, a
        kv, rows, held, window, sinks, first, last = a
        assert idle == 0 and count <= max(min(kv - rows + last + 1, held), 0), a


def test_a_tile_far_from_the_first_position(tiles):
    kv = 2**30
    (got,) = tiles([(kv, 64, kv, 3, 2, 0, 63)])
    assert got == [-1, 2 + 3 + 63, 0]
