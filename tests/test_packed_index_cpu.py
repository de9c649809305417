"""The index arithmetic of the packed operators (csrc/packed_index.h), compiled for
the host: every tile of every sequence has one work slot of its own, nothing leaves
its range whatever the offsets hold, and the key ranges are the formula's."""
import os
import random
import subprocess

import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(REPO, "vpipe-ltx-2.5_b200", "csrc")

HOST = r"""
#include "packed_index.h"
extern "C" {
int t_base(int a, int s, int t, int x) { return ltx::slot_base(a, s, t, x); }
int t_count(int r, int s, int t, int x) { return ltx::slot_count(r, s, t, x); }
int t_high(int p, int m, int c) { return ltx::key_high(p, m, c); }
int t_low(int p, int w) { return ltx::key_low(p, w); }
int t_clamp(int v, int lo, int hi) { return ltx::clamp_int(v, lo, hi); }
}
"""


@pytest.fixture(scope="module")
def idx(tmp_path_factory):
    import ctypes
    d = tmp_path_factory.mktemp("idx")
    src = d / "t.cc"
    src.write_text(HOST)
    lib = d / "t.so"
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Wextra", "-Werror", "-shared", "-fPIC", "-I",
                    CSRC, str(src), "-o", str(lib)], check=True)
    return ctypes.CDLL(str(lib))


def test_every_tile_has_a_slot_of_its_own(idx):
    rng = random.Random(1)
    for _ in range(300):
        tile = rng.choice([1, 2, 3, 25, 32, 64, 128, 256])
        lens = [rng.choice([0, 1, 2, tile - 1, tile, tile + 1, rng.randint(0, 5 * tile)])
                for _ in range(rng.randint(1, 12))]
        cu = [rng.randint(0, 9)]
        for n in lens:
            cu.append(cu[-1] + n)
        rows = cu[-1] + rng.randint(0, 9)
        for extra in (1, 2):
            used = set()
            for s, n in enumerate(lens):
                base = idx.t_base(cu[s], s, tile, extra)
                # extra 2: the run starts anywhere inside a tile
                tiles = -(-n // tile) if extra == 1 else (0 if n == 0 else 1 if n == 1
                                                          else -(-n // tile) + 1)
                for i in range(tiles):
                    assert base + i < idx.t_base(cu[s + 1], s + 1, tile, extra)
                    assert base + i not in used
                    used.add(base + i)
            assert not used or max(used) < idx.t_count(rows, len(lens), tile, extra)


def test_key_ranges(idx):
    big = 2 ** 31 - 1
    for n in range(0, 9):
        for m in range(0, 9):
            for w in (0, 1, 3, 100, big):
                for causal in (0, 1):
                    for i in range(n):
                        pos = m - n + i
                        got = range(idx.t_low(pos, w), idx.t_high(pos, m, causal))
                        want = [j for j in range(m) if (not causal or j <= pos) and
                                (not w or j > pos - w)]
                        assert list(got) == want, (n, m, w, causal, i)


def test_clamp(idx):
    for v in (-2 ** 31, -1, 0, 5, 7, 2 ** 31 - 1):
        assert 0 <= idx.t_clamp(v, 0, 7) <= 7
