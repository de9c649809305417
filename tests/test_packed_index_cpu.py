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
int t_span_ok(int s, int n, int c) { return ltx::span_ok(s, n, c); }
int t_page_ok(int g, int n) { return ltx::page_ok(g, n); }
void t_span(int s, int n, int i, int* o) {
  const ltx::PageSpan r = ltx::page_span(s, n, i);
  o[0] = r.block; o[1] = r.a; o[2] = r.b;
}
unsigned long long t_bound(unsigned long long a, unsigned long long w, unsigned long long i)
{ return ltx::work_bound(a, w, i); }
unsigned long long t_owner(unsigned long long a, unsigned long long w, unsigned long long x)
{ return ltx::work_owner(a, w, x); }
int t_top(int n, int m, int t, int c, int w) { return ltx::top_level(ltx::tile_levels(n, m, t, c, w)); }
int t_above(int n, int m, int t, int c, int w, int l)
{ return ltx::tiles_above(ltx::tile_levels(n, m, t, c, w), l); }
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


def test_pages_of_a_run_of_tokens(idx):
    """Every token of a run lies on one of the pages that its work slots cover, and
    what leaves the table, or names no page, is told apart."""
    import ctypes
    out = (ctypes.c_int * 3)()
    rng = random.Random(2)
    for _ in range(400):
        start, n = rng.randint(0, 300), rng.choice([1, 2, 63, 64, 65, 66, rng.randint(1, 500)])
        tokens = []
        for i in range(1 if n == 1 else -(-n // 64) + 1):
            idx.t_span(start, n, i, out)
            block, a, b = out
            if b > a:
                assert a // 64 == (b - 1) // 64 == block
                tokens += range(a, b)
        assert tokens == list(range(start, start + n))
        idx.t_span(start, n, -(-n // 64) + 1, out)     # past the last
        assert out[2] <= out[1]
    big = 2 ** 31 - 1
    assert idx.t_span_ok(0, 64, 64) and idx.t_span_ok(64, 0, 64) and idx.t_span_ok(10, 54, 64)
    for start, n, cap in ((-1, 1, 64), (-2 ** 31, 1, 64), (64, 1, 64), (10, 55, 64), (65, 0, 64),
                          (big, 1, 64), (big, big, 64), (1, big, 64)):
        assert not idx.t_span_ok(start, n, cap), (start, n, cap)
    assert idx.t_page_ok(0, 3) and idx.t_page_ok(2, 3)
    for page, pages in ((-1, 3), (3, 3), (0, 0), (big, 3), (-2 ** 31, 3)):
        assert not idx.t_page_ok(page, pages)


def test_equal_runs_of_work(idx):
    """Runs cover the list in order, each of at least one item and of sizes that
    differ by one; the owner of an item is the run it lies in."""
    import ctypes
    u = ctypes.c_ulonglong
    idx.t_bound.restype = idx.t_owner.restype = u
    rng = random.Random(3)
    for _ in range(200):
        all_ = rng.choice([1, 2, 7, rng.randint(1, 5000)])
        workers = min(all_, rng.choice([1, 2, 1184, rng.randint(1, 1184)]))
        b = [idx.t_bound(u(all_), u(workers), u(i)) for i in range(workers + 1)]
        assert b[0] == 0 and b[-1] == all_
        sizes = {y - x for x, y in zip(b, b[1:])}
        assert min(sizes) >= 1 and max(sizes) - min(sizes) <= 1
        for i in range(workers):
            for x in {b[i], b[i + 1] - 1}:
                assert idx.t_owner(u(all_), u(workers), u(x)) == i
    big = 1 << 40                                       # beyond 32 bits
    assert idx.t_owner(u(big), u(1184), u(big - 1)) == 1183
    assert idx.t_bound(u(big), u(1184), u(1184)) == big


def test_tiles_come_in_order_of_their_keys(idx):
    """tiles_above is the number of tiles whose level is higher, all of them at -1, none
    at the top; a causal sequence's are its last ones."""
    rng = random.Random(5)
    big = 2 ** 31 - 1
    for i in range(3000):
        t = rng.choice([1, 4, 25, 64, 128, 512])
        n, m = rng.choice([0, 1, t, rng.randint(0, 9 * t)]), rng.randint(0, 12 * t)
        window = rng.choice([0, 0, 1, t, 3 * t + 5, big])
        causal = rng.randint(0, 1)
        tiles = -(-n // t)
        cap = big if window == 0 else min(big, (window + t) // t + 1)
        level = []
        for k in range(tiles):
            reach = m - n + (k + 1) * t if causal else m
            level.append(min(cap, max(0, -(-reach // t))))
        assert level == sorted(level)
        top = idx.t_top(n, m, t, causal, window)
        assert top == max(level + [0])
        for lv in range(-1, top + 2):
            assert idx.t_above(n, m, t, causal, window, lv) == sum(x > lv for x in level)
    # the largest sizes stay in range
    for n, m, t in ((big, big, 1), (big, 0, 1), (0, big, 1), (big, big, 512), (1, big, 4)):
        for causal in (0, 1):
            tiles = -(-n // t)
            top = idx.t_top(n, m, t, causal, 0)
            assert 0 <= top and idx.t_above(n, m, t, causal, 0, top) == 0
            assert idx.t_above(n, m, t, causal, 0, -1) == tiles
            assert all(0 <= idx.t_above(n, m, t, causal, 0, lv) <= tiles
                       for lv in (0, 1, top // 2, max(0, top - 1)))
