// packed_index.h -- where things are in packed sequences: row tiles, the keys
// a row sees, cache pages.  Plain integer code without CUDA types, shared by
// the kernels and compiled on its own by the CPU tests.
//
// Sequence s of a packed tensor has rows [cu[s], cu[s + 1]).  cu is device
// data that no host code has looked at: every value goes through
// clamp_int(cu, 0, rows) before it is used, so that a wrong one costs rows,
// never an access out of bounds.
#pragma once

#if defined(__CUDACC__)
#define LTX_HD __host__ __device__ __forceinline__
#else
#define LTX_HD inline
#endif

namespace ltx {

LTX_HD int clamp_int(int v, int lo, int hi) { return v < lo ? lo : (v > hi ? hi : v); }

// Work slots of a tensor of `rows` packed rows: sequence s owns the slots from
// slot_base(cu[s], s) up to slot_base(cu[s + 1], s + 1), computed from its own
// offset alone (no prefix sum over the sequences before it).  A sequence of n
// rows gets at least n / tile + extra - 1 slots, rounded up:
//   floor((a + n) / t) + x - floor(a / t)  >=  floor(n / t) + x.
// extra 1 covers ceil(n / t) row tiles; extra 2 covers the tiles of a run that
// starts anywhere inside a tile (ceil(n / t) + 1 of them for n > 0, and one
// where n < 2).  Slots past a sequence's last tile are empty.
LTX_HD int slot_base(int start, int seq, int tile, int extra) { return start / tile + extra * seq; }
LTX_HD int slot_count(int rows, int seqs, int tile, int extra)
{
  return slot_base(rows, seqs, tile, extra);
}

// Row i of n rows over m keys stands at position m - n + i.
// The keys it sees are [key_low, key_high).
LTX_HD int key_high(int pos, int m, int causal)
{
  if (!causal) return m;
  return pos < 0 ? 0 : (pos < m ? pos + 1 : m);
}
LTX_HD int key_low(int pos, int window)
{
  return window > 0 && pos >= window ? pos - window + 1 : 0;
}

// The query tiles of a sequence, `t` rows each, by how far their keys reach: tile i
// is of level ceil(reach / t), where reach is the m keys, or causal those up to its
// last row's position, m - n + (i + 1) t, and `cap` at most (a window's).  Levels are
// for ordering alone; the last tile counts as a whole one.
struct TileLevels {
  int tiles, t, cap, whole;       // whole: all tiles reach all of m
  long long shift;                // m - n, or m
};
LTX_HD TileLevels tile_levels(int n, int m, int t, int causal, int window)
{
  TileLevels l;
  l.tiles = (int)(((unsigned)n + (unsigned)t - 1u) / (unsigned)t);
  l.t = t;
  l.cap = 0x7fffffff;
  if (window > 0) {
    const unsigned cap = ((unsigned)window + (unsigned)t) / (unsigned)t + 1u;
    if (cap < 0x7fffffffu) l.cap = (int)cap;
  }
  l.whole = !causal;
  l.shift = causal ? (long long)m - n : m;
  return l;
}
// The largest level; the number of tiles above a level (-1: all).
LTX_HD int top_level(const TileLevels& l)
{
  if (l.tiles == 0) return 0;
  const long long reach = l.shift + (l.whole ? 0 : (long long)l.tiles * l.t);
  if (reach <= 0) return 0;
  const unsigned top = ((unsigned)reach + (unsigned)l.t - 1u) / (unsigned)l.t;   // reach <= m + t
  return top < (unsigned)l.cap ? (int)top : l.cap;
}
LTX_HD int tiles_above(const TileLevels& l, int level)
{
  if (level < 0) return l.tiles;
  if (level >= l.cap) return 0;
  const long long most = (long long)level * l.t - l.shift;  // tile i is above: (i + 1) t > most
  if (l.whole) return most < 0 ? l.tiles : 0;
  if (most >= (long long)l.tiles * l.t) return 0;
  return l.tiles - (most < 0 ? 0 : (int)((unsigned)most / (unsigned)l.t));
}

// ---- the paged cache -------------------------------------------------------

constexpr int kPage = 64;         // tokens of a page

// Whether n tokens from `start` on lie inside a table of `cap` tokens.
LTX_HD bool span_ok(int start, int n, int cap)
{
  return start >= 0 && start <= cap && n <= cap - start;
}
LTX_HD bool page_ok(int page, int pages) { return page >= 0 && page < pages; }

// The tokens [a, b) of [start, start + n) on the i-th page they touch, page
// `block` of the sequence; b <= a where there is no i-th page.
struct PageSpan {
  int block, a, b;
};
LTX_HD PageSpan page_span(int start, int n, int i)
{
  PageSpan r;
  r.block = start / kPage + i;
  const int from = r.block * kPage;
  r.a = start > from ? start : from;
  r.b = start + n < from + kPage ? start + n : from + kPage;
  return r;
}

// A list of `all` work items in equal runs: worker i of `workers` (at most
// `all`) has the items [work_bound(i), work_bound(i + 1)); item x is
// work_owner's.
typedef unsigned long long u64;
LTX_HD u64 work_bound(u64 all, u64 workers, u64 i) { return all * i / workers; }
LTX_HD u64 work_owner(u64 all, u64 workers, u64 x) { return ((x + 1) * workers - 1) / all; }

}  // namespace ltx
