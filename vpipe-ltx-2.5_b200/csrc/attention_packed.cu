// attention_packed.cu -- attention over packed prompts on the 5th-generation
// tensor cores: causal or full, grouped heads, sliding window, head widths
// 64, 128 and 256.
//
// Query row i of a sequence with n queries and m keys, at position
// pos = m - n + i, sees the keys j in [key_low, key_high) (packed_index.h):
//   o = sum_j 2^(c q.k_j - r) v_j / sum_j 2^(c q.k_j - r),   c = scale log2 e,
// r a running maximum of the row, and o = 0 where it sees none.
//
// Grouped heads share one stream of keys: the 128 rows of a query tile are
// TQ = floor(128 / G) tokens times the G query heads of one key/value head
// (row = token * G + head, one 3-D TMA box), so K and V are read once for the
// group and a causal tile ends TQ tokens, not 128, past its first row.
//
// A CTA holds four query tiles of 64-key steps (head width 64), two of 128-key
// steps (128) or one (256: its O takes 256 of the 512 TMEM columns), the layout
// of attention_tc.cu:
//   warp 0      TMA: Q, then K and V tiles in the order the MMAs use them,
//               through one ring of equal slots
//   warp 1      MMA: S = Q K^T, O += P V with P read from TMEM
//   warp 2      takes work: finds an item's sequence and keys and hands them to
//               the others through shared memory, one item ahead
//   warp 3      zeroes what is not the sequence's of an item's last V tile: told by a
//               barrier of its own (`cut`) that the tile is there, it tells `full`.
//               The same by the MMA warp made D = 64 4 % slower, stopping the
//               products at the last 16 keys 8 %
//   warps 4-..  softmax, 64 score columns a thread: eight warps a query tile,
//               two for each TMEM lane quarter, or four with a row a thread
// An item is a CTA's query tiles of one key head.  The grid has a CTA
// for each; a CTA that runs takes over the next one not yet launched (cluster
// launch control), so that barriers and TMEM are set up once, the next item's
// loads and first scores run under this one's last softmax and store, and the
// items, longest first in a causal sequence or in the whole call (PkOrder), go to
// whoever is free.
// Few items over long keys (a prompt's next chunk) go to clusters of 2, 4 or 8 CTAs,
// each with a run of the keys; their parts of O are joined through distributed shared
// memory (pk_join), so that no workspace is needed.
// With several tiles one's MMAs run under the others' softmax; with one tile the
// scores are double-buffered, so S of key tile j + 1 runs under softmax j.
// V is used as TMA lays it down, [key][64 dims] in 128-byte swizzled rows: the
// MN-major form of the MMA's B operand, no transposed copy.
//
// P is rounded to bf16, as the MMA takes it beside a bf16 V, while its sum stays f32:
// 2^-8 of a term and independent from term to term, so prompts of normal values are off by
// 0.0019 to 0.0023 rms against 64 bits, where rounding the result alone makes 0.0016.
//
// What P multiplies must not matter where P is 0, but 0 * NaN is NaN.  V rows behind
// a sequence's last key are zeroed in shared memory before the products see them
// (warp 3).  V rows of the sequence's own that this row, but not all of its tile, may
// not see (later tokens', those before its window) stay: a row that ends up with a NaN
// is computed again by repair_row from the keys it sees alone; a NaN that belongs
// there comes out the same.  That takes 50, 145, 240 ns a row and key at head width 64,
// 128, 256 (a warp's rows follow each other).
//
// Every wait is bounded; a timeout sets the context's error word and the CTA
// drains and exits.  While a warp computes rows again (32 of 300000 keys each take 2.3 s
// at width 256) the others' time runs from its last beat (pk_wait).
#include <cuda.h>

#include <climits>
#include <cstring>

#include "attention_tc.cuh"
#include "block_ops.h"
#include "kernels.h"
#include "packed_index.h"
#include "packed_seq.cuh"
#include "ptx.cuh"

namespace ltx {

namespace {

constexpr int kRows = 128;        // query rows of a tile = TMEM lanes
constexpr float kGrow = 8.0f;     // log2 of the largest P before O is rescaled

enum : int {
  PERR_PRODUCER = 0x65,
  PERR_MMA = 0x66,
  PERR_SOFTMAX = 0x67,
  PERR_DRAIN = 0x68,
  PERR_ITEM = 0x6A,
  PERR_CUT = 0x6B,
};

// Width 128 has two forms.  Wide: two query tiles a CTA, so that K and V are read
// once for 256 rows; a tile's softmax (1980 clocks) and its products (1490) follow
// each other, 3720 clocks for both tiles' 128 keys.  Narrow: one tile and three
// score buffers, two groups of softmax warps by turns, 1525 clocks for one tile's
// 128 keys; half the rows an item.  Under the power cap the wide form runs long
// prompts faster all the same (528 against 544 us, 8192 tokens, at 1.69 against
// 1.55 GHz), so the narrow one takes calls whose wide items would not fill the SMs.
// That rule is plain, not the best where wide items fill the SMs once and a little,
// since wide items share no keys.  32/8 heads, one sequence, us (wide / narrow):
//   new tokens on 8000       1100       1151       1153       1300       1600       2300
//                         140 / 132  141 / 134  263 / 149  262 / 185  270 / 205  294 / 302
//   prompts                  1300       2000       2400       4000       8192
//                        32.4 / 28.4  51.6 / 46.5  68 / 59   141 / 127  483 / 507
template <int D, bool NARROW>
struct PkCfg {
  static_assert(D == 128 || !NARROW, "forms");
  static constexpr int kTiles = D == 64 ? 4 : D == 128 && !NARROW ? 2 : 1;  // query tiles of a CTA
  static constexpr int kKeys = D == 64 ? 64 : 128;     // keys of a tile
  static constexpr int kBufs = D == 256 ? 2 : NARROW ? 3 : 1;     // score buffers of a query tile
  static constexpr int kSplit = kKeys / 64;            // softmax threads of a row, and
  static constexpr int kAlt = NARROW ? 2 : 1;          // groups that take key tiles in turn
  static constexpr int kGroup = 4 * kSplit * kAlt;     // softmax warps of a query tile
  static constexpr int kThreads = 128 + 32 * kGroup * kTiles;
  static constexpr int kQAtom = kRows * 128;           // 128 rows x 128 B (64 dims)
  static constexpr int kQTile = (D / 64) * kQAtom;
  // One ring slot: a K or V tile, or half of one at width 256 (K: 128 dims
  // of 128 keys; V: all dims of 64 keys).
  static constexpr int kParts = D == 256 ? 2 : 1;
  static constexpr int kKAtom = kKeys * 128;
  static constexpr int kSlot = (D / 64) * kKAtom / kParts;
  static constexpr int kSlots = D == 64 ? 16 : D == 128 && !NARROW ? 4 : 5;
  static constexpr int kVKeys = kKeys / kParts;        // keys of a V slot
  // row maxima and sums on their way between the threads of a row:
  // [group][parity][half][row], and the maxima handed from group to group
  static constexpr int kGroups = kTiles * kAlt;
  static constexpr int kMaxBytes =
      kSplit == 1 ? 0 : (kGroups * 4 + (kAlt == 2 ? 4 : 0)) * kRows * 4;
  static constexpr int kScores = kTiles * kBufs;       // score buffers
  static constexpr int kBars = 2 * kSlots + 2 * kScores + 4 * kTiles + 8 + 2 * kParts +
                               (kAlt == 2 ? 16 : 0);
  static constexpr int kBarBytes = (kBars * 8 + 16 + 15) / 16 * 16;
  static constexpr int kSmem = kTiles * kQTile + kSlots * kSlot + kMaxBytes + kBarBytes + 256;
  static constexpr uint32_t kOCol = 0;                 // O_t at t * D
  static constexpr uint32_t kSCol = kTiles * D;        // tile t's buffer i at t * kBufs + i
  static_assert(kSCol + kScores * kKeys <= 512, "TMEM columns");
  static_assert(kSmem <= 232448, "shared memory");
};

struct PkParams {
  const __nv_bfloat16 *q, *k, *v;
  __nv_bfloat16* o;
  int ldq, ldk, ldv, ldo;
  const int *cu_q, *cu_k;
  int seqs, rows, keys;     // rows of q and o, rows of k and v
  int kv_heads, group, tq;  // tq: tokens of a query tile
  int causal, window;
  int by_reach;             // items in the order of PkOrder
  int base;                 // the grid's first item
  int split;                // CTAs that share an item's keys
  float c;                  // scale log2 e
  int* err;
};

// B in MN-major form (rows of 64 dims, 128 B, swizzled; 8-key groups 1024 B
// apart, 64-dim blocks `block` bytes apart).
__device__ __forceinline__ uint64_t sdesc_mn_sw128(uint32_t saddr, uint32_t block)
{
  uint64_t d = 0;
  d |= (uint64_t)((saddr & 0x3FFFF) >> 4);
  d |= (uint64_t)(block >> 4) << 16;             // LBO: next 64 dims
  d |= (uint64_t)(1024 >> 4) << 32;              // SBO: next 8 keys
  d |= (uint64_t)1 << 46;                        // descriptor version (sm100)
  d |= (uint64_t)2 << 61;                        // SWIZZLE_128B
  return d;
}

// idesc_bf16 with B MN-major.
__host__ __device__ constexpr uint32_t idesc_bf16_bmn(int M, int N)
{
  return idesc_bf16(M, N) | (1u << 16);
}

// The MMA warp runs as a whole, so that the operands' descriptors stay in uniform
// registers, and one lane of it (`lead`) issues: one lane running the loop alone
// moves every operand there anew, which made 1200-1700 clocks of a query tile's
// 500-1000 on the tensor pipe.
__device__ __forceinline__ uint32_t elect_lane()
{
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r));
  return r;
}

__device__ __forceinline__ void umma_ss_by(uint32_t lead, uint32_t d, uint64_t a, uint64_t b,
                                           uint32_t idesc, uint32_t acc)
{
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(lead)
      : "memory");
}

__device__ __forceinline__ void umma_ts_by(uint32_t lead, uint32_t d, uint32_t a_tmem, uint64_t b,
                                           uint32_t idesc, uint32_t acc)
{
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a_tmem), "l"(b), "r"(idesc), "r"(acc), "r"(lead)
      : "memory");
}

__device__ __forceinline__ void umma_commit_by(uint32_t lead, uint64_t* bar)
{
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(
          smem_u32(bar)),
      "r"(lead)
      : "memory");
}

// 3-D tiled load, coordinates (x, y, z); x * element size a multiple of 16.
__device__ __forceinline__ void tma_load_3d(const void* map, uint64_t* bar, void* dst, int x,
                                            int y, int z)
{
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_"
      "tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(dst)),
      "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}

// A CTA's words for its waits.
struct PkState {
  uint32_t tmem;
  int abort;                      // not 0: the error for which all roles leave
  unsigned long long beat;        // when rows were last seen being computed again
};

// mbar_wait whose time runs from the last beat.  The CTA reports the error when it
// ends: a report at each wait made captions at width 64 3 % slower.
__device__ __forceinline__ bool pk_wait(uint64_t* bar, uint32_t parity, volatile PkState* s,
                                        int code)
{
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = globaltimer_ns();
  while (true) {
    if (mbar_try_wait(bar, parity)) return true;
    if (s->abort) return false;
    // (signed: a beat may come between the two reads)
    if (globaltimer_ns() - t0 > kWaitNs &&
        (long long)(globaltimer_ns() - s->beat) > (long long)kWaitNs) {
      s->abort = code;
      return false;
    }
  }
}

// The NaNs among columns [col0, col0 + N) of an output row that this warp has
// stored, looked into: a column with a NaN among its row's own values (rows
// key0 + j of v, j in [lo, hi)) keeps it; if any is left, the row is computed again
// from its own keys alone, in f32.  The first pass costs 1/10 of the second, so
// that a NaN every row sees stays cheap.  Beats every 4096 keys.
template <int D, int N>
__device__ __noinline__ void repair_row(const PkParams& p, volatile PkState* s, int row, int head,
                                        int kvh, int key0, int lo, int hi, int col0)
{
  constexpr int W = N / 32;                       // columns of a lane, 2 or 4
  const int lane = (int)lane_id();
  __nv_bfloat16* o = p.o + (size_t)row * p.ldo + (size_t)head * D + col0 + lane * W;
  const __nv_bfloat16* v0 = p.v + (size_t)key0 * p.ldv + (size_t)kvh * D + col0 + lane * W;
  bool bad[W], open = false;
  for (int e = 0; e < W; ++e) {
    const float x = __bfloat162float(o[e]);
    bad[e] = x != x;
    open |= bad[e];
  }
  bool found[W] = {};
  for (int j = lo; j < hi && __any_sync(0xffffffffu, open); j += 16) {
    if (((j - lo) & 4095) == 0) s->beat = globaltimer_ns();
    open = false;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const __nv_bfloat162* v =
          reinterpret_cast<const __nv_bfloat162*>(v0 + (size_t)min(j + i, hi - 1) * p.ldv);
#pragma unroll
      for (int e = 0; e < W; e += 2) {
        const float2 x = __bfloat1622float2(v[e / 2]);
        found[e] |= x.x != x.x;
        found[e + 1] |= x.y != x.y;
      }
    }
#pragma unroll
    for (int e = 0; e < W; ++e) open |= bad[e] && !found[e];
  }
  if (!__any_sync(0xffffffffu, open)) return;

  const uint4* q = reinterpret_cast<const uint4*>(p.q + (size_t)row * p.ldq + (size_t)head * D);
  float m = -INFINITY, l = 0.0f, acc[W];
  for (int e = 0; e < W; ++e) acc[e] = 0.0f;
  for (int j0 = lo; j0 < hi; j0 += 32) {
    if (((j0 - lo) & 4095) == 0) s->beat = globaltimer_ns();
    const int n = min(32, hi - j0);
    const uint4* k = reinterpret_cast<const uint4*>(
        p.k + (size_t)(key0 + j0 + min(lane, n - 1)) * p.ldk + (size_t)kvh * D);
    float dot = 0.0f;
#pragma unroll 4
    for (int d = 0; d < D / 8; ++d) {
      const uint4 a = q[d], b = k[d];
      const uint32_t aw[4] = {a.x, a.y, a.z, a.w}, bw[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        dot = fmaf(__uint_as_float(aw[i] << 16), __uint_as_float(bw[i] << 16), dot);
        dot = fmaf(__uint_as_float(aw[i] & 0xffff0000u), __uint_as_float(bw[i] & 0xffff0000u), dot);
      }
    }
    const float score = lane < n ? dot * p.c : -INFINITY;
    float mx = score;
    for (int w = 16; w > 0; w >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
    const float m_new = fmaxf(m, mx);
    const float r = m_new == -INFINITY ? 0.0f : m_new;
    const float f = m == -INFINITY ? 0.0f : exp2f(m - r);
    const float pj = lane < n ? exp2f(score - r) : 0.0f;
    m = m_new;
    l = l * f + pj;                               // this lane's share
    for (int e = 0; e < W; ++e) acc[e] *= f;
#pragma unroll 8
    for (int i = 0; i < n; ++i) {
      const float pi = __shfl_sync(0xffffffffu, pj, i);
      const __nv_bfloat162* v =
          reinterpret_cast<const __nv_bfloat162*>(v0 + (size_t)(j0 + i) * p.ldv);
#pragma unroll
      for (int e = 0; e < W; e += 2) {
        const float2 x = __bfloat1622float2(v[e / 2]);
        acc[e] = fmaf(pi, x.x, acc[e]);
        acc[e + 1] = fmaf(pi, x.y, acc[e + 1]);
      }
    }
  }
  for (int w = 16; w > 0; w >>= 1) l += __shfl_xor_sync(0xffffffffu, l, w);
  for (int e = 0; e < W; ++e)
    if (bad[e]) o[e] = __float2bfloat16_rn(acc[e] / l);
}

// Bits [from, to) of 32, both bounds anywhere.
__device__ __forceinline__ uint32_t bits_from_to(int from, int to)
{
  const uint32_t below = to >= 32 ? 0xffffffffu : to <= 0 ? 0u : (1u << to) - 1u;
  const uint32_t skip = from >= 32 ? 0xffffffffu : from <= 0 ? 0u : (1u << from) - 1u;
  return below & ~skip;
}

// N columns of this thread's row of O out of TMEM, scaled, to o + at (at < 0:
// nowhere); tells `o_free` once the warp has read it.  Returns whether a NaN was
// among it.  Eight lanes exchange their rows' 16-byte pieces so that a store
// writes 128 bytes of four rows; 16 bytes of 32 rows took 4000 clocks an item.
template <int N>
__device__ __forceinline__ bool store_row(uint32_t ocol, bool there, bool sees, float g,
                                          __nv_bfloat16* o, long long at, uint64_t* o_free)
{
  const uint32_t lane = lane_id();
  bool nan = false;
#pragma unroll
  for (int c8 = 0; c8 < N / 64; ++c8) {
    uint32_t w[8][4];                                  // eight pieces of 8 columns
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t v[32];
      tmem_ld32(ocol + (uint32_t)(c8 * 64 + h * 32), v);   // whatever it holds, where no key was seen
      tmem_wait_ld();
#pragma unroll
      for (int e = 0; e < 32; ++e) {
        const float x = sees ? __uint_as_float(v[e]) * g : 0.0f;
        nan |= x != x;
        v[e] = __float_as_uint(x);
      }
#pragma unroll
      for (int e = 0; e < 16; ++e)
        w[h * 4 + e / 4][e % 4] = pack_bf16(__uint_as_float(v[2 * e]), __uint_as_float(v[2 * e + 1]));
    }
    if (there && c8 + 1 == N / 64) {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(o_free);
    }
    // piece k of lane i becomes piece i of lane k, in eights
#pragma unroll
    for (int s = 4; s > 0; s >>= 1) {
      const bool up = (lane & (uint32_t)s) != 0;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        if ((k & s) != 0) continue;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t got = __shfl_xor_sync(0xffffffffu, up ? w[k][e] : w[k | s][e], s);
          if (up) w[k][e] = got;
          else w[k | s][e] = got;
        }
      }
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const long long to = __shfl_sync(0xffffffffu, at, (int)(lane & 24u) + k);
      if (to >= 0)
        *reinterpret_cast<uint4*>(o + to + c8 * 64 + (lane & 7u) * 8) =
            make_uint4(w[k][0], w[k][1], w[k][2], w[k][3]);
    }
  }
  return nan;
}

// Two to 32 sequences of a call, one a lane, with their tiles of T * tq rows in the
// order of how many keys they read, most first, whichever sequence they are of: a
// long tile that starts late is what a call of a few ragged prompts ends on.  Not
// where all items start at once (finding the first takes 1 us longer), nor where
// keys and values leave the L2 that going sequence by sequence keeps them in and
// fewer than 512 rows share a read.  Measured, by reach against by sequence:
// 16 prompts of 22 to 946 tokens, head width 64: 61 against 77 us; at width 128,
// 20 to 2500 tokens, 41 MB of keys and values: 174 against 209, 82 MB: 348 against
// 359, 165 MB: 693 against 645; at 256, 62 MB: 101 against 117, 124 MB: 237 against
// 235, 248 MB: 490 against 412; at 64, 82 MB: 171 against 204, 400 MB: 1143 against
// 1170.
struct PkOrder {
  int row0, nq, key0, nk;         // this lane's sequence
  TileLevels levels;
  int top;                        // the highest level of all

  __device__ __forceinline__ void read(const PkParams& p, int t)
  {
    const int s = (int)lane_id();
    row0 = nq = key0 = nk = 0;
    if (s < p.seqs) {
      const int a = p.cu_q[s], b = p.cu_q[s + 1], c = p.cu_k[s], d = p.cu_k[s + 1];
      row0 = clamp_int(a, 0, p.rows);
      nq = clamp_int(b, row0, p.rows) - row0;
      key0 = clamp_int(c, 0, p.keys);
      nk = clamp_int(d, key0, p.keys) - key0;
    }
    levels = tile_levels(nq, nk, t, p.causal, p.window);
    top = __reduce_max_sync(0xffffffffu, top_level(levels));
  }

  // The sequence (lane) and tile of place `rank`; -1 past the last.
  __device__ __forceinline__ int find(int rank, int* tile) const
  {
    int lo = 0, hi = top;         // the lowest level with no more than `rank` tiles above it
    while (lo < hi) {
      const int mid = lo + (hi - lo) / 2;
      if (__reduce_add_sync(0xffffffffu, tiles_above(levels, mid)) <= rank) hi = mid;
      else lo = mid + 1;
    }
    const int above = tiles_above(levels, lo), in = tiles_above(levels, lo - 1) - above;
    const int r = rank - __reduce_add_sync(0xffffffffu, above);
    int upto = in;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, upto, d);
      if ((int)lane_id() >= d) upto += x;
    }
    const int s = __ffs((int)__ballot_sync(0xffffffffu, upto > r)) - 1;
    *tile = __shfl_sync(0xffffffffu, levels.tiles - 1 - above - (r - (upto - in)), s & 31);
    return s;
  }
};

// One item of work as warp 2 hands it on (head < 0: no more).
struct PkItem {
  int head;                       // key/value head
  int row0, nq, tok0;             // the sequence's rows, the item's first token
  int key0, nk;                   // the sequence's keys
  int first, tiles[4];            // first key of the key tiles, their number for each query tile
};

// Keys of the sequence from the first one of key tile n - 1 on.
__device__ __forceinline__ int pk_left(const PkItem& w, int n, int keys)
{
  return w.nk - w.first - (n - 1) * keys;
}

// Ask for the next CTA of the grid that has not been launched; the 16-byte answer
// arrives in shared memory and on the barrier.
__device__ __forceinline__ void ask_next(void* answer, uint64_t* bar)
{
  mbar_arrive_expect_tx(bar, 16);
  asm volatile(
      "clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], "
      "[%1];" ::"r"(smem_u32(answer)),
      "r"(smem_u32(bar))
      : "memory");
}

// The answer's blockIdx.x, or -1: none was left.
__device__ __forceinline__ int next_index(const void* answer)
{
  uint32_t x = 0, ok = 0;
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b128 r;\n\t"
      "ld.shared.b128 r, [%2];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n\t"
      "selp.u32 %1, 1, 0, p;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %0, r;\n\t}"
      : "+r"(x), "=r"(ok)
      : "r"(smem_u32(answer))
      : "memory");
  return ok != 0 ? (int)x : -1;
}

constexpr int kMaxSplit = 8;      // CTAs of a cluster

__device__ __forceinline__ float2 ld_dsmem_f2(uint32_t caddr)
{
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];"
               : "=f"(v.x), "=f"(v.y)
               : "r"(caddr)
               : "memory");
  return v;
}

// Where 16-byte piece c of row `row` of a CTA's part of O lies.
template <int D>
__device__ __forceinline__ uint32_t pk_part(int row, int c)
{
  return (uint32_t)(row * (D / 4) + (c ^ (row & 7))) * 16u;
}

// This CTA's share of an item's rows (every S-th) out of the parts of the S CTAs of
// the cluster: with M the largest of their maxima,
//   o = sum 2^(m_i - M) O_i / sum 2^(m_i - M) l_i,
// in the CTAs' order.  A thread has 4 columns at a time, a warp whole rows or 128
// columns, and asks for 4 parts at once.
template <int D, int T, int S>
__device__ __forceinline__ void pk_join(const PkParams& p, volatile PkState* s, const PkItem& w,
                                        uint32_t parts, uint32_t sums, int tid, int threads)
{
  constexpr int kPieces = D / 4, kSpan = D < 128 ? D : 128;
  constexpr int kBatch = S < 4 ? S : 4, kAhead = 4 / kBatch;
  constexpr int kShare = kRows / S, kTotal = T * kShare * kPieces;
  const int rank = (int)cluster_ctarank(), rows = p.tq * p.group, shift = w.nk - w.nq;
#pragma unroll 1
  for (int u0 = tid; u0 < kTotal; u0 += kAhead * threads) {
    float2 ml[kAhead][S];
    float4 o[kAhead][kBatch];
    uint32_t part[kAhead];
    int at[kAhead];                                    // the row's place in its item, or -1
    bool any = false;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int u = u0 + i * threads, n = u / kPieces;
      const int t = n / kShare, r = n % kShare * S + rank;
      at[i] = -1;
      if (u < kTotal && r < rows) {
        const int tok = t * p.tq + r / p.group;
        if (w.tok0 + tok < w.nq) at[i] = tok * p.group + r % p.group;
      }
      if (at[i] >= 0) {
        any = true;
        const int place = t * kRows + r;
        const uint32_t sum = sums + (uint32_t)place * 8u;
        part[i] = parts + pk_part<D>(place, u % kPieces);
#pragma unroll
        for (int k = 0; k < S; ++k) ml[i][k] = ld_dsmem_f2(mapa_shared(sum, (uint32_t)k));
#pragma unroll
        for (int k = 0; k < kBatch; ++k) o[i][k] = ld_dsmem_f4(mapa_shared(part[i], (uint32_t)k));
      }
    }
    if (!__any_sync(0xffffffffu, any)) continue;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int c = (u0 + i * threads) % kPieces;
      float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      float l = 0.0f;
      int lo = 0, hi = 0, row = 0, head = 0;
      if (at[i] >= 0) {
        const int tok = w.tok0 + at[i] / p.group;
        row = w.row0 + tok;
        head = w.head * p.group + at[i] % p.group;
        lo = key_low(shift + tok, p.window);
        hi = key_high(shift + tok, w.nk, p.causal);
        float top = -INFINITY;
#pragma unroll
        for (int k = 0; k < S; ++k) top = fmaxf(top, ml[i][k].x);
#pragma unroll
        for (int k = 0; k < S; ++k) {
          if (k > 0 && k % kBatch == 0) {
#pragma unroll
            for (int j = 0; j < kBatch; ++j)
              o[i][j] = ld_dsmem_f4(mapa_shared(part[i], (uint32_t)(k + j)));
          }
          const float2 y = ml[i][k];
          const float4 z = o[i][k % kBatch];
          if (y.x == -INFINITY && y.y == 0.0f) continue; // saw nothing; what was read is no O
          const float f = y.x == -INFINITY ? 1.0f : fast_exp2(y.x - top);
          l = fmaf(f, y.y, l);
          x.x = fmaf(f, z.x, x.x);
          x.y = fmaf(f, z.y, x.y);
          x.z = fmaf(f, z.z, x.z);
          x.w = fmaf(f, z.w, x.w);
        }
        const float g = 1.0f / l;
        x = hi > lo ? make_float4(x.x * g, x.y * g, x.z * g, x.w * g)
                    : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        *reinterpret_cast<uint2*>(p.o + (size_t)row * p.ldo + (size_t)head * D + c * 4) =
            make_uint2(pack_bf16(x.x, x.y), pack_bf16(x.z, x.w));
      }
      const bool nan = x.x != x.x || x.y != x.y || x.z != x.z || x.w != x.w;
      __syncwarp();                                    // repair_row follows on these stores
      // one lane of each row asks
      uint32_t bad = __ballot_sync(0xffffffffu, nan && l > 0.0f);
      while (bad != 0) {
        const int src = __ffs((int)bad) - 1;
        bad &= kPieces < 32 ? ~(((1u << (kPieces & 31)) - 1u) << (src / kPieces * kPieces)) : 0u;
        repair_row<D, kSpan>(p, s, __shfl_sync(0xffffffffu, row, src),
                             __shfl_sync(0xffffffffu, head, src), w.head, w.key0,
                             __shfl_sync(0xffffffffu, lo, src), __shfl_sync(0xffffffffu, hi, src),
                             __shfl_sync(0xffffffffu, c * 4 / kSpan * kSpan, src));
      }
    }
  }
}

// SPLIT: a cluster of p.split CTAs has one item, each a run of its key tiles, and
// ends with it.
template <int D, bool NARROW, bool SPLIT>
__global__ void __launch_bounds__(PkCfg<D, NARROW>::kThreads, 1)
    pk_attention_kernel(const __grid_constant__ CUtensorMap tm_q,
                        const __grid_constant__ CUtensorMap tm_k,
                        const __grid_constant__ CUtensorMap tm_v,
                        const __grid_constant__ PkParams p)
{
  using C = PkCfg<D, NARROW>;
  constexpr int T = C::kTiles, R = C::kSlots, NB = C::kBufs, kKeys = C::kKeys;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* s_q = smem_raw;                             // tile t at t * kQTile
  uint8_t* s_ring = s_q + T * C::kQTile;
  float (*s_mx)[2][2][kRows] =                         // [group][parity][half][row]
      reinterpret_cast<float (*)[2][2][kRows]>(s_ring + R * C::kSlot);
  float (*s_m)[2][kRows] =                             // [group][half][row]
      reinterpret_cast<float (*)[2][kRows]>(s_mx + C::kGroups);
  uint64_t* bars = reinterpret_cast<uint64_t*>(s_ring + R * C::kSlot + C::kMaxBytes);
  uint64_t* q_full = bars;
  uint64_t* q_empty = q_full + 1;
  uint64_t* full = q_empty + 1;
  uint64_t* empty = full + R;
  uint64_t* s_full = empty + R;
  uint64_t* p_full = s_full + C::kScores;
  uint64_t* o_done = p_full + C::kScores;
  uint64_t* o_free = o_done + 2 * T;                   // o_done: two a tile, by turns
  uint64_t* o_last = o_free + T;
  uint64_t* item_full = o_last + T;
  uint64_t* item_empty = item_full + 2;
  uint64_t* asked = item_empty + 2;
  uint64_t* drain = asked + 1;
  uint64_t* cut = drain + 1;                           // [item's place][part]
  uint64_t* m_full = cut + 2 * C::kParts;              // [group][half][lane quarter] (kAlt 2)
  volatile PkState* s_state = reinterpret_cast<volatile PkState*>(bars + C::kBars);
  uint8_t* tail = s_ring + R * C::kSlot + C::kMaxBytes + C::kBarBytes;
  uint8_t* s_answer = tail;                            // 16 bytes
  volatile int* s_fail = reinterpret_cast<volatile int*>(tail + 16);    // one a query tile
  volatile int* s_swap = s_fail + 2;                   // one a group
  PkItem* s_item = reinterpret_cast<PkItem*>(tail + 32);                // two
  static_assert(32 + 2 * sizeof(PkItem) <= 256, "tail");

  // the same for all lanes, and known to be
  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0);
  const uint32_t lane = threadIdx.x & 31;
  if ((smem_u32(smem_raw) & 1023u) != 0) {             // the swizzle's atom
    if (threadIdx.x == 0) atomicCAS(p.err, 0, PERR_DRAIN);
    return;
  }

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int i = 0; i < R; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < C::kScores; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4 * C::kSplit);
    }
    for (int i = 0; i < T; ++i) {
      mbar_init(&o_done[2 * i], 1);
      mbar_init(&o_done[2 * i + 1], 1);
      mbar_init(&o_free[i], 4 * C::kSplit);
      mbar_init(&o_last[i], 1);
    }
    if (C::kAlt == 2)
      for (int i = 0; i < 16; ++i) mbar_init(&m_full[i], 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&item_full[i], 1);
      mbar_init(&item_empty[i], 3 + C::kGroup * T);
    }
    for (int i = 0; i < 2 * C::kParts; ++i) mbar_init(&cut[i], 1);
    s_fail[0] = s_fail[1] = 0;
    mbar_init(asked, 1);
    mbar_init(drain, 1);
    s_state->abort = 0;
    s_state->beat = 0;
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  if (warp == 1) {
    tmem_alloc(const_cast<uint32_t*>(&s_state->tmem), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_state->tmem;
  pdl_wait();
  pdl_trigger();

  // Items pass through two places in turn; each role counts them (`it`) and what
  // it has waited for and signalled since the CTA began, so that the barriers'
  // phases run on from item to item.
  if (warp == 2) {
    // ------------------------------------------------------------ items
    const int slots = slot_count(p.rows, p.seqs, T * p.tq, 1);
    PkOrder order;
    if (p.by_reach) order.read(p, T * p.tq);
    int index = p.base + (int)(SPLIT ? blockIdx.x / (unsigned)p.split : blockIdx.x);
    bool ok = true;
    for (int it = 0; ok; ++it) {
      // the answer is read before the next question goes out to its place
      if (!SPLIT && index >= 0 && lane == 0) {
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        ask_next(s_answer, asked);
      }
      PkItem w;
      w.head = -1;
      if (index >= 0) {
        w.head = (int)((unsigned)index % (unsigned)p.kv_heads);
        const int rank = (int)((unsigned)index / (unsigned)p.kv_heads);
        if (p.by_reach) {
          int tile;
          const int seq = order.find(rank, &tile);
          w.row0 = __shfl_sync(0xffffffffu, order.row0, seq & 31);
          w.nq = __shfl_sync(0xffffffffu, order.nq, seq & 31);
          w.key0 = __shfl_sync(0xffffffffu, order.key0, seq & 31);
          w.nk = __shfl_sync(0xffffffffu, order.nk, seq & 31);
          if (seq < 0) w.nq = tile = 0;
          w.tok0 = tile * (T * p.tq);
        } else {
          // slots run backwards, so that a causal sequence's longest items are first
          const int slot = slots - 1 - rank;
          const int seq = find_seq(p.cu_q, p.seqs, p.rows, T * p.tq, 1, slot);
          w.row0 = clamp_int(p.cu_q[seq], 0, p.rows);
          w.nq = clamp_int(p.cu_q[seq + 1], w.row0, p.rows) - w.row0;
          w.key0 = clamp_int(p.cu_k[seq], 0, p.keys);
          w.nk = clamp_int(p.cu_k[seq + 1], w.key0, p.keys) - w.key0;
          int tile = slot - slot_base(w.row0, seq, T * p.tq, 1);
          if (tile < 0) w.nq = tile = 0;               // rows before the first sequence
          w.tok0 = tile * (T * p.tq);
        }
        // keys any of the rows sees: from the first row's low to the last one's high
        const int shift = w.nk - w.nq;
        w.first = key_low(shift + w.tok0, p.window);
#pragma unroll
        for (int t = 0; t < 4; ++t) w.tiles[t] = 0;
#pragma unroll
        for (int t = 0; t < T; ++t) {
          const int a = w.tok0 + t * p.tq, b = min(a + p.tq, w.nq);
          if (b > a) {
            const int end = key_high(shift + b - 1, w.nk, p.causal);
            w.tiles[t] = end > w.first ? (end - w.first + kKeys - 1) / kKeys : 0;
          }
        }
        if constexpr (SPLIT) {
          const int n = max(max(w.tiles[0], w.tiles[1]), max(w.tiles[2], w.tiles[3]));
          const u64 rank = cluster_ctarank(), of = (u64)p.split;
          const int from = (int)work_bound((u64)n, of, rank), to = (int)work_bound((u64)n, of, rank + 1);
#pragma unroll
          for (int t = 0; t < 4; ++t) w.tiles[t] = clamp_int(w.tiles[t] - from, 0, to - from);
          w.first += from * kKeys;
        }
      }
      ok = __all_sync(0xffffffffu, pk_wait(&item_empty[it & 1], ((uint32_t)(it >> 1) & 1u) ^ 1u,
                                           s_state, PERR_ITEM));
      if (ok && lane == 0) {
        s_item[it & 1] = w;
        mbar_arrive(&item_full[it & 1]);
      }
      if (index < 0) break;
      if (SPLIT) {
        index = -1;
        continue;
      }
      // every question is waited for, so that no answer is under way at the end
      volatile int no_abort = 0;
      const bool told = __all_sync(
          0xffffffffu, mbar_wait(asked, (uint32_t)it & 1u, &no_abort, p.err, PERR_DRAIN));
      ok = ok && told;
      if (ok) {
        index = next_index(s_answer);
        if (index >= 0) index += p.base;
      }
      __syncwarp();
    }
  } else if (warp == 0) {
    // ------------------------------------------------------------- TMA
    if (lane == 0) {
      uint32_t armed = 0, armed_par = 0, q_armed = 0, cut_armed = 0, cut_par = 0;
      int used = 0, with_keys = 0;                     // ring slots, items that have keys
      bool ok = true;
      for (int it = 0; ok; ++it) {
        ok = pk_wait(&item_full[it & 1], (uint32_t)(it >> 1) & 1u, s_state, PERR_PRODUCER);
        if (!ok) break;
        const PkItem w = s_item[it & 1];
        mbar_arrive(&item_empty[it & 1]);
        if (w.head < 0) break;
        const int n = max(max(w.tiles[0], w.tiles[1]), max(w.tiles[2], w.tiles[3]));
        if (n == 0) continue;
        const bool cuts = pk_left(w, n, kKeys) < kKeys;
        // Q's place is free once the item before has its last scores
        ok = pk_wait(q_empty, ((uint32_t)with_keys & 1u) ^ 1u, s_state, PERR_PRODUCER);
        if (!ok) break;
        mbar_arrive_expect_tx(q_full, (uint32_t)(T * (D / 64) * p.group * p.tq * 128));
        for (int t = 0; t < T; ++t)
          for (int a = 0; a < D / 64; ++a)
            tma_load_3d(&tm_q, q_full, s_q + t * C::kQTile + a * C::kQAtom, a * 64,
                        w.head * p.group, w.row0 + w.tok0 + t * p.tq);
        ++with_keys;
        q_armed = 1;
        // one slot: `v` selects V, part its half at width 256
        auto load = [&](bool v, int j) {
          for (int part = 0; ok && part < C::kParts; ++part, ++used) {
            const int st = used % R;
            const uint32_t ph = (uint32_t)(used / R) & 1u;
            ok = pk_wait(&empty[st], ph ^ 1u, s_state, PERR_PRODUCER);
            if (!ok) break;
            uint8_t* dst = s_ring + st * C::kSlot;
            const int key = w.key0 + w.first + j * kKeys;
            uint64_t* bar = &full[st];
            armed |= 1u << st;
            armed_par = (armed_par & ~(1u << st)) | (ph << st);
            if (v && cuts && j + 1 == n) {             // warp 3 tells `full`
              const int i = (it & 1) * C::kParts + part;
              bar = &cut[i];
              armed &= ~(1u << st);
              cut_par ^= cut_armed & (1u << i);        // 0 the first time, then the other
              cut_armed |= 1u << i;
            }
            mbar_arrive_expect_tx(bar, C::kSlot);
            if (v) {
              for (int a = 0; a < D / 64; ++a)
                tma_load_3d(&tm_v, bar, dst + a * C::kVKeys * 128, a * 64, w.head,
                            key + part * C::kVKeys);
            } else {
              constexpr int A = D / 64 / C::kParts;
              for (int a = 0; a < A; ++a)
                tma_load_3d(&tm_k, bar, dst + a * C::kKAtom, (part * A + a) * 64, w.head, key);
            }
          }
        };
        for (int j = 0; ok && j < min(NB, n); ++j) load(false, j);
        for (int j = 0; ok && j < n; ++j) {
          load(true, j);
          if (j + NB < n) load(false, j + NB);
        }
      }
      // Every load lands before the CTA may exit.
      volatile int no_abort = 0;
      if (q_armed)
        mbar_wait(q_full, (uint32_t)(with_keys - 1) & 1u, &no_abort, p.err, PERR_DRAIN);
      for (int st = 0; st < R; ++st)
        if (armed & (1u << st))
          mbar_wait(&full[st], (armed_par >> st) & 1u, &no_abort, p.err, PERR_DRAIN);
      for (int i = 0; i < 2 * C::kParts; ++i)
        if (cut_armed & (1u << i))
          mbar_wait(&cut[i], (cut_par >> i) & 1u, &no_abort, p.err, PERR_DRAIN);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------- MMA
    constexpr uint32_t idesc_s = idesc_bf16(kRows, kKeys);
    constexpr uint32_t idesc_o = idesc_bf16_bmn(kRows, D);
    const uint32_t lead = elect_lane();
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      return __all_sync(0xffffffffu, pk_wait(bar, parity, s_state, PERR_MMA)) != 0;
    };
    // a place in the ring of slots and the parity of its round
    struct Ring {
      uint32_t slot, round;
      __device__ __forceinline__ void next()
      {
        if (++slot == (uint32_t)R) {
          slot = 0;
          round ^= 1u;
        }
      }
    };
    Ring ring = {0, 0};
    const uint64_t q_desc = sdesc_k128_sw128(smem_u32(s_q));
    const uint64_t k_desc = sdesc_k128_sw128(smem_u32(s_ring));
    const uint64_t v_desc = sdesc_mn_sw128(smem_u32(s_ring), C::kVKeys * 128);
    // scores for query tile t into buffer b of the k steps that key slot `at`
    // holds (part: its half at width 256)
    auto issue_s = [&](int t, uint32_t b, uint32_t at, int part) {
      constexpr int A = D / 64 / C::kParts;            // 64-dim atoms of a slot
      const uint32_t d = tm + C::kSCol + b * (uint32_t)kKeys;
      const uint64_t qd = q_desc + (uint64_t)(((t * C::kQTile + part * A * C::kQAtom) >> 4));
      const uint64_t kd = k_desc + (uint64_t)(at * (uint32_t)(C::kSlot >> 4));
#pragma unroll
      for (int kk = 0; kk < A * 4; ++kk)
        umma_ss_by(lead, d, qd + (uint64_t)((kk >> 2) * (C::kQAtom >> 4) + 2 * (kk & 3)),
                   kd + (uint64_t)((kk >> 2) * (C::kKAtom >> 4) + 2 * (kk & 3)), idesc_s,
                   part > 0 || kk > 0 ? 1u : 0u);
    };
    // O += P V over the keys of value slot `at`
    auto issue_pv = [&](int t, uint32_t b, uint32_t at, int part, bool first) {
      const uint32_t pa = tm + C::kSCol + b * (uint32_t)kKeys + (uint32_t)(part * C::kVKeys / 2);
      const uint64_t vd = v_desc + (uint64_t)(at * (uint32_t)(C::kSlot >> 4));
#pragma unroll
      for (int kk = 0; kk < C::kVKeys / 16; ++kk)
        umma_ts_by(lead, tm + C::kOCol + (uint32_t)(t * D), pa + (uint32_t)(kk * 8),
                   vd + (uint64_t)(kk * (16 * 128 >> 4)), idesc_o,
                   !first || part > 0 || kk > 0 ? 1u : 0u);
    };
    uint32_t with_keys = 0;                            // items that have keys
    uint32_t step[T] = {}, opened[T] = {};             // score tiles and items, a query tile
    bool ok = true;
    for (uint32_t it = 0; ok; ++it) {
      ok = wait(&item_full[it & 1], (it >> 1) & 1u);
      if (!ok) break;
      const PkItem* w = &s_item[it & 1];
      const int head = __shfl_sync(0xffffffffu, w->head, 0);
      int tiles[T], n = 0;
#pragma unroll
      for (int t = 0; t < T; ++t) {
        tiles[t] = __shfl_sync(0xffffffffu, w->tiles[t], 0);
        n = max(n, tiles[t]);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&item_empty[it & 1]);
      if (head < 0) break;
      if (n == 0) continue;
      ok = wait(q_full, with_keys & 1u);
      if (!ok) break;
      ++with_keys;
      // scores of key tile j for every query tile that has it, from the slots at k
      auto scores = [&](int t, int j, Ring k, bool first) {
        const uint32_t buf = (uint32_t)(t * NB) + ((step[t] + (uint32_t)j) % (uint32_t)NB);
#pragma unroll
        for (int part = 0; part < C::kParts; ++part) {
          if (ok && first) ok = wait(&full[k.slot], k.round);
          if (!ok) return;
          tc_fence_after();
          issue_s(t, buf, k.slot, part);
          if (T == 1) umma_commit_by(lead, &empty[k.slot]);
          k.next();
        }
        umma_commit_by(lead, &s_full[buf]);
      };
      auto release = [&](Ring k) {                     // with one query tile each use does it
        if (T > 1) umma_commit_by(lead, &empty[k.slot]);
      };
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        if (!ok || j >= n) continue;
        bool first = true;
#pragma unroll
        for (int t = 0; t < T; ++t)
          if (ok && j < tiles[t]) {
            scores(t, j, ring, first);
            first = false;
          }
        if (!ok) continue;
        release(ring);
#pragma unroll
        for (int part = 0; part < C::kParts; ++part) ring.next();
        if (j + 1 == n) umma_commit_by(lead, q_empty);
      }
      for (int j = 0; ok && j < n; ++j) {
        const Ring v = ring;                           // V_j, then K_{j + NB}
#pragma unroll
        for (int part = 0; part < C::kParts; ++part) ring.next();
        const Ring k = ring;
        const bool more = j + NB < n;
        bool have_v = false, have_k = false;
#pragma unroll
        for (int t = 0; t < T; ++t) {
          if (!ok || j >= tiles[t]) continue;
          // P V, then the scores that take its buffer (in order: they overwrite it
          // only after this P V has read P from it); an item's first P V overwrites
          // O, which the softmax must have read
          const uint32_t at = step[t] + (uint32_t)j;
          const uint32_t buf = (uint32_t)(t * NB) + at % (uint32_t)NB;
          ok = wait(&p_full[buf], (at / (uint32_t)NB) & 1u);
          if (ok && j == 0) ok = wait(&o_free[t], (opened[t]++ & 1u) ^ 1u);
          Ring vv = v;
#pragma unroll
          for (int part = 0; part < C::kParts; ++part) {
            if (ok && !have_v) ok = wait(&full[vv.slot], vv.round);
            if (!ok) continue;
            tc_fence_after();
            issue_pv(t, buf, vv.slot, part, j == 0);
            if (T == 1) umma_commit_by(lead, &empty[vv.slot]);
            vv.next();
          }
          have_v = true;
          if (!ok) continue;
          umma_commit_by(lead, &o_done[2 * t + (int)(at & 1u)]);
          if (j + 1 == tiles[t]) umma_commit_by(lead, &o_last[t]);
          if (j + NB < tiles[t]) {
            scores(t, j + NB, k, !have_k);
            have_k = true;
          }
        }
        if (!ok) break;
        release(v);
        if (more) {
          release(k);
#pragma unroll
          for (int part = 0; part < C::kParts; ++part) ring.next();
        }
        if (j + NB + 1 == n) umma_commit_by(lead, q_empty);
      }
#pragma unroll
      for (int t = 0; t < T; ++t) step[t] += (uint32_t)tiles[t];
    }
    umma_commit_by(lead, drain);
    volatile int no_abort = 0;
    mbar_wait(drain, 0, &no_abort, p.err, PERR_DRAIN);
    __syncwarp();
  } else if (warp == 3) {
    // ------------------------------------------------------------- cuts
    int used = 0;                                      // ring slots
    uint32_t seen[2] = {};                             // cuts of each place
    bool ok = true;
    for (int it = 0; ok; ++it) {
      ok = __all_sync(0xffffffffu, pk_wait(&item_full[it & 1], (uint32_t)(it >> 1) & 1u, s_state,
                                           PERR_CUT));
      if (!ok) break;
      const PkItem* w = &s_item[it & 1];
      const int head = w->head;
      const int n = max(max(w->tiles[0], w->tiles[1]), max(w->tiles[2], w->tiles[3]));
      const int left = pk_left(*w, n, kKeys);
      if (head >= 0 && n > 0) {
        used += 2 * n * C::kParts;                     // the last V tile is its last
        if (left < kKeys) {
          const uint32_t parity = seen[it & 1]++ & 1u;
#pragma unroll
          for (int part = 0; part < C::kParts; ++part) {
            const int st = (used - C::kParts + part) % R;
            ok = ok && __all_sync(0xffffffffu, pk_wait(&cut[(it & 1) * C::kParts + part], parity,
                                                       s_state, PERR_CUT));
            if (!ok) break;
            // whole 128-byte rows of each 64 dims, from the first key that is not
            // the sequence's
            const int from = clamp_int(left - part * C::kVKeys, 0, C::kVKeys);
            for (int i = (int)lane; i < (C::kVKeys - from) * (D / 8); i += 32)
              *reinterpret_cast<uint4*>(s_ring + st * C::kSlot +
                                        i % (D / 8) / 8 * (C::kVKeys * 128) +
                                        (from + i / (D / 8)) * 128 + i % 8 * 16) =
                  make_uint4(0, 0, 0, 0);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&full[st]);
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&item_empty[it & 1]);
      if (head < 0) break;
    }
  } else if (warp >= 4) {
    // ---------------------------------------------------------- softmax
    // Four warps a tile with a row a thread; or eight with two threads a row (hh:
    // score columns [0, 64) and [64, 128) of a key tile), or two such groups that
    // take the key tiles in turn (`alt`), so that one's exponentials run under the
    // other's maxima, stores and waits.
    constexpr int kSplit = C::kSplit, kAlt = C::kAlt;
    const int t = (warp - 4) / C::kGroup;
    const int hh = ((warp - 4) >> 2) & (kSplit - 1);
    const int alt = (warp - 4) / (4 * kSplit) & (kAlt - 1);
    const int gx = t * kAlt + alt;                     // this group, of kGroups
    const int quarter = warp & 3;
    const int r = quarter * 32 + (int)lane;
    const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
    const uint32_t orow = tmem + lane_base + C::kOCol + (uint32_t)(t * D);
    const float c = p.c;
    // score tiles of this query tile so far, and exchanges (kSplit 2)
    uint32_t step = 0, swap = 0, closed = 0;           // closed: items with keys
    bool ok = true, joins = false;
#pragma unroll 1
    for (int it = 0;; ++it) {
      // Two warps a row meet at barriers, so all warps of a tile agree on going on:
      // a wait that failed is told before one, and their number in an item is the
      // same for all.
      ok = __all_sync(0xffffffffu, ok && pk_wait(&item_full[it & 1], (uint32_t)(it >> 1) & 1u,
                                                 s_state, PERR_SOFTMAX));
      if (kSplit * kAlt == 1) {
        if (!ok) break;
      } else {
        if (!ok && lane == 0) s_fail[t] = 1;
        named_bar_sync(1 + t, 32 * C::kGroup);
        if (s_fail[t] != 0) break;
      }
      // the item stays in its place until this role is through with it
      const PkItem* w = &s_item[it & 1];
      if (w->head < 0) break;
      const int nt = w->tiles[t];
      const int first = w->first;
      // the keys this thread's row sees, and those that all valid rows of the
      // query tile see
      int lo, hi, all_lo, all_hi;
      {
        const int tok = w->tok0 + t * p.tq + r / p.group, shift = w->nk - w->nq;
        const bool valid_row = r < p.tq * p.group && tok < w->nq;
        lo = key_low(shift + tok, p.window);
        hi = valid_row ? key_high(shift + tok, w->nk, p.causal) : 0;
        const int a_tok = w->tok0 + t * p.tq, b_tok = min(a_tok + p.tq, w->nq) - 1;
        all_lo = key_low(shift + b_tok, p.window);
        all_hi = key_high(shift + a_tok, w->nk, p.causal);
      }
      // m_run: what this thread's sum refers to.  kAlt 2: the row's maximum goes
      // from group to group with the key tiles (s_mx[t][1][group]).
      float m_run = -INFINITY, l_run = 0.0f;
#pragma unroll 1
      for (int i = kAlt == 2 ? (int)((step ^ (uint32_t)alt) & 1u) : 0; i < nt; i += kAlt) {
        const uint32_t at = step + (uint32_t)i;        // this score tile
        const int sb = t * NB + (int)(at % (uint32_t)NB);
        const uint32_t scol = tmem + lane_base + C::kSCol + (uint32_t)(sb * kKeys);
        ok = __all_sync(0xffffffffu, ok && pk_wait(&s_full[sb], (at / (uint32_t)NB) & 1u, s_state,
                                                   PERR_SOFTMAX));
        uint32_t a[32], b[32];
        tc_fence_after();
        tmem_ld32(scol + (uint32_t)(hh * 64), a);
        tmem_ld32(scol + (uint32_t)(hh * 64 + 32), b);
        tmem_wait_ld();
        const int j0 = first + i * kKeys;
        if (j0 < all_lo || j0 + kKeys > all_hi) {
          // bit e of (ma, mb): this row sees score e; one test a score, where two
          // comparisons took 1500 clocks a tile
          const int from = lo - j0 - hh * 64, to = hi - j0 - hh * 64;
          const uint32_t ma = bits_from_to(from, to), mb = bits_from_to(from - 32, to - 32);
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            a[e] = (ma >> e) & 1u ? a[e] : 0xff800000u;              // -inf
            b[e] = (mb >> e) & 1u ? b[e] : 0xff800000u;
          }
        }
        float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
          m4[0] = max3f(m4[0], __uint_as_float(a[e]), __uint_as_float(a[e + 1]));
          m4[1] = max3f(m4[1], __uint_as_float(a[e + 2]), __uint_as_float(a[e + 3]));
          m4[2] = max3f(m4[2], __uint_as_float(b[e]), __uint_as_float(b[e + 1]));
          m4[3] = max3f(m4[3], __uint_as_float(b[e + 2]), __uint_as_float(b[e + 3]));
        }
        float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
        float m_old = m_run;                           // what O refers to
        if (kSplit == 2) {
          // the row's max over both halves: exchange through shared memory (both
          // halves have their scores in registers after this barrier, so either
          // may then overwrite the TMEM columns with P)
          s_mx[gx][swap & 1u][hh][r] = mx;
          named_bar_sync(3 + gx, 256);
          mx = fmaxf(s_mx[gx][swap & 1u][0][r], s_mx[gx][swap & 1u][1][r]);
          ++swap;
        }
        if (kAlt == 2) {
          // the maximum that the other group's key tile left
          if (i == 0) {
            m_old = -INFINITY;
          } else {
            ok = __all_sync(0xffffffffu,
                            ok && pk_wait(&m_full[((alt ^ 1) * 2 + hh) * 4 + quarter],
                                          ((at - 1u) >> 1) & 1u, s_state, PERR_SOFTMAX));
            m_old = s_m[alt ^ 1][hh][r];
          }
        }
        if (!ok) continue;
        const float m_tile = mx * c;
        // a row's first visible tile sets its maximum; later it moves only when
        // it grows by more than 2^kGrow (until then P stays below 2^kGrow)
        const bool need = m_tile > m_old + kGrow;
        const bool rescale = i > 0 && __any_sync(0xffffffffu, need);
        const float m_new = need ? m_tile : m_old;
        if (kAlt == 2) {
          s_m[alt][hh][r] = m_new;
          __syncwarp();
          if (lane == 0) mbar_arrive(&m_full[(alt * 2 + hh) * 4 + quarter]);
        }
        float f = 1.0f;
        if (need) f = fast_exp2(m_old - m_new);
        if (kAlt == 2) {
          // this group's sum may refer to an older maximum than O
          if (m_run != m_new) l_run *= fast_exp2(m_run - m_new);
        } else {
          l_run *= f;
        }
        m_run = m_new;
        const float nm = m_run == -INFINITY ? 0.0f : -m_run;
        const unsigned long long c2 = pair2(__float_as_uint(c), __float_as_uint(c));
        const unsigned long long nm2 = pair2(__float_as_uint(nm), __float_as_uint(nm));
        unsigned long long sa = 0ull, sb2 = 0ull;
        uint32_t pk[32];
        fa3_exp(a, b, c2, nm2, pk, sa, sb2);
        tmem_st32(scol + (uint32_t)(hh * 32), pk);
        const unsigned long long st2 = fadd2(sa, sb2);
        l_run += __uint_as_float((uint32_t)st2) + __uint_as_float((uint32_t)(st2 >> 32));
        if (rescale) {
          // All of O but this key tile's part.  Of the barrier's two rounds back the
          // P V at - 3 is done (these scores came after it), so the parity is plain;
          // with one barrier P V at - 2, under way or done, would leave it open.
          ok = __all_sync(0xffffffffu, pk_wait(&o_done[2 * t + (int)((at - 1u) & 1u)],
                                               ((at - 1u) >> 1) & 1u, s_state, PERR_SOFTMAX));
          if (ok) {
            tc_fence_after();
#pragma unroll
            for (int c4 = 0; c4 < D / kSplit / 32; ++c4) {
              uint32_t v[32];
              const uint32_t oc = orow + (uint32_t)(hh * (D / kSplit) + c4 * 32);
              tmem_ld32(oc, v);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 32; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) * f);
              tmem_st32(oc, v);
            }
          }
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (ok && lane == 0) mbar_arrive(&p_full[sb]);
      }
      // the row's sum over its threads, under the last maximum
      float l_row = l_run, m_end = m_run;
      if (kAlt == 2 && nt > 0) {
        const uint32_t end = step + (uint32_t)nt - 1u;
        if ((int)(end & 1u) != alt) {
          ok = __all_sync(0xffffffffu,
                          ok && pk_wait(&m_full[((alt ^ 1) * 2 + hh) * 4 + quarter],
                                        (end >> 1) & 1u, s_state, PERR_SOFTMAX));
          m_end = s_m[alt ^ 1][hh][r];
        }
        if (m_run != m_end) l_row *= fast_exp2(m_run - m_end);
      }
      if (kSplit * kAlt > 1) {
        // (the last exchange's reads of this place were before the barrier at the
        // start of this item or an exchange in it)
        s_mx[gx][swap & 1u][hh][r] = l_row;
        if (kAlt == 2) s_swap[alt] = (int)(swap & 1u);
        named_bar_sync(1 + t, 32 * C::kGroup);
        l_row = s_mx[gx][swap & 1u][0][r] + s_mx[gx][swap & 1u][1][r];
        if (kAlt == 2) {
          const int at = s_swap[alt ^ 1];
          l_row += s_mx[alt ^ 1][at][0][r] + s_mx[alt ^ 1][at][1][r];
        }
        ++swap;
      }
      step += (uint32_t)nt;
      // The rows go out; of two groups the one without the last key tile does it.
      // (All of O is waited for by a barrier of its own: by o_done the P V before the
      // last may be under way still, or both be done, and a parity tells neither.)
      const bool stores = kAlt == 1 || (nt > 0 ? (int)((step - 1u) & 1u) != alt : alt == 0);
      if (nt > 0) {
        if (stores)
          ok = __all_sync(0xffffffffu, ok && pk_wait(&o_last[t], closed & 1u, s_state,
                                                     PERR_SOFTMAX));
        ++closed;
      }
      if constexpr (SPLIT) {
        // O and (maximum, sum) to this CTA's shared memory, once the products of all
        // query tiles are through with it; 16-byte pieces in turn against bank conflicts
        constexpr int kCols = D / kSplit;
        ok = __all_sync(0xffffffffu, ok && pk_wait(drain, 0, s_state, PERR_SOFTMAX));
        if (ok && stores) {
          tc_fence_after();
#pragma unroll
          for (int c4 = 0; c4 < kCols / 32; ++c4) {
            uint32_t v[32];
            tmem_ld32(orow + (uint32_t)(hh * kCols + c4 * 32), v);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 8; ++e)
              *reinterpret_cast<uint4*>(
                  s_ring + pk_part<D>(t * kRows + r, hh * (kCols / 4) + c4 * 8 + e)) =
                  make_uint4(v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]);
          }
          if (hh == 0)                                 // (Q's place)
            reinterpret_cast<float2*>(s_q)[t * kRows + r] = make_float2(m_end, nt > 0 ? l_row : 0.0f);
        }
        joins = true;
        break;
      }
      if (!ok) continue;
      if (stores) {
        tc_fence_after();
        constexpr int kCols = D / kSplit;
        const bool sees = nt > 0 && hi > lo;
        const int tok = w->tok0 + t * p.tq + r / p.group;
        const bool valid_row = r < p.tq * p.group && tok < w->nq;
        const int row = w->row0 + tok, head = w->head * p.group + r % p.group;
        const float g = 1.0f / l_row;
        // a sum of 0 or NaN is of the row's own keys and makes all of it NaN
        const bool fix = valid_row && l_row > 0.0f;
        const long long to = (long long)row * p.ldo + (long long)head * D + hh * kCols;
        const bool nan = store_row<kCols>(orow + (uint32_t)(hh * kCols), nt > 0, sees, g, p.o,
                                          valid_row ? to : -1, &o_free[t]);
        __syncwarp();                                  // repair_row follows on these stores
        uint32_t bad = __ballot_sync(0xffffffffu, nan && fix);
        while (bad != 0) {
          const int src = __ffs((int)bad) - 1;
          bad &= bad - 1;
          repair_row<D, kCols>(p, s_state, __shfl_sync(0xffffffffu, row, src),
                               __shfl_sync(0xffffffffu, head, src), w->head, w->key0,
                               __shfl_sync(0xffffffffu, lo, src),
                               __shfl_sync(0xffffffffu, hi, src), hh * kCols);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&item_empty[it & 1]);
    }
    if constexpr (SPLIT) {
      cluster_sync_all();                              // every CTA's part is there
      if (joins) {
        const uint32_t parts = smem_u32(s_ring), sums = smem_u32(s_q);
        const int tid = (int)threadIdx.x - 128, threads = C::kThreads - 128;
        if (p.split == 2) pk_join<D, T, 2>(p, s_state, s_item[0], parts, sums, tid, threads);
        else if (p.split == 4) pk_join<D, T, 4>(p, s_state, s_item[0], parts, sums, tid, threads);
        else pk_join<D, T, 8>(p, s_state, s_item[0], parts, sums, tid, threads);
      }
    }
  }
  if constexpr (SPLIT) {
    if (warp < 4) cluster_sync_all();
    cluster_sync_all();                                // parts are read, CTAs may go
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (threadIdx.x == 0 && s_state->abort != 0) atomicCAS(p.err, 0, s_state->abort);
  if (warp == 1) tmem_dealloc(tmem, 512);
}

PFN_encodeTiled g_pk_encode = nullptr;

// bf16 [rows][heads][D] with row stride ld as boxes of 64 dims x box_heads x
// box_rows, 128B-swizzled; out of range reads as zero.
bool pk_encode(CUtensorMap* map, const __nv_bfloat16* x, int D, int heads, int rows, int ld,
               int box_heads, int box_rows)
{
  if (g_pk_encode == nullptr) {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult qr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &qr) !=
            cudaSuccess ||
        fn == nullptr)
      return false;
    g_pk_encode = reinterpret_cast<PFN_encodeTiled>(fn);
  }
  const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)heads, (cuuint64_t)rows};
  const cuuint64_t strides[2] = {(cuuint64_t)D * 2, (cuuint64_t)ld * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)box_heads, (cuuint32_t)box_rows};
  const cuuint32_t estr[3] = {1, 1, 1};
  return g_pk_encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<__nv_bfloat16*>(x), dims,
                     strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                     CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

constexpr long long kOrderBytes = 96ll << 20;    // keys and values that stay in L2 (126 MB)

// The items of a call, and `count` of them from `base` on as one grid.
template <int D, bool NARROW>
long long pk_items(const PackedAttention& a)
{
  return (long long)slot_count(a.rows, a.seqs,
                               PkCfg<D, NARROW>::kTiles * (kRows / (a.heads / a.kv_heads)), 1) *
         a.kv_heads;
}

template <int D, bool NARROW, bool SPLIT>
int pk_launch(const PackedAttention& a, int num_sms, long long base, long long count, int split,
              int* err, cudaStream_t s)
{
  using C = PkCfg<D, NARROW>;
  PkParams p;
  memset(&p, 0, sizeof(p));
  p.q = a.q;
  p.k = a.k;
  p.v = a.v;
  p.o = a.o;
  p.ldq = a.ldq;
  p.ldk = a.ldk;
  p.ldv = a.ldv;
  p.ldo = a.ldo;
  p.cu_q = a.cu_q;
  p.cu_k = a.cu_k;
  p.seqs = a.seqs;
  p.rows = a.rows;
  p.keys = a.keys;
  p.kv_heads = a.kv_heads;
  p.group = a.heads / a.kv_heads;
  p.tq = kRows / p.group;
  p.causal = a.causal;
  p.window = a.window;
  p.c = a.scale * 1.4426950408889634f;
  p.err = err;
  CUtensorMap mq, mk, mv;
  // no keys at all: every row is empty and nothing loads through mk and mv, which
  // describe q then (k and v may be anything, and so may their strides)
  const bool none = a.keys == 0;
  if (!pk_encode(&mq, a.q, D, a.heads, a.rows, a.ldq, p.group, p.tq) ||
      !pk_encode(&mk, none ? a.q : a.k, D, a.kv_heads, none ? 1 : a.keys, none ? a.ldq : a.ldk, 1,
                 C::kKeys) ||
      !pk_encode(&mv, none ? a.q : a.v, D, a.kv_heads, none ? 1 : a.keys, none ? a.ldq : a.ldv, 1,
                 C::kVKeys))
    return -1;
  if (base + count > INT_MAX || count * split > INT_MAX) return -2;
  p.by_reach = a.seqs > 1 && a.seqs <= 32 && pk_items<D, NARROW>(a) > num_sms &&
               (D == 64 || (long long)a.keys * a.kv_heads * (D * 4) <= kOrderBytes);
  static std::atomic<unsigned long long> attr{0};
  if (!smem_limit_once(pk_attention_kernel<D, NARROW, SPLIT>, C::kSmem, attr)) return -1;
  p.base = (int)base;
  p.split = split;
  launch_k(pk_attention_kernel<D, NARROW, SPLIT>, dim3((unsigned)(count * split)), dim3(C::kThreads),
           C::kSmem, s, split, mq, mk, mv, p);
  return launched();
}

// Clusters of n CTAs that the current device holds at once (0: none), asked once.
template <int D, bool NARROW>
int pk_clusters(int n)
{
  using C = PkCfg<D, NARROW>;
  static std::atomic<int> known[64][kMaxSplit + 1];    // count + 1
  static std::atomic<unsigned long long> attr{0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  int have = known[dev][n].load(std::memory_order_relaxed);
  if (have == 0) {
    if (!smem_limit_once(pk_attention_kernel<D, NARROW, true>, C::kSmem, attr)) return 0;
    cudaLaunchAttribute size;
    size.id = cudaLaunchAttributeClusterDimension;
    size.val.clusterDim.x = (unsigned)n;
    size.val.clusterDim.y = size.val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)n);
    cfg.blockDim = dim3(C::kThreads);
    cfg.dynamicSmemBytes = C::kSmem;
    cfg.attrs = &size;
    cfg.numAttrs = 1;
    int count = 0;
    if (cudaOccupancyMaxActiveClusters(&count, pk_attention_kernel<D, NARROW, true>, &cfg) !=
        cudaSuccess) {
      cudaGetLastError();
      count = 0;
    }
    have = count + 1;
    known[dev][n].store(have, std::memory_order_relaxed);
  }
  return have - 1;
}

// CTAs an item: where the items alone leave SMs idle and the keys are long, clusters
// share them.  Measured: a key tile takes kStep us, the join kJoin, and a further
// round of clusters, which start anew, 12 (a CTA on its own goes on to its next item).
// 32/8 heads of 128, one sequence, us (alone / by the rule):
//   new tokens, keys before      500           2000          8000          32000
//   16                        9.6 /  8.6   19.1 /  9.8   56.1 / 15.9   204.3 / 35.6
//   64                       11.1 / 10.7   19.8 / 12.4   58.0 / 23.1   206.7 / 61.8
// and, 16 tokens, 32/8 heads of 64:
//                            12.3 /  9.4   33.8 / 11.9    116 / 21.7     449 / 60.8
// 16/8 heads of 256:         12.0 / 12.0   27.7 / 11.2   89.0 / 20.6     333 / 52.8
// (kStep is a whole item's; at width 64 one with few rows, one query tile of four,
// takes less: 115 us for the 8000 keys against 136 for 64 tokens.)
template <int D, bool NARROW>
int pk_split(long long items, float alone, float start, int num_sms)
{
  constexpr float kJoin = D == 64 ? 4.3f : D == 128 ? 2.5f : 6.3f, kRound = 12.0f;
  float best = 0.95f * (float)((items + num_sms - 1) / num_sms) * alone;
  int split = 1;
  for (int n = 2; n <= kMaxSplit && start + kJoin + alone / (float)n < best; n *= 2) {
    const int fit = pk_clusters<D, NARROW>(n);
    if (fit <= 0) break;
    const float rounds = (float)((items + fit - 1) / fit);
    const float t = start + kJoin + rounds * alone / (float)n + (rounds - 1.0f) * kRound;
    if (t < best) {
      best = t;
      split = n;
    }
  }
  return split;
}

template <int D, bool NARROW>
int pk_form(const PackedAttention& a, int num_sms, int* err, cudaStream_t s)
{
  constexpr float kStep = D == 128 ? 0.82f : 1.33f;
  constexpr float kStart = 8.0f;                       // us of a second launch
  float keys = (float)a.keys / (float)a.seqs;
  if (a.window > 0) keys = fminf(keys, (float)a.window + (float)kRows);
  const float alone = keys / (float)PkCfg<D, NARROW>::kKeys * kStep;      // us an item
  const long long items = pk_items<D, NARROW>(a);
  int split = pk_split<D, NARROW>(items, alone, 0.0f, num_sms);
  if (split > 1) return pk_launch<D, NARROW, true>(a, num_sms, 0, items, split, err, s);
  // items of about the same length that end in a round of few: these by clusters, in a
  // launch of their own (2 chunks of 333 to 777 tokens on 6990, 20/4 heads of 128: 92
  // against 101 us; 1200 tokens on 8000, 16/4 heads: 86 against 122)
  const long long last = items % num_sms;
  if (items > num_sms && last > 0 && (long long)a.rows * 2 <= a.keys) {
    split = pk_split<D, NARROW>(last, alone, kStart, num_sms);
    if (split > 1) {
      const int rc = pk_launch<D, NARROW, false>(a, num_sms, 0, items - last, 1, err, s);
      return rc != 0 ? rc
                     : pk_launch<D, NARROW, true>(a, num_sms, items - last, last, split, err, s);
    }
  }
  return pk_launch<D, NARROW, false>(a, num_sms, 0, items, 1, err, s);
}

}  // namespace

int launch_attention_packed(const PackedAttention& a, int num_sms, int* err, cudaStream_t s)
{
  switch (a.head_dim) {
    case 64: return pk_form<64, false>(a, num_sms, err, s);
    case 128: {
      const long long wide = pk_items<128, false>(a);
      return wide <= num_sms ? pk_form<128, true>(a, num_sms, err, s)
                             : pk_launch<128, false, false>(a, num_sms, 0, wide, 1, err, s);
    }
    case 256: return pk_form<256, false>(a, num_sms, err, s);
    default: return -2;
  }
}

}  // namespace ltx
