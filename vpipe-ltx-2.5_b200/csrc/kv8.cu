// kv8.cu -- the 8-bit key/value cache: append, read back, attention over it.
//
// A cache is pages of 64 tokens: int8 codes [pages][kv_heads][64][D] and one
// bf16 scale for each page and head, for keys and for values.  Token t of a
// sequence is slot t % 64 of page table[t / 64].  A code c stands for c * s.
//
// The scale has 8 significant bits so that every decision here is exact.  An
// appended value x (8 bits too) gets the code rint(x / s); the quotient of two
// 8-bit numbers is either a half-integer exactly or at least 2^-9 away from
// one (the difference is a multiple of 1 / (2 s's integer)), so f32 decides it
// as real numbers would.
#include <cfloat>
#include <climits>
#include <cstring>

#include <cuda_fp16.h>

#include "attention_tc.cuh"
#include "block_ops.h"
#include "kernels.h"
#include "packed_index.h"
#include "packed_seq.cuh"
#include "ptx.cuh"

namespace ltx {

namespace {

enum : int {
  KERR_PLACE = 0x69,              // a start, length or page outside the cache
};

__device__ __forceinline__ float bf16_bits(uint32_t b) { return __uint_as_float(b << 16); }

// The smallest bf16 s with 127 s >= most (bits of a finite bf16 >= 0).
// 127 * s has 15 significant bits: exact in f32.
__device__ __forceinline__ uint32_t page_scale(uint32_t most_bits)
{
  const float most = bf16_bits(most_bits);
  uint32_t s = __float_as_uint(__fdiv_rn(most, 127.0f)) >> 16;
  if (127.0f * bf16_bits(s) < most) ++s;
  return s;
}

// ---- append and read back ------------------------------------------------

struct KvPages {
  int8_t *k, *v;
  uint16_t *ks, *vs;
  const int* table;
  const int* starts;
  const int* cu;
  int table_ld, pages, kv_heads, seqs, rows;
  int* err;
};

// A run of new tokens on one page.
struct KvSpan {
  int seq, row, block;            // sequence, packed row of the first token, its page's place
  int from, count;                // slot of the first token, tokens
};

// The tokens of the page that work slot `slot` covers; count 0 where it has none.
// Whole warps call it.  Up to 32 sequences each lane looks at one, so that one
// round of loads answers.
__device__ __forceinline__ KvSpan kv_span(const KvPages& p, int slot)
{
  KvSpan w;
  int s, row0, end, start;
  if (p.seqs <= 32) {
    const int lane = (int)lane_id();
    int a = 0, b = 0, c = 0;
    if (lane < p.seqs) {
      a = p.cu[lane];
      b = p.cu[lane + 1];
      c = p.starts[lane];
    }
    a = clamp_int(a, 0, p.rows);
    const bool below = lane == 0 || (lane < p.seqs && slot_base(a, lane, kPage, 2) <= slot);
    s = 31 - __clz((int)__ballot_sync(0xffffffffu, below));
    row0 = __shfl_sync(0xffffffffu, a, s);
    end = __shfl_sync(0xffffffffu, b, s);
    start = __shfl_sync(0xffffffffu, c, s);
  } else {
    s = find_seq(p.cu, p.seqs, p.rows, kPage, 2, slot);
    row0 = clamp_int(p.cu[s], 0, p.rows);
    end = p.cu[s + 1];
    start = p.starts[s];
  }
  const int n = clamp_int(end, row0, p.rows) - row0;
  const int i = slot - slot_base(row0, s, kPage, 2);
  w.seq = s;
  w.count = 0;
  if (n == 0 || i < 0) return w;
  if (!span_ok(start, n, p.table_ld * kPage)) {
    if (threadIdx.x == 0) atomicCAS(p.err, 0, KERR_PLACE);
    return w;
  }
  const PageSpan span = page_span(start, n, i);
  w.block = span.block;
  w.row = row0 + (span.a - start);
  w.from = span.a - span.block * kPage;
  w.count = max(0, span.b - span.a);
  return w;
}

// The span's page, or -1 where the table names none.
__device__ __forceinline__ int kv_page(const KvPages& p, const KvSpan& w)
{
  const int page = p.table[(size_t)w.seq * p.table_ld + w.block];
  if (page_ok(page, p.pages)) return page;
  if ((threadIdx.x & 31) == 0) atomicCAS(p.err, 0, KERR_PLACE);
  return -1;
}

__device__ __forceinline__ uint32_t max_bits(uint4 v)
{
  const uint32_t a = __vmaxu2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu);
  const uint32_t b = __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu);
  return __vmaxu2(a, b);
}

// The scale of a page and head once values of magnitude `most` join it.  bf16
// magnitudes order like their bits; a NaN or infinity is above 0x7f7f and makes the
// scale NaN.
__device__ __forceinline__ uint32_t joined_scale(uint32_t most, uint32_t was, bool held)
{
  const uint32_t now = most > 0x7f7fu ? 0x7fc0u : page_scale(most);
  return held ? max(now, was) : now;
}

// The page's own codes, brought to a grown scale: c * was / now, a quotient of 15
// by 8 bits, decided by the correctly rounded f32 division.  Each growth rounds them
// anew.  A page of 64 normal values a column filled token by token is off by 0.38 of
// its scale rms (2.1 at most of 64k values), filled at once by 0.29 (0.5); where the
// values grow threefold along the page by 0.57 (2.7), 64-fold by 0.71 (2.2).
__device__ __forceinline__ void rescale_codes(int8_t* codes, int count4, uint32_t was, uint32_t now,
                                              int at, int step)
{
  const float s0 = bf16_bits(was), s1 = bf16_bits(now);
  for (int i = at; i < count4; i += step) {
    char4 c = reinterpret_cast<char4*>(codes)[i];
    c.x = (signed char)__float2int_rn(__fdiv_rn((float)c.x * s0, s1));
    c.y = (signed char)__float2int_rn(__fdiv_rn((float)c.y * s0, s1));
    c.z = (signed char)__float2int_rn(__fdiv_rn((float)c.z * s0, s1));
    c.w = (signed char)__float2int_rn(__fdiv_rn((float)c.w * s0, s1));
    reinterpret_cast<char4*>(codes)[i] = c;
  }
}

__device__ __forceinline__ unsigned long long fmul2(unsigned long long a, unsigned long long b)
{
  unsigned long long d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// x / s to the nearest integer, ties to even, for the bf16 values x and scale s:
//   t = x / s by one product with 1 / s, within 2^-15 of the quotient;
//   adding 1.5 * 2^12 rounds it to a multiple of 2^-11, which puts a tie back on
//   the tie and leaves all others on their side (2^-9);
//   adding 1.5 * 2^23 - 1.5 * 2^12 rounds to the nearest integer, ties to even,
//   and leaves the code in the sum's low byte.
// Two values at a time (a value at a time, with the two last additions apart and the
// old scale read for new pages too, 90 MB of prompts took 25 us, now 18).  1 / s may
// not be finite for a tiny s: x goes through 2^64 / (2^64 s) there.
struct KvCoder {
  unsigned long long inv;
  float mul;                      // 1, or 2^64 ahead of inv
  __device__ __forceinline__ explicit KvCoder(uint32_t scale)
  {
    const float s = bf16_bits(scale);
    const bool none = scale > 0x7f7fu || s == 0.0f;
    mul = !none && s < 0x1p-64f ? 0x1p64f : 1.0f;
    const uint32_t i = __float_as_uint(none ? 0.0f : __frcp_rn(s * mul));
    inv = pair2(i, i);
  }
  // the codes of a word's two values in the low bytes of two words
  __device__ __forceinline__ unsigned long long two(uint32_t w) const
  {
    uint32_t a = w << 16, b = w & 0xffff0000u;
    if (mul != 1.0f) {
      a = __float_as_uint(__uint_as_float(a) * mul);
      b = __float_as_uint(__uint_as_float(b) * mul);
    }
    unsigned long long t = fmul2(pair2(a, b), inv);
    t = fadd2(t, pair2(0x45c00000u, 0x45c00000u));           // 6144
    return fadd2(t, pair2(0x4b3fe800u, 0x4b3fe800u));        // 12582912 - 6144
  }
  __device__ __forceinline__ uint32_t four(uint32_t a, uint32_t b) const
  {
    const unsigned long long c = two(a), d = two(b);
    return __byte_perm(__byte_perm((uint32_t)c, (uint32_t)(c >> 32), 0x0040),
                       __byte_perm((uint32_t)d, (uint32_t)(d >> 32), 0x0040), 0x5410);
  }
  __device__ __forceinline__ uint2 eight(uint4 v) const
  {
    return make_uint2(four(v.x, v.y), four(v.z, v.w));
  }
};

constexpr int kAppendThreads = 256;

// Many rows: one page, one head, keys (blockIdx.z 0) or values (1) a block.  The new
// rows stay in registers between the search for their maximum and their rounding,
// so they are read once; they are on their way before the page is known.
template <int D>
__global__ void __launch_bounds__(kAppendThreads)
    kv8_append_kernel(KvPages p, const __nv_bfloat16* k, int ldk, const __nv_bfloat16* v, int ldv)
{
  constexpr int kChunks = D / 8;                       // 16-byte pieces of a row
  constexpr int kRowsAt = kAppendThreads / kChunks;    // rows a pass
  constexpr int kPasses = kPage / kRowsAt;
  __shared__ uint32_t s_most[kAppendThreads / 32];
  pdl_wait();
  pdl_trigger();
  // heads of a page are neighbours in the grid, as their columns are in a row
  const int head = (int)(blockIdx.x % (unsigned)p.kv_heads);
  const KvSpan w = kv_span(p, (int)(blockIdx.x / (unsigned)p.kv_heads));
  if (w.count == 0) return;
  const bool val = blockIdx.z != 0;
  const __nv_bfloat16* x = val ? v : k;
  const int ld = val ? ldv : ldk;
  const int chunk = (int)threadIdx.x % kChunks, r0 = (int)threadIdx.x / kChunks;
  uint4 in[kPasses];
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    const int r = r0 + i * kRowsAt;
    in[i] = make_uint4(0, 0, 0, 0);
    if (r < w.count)
      in[i] = *reinterpret_cast<const uint4*>(x + (size_t)(w.row + r) * ld +
                                              (size_t)head * D + chunk * 8);
  }
  const int page = kv_page(p, w);
  if (page < 0) return;
  const size_t line = (size_t)page * p.kv_heads + head;
  int8_t* codes = (val ? p.v : p.k) + line * (size_t)(kPage * D);
  uint16_t* scale = (val ? p.vs : p.ks) + line;
  const uint32_t was = w.from > 0 ? *scale : 0u;       // of no use on a new page
  uint32_t most = 0;
#pragma unroll
  for (int i = 0; i < kPasses; ++i) most = __vmaxu2(most, max_bits(in[i]));
  most = max(most & 0xffffu, most >> 16);
  most = __reduce_max_sync(0xffffffffu, most);
  if ((threadIdx.x & 31) == 0) s_most[threadIdx.x >> 5] = most;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kAppendThreads / 32; ++i) most = max(most, s_most[i]);
  const uint32_t now = joined_scale(most, was, w.from > 0);
  if (w.from > 0 && now != was && now <= 0x7f7fu)
    rescale_codes(codes, w.from * (D / 4), was, now, (int)threadIdx.x, kAppendThreads);
  if (threadIdx.x == 0 && (w.from == 0 || now != was)) *scale = (uint16_t)now;
  const KvCoder coder(now);
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    const int r = r0 + i * kRowsAt;
    if (r >= w.count) break;
    *reinterpret_cast<uint2*>(codes + (size_t)(w.from + r) * D + chunk * 8) =
        now > 0x7f7fu ? make_uint2(0, 0) : coder.eight(in[i]);
  }
}

// Few rows (a token for each sequence): a block a page, a warp for each head's keys
// or values by turns.
template <int D>
__global__ void __launch_bounds__(kAppendThreads)
    kv8_append_few_kernel(KvPages p, const __nv_bfloat16* k, int ldk, const __nv_bfloat16* v,
                          int ldv)
{
  constexpr int kChunks = D / 8, kRowsAt = 32 / kChunks;
  pdl_wait();
  pdl_trigger();
  const KvSpan w = kv_span(p, (int)blockIdx.x);
  if (w.count == 0) return;
  const int lane = (int)threadIdx.x & 31, warp = (int)threadIdx.x >> 5;
  const int chunk = lane % kChunks, r0 = lane / kChunks;
  int page = -2;
  for (int i = warp; i < 2 * p.kv_heads; i += kAppendThreads / 32) {
    const bool val = i >= p.kv_heads;
    const int head = val ? i - p.kv_heads : i;
    const __nv_bfloat16* x = (val ? v : k) + (size_t)w.row * (val ? ldv : ldk) + (size_t)head * D +
                             chunk * 8;
    const int ld = val ? ldv : ldk;
    uint4 first = make_uint4(0, 0, 0, 0);
    if (r0 < w.count) first = *reinterpret_cast<const uint4*>(x + (size_t)r0 * ld);
    if (page == -2) page = kv_page(p, w);
    if (page < 0) return;
    const size_t line = (size_t)page * p.kv_heads + head;
    int8_t* codes = (val ? p.v : p.k) + line * (size_t)(kPage * D);
    uint16_t* scale = (val ? p.vs : p.ks) + line;
    const uint32_t was = *scale;
    uint32_t most = max_bits(first);
    for (int r = r0 + kRowsAt; r < w.count; r += kRowsAt)
      most = __vmaxu2(most, max_bits(*reinterpret_cast<const uint4*>(x + (size_t)r * ld)));
    most = max(most & 0xffffu, most >> 16);
    most = __reduce_max_sync(0xffffffffu, most);
    const uint32_t now = joined_scale(most, was, w.from > 0);
    if (w.from > 0 && now != was && now <= 0x7f7fu)
      rescale_codes(codes, w.from * (D / 4), was, now, lane, 32);
    __syncwarp();                                      // all have read `was`
    if (lane == 0 && (w.from == 0 || now != was)) *scale = (uint16_t)now;
    const KvCoder coder(now);
    for (int r = r0; r < w.count; r += kRowsAt) {
      const uint4 in = r == r0 ? first : *reinterpret_cast<const uint4*>(x + (size_t)r * ld);
      *reinterpret_cast<uint2*>(codes + (size_t)(w.from + r) * D + chunk * 8) =
          now > 0x7f7fu ? make_uint2(0, 0) : coder.eight(in);
    }
  }
}

// Rows of a cache back as bf16: bf16(c * s).  Eight codes a lane at a time, so that a
// warp stores 512 adjacent bytes: 13.8 us for 90 MB (6.5 TB/s), 19.7 with sixteen
// codes and every other 16 bytes a store.
template <int D>
__global__ void __launch_bounds__(kAppendThreads)
    kv8_read_kernel(KvPages p, __nv_bfloat16* k, int ldk, __nv_bfloat16* v, int ldv)
{
  constexpr int kChunks = D / 8, kMost = kPage * kChunks / kAppendThreads;
  pdl_wait();
  pdl_trigger();
  const int head = (int)(blockIdx.x % (unsigned)p.kv_heads);
  const KvSpan w = kv_span(p, (int)(blockIdx.x / (unsigned)p.kv_heads));
  if (w.count == 0) return;
  const int page = kv_page(p, w);
  if (page < 0) return;
  const bool val = blockIdx.z != 0;
  __nv_bfloat16* x = val ? v : k;
  const int ld = val ? ldv : ldk;
  const size_t line = (size_t)page * p.kv_heads + head;
  const int8_t* codes = (val ? p.v : p.k) + line * (size_t)(kPage * D) + (size_t)w.from * D;
  const float s = bf16_bits((val ? p.vs : p.ks)[line]);
  uint2 c[kMost];
#pragma unroll
  for (int j = 0; j < kMost; ++j) {
    const int i = (int)threadIdx.x + j * kAppendThreads;
    if (i < w.count * kChunks) c[j] = reinterpret_cast<const uint2*>(codes)[i];
  }
#pragma unroll
  for (int j = 0; j < kMost; ++j) {
    const int i = (int)threadIdx.x + j * kAppendThreads;
    if (i >= w.count * kChunks) break;
    const uint32_t words[2] = {c[j].x, c[j].y};
    uint32_t o[4];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const char4 b = *reinterpret_cast<const char4*>(&words[e]);
      o[2 * e] = pack_bf16((float)b.x * s, (float)b.y * s);
      o[2 * e + 1] = pack_bf16((float)b.z * s, (float)b.w * s);
    }
    uint4* dst = reinterpret_cast<uint4*>(x + (size_t)(w.row + i / kChunks) * ld +
                                          (size_t)head * D + (i % kChunks) * 8);
    *dst = make_uint4(o[0], o[1], o[2], o[3]);
  }
}

// ---- attention over the cache ----------------------------------------------
//
// The new rows of a sequence (n tokens, the last n of its `length`) times the
// G query heads of a key/value head are rows token * G + head, in tiles of 8
// or 16.  The work is the list of all (sequence, kv head, row tile, 8 KB stage
// of keys and values) in that order, and every warp of the grid takes an equal
// run of it, whatever the lengths, and works on it alone: no barrier, no shared
// result.  A tile that one warp has whole goes straight to o; of the others
// (a warp's first and last, at most) each part goes to the workspace as (max,
// sum, O) for kv8_merge_kernel.  Measured beside this on 64 ragged sequences
// and on 32 of one-row tiles (8192 and 4096 tokens at most): runs shared by a
// block's four warps with a join in shared memory, and parts joined by the last
// block to arrive, which saves the second launch: 104 and 53 us against 91 and 34,
// the difference spent at barriers, fences and counters in the middle of a run.
// Few short tiles are a block's each instead, in one launch (kv_attn_launch).
//
// This reads 2 D bytes a token and key head and is bound by HBM as long as a
// code costs few instructions.  The products run transposed, S^T = K Q^T and
// O^T = V^T P^T, on warp MMAs with f32 sums (m16n8k16, f16 operands): 16 keys or
// 16 output columns by 8 query rows, since a decoded token has no more rows than
// query heads share a key head.  Against 16 query rows in the M place that halves
// the MMAs, the exponentials and the registers.  f16 is what the MMA takes beside the
// codes: P rounds at 2^-11, under the result's own bf16 rounding of 2^-8 (against 64
// bits normal values are off by 0.00165 rms, the f32 form by the same); q's 8 bits are
// exact once its row is brought near 2^8 by a power of two.  Measured on 131072
// tokens, 8 key heads of 128 under 4 query heads each: 48.8 us for 268 MB (5.5 TB/s),
// 739 warp instructions a stage (903 that way), 55 % of the issue slots, tensor pipe
// 19 %.  5 us of it are the start (offsets, pages, then keys wait for one another); the
// rest is HBM at 6.1 TB/s.
//   K  byte 128 + c in the low half of an f16 is the subnormal (128 + c) 2^-24:
//      one byte permute a pair, and 128 sum(q) leaves the score with the
//      exponent's other constants.
//   V  the pair becomes 1024 + 128 + c by a permute, and c by one packed
//      subtraction (exact): here 128 sum(P) would swamp the f32 sums.
//   P  leaves S^T's accumulators key by lane group and enters the second product
//      row by lane group: one 8x8 transposition a 16-bit register.
// K's scale goes into the exponent's factor, V's as a power of two into P's
// exponent, so neither costs an instruction a score.
//
// Each warp streams its stages through a ring of its own, keys and values in
// turn, two stages ahead, with 16-byte asynchronous copies (no barrier between
// warps before a tile ends).  Shared memory is swizzled by 16-byte pieces so
// that the fragment reads below are free of conflicts: eight keys for K, pairs
// of keys for V.

template <int D, int NR>
struct KvCfg {
  static constexpr int kTok = 4096 / D;                // tokens of a stage
  // warps of the block that has an SM to itself: as many as the registers allow
  static constexpr int kWarps = D == 256 || NR == 2 ? 8 : 12;
  static constexpr int kThreads = kWarps * 32;
  static constexpr int kStageBytes = 8192;             // K, then V
  static constexpr int kSmem = kWarps * 2 * kStageBytes;
  static constexpr int kMT = kTok / 16;                // key tiles of a stage
  static constexpr int kOT = D / 16;                   // output column tiles
};

constexpr float kKvGrow = 6.0f;   // log2 of the largest P before O is rescaled

struct KvAttn {
  const int8_t *k, *v;
  const uint16_t *ks, *vs;
  const __nv_bfloat16* q;
  __nv_bfloat16* o;
  int ldq, ldo;
  const int *cu, *lengths, *table;
  int table_ld, pages, kv_heads, group, seqs, rows, window;
  float c;                        // scale log2 e
  int workers;                    // warps of the attention grid
  float* part_o;                  // [workers][2][tile rows][D]
  float* part_ml;                 // [workers][2][tile rows][2]
  int* err;
};

// What one sequence asks for.
struct KvSeq {
  int row0, n, len;               // its new rows, its length
  int tiles, first, units;        // row tiles; first stage and stages of each
};

template <int D, int TR>
__device__ __forceinline__ KvSeq kv_seq(const KvAttn& p, int s)
{
  constexpr int T = 4096 / D;                          // tokens of a stage
  KvSeq q;
  q.row0 = clamp_int(p.cu[s], 0, p.rows);
  q.n = clamp_int(p.cu[s + 1], q.row0, p.rows) - q.row0;
  const int len = p.lengths[s], cap = p.table_ld * kPage;
  q.len = clamp_int(len, 0, cap);
  if (len != q.len) atomicCAS(p.err, 0, KERR_PLACE);
  q.tiles = (q.n * p.group + TR - 1) / TR;
  const int lo = key_low(q.len - q.n, p.window);
  q.first = lo / T;
  q.units = q.len > lo ? (q.len + T - 1) / T - q.first : 0;
  return q;
}

__device__ __forceinline__ u64 kv_work(const KvAttn& p, const KvSeq& q)
{
  return (u64)q.tiles * (u64)p.kv_heads * (u64)q.units;
}

// Warps that share `all` stages: one at least for each.
__device__ __forceinline__ u64 kv_workers(const KvAttn& p, u64 all)
{
  return min((u64)p.workers, all);
}

// All sequences of a call as the first N threads of a block see them: the work
// before each thread's run of them (`each` from threadIdx * each on) and, where a
// thread has one at most, what they ask for.
template <int N>
struct KvTable {
  u64 before[N + 1];
  u64 warp_sum[N / 32];
  KvSeq q[N];
};

// Fills it; every thread of the block calls this.
template <int D, int TR, int N>
__device__ __forceinline__ void kv_scan(const KvAttn& p, KvTable<N>& tab)
{
  const int each = (p.seqs + N - 1) / N;
  const int t = (int)threadIdx.x, lane = t & 31;
  u64 mine = 0;
  for (int i = 0; t < N && i < each; ++i) {
    const int s = t * each + i;
    if (s >= p.seqs) break;
    const KvSeq q = kv_seq<D, TR>(p, s);
    if (each == 1) tab.q[t] = q;
    mine += kv_work(p, q);
  }
  u64 sum = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const u64 o = __shfl_up_sync(0xffffffffu, sum, d);
    if (lane >= d) sum += o;
  }
  if (lane == 31 && t < N) tab.warp_sum[t >> 5] = sum;
  __syncthreads();
  u64 earlier = 0;
#pragma unroll
  for (int w = 0; w < N / 32; ++w)
    if (w < (t >> 5)) earlier += tab.warp_sum[w];
  if (t < N) tab.before[t] = earlier + sum - mine;
  if (t == N - 1) tab.before[N] = earlier + sum;
  __syncthreads();
}

template <int D, int TR, int N>
__device__ __forceinline__ KvSeq kv_get(const KvAttn& p, const KvTable<N>& tab, int s)
{
  return p.seqs <= N ? tab.q[s] : kv_seq<D, TR>(p, s);
}

// A place in the list of work.
struct KvPlace {
  KvSeq q;
  int s, head, tile, unit;
};

// The place of stage x.
template <int D, int TR, int N>
__device__ __forceinline__ KvPlace kv_locate(const KvAttn& p, const KvTable<N>& tab, u64 x)
{
  int lo = 0, hi = N;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (tab.before[mid] <= x) lo = mid;
    else hi = mid;
  }
  const int each = (p.seqs + N - 1) / N;
  KvPlace a;
  u64 at = tab.before[lo];
  a.s = lo * each;
  const int last = min(p.seqs, a.s + each) - 1;
  while (true) {
    a.q = kv_get<D, TR, N>(p, tab, a.s);
    const u64 w = kv_work(p, a.q);
    if (x < at + w || a.s == last) break;
    at += w;
    ++a.s;
  }
  const u64 per = (u64)a.q.tiles * (u64)a.q.units, in = x - at;
  a.head = (int)(in / per);
  a.tile = (int)(in % per / (u64)a.q.units);
  a.unit = (int)(in % per % (u64)a.q.units);
  return a;
}

// k stages on (k at most what is left of the tile); past the list's end s
// reaches seqs.
template <int D, int TR, int N>
__device__ __forceinline__ void kv_move(const KvAttn& p, const KvTable<N>& tab, KvPlace& a, int k)
{
  a.unit += k;
  if (a.unit < a.q.units) return;
  a.unit = 0;
  if (++a.tile < a.q.tiles) return;
  a.tile = 0;
  if (++a.head < p.kv_heads) return;
  a.head = 0;
  do {
    if (++a.s >= p.seqs) return;
    a.q = kv_get<D, TR, N>(p, tab, a.s);
  } while (kv_work(p, a.q) == 0);
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src)
{
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit()
{
  asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void cp_async_wait()
{
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Offset of 16-byte piece ch of row r in a stage's K or V.
template <int D, bool V>
__device__ __forceinline__ uint32_t kv_place(int r, int ch)
{
  if constexpr (D == 64) {
    const int piece = ((r & 1) * 4 + ch) ^ (((r >> 1) & 3) * 2);
    return (uint32_t)((r >> 1) * 128 + piece * 16);
  } else {
    const int flip = V ? ((r >> 1) & 3) * 2 : (r & 1) * 4;
    return (uint32_t)(r * D + (ch & ~7) * 16 + ((ch & 7) ^ flip) * 16);
  }
}

__device__ __forceinline__ uint4 lds128(const uint8_t* a)
{
  return *reinterpret_cast<const uint4*>(a);
}
__device__ __forceinline__ uint2 lds64(const uint8_t* a)
{
  return *reinterpret_cast<const uint2*>(a);
}

// A constant the compiler keeps in a register.
__device__ __forceinline__ uint32_t held(uint32_t v)
{
  uint32_t r;
  asm volatile("mov.b32 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// Bytes 0, 1 (hi = false) or 2, 3 of w, each u = 128 + c, as the f16 pair u 2^-24.
__device__ __forceinline__ uint32_t f16_tiny(uint32_t w, bool hi)
{
  return __byte_perm(w, 0u, hi ? 0x4342 : 0x4140);
}
// The same bytes as the f16 pair c; k64 holds 0x64646464.
__device__ __forceinline__ uint32_t f16_pair(uint32_t w, uint32_t k64, bool hi)
{
  const uint32_t u = __byte_perm(w, k64, hi ? 0x4342 : 0x4140);           // 1024 + 128 + c
  uint32_t r;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(u), "r"(0x64806480u));   // 1152
  return r;
}

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                        uint32_t a3, uint32_t b0, uint32_t b1)
{
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi)
{
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// Rows and columns of an 8x8 matrix of 16-bit values, a pair a lane, exchanged.
__device__ __forceinline__ uint32_t transpose8(uint32_t v)
{
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// The factor of a part (max m, sum l) under the joint maximum: a part that saw
// nothing has sum 0 and O 0.
__device__ __forceinline__ float kv_weight(float m, float l, float top)
{
  return m == -INFINITY ? (l == 0.0f ? 0.0f : 1.0f) : fast_exp2(m - top);
}

// One row of a tile out of f32: columns 2 (32 e + lane) and the next of this lane.  A
// row that met no key, because it sees none or their pages are not there, has the sum
// 0 (else its largest weight alone makes 1, or the sum is NaN) and is zero.
template <int D>
__device__ __forceinline__ void kv_put_row(const KvAttn& p, const KvSeq& q, int head, int rt,
                                           const float2 (&acc)[D / 64], float l)
{
  const int tok = rt / p.group, lane = (int)lane_id();
  const float norm = 1.0f / l;
  __nv_bfloat16* dst = p.o + (size_t)(q.row0 + tok) * p.ldo +
                       (size_t)(head * p.group + rt % p.group) * D;
#pragma unroll
  for (int e = 0; e < D / 64; ++e)
    *reinterpret_cast<uint32_t*>(dst + (e * 32 + lane) * 2) =
        l != 0.0f ? pack_bf16(acc[e].x * norm, acc[e].y * norm) : 0u;
}

// NR: groups of 8 query rows of a tile.  TEAM: a block has a tile and its warps
// share the stages, joined in shared memory; no second launch, no workspace.
template <int D, int NR, bool TEAM>
__global__ void __launch_bounds__(KvCfg<D, NR>::kThreads, 1)
    kv8_attention_kernel(const __grid_constant__ KvAttn p)
{
  using C = KvCfg<D, NR>;
  constexpr int T = C::kTok, W = C::kWarps, N = C::kThreads, TR = 8 * NR, MT = C::kMT, OT = C::kOT;
  extern __shared__ __align__(128) uint8_t smem_raw[];
  __shared__ KvTable<N> s_tab;
  __shared__ __align__(8) float s_ml[TEAM ? W : 1][TEAM ? TR : 1][2];
  static_assert(TR * D * 4 <= 2 * C::kStageBytes && W <= 32, "a part takes the place of the stages");
  const int warp = (int)threadIdx.x >> 5, lane = (int)threadIdx.x & 31;
  const int g = lane >> 2, cc = lane & 3;
  uint8_t* const mine = smem_raw + warp * 2 * C::kStageBytes;
  const uint32_t ring = smem_u32(mine);
  const uint32_t k64 = held(0x64646464u);
  // This lane's places in a stage.  Pieces swizzle by bits that only the lane
  // sets, so all of a stage is at constants from these: K row g (piece cc, and
  // 4 + cc of 8), V rows 2 cc of 16 (piece g), the pieces it copies.
  const uint32_t k_at[2] = {kv_place<D, false>(g, cc), kv_place<D, false>(g, D == 64 ? cc : 4 + cc)};
  const uint32_t v_at = kv_place<D, true>(2 * cc, D == 64 ? g >> 1 : g) +
                        (D == 64 ? (uint32_t)(g & 1) * 8u : 0u);
  const uint32_t k_to = kv_place<D, false>(lane / (D / 16), lane % (D / 16));
  const uint32_t v_to = kv_place<D, true>(lane / (D / 16), lane % (D / 16));
  pdl_wait();
  pdl_trigger();

  kv_scan<D, TR, N>(p, s_tab);
  KvPlace at;
  uint32_t count;
  size_t site = 0;                                     // of this warp's parts
  int team = 0;
  if constexpr (TEAM) {
    const int slot = (int)(blockIdx.x / (unsigned)p.kv_heads);
    int hi = p.seqs;                                   // N at most
    at.s = 0;
    while (hi - at.s > 1) {
      const int mid = (at.s + hi) / 2;
      if (slot_base(s_tab.q[mid].row0 * p.group, mid, TR, 1) <= slot) at.s = mid;
      else hi = mid;
    }
    at.q = s_tab.q[at.s];
    at.head = (int)(blockIdx.x % (unsigned)p.kv_heads);
    at.tile = slot - slot_base(at.q.row0 * p.group, at.s, TR, 1);
    if (at.tile < 0 || at.tile >= at.q.tiles) return;  // the whole block
    team = min(W, at.q.units);                         // warps with a part
    at.unit = 0;
    count = 0;
    if (warp < team) {
      at.unit = (int)work_bound((u64)at.q.units, (u64)team, (u64)warp);
      count = (uint32_t)((int)work_bound((u64)at.q.units, (u64)team, (u64)warp + 1) - at.unit);
    }
  } else {
    // this warp's run of the work; neighbours in it are on different SMs
    const u64 all = s_tab.before[N];
    const u64 workers = kv_workers(p, all);
    const u64 me = (u64)warp * gridDim.x + blockIdx.x;
    if (me >= workers) return;
    const u64 begin = work_bound(all, workers, me);
    count = (uint32_t)(work_bound(all, workers, me + 1) - begin);
    at = kv_locate<D, TR, N>(p, s_tab, begin);
    site = me * 2 * TR;
  }

  // The loading side: the next stage, and the pages of 32 blocks of its
  // sequence, one a lane.  Scales arrive in registers two stages ahead of their
  // use (a page that is not there is marked by an impossible one).
  KvPlace ld = at;
  uint32_t loaded = 0;
  int c_s = -1, c_group = 0, c_page = -1;
  const int8_t* v_src = nullptr;                       // values of the stage begun
  uint32_t ks_next[2], vs_next[2];
  auto load_k = [&](int stage, uint32_t& ks, uint32_t& vs) {
    v_src = nullptr;
    ks = 0xbf80u;                                      // -1
    vs = 0;
    if (loaded < count) {
      const int tok = (ld.q.first + ld.unit) * T;
      const int block = tok / kPage, group = block & ~31;
      if (ld.s != c_s || group != c_group) {
        c_s = ld.s;
        c_group = group;
        c_page = -1;
        if ((group + lane) * kPage < ld.q.len) {
          c_page = p.table[(size_t)ld.s * p.table_ld + group + lane];
          if (!page_ok(c_page, p.pages)) {
            atomicCAS(p.err, 0, KERR_PLACE);
            c_page = -1;
          }
        }
      }
      const int page = __shfl_sync(0xffffffffu, c_page, block - group);
      if (page >= 0) {
        const size_t line = (size_t)page * p.kv_heads + ld.head;
        const size_t off = line * (size_t)(kPage * D) + (size_t)(tok % kPage) * D +
                           (size_t)lane * 16;
        const int8_t* src = p.k + off;
        v_src = p.v + off;
        const uint32_t dst = ring + (uint32_t)(stage * C::kStageBytes) + k_to;
        // piece i * 32 + lane: row i * (512 / D) further
#pragma unroll
        for (int i = 0; i < 8; ++i) cp_async16(dst + i * 512, src + i * 512);
        ks = p.ks[line];
        vs = p.vs[line];
      }
      if (++loaded < count) kv_move<D, TR, N>(p, s_tab, ld, 1);
    }
    cp_async_commit();
  };
  auto load_v = [&](int stage) {
    if (v_src != nullptr) {
      const uint32_t dst = ring + (uint32_t)(stage * C::kStageBytes) + 4096u;
      // the flip of V's rows moves with i
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t flip = D == 64 ? 0u : D == 128 ? (uint32_t)(i & 1) * 64u
                                                      : (uint32_t)(i & 3) * 32u;
        cp_async16(dst + (v_to ^ flip) + i * 512, v_src + i * 512);
      }
    }
    cp_async_commit();
  };
  // queries of a tile as they lie: row g of each group of 8, 16 of every 64
  // columns; rows past the tile's last are zeros, computed and never stored
  uint4 raw[NR][D / 64][2];
  auto fetch_q = [&]() {
    const int row0 = at.tile * TR, rows = min(TR, at.q.n * p.group - row0);
#pragma unroll
    for (int h = 0; h < NR; ++h) {
      const int r = g + 8 * h;
      const int tok = (row0 + r) / p.group, head = at.head * p.group + (row0 + r) % p.group;
      const __nv_bfloat16* q = p.q + (size_t)(at.q.row0 + tok) * p.ldq + (size_t)head * D;
#pragma unroll
      for (int j = 0; j < D / 64; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          raw[h][j][i] = make_uint4(0, 0, 0, 0);
          if (r < rows) raw[h][j][i] = *reinterpret_cast<const uint4*>(q + j * 64 + cc * 16 + i * 8);
        }
    }
  };
  fetch_q();                                           // ahead of the first stages
  load_k(0, ks_next[0], vs_next[0]);
  load_v(0);
  load_k(1, ks_next[1], vs_next[1]);
  load_v(1);

  int stage = 0;
  for (uint32_t x = 0; x < count;) {
    // ---- a tile, or this warp's share of it
    const uint32_t share = min((uint32_t)(at.q.units - at.unit), count - x);
    const int row0 = at.tile * TR;
    const int rows = min(TR, at.q.n * p.group - row0);
    const int shift = at.q.len - at.q.n;
    // keys that all of its rows see
    const int all_lo = key_low(shift + (row0 + rows - 1) / p.group, p.window);
    const int all_hi = key_high(shift + row0 / p.group, at.q.len, 1);

    if (x > 0) fetch_q();
    uint32_t qf[NR][D / 16][2];
    float qs[NR][2], qb[NR][2];                        // exponent's factor, 128 sum(q) 2^-24
#pragma unroll
    for (int h = 0; h < NR; ++h) {
      uint32_t most = 0;
#pragma unroll
      for (int j = 0; j < D / 64; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint4 w = raw[h][j][i];
          const uint32_t a = __vmaxu2(w.x & 0x7fff7fffu, w.y & 0x7fff7fffu);
          const uint32_t b = __vmaxu2(w.z & 0x7fff7fffu, w.w & 0x7fff7fffu);
          most = __vmaxu2(most, __vmaxu2(a, b));
        }
      most = max(most & 0xffffu, most >> 16);
      most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
      most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
      // 2^(8 - exponent of the row's largest), 1 where that is zero or not finite
      int ex = (int)(most >> 7) - 127;
      if (most == 0 || most > 0x7f7fu) ex = 8;
      ex = max(ex, -100);
      const float up = __uint_as_float((uint32_t)(127 + 8 - ex) << 23);
      // (2^24 of K's codes comes in with K's scale, so that this stays finite)
      const float factor = p.c * __uint_as_float((uint32_t)(127 - 8 + ex) << 23);
      float sum = 0.0f;
#pragma unroll
      for (int j = 0; j < D / 64; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t words[4] = {raw[h][j][i].x, raw[h][j][i].y, raw[h][j][i].z, raw[h][j][i].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            // 8 values of half i of the lane's 16: k steps 2 i and 2 i + 1
            const uint32_t f = pack_f16(__uint_as_float(words[e] << 16) * up,
                                        __uint_as_float(words[e] & 0xffff0000u) * up);
            const float2 back = __half22float2(*reinterpret_cast<const __half2*>(&f));
            sum += back.x + back.y;
            qf[h][j * 4 + i * 2 + (e >> 1)][e & 1] = f;
          }
        }
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      // scores come to this lane for rows 2 cc and 2 cc + 1
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        qs[h][e] = __shfl_sync(0xffffffffu, factor, (2 * cc + e) * 4);
        qb[h][e] = __shfl_sync(0xffffffffu, sum, (2 * cc + e) * 4) * 7.62939453125e-6f;
      }
    }

    float o[NR][OT][4];
#pragma unroll
    for (int h = 0; h < NR; ++h)
#pragma unroll
      for (int t = 0; t < OT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[h][t][e] = 0.0f;
    float m[NR][2], l[NR][2];
#pragma unroll
    for (int h = 0; h < NR; ++h)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        m[h][e] = -INFINITY;
        l[h][e] = 0.0f;
      }
    // O is held in units of `ref`, 1/32 of a V scale met before (0: none yet), but no
    // less than `low`: 2^-64 of the largest unit so far, so that O, 2^22 units a key at
    // most in the largest, stays finite in any; and a normal number, as the divisions by
    // it require
    float ref = 0.0f, low = FLT_MIN;

    for (uint32_t u = 0; u < share; ++u) {
      const uint8_t* const kb = mine + stage * C::kStageBytes;
      const uint8_t* const vb = kb + 4096 + v_at;
      cp_async_wait<3>();
      __syncwarp();
      const float ks = bf16_bits(ks_next[0]), vs = bf16_bits(vs_next[0]);
      ks_next[0] = ks_next[1];
      vs_next[0] = vs_next[1];
      const bool there = ks != -1.0f;

      // S^T.  A key tile's steps depend on each other: kSums sums of each keep
      // four products in flight.
      constexpr int kSums = MT * NR >= 4 ? 1 : 4 / (MT * NR);
      float sc[NR][MT][kSums][4];
#pragma unroll
      for (int h = 0; h < NR; ++h)
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int k = 0; k < kSums; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[h][t][k][e] = 0.0f;
      if (there) {
#pragma unroll
        for (int j = 0; j < D / 64; ++j) {
          uint4 w0[MT], w8[MT];
#pragma unroll
          for (int t = 0; t < MT; ++t) {
            const uint8_t* row = kb + k_at[j & 1] + t * 16 * D + (j >> 1) * 128;
            w0[t] = lds128(row);
            w8[t] = lds128(row + 8 * D);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int t = 0; t < MT; ++t) {
              const uint32_t y0 = 0x80808080u ^
                  (i == 0 ? w0[t].x : i == 1 ? w0[t].y : i == 2 ? w0[t].z : w0[t].w);
              const uint32_t y8 = 0x80808080u ^
                  (i == 0 ? w8[t].x : i == 1 ? w8[t].y : i == 2 ? w8[t].z : w8[t].w);
              const uint32_t a0 = f16_tiny(y0, false), a1 = f16_tiny(y8, false);
              const uint32_t a2 = f16_tiny(y0, true), a3 = f16_tiny(y8, true);
#pragma unroll
              for (int h = 0; h < NR; ++h)
                mma_f16(sc[h][t][i % kSums], a0, a1, a2, a3, qf[h][j * 4 + i][0],
                        qf[h][j * 4 + i][1]);
            }
        }
      }
      __syncwarp();
      load_k(stage, ks_next[1], vs_next[1]);

      uint32_t pf[NR][MT][2];
      if (there) {
        const int j0 = (at.q.first + at.unit + (int)u) * T;
        const bool masked = j0 + T > all_hi || j0 < all_lo;
        // P carries the page's V scale over ref.  ref moves when that leaves
        // [1/2, 512]: P, at most 2^kKvGrow, then stays inside f16's range and
        // loses bits (below its normal 2^-14) only 2^13 under the row's largest.  A V
        // scale under ref's lowest loses them sooner (2^-25 of that unit), and one
        // 2^-8 of it counts as zero.
        const bool usual = vs >= low * 0x1p-8f && vs <= FLT_MAX;   // not zero, not NaN
        float turn = 1.0f;
        if (usual && !(vs <= ref * 512.0f && vs >= ref * 0.5f)) {
          const float to = fmaxf(vs * 0.03125f, low);
          turn = __fdividef(ref, to);
          ref = to;
          low = fmaxf(low, to * 0x1p-64f);
        }
        const float ratio = usual ? __fdividef(vs, ref) : 1.0f;
        const float lift = __log2f(ratio), unlift = __fdividef(1.0f, ratio);
#pragma unroll
        for (int h = 0; h < NR; ++h) {
          int lo[2] = {0, 0}, hi[2] = {INT_MAX, INT_MAX};
          float s[MT][4];
#pragma unroll
          for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              s[t][e] = sc[h][t][0][e];
#pragma unroll
              for (int k = 1; k < kSums; ++k) s[t][e] += sc[h][t][k][e];
            }
          if (masked) {
            // the keys each row sees
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int r = 8 * h + 2 * cc + e;
              if (r < rows) {
                const int pos = shift + (row0 + r) / p.group;
                lo[e] = key_low(pos, p.window);
                hi[e] = key_high(pos, at.q.len, 1);
              }
            }
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int j = j0 + t * 16 + g + (e >> 1) * 8;
                if (j < lo[e & 1] || j >= hi[e & 1]) s[t][e] = -INFINITY;
              }
          }
          // exponent of two of a score: (s - qb) * qs * K's scale
          float f[2], n[2];
          bool moved = turn != 1.0f;
          float fo[2] = {turn, turn};
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            f[e] = qs[h][e] * ks * 16777216.0f;
            float mx = fmaxf(s[0][e], s[0][2 + e]);
#pragma unroll
            for (int t = 1; t < MT; ++t) mx = max3f(mx, s[t][e], s[t][2 + e]);
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            mx = mx == -INFINITY ? mx : (mx - qb[h][e]) * f[e];
            if (mx > m[h][e] + kKvGrow) {
              const float d = fast_exp2(m[h][e] - mx);
              m[h][e] = mx;
              l[h][e] *= d;
              fo[e] *= d;
              moved = true;
            }
            n[e] = fmaf(-qb[h][e], f[e], lift - (m[h][e] == -INFINITY ? 0.0f : m[h][e]));
          }
          if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
            for (int t = 0; t < OT; ++t)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[h][t][e] *= fo[e & 1];
          }
#pragma unroll
          for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[t][e] = fast_exp2(fmaf(s[t][e], f[e & 1], n[e & 1]));
          if (masked) {
            // -inf * 0 is no 0: what a row does not see leaves here
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int j = j0 + t * 16 + g + (e >> 1) * 8;
                if (j < lo[e & 1] || j >= hi[e & 1]) s[t][e] = 0.0f;
              }
          }
          float sum[2] = {0.0f, 0.0f};
#pragma unroll
          for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int e = 0; e < 2; ++e) sum[e] += s[t][e] + s[t][2 + e];
#pragma unroll
          for (int e = 0; e < 2; ++e) l[h][e] = fmaf(sum[e], unlift, l[h][e]);
          if (!usual) {
            // values of zero, or so small, count in the sum alone; a NaN or an infinity
            // reaches the rows that see the page
            const float over = vs < low ? 0.0f : vs;
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int j = j0 + t * 16 + g + (e >> 1) * 8;
                s[t][e] = j < lo[e & 1] || j >= hi[e & 1] ? 0.0f : s[t][e] * over;
              }
          }
#pragma unroll
          for (int t = 0; t < MT; ++t) {
            pf[h][t][0] = transpose8(pack_f16(s[t][0], s[t][1]));
            pf[h][t][1] = transpose8(pack_f16(s[t][2], s[t][3]));
          }
        }
      }

      // O^T
      cp_async_wait<3>();
      __syncwarp();
      if (there) {
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          const uint8_t* const vr = vb + t * 16 * D;
          // four output columns from one word of each of the lane's four keys
          auto four = [&](int base, uint32_t w0, uint32_t w1, uint32_t w8, uint32_t w9) {
            w0 ^= 0x80808080u;
            w1 ^= 0x80808080u;
            w8 ^= 0x80808080u;
            w9 ^= 0x80808080u;
            const uint32_t x0 = __byte_perm(w0, w1, 0x5140), x1 = __byte_perm(w0, w1, 0x7362);
            const uint32_t y0 = __byte_perm(w8, w9, 0x5140), y1 = __byte_perm(w8, w9, 0x7362);
            const uint32_t a0 = f16_pair(x0, k64, false), a1 = f16_pair(x0, k64, true);
            const uint32_t a2 = f16_pair(y0, k64, false), a3 = f16_pair(y0, k64, true);
            const uint32_t b0 = f16_pair(x1, k64, false), b1 = f16_pair(x1, k64, true);
            const uint32_t b2 = f16_pair(y1, k64, false), b3 = f16_pair(y1, k64, true);
#pragma unroll
            for (int h = 0; h < NR; ++h) {
              mma_f16(o[h][base], a0, a1, a2, a3, pf[h][t][0], pf[h][t][1]);
              mma_f16(o[h][base + 1], b0, b1, b2, b3, pf[h][t][0], pf[h][t][1]);
            }
          };
          if constexpr (D == 64) {
            // key 2 cc + 1 is 64 bytes on in the same 128, swizzled alike
            const uint8_t* const odd = kb + 4096 + (v_at ^ 64u) + t * 16 * D;
            const uint2 w0 = lds64(vr), w1 = lds64(odd);
            const uint2 w8 = lds64(vr + 8 * D), w9 = lds64(odd + 8 * D);
            four(0, w0.x, w1.x, w8.x, w9.x);
            four(2, w0.y, w1.y, w8.y, w9.y);
          } else {
#pragma unroll
            for (int w = 0; w < D / 128; ++w) {
              const uint4 w0 = lds128(vr + w * 128), w1 = lds128(vr + D + w * 128);
              const uint4 w8 = lds128(vr + 8 * D + w * 128), w9 = lds128(vr + 9 * D + w * 128);
              four(w * 8 + 0, w0.x, w1.x, w8.x, w9.x);
              four(w * 8 + 2, w0.y, w1.y, w8.y, w9.y);
              four(w * 8 + 4, w0.z, w1.z, w8.z, w9.z);
              four(w * 8 + 6, w0.w, w1.w, w8.w, w9.w);
            }
          }
        }
      }
      __syncwarp();
      load_v(stage);
      stage ^= 1;
    }

    // ---- the tile's rows, or this share's part of them
    const bool whole = !TEAM && at.unit == 0 && share == (uint32_t)at.q.units;
    // a warp's first tile goes to place 0, another to 1; TEAM: over the stages, which
    // all lanes have read
    float* part_o = p.part_o + site * D;
    float* part_ml = p.part_ml + site * 2;
    if constexpr (TEAM) {
      part_o = reinterpret_cast<float*>(mine);
      part_ml = s_ml[warp][0];
      __syncwarp();
    }
    const float unit = ref > 0.0f ? ref : 1.0f;
#pragma unroll
    for (int h = 0; h < NR; ++h)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        l[h][e] += __shfl_xor_sync(0xffffffffu, l[h][e], 4);
        l[h][e] += __shfl_xor_sync(0xffffffffu, l[h][e], 8);
        l[h][e] += __shfl_xor_sync(0xffffffffu, l[h][e], 16);
        const int r = 8 * h + 2 * cc + e;
        if (r >= rows) continue;
        // this lane has columns g * 16 .. + 15 of every 128 (g * 8 .. + 7 of 64)
        constexpr int J = D == 64 ? 4 : 8;             // tiles of a V piece
        if (whole) {
          const int tok = (row0 + r) / p.group, head = at.head * p.group + (row0 + r) % p.group;
          const bool any = l[h][e] != 0.0f;            // see kv_put_row
          const float norm = unit / l[h][e];
          __nv_bfloat16* dst = p.o + (size_t)(at.q.row0 + tok) * p.ldo + (size_t)head * D;
#pragma unroll
          for (int t = 0; t < OT; t += 4) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
              w[i] = any ? pack_bf16(o[h][t + i][e] * norm, o[h][t + i][2 + e] * norm) : 0u;
            *reinterpret_cast<uint4*>(dst + t / J * 128 + g * 2 * J + t % J * 2) =
                make_uint4(w[0], w[1], w[2], w[3]);
          }
        } else {
          float* dst = part_o + r * D;
#pragma unroll
          for (int t = 0; t < OT; t += 2)
            *reinterpret_cast<float4*>(dst + t / J * 128 + g * 2 * J + t % J * 2) =
                make_float4(o[h][t][e] * unit, o[h][t][2 + e] * unit, o[h][t + 1][e] * unit,
                            o[h][t + 1][2 + e] * unit);
          if (g == 0)
            *reinterpret_cast<float2*>(part_ml + r * 2) = make_float2(m[h][e], l[h][e]);
        }
      }
    x += share;
    if (!TEAM && x < count) {
      if (x == share) site += TR;
      kv_move<D, TR, N>(p, s_tab, at, (int)share);
    }
  }
  cp_async_wait<0>();

  if constexpr (TEAM) {
    __syncthreads();
    const int rows = min(TR, at.q.n * p.group - at.tile * TR);
    for (int r = warp; r < rows; r += W) {
      float2 ml = make_float2(-INFINITY, 0.0f);
      if (lane < team) ml = *reinterpret_cast<const float2*>(s_ml[lane][r]);
      float top = ml.x;
      for (int w = 16; w > 0; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
      const float f = kv_weight(ml.x, ml.y, top);
      float sum = f * ml.y;
      for (int w = 16; w > 0; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
      float2 acc[D / 64];
#pragma unroll
      for (int e = 0; e < D / 64; ++e) acc[e] = make_float2(0.0f, 0.0f);
#pragma unroll 4
      for (int w = 0; w < team; ++w) {
        const float fw = __shfl_sync(0xffffffffu, f, w);
        const float2* src =
            reinterpret_cast<const float2*>(smem_raw + w * 2 * C::kStageBytes) + r * (D / 2);
#pragma unroll
        for (int e = 0; e < D / 64; ++e) {
          const float2 v = src[e * 32 + lane];
          acc[e].x = fmaf(fw, v.x, acc[e].x);
          acc[e].y = fmaf(fw, v.y, acc[e].y);
        }
      }
      kv_put_row<D>(p, at.q, at.head, at.tile * TR + r, acc, sum);
    }
  }
}

// Joins the tiles that several warps share: with M the largest of their
// maxima, o = sum 2^(m_i - M) O_i / sum 2^(m_i - M) l_i, in a fixed order.
// Writes zeros for the rows of sequences without keys, which no warp has.  A
// block a (row tile, kv head), or each of its rows where the tiles alone leave SMs
// idle (grid z); its warps share the rows and, where those are fewer, the parts of
// a row.  It is a chain of latencies (no SM has room for it before the attention
// ends), so a warp asks for its parts' maxima and their O at once and joins them
// under its own maximum; the warps of a row join theirs in shared memory (all under
// the row's maximum, read first: 58.5 against 54.8 us for the case below).
// Everything up to pdl_wait reads only what the attention kernel had waited for
// itself.
template <int D, int NR, int W>
__global__ void __launch_bounds__(W * 32) kv8_merge_kernel(const __grid_constant__ KvAttn p)
{
  constexpr int N = 128, E = D / 64, P = E == 4 ? 4 : 8, TR = 8 * NR;
  __shared__ KvTable<N> s_tab;
  __shared__ float2 s_o[W][D / 2];
  __shared__ float2 s_ml[W];
  const int warp = (int)threadIdx.x >> 5, lane = (int)threadIdx.x & 31;
  const int head = (int)blockIdx.y, slot = (int)blockIdx.x;
  // the slot's sequence: tiles of rows are slots of cu * group rows
  int lo = 0, hi = p.seqs;
  if (p.seqs > N)
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (slot_base(clamp_int(p.cu[mid], 0, p.rows) * p.group, mid, TR, 1) <= slot) lo = mid;
      else hi = mid;
    }
  kv_scan<D, TR, N>(p, s_tab);
  if (p.seqs <= N)
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (slot_base(s_tab.q[mid].row0 * p.group, mid, TR, 1) <= slot) lo = mid;
      else hi = mid;
    }
  const int s = lo;
  const KvSeq q = kv_get<D, TR, N>(p, s_tab, s);
  const int tile = slot - slot_base(q.row0 * p.group, s, TR, 1);
  int rows = tile < 0 || tile >= q.tiles ? 0 : min(TR, q.n * p.group - tile * TR);
  // this block's rows: r_from .. rows - 1
  const int r_from = (int)blockIdx.z * (TR / (int)gridDim.z);
  rows = min(rows, r_from + TR / (int)gridDim.z);
  const u64 all = s_tab.before[N], workers = kv_workers(p, all);
  const int each = (p.seqs + N - 1) / N;
  u64 at = s_tab.before[s / each];
  for (int i = s / each * each; i < s; ++i) at += kv_work(p, kv_get<D, TR, N>(p, s_tab, i));
  at += ((u64)head * q.tiles + tile) * (u64)q.units;
  int first = 0, last = 0, place0 = 0;                 // workers, the first one's place
  if (rows > r_from && q.units > 0) {
    first = (int)work_owner(all, workers, at);
    last = (int)work_owner(all, workers, at + q.units - 1);
    place0 = work_bound(all, workers, (u64)first) < at ? 1 : 0;
  }
  pdl_wait();
  pdl_trigger();
  if (rows <= r_from) return;
  if (q.units == 0) {
    for (int i = r_from * D + (int)threadIdx.x; i < rows * D; i += W * 32) {
      const int r = tile * TR + i / D;
      p.o[(size_t)(q.row0 + r / p.group) * p.ldo + (size_t)(head * p.group + r % p.group) * D +
          i % D] = __float2bfloat16_rn(0.0f);
    }
    return;
  }
  if (first == last) return;                           // written by its warp
  const int parts = last - first + 1;
  auto site = [&](int i, int r) { return ((first + i) * 2 + (i == 0 ? place0 : 0)) * TR + r; };
  // `wide` warps a row, a power of two
  const int own = rows - r_from;
  const int wide = max(1, W / (own > 8 ? 16 : own > 4 ? 8 : own > 2 ? 4 : own > 1 ? 2 : 1));
  for (int r0 = r_from; r0 < rows; r0 += W / wide) {
    const int r = r0 + warp / wide, mine = warp % wide;
    float2 acc[E];
    float l = 0.0f, top = -INFINITY;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = make_float2(0.0f, 0.0f);
    if (r < rows) {
      // parts [mine per, end), 32 at a time, a lane each for their factors under the
      // maximum so far; O of P of them is on its way with the maxima
      const int per = (parts + wide - 1) / wide;
      const int end = min(parts, (mine + 1) * per);
      for (int i0 = mine * per; i0 < end; i0 += 32) {
        const int n = min(32, end - i0);
        float2 ml = make_float2(-INFINITY, 0.0f);
        if (lane < n) ml = *reinterpret_cast<const float2*>(p.part_ml + site(i0 + lane, r) * 2);
        for (int b = 0; b < n; b += P) {
          float2 v[P][E];
#pragma unroll
          for (int i = 0; i < P; ++i) {
            const float2* src =
                reinterpret_cast<const float2*>(p.part_o + (size_t)site(min(i0 + b + i, end - 1), r) * D);
#pragma unroll
            for (int e = 0; e < E; ++e) v[i][e] = src[e * 32 + lane];
          }
          if (b == 0) {
            float most = ml.x;
            for (int w = 16; w > 0; w >>= 1)
              most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, w));
            if (most > top) {
              const float d = top == -INFINITY ? 1.0f : fast_exp2(top - most);
              l *= d;
#pragma unroll
              for (int e = 0; e < E; ++e) acc[e] = make_float2(acc[e].x * d, acc[e].y * d);
              top = most;
            }
            ml.x = kv_weight(ml.x, ml.y, top);
            l = fmaf(ml.x, ml.y, l);
          }
#pragma unroll
          for (int i = 0; i < P; ++i) {
            const float f = __shfl_sync(0xffffffffu, ml.x, (b + i) & 31);
            if (b + i < n) {
#pragma unroll
              for (int e = 0; e < E; ++e) {
                acc[e].x = fmaf(f, v[i][e].x, acc[e].x);
                acc[e].y = fmaf(f, v[i][e].y, acc[e].y);
              }
            }
          }
        }
      }
      for (int w = 16; w > 0; w >>= 1) l += __shfl_xor_sync(0xffffffffu, l, w);
    }
    if (wide > 1) {
      if (r < rows) {
#pragma unroll
        for (int e = 0; e < E; ++e) s_o[warp][e * 32 + lane] = acc[e];
        if (lane == 0) s_ml[warp] = make_float2(top, l);
      }
      __syncthreads();
      if (r < rows && mine == 0) {
        float2 ml = make_float2(-INFINITY, 0.0f);
        if (lane < wide) ml = s_ml[warp + lane];
        float most = ml.x;
        for (int w = 16; w > 0; w >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, w));
        const float f = kv_weight(ml.x, ml.y, most);
        l = f * ml.y;
        for (int w = 16; w > 0; w >>= 1) l += __shfl_xor_sync(0xffffffffu, l, w);
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = make_float2(0.0f, 0.0f);
#pragma unroll 8
        for (int w = 0; w < wide; ++w) {
          const float fw = __shfl_sync(0xffffffffu, f, w);
#pragma unroll
          for (int e = 0; e < E; ++e) {
            const float2 v = s_o[warp + w][e * 32 + lane];
            acc[e].x = fmaf(fw, v.x, acc[e].x);
            acc[e].y = fmaf(fw, v.y, acc[e].y);
          }
        }
      }
    }
    if (r < rows && mine == 0) kv_put_row<D>(p, q, head, tile * TR + r, acc, l);
  }
}

KvPages kv_pages(const Kv8Cache& c, const Kv8Rows& r, int* err)
{
  KvPages p;
  memset(&p, 0, sizeof(p));
  p.k = c.k;
  p.v = c.v;
  p.ks = c.ks;
  p.vs = c.vs;
  p.table = r.table;
  p.starts = r.starts;
  p.cu = r.cu;
  p.table_ld = r.table_ld;
  p.pages = c.pages;
  p.kv_heads = c.kv_heads;
  p.seqs = r.seqs;
  p.rows = r.rows;
  p.err = err;
  return p;
}

// blocks of a page and head, keys and values
bool kv_pages_grid(const Kv8Cache& c, const Kv8Rows& r, dim3* grid)
{
  const long long n = (long long)slot_count(r.rows, r.seqs, kPage, 2) * c.kv_heads;
  if (n > INT_MAX) return false;
  *grid = dim3((unsigned)n, 1, 2);
  return true;
}

template <int D, int NR>
int kv_attn_launch(const Kv8Attention& a, int num_sms, int* err, cudaStream_t s)
{
  using C = KvCfg<D, NR>;
  KvAttn p;
  memset(&p, 0, sizeof(p));
  p.k = a.cache.k;
  p.v = a.cache.v;
  p.ks = a.cache.ks;
  p.vs = a.cache.vs;
  p.q = a.q;
  p.o = a.o;
  p.ldq = a.ldq;
  p.ldo = a.ldo;
  p.cu = a.rows.cu;
  p.lengths = a.rows.starts;
  p.table = a.rows.table;
  p.table_ld = a.rows.table_ld;
  p.pages = a.cache.pages;
  p.kv_heads = a.cache.kv_heads;
  p.group = a.heads / a.cache.kv_heads;
  p.seqs = a.rows.seqs;
  p.rows = a.rows.rows;
  p.window = a.window;
  p.c = a.scale * 1.4426950408889634f;
  p.err = err;
  const int slots = slot_count(p.rows * p.group, p.seqs, 8 * NR, 1);
  const long long tiles = (long long)slots * p.kv_heads;
  const long long reach = a.window > 0 && a.window < a.max_len - p.rows ? (long long)a.window + p.rows
                                                                       : a.max_len;
  const long long units = (reach + C::kTok - 1) / C::kTok;          // of a tile, at most
  // A block a tile (TEAM) where the tiles fit the SMs and the longest is short: 5 us and
  // 1.3 to 1.8 for each stage of a warp, against 9 us and the bytes at HBM's rate for
  // equal runs of all the work.  Measured, one token a sequence at head width 128, 4
  // query heads a key head, us (TEAM / equal runs):
  //   tokens        300          1000          2000         4000
  //   8 tiles     6.2 /  8.2    9.6 /  9.2   15.6 /  9.4   24.1 / 10.0
  //   32          6.6 / 11.8   10.1 / 12.3   16.2 / 14.4   24.9 / 16.8
  //   64          6.7 / 11.0   10.4 / 15.3   16.8 / 19.4   25.6 / 24.4
  // and not beyond 6 stages a warp, since lengths may be anything up to max_len.  The same
  // numbers serve the other widths and tiles of 16 rows (us for 300, 1000, 2000, 4000
  // tokens, TEAM / equal runs, * the rule's choice):
  //   width  64,  8 tiles    5.4* 7.9   7.2*  9.0   9.5* 10.1  15.1  10.3*
  //              64          5.9*10.5   7.9* 11.5  10.3* 13.9  16.0* 17.1
  //   width 256,  8          8.3* 9.2  15.9   9.4* 27.2  10.5* 50.0  12.3*
  //              64          8.9*12.6  16.6  15.8* 28.5  22.1* 51.9  33.1*
  //   128, 16 rows, 8       10.1*13.0  14.3  13.5* 21.7  13.9* 36.5  14.9*
  //              32         10.3*26.6  14.5* 28.8  21.9  31.1* 36.6  34.4*
  //              64         10.4*15.1  14.6* 19.8  22.2  25.5* 37.5  33.1*
  // Equal runs of 32 tiles of 16 rows pay for a join of a warp a row that is slow for so
  // many; there and with 64 the rule gives up on TEAM too early at 2000 tokens.
  const long long used = p.rows == p.seqs ? (long long)p.seqs * ((p.group + 8 * NR - 1) / (8 * NR))
                                          : slots;                  // slots with rows
  const long long rounds = (units + C::kWarps - 1) / C::kWarps;
  if (used * p.kv_heads <= num_sms && p.seqs <= C::kThreads && rounds <= 6 &&
      (rounds - 3) * 1200 <= NR * used * p.kv_heads * units) {
    static std::atomic<unsigned long long> attr{0};
    if (!smem_limit_once(kv8_attention_kernel<D, NR, true>, C::kSmem, attr)) return -1;
    launch_k(kv8_attention_kernel<D, NR, true>, dim3((unsigned)tiles), dim3(C::kThreads), C::kSmem,
             s, 1, p);
    return launched();
  }
  // a block for each SM, fewer where the longest sequences cannot fill them
  const long long most = tiles * (units + 1);
  const int grid = (int)(most < num_sms ? (most < 1 ? 1 : most) : num_sms);
  p.workers = grid * C::kWarps;
  p.part_o = a.workspace;
  p.part_ml = p.part_o + (size_t)p.workers * 2 * (8 * NR) * D;
  static std::atomic<unsigned long long> attr{0};
  if (!smem_limit_once(kv8_attention_kernel<D, NR, false>, C::kSmem, attr)) return -1;
  launch_k(kv8_attention_kernel<D, NR, false>, dim3((unsigned)grid), dim3(C::kThreads), C::kSmem, s, 1,
           p);
  if (launched() != 0) return -1;
  // few tiles have many parts each: 16 warps a row (1 sequence of 131072 tokens, 222
  // parts a row: 53.5 us with the attention, 54.8 with 32 warps, 57.1 with 8); else a
  // warp a row
  if ((long long)slots * p.kv_heads * 2 <= num_sms)
    launch_k(kv8_merge_kernel<D, NR, 16>, dim3((unsigned)slots, (unsigned)p.kv_heads, 8 * NR),
             dim3(512), 0, s, 1, p);
  else if ((long long)p.rows * p.group > 4ll * p.seqs)
    launch_k(kv8_merge_kernel<D, NR, 8>, dim3((unsigned)slots, (unsigned)p.kv_heads), dim3(256), 0,
             s, 1, p);
  else
    launch_k(kv8_merge_kernel<D, NR, 4>, dim3((unsigned)slots, (unsigned)p.kv_heads), dim3(128), 0,
             s, 1, p);
  return launched();
}

// Tiles of 8 rows where the sequences have no more on the average (a decoded
// token under up to 8 query heads a key head), else of 16 (64 sequences of 100 to
// 8192 tokens, 16 rows: 142 against 183 us at width 128, 91 against 106 at 64).
// At width 256 a second group of rows does not fit the registers beside O and q
// and two tiles are faster (16 sequences, 16 rows, 4096 keys: 88 against 100 us).
template <int D>
int kv_attn_tiles(const Kv8Attention& a, int num_sms, int* err, cudaStream_t s)
{
  if constexpr (D < 256) {
    const long long rows = (long long)a.rows.rows * (a.heads / a.cache.kv_heads);
    if (rows > 8ll * a.rows.seqs) return kv_attn_launch<D, 2>(a, num_sms, err, s);
  }
  return kv_attn_launch<D, 1>(a, num_sms, err, s);
}

}  // namespace

int launch_kv8_append(const Kv8Cache& c, const Kv8Rows& r, const __nv_bfloat16* k, int ldk,
                      const __nv_bfloat16* v, int ldv, int* err, cudaStream_t s)
{
  const KvPages p = kv_pages(c, r, err);
  // few rows a sequence: a block a page; else one for each of its heads, keys and values
  const bool few = (long long)r.rows <= 4ll * r.seqs;
  dim3 grid;
  if (few) grid = dim3((unsigned)slot_count(r.rows, r.seqs, kPage, 2));
  else if (!kv_pages_grid(c, r, &grid)) return -2;
  const dim3 block(kAppendThreads);
  switch (c.head_dim) {
    case 64:
      launch_k(few ? kv8_append_few_kernel<64> : kv8_append_kernel<64>, grid, block, 0, s, 1, p, k,
               ldk, v, ldv);
      break;
    case 128:
      launch_k(few ? kv8_append_few_kernel<128> : kv8_append_kernel<128>, grid, block, 0, s, 1, p,
               k, ldk, v, ldv);
      break;
    case 256:
      launch_k(few ? kv8_append_few_kernel<256> : kv8_append_kernel<256>, grid, block, 0, s, 1, p,
               k, ldk, v, ldv);
      break;
    default: return -2;
  }
  return launched();
}

int launch_kv8_read(const Kv8Cache& c, const Kv8Rows& r, __nv_bfloat16* k, int ldk,
                    __nv_bfloat16* v, int ldv, int* err, cudaStream_t s)
{
  const KvPages p = kv_pages(c, r, err);
  dim3 grid;
  if (!kv_pages_grid(c, r, &grid)) return -2;
  switch (c.head_dim) {
    case 64: launch_k(kv8_read_kernel<64>, grid, dim3(kAppendThreads), 0, s, 1, p, k, ldk, v, ldv); break;
    case 128: launch_k(kv8_read_kernel<128>, grid, dim3(kAppendThreads), 0, s, 1, p, k, ldk, v, ldv); break;
    case 256: launch_k(kv8_read_kernel<256>, grid, dim3(kAppendThreads), 0, s, 1, p, k, ldk, v, ldv); break;
    default: return -2;
  }
  return launched();
}

size_t kv8_attention_workspace(int head_dim, int num_sms)
{
  // a first and a last part a warp: 12 warps with 8 rows at most, 8 with 16
  const size_t rows = (size_t)num_sms * 2 * 16 * KvCfg<128, 2>::kWarps;
  static_assert(KvCfg<128, 1>::kWarps * 8 <= KvCfg<128, 2>::kWarps * 16 &&
                KvCfg<64, 1>::kWarps == KvCfg<128, 1>::kWarps &&
                KvCfg<64, 2>::kWarps == KvCfg<128, 2>::kWarps &&
                KvCfg<256, 1>::kWarps <= KvCfg<128, 1>::kWarps, "rows of the workspace");
  return rows * (size_t)(head_dim + 2) * sizeof(float);
}

int launch_kv8_attention(const Kv8Attention& a, int num_sms, int* err, cudaStream_t s)
{
  switch (a.cache.head_dim) {
    case 64: return kv_attn_tiles<64>(a, num_sms, err, s);
    case 128: return kv_attn_tiles<128>(a, num_sms, err, s);
    case 256: return kv_attn_tiles<256>(a, num_sms, err, s);
    default: return -2;
  }
}

}  // namespace ltx
