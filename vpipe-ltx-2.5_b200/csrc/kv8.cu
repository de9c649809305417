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

struct KvSpan {
  int row, from, count;           // packed row of the first token, its slot, tokens
  size_t page;                    // page * kv_heads + head
};

// The tokens of one page that work slot `slot` covers, false where it has none.
// Every thread of the block calls it.
__device__ __forceinline__ bool kv_span(const KvPages& p, int slot, int head, KvSpan* out)
{
  const int s = find_seq(p.cu, p.seqs, p.rows, kPage, 2, slot);
  const int row0 = clamp_int(p.cu[s], 0, p.rows);
  const int n = clamp_int(p.cu[s + 1], row0, p.rows) - row0;
  const int i = slot - slot_base(row0, s, kPage, 2);
  const int start = p.starts[s];
  if (n == 0 || i < 0) return false;
  const int cap = p.table_ld * kPage;
  if (!span_ok(start, n, cap)) {
    if (threadIdx.x == 0) atomicCAS(p.err, 0, KERR_PLACE);
    return false;
  }
  const PageSpan span = page_span(start, n, i);
  if (span.b <= span.a) return false;
  const int page = p.table[(size_t)s * p.table_ld + span.block];
  if (!page_ok(page, p.pages)) {
    if (threadIdx.x == 0) atomicCAS(p.err, 0, KERR_PLACE);
    return false;
  }
  out->row = row0 + (span.a - start);
  out->from = span.a - span.block * kPage;
  out->count = span.b - span.a;
  out->page = (size_t)page * p.kv_heads + head;
  return true;
}

constexpr int kAppendThreads = 256;

// One page, one head, keys (blockIdx.z 0) or values (1) a block: the new rows
// stay in registers between the search for their maximum and their rounding,
// so they are read once.
//   t = x / s by one product with 1 / s, within 2^-15 of the quotient;
//   adding and taking away 1.5 * 2^12 rounds it to a multiple of 2^-11, which
//   puts a tie back on the tie and leaves all others on their side (2^-9);
//   adding 1.5 * 2^23 rounds to the nearest integer, ties to even, and leaves
//   the code in the sum's low byte.
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
  KvSpan w;
  if (!kv_span(p, (int)blockIdx.x, (int)blockIdx.y, &w)) return;
  const bool val = blockIdx.z != 0;
  const __nv_bfloat16* x = val ? v : k;
  const int ld = val ? ldv : ldk;
  int8_t* codes = (val ? p.v : p.k) + w.page * (size_t)(kPage * D);
  uint16_t* scale = (val ? p.vs : p.ks) + w.page;
  const int chunk = (int)threadIdx.x % kChunks, r0 = (int)threadIdx.x / kChunks;

  uint4 in[kPasses];
  uint32_t most = 0;
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    const int r = r0 + i * kRowsAt;
    in[i] = make_uint4(0, 0, 0, 0);
    if (r < w.count)
      in[i] = *reinterpret_cast<const uint4*>(x + (size_t)(w.row + r) * ld +
                                              (size_t)blockIdx.y * D + chunk * 8);
    const uint32_t a = __vmaxu2(in[i].x & 0x7fff7fffu, in[i].y & 0x7fff7fffu);
    const uint32_t b = __vmaxu2(in[i].z & 0x7fff7fffu, in[i].w & 0x7fff7fffu);
    most = __vmaxu2(most, __vmaxu2(a, b));
  }
  most = max(most & 0xffffu, most >> 16);
  most = __reduce_max_sync(0xffffffffu, most);
  if ((threadIdx.x & 31) == 0) s_most[threadIdx.x >> 5] = most;
  const uint32_t was = *scale;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kAppendThreads / 32; ++i) most = max(most, s_most[i]);

  // bf16 magnitudes order like their bits; a NaN or infinity is above 0x7f7f
  // and makes the page's scale NaN
  uint32_t now = most > 0x7f7fu ? 0x7fc0u : page_scale(most);
  if (w.from > 0) now = max(now, was);
  const bool bad = now > 0x7f7fu;
  if (w.from > 0 && now != was && !bad) {
    // the page's own codes, brought to the grown scale: c * was / now, a
    // quotient of 15 by 8 bits, decided by the correctly rounded f32 division
    const float s0 = bf16_bits(was), s1 = bf16_bits(now);
    for (int i = (int)threadIdx.x; i < w.from * (D / 4); i += kAppendThreads) {
      char4 c = reinterpret_cast<char4*>(codes)[i];
      c.x = (signed char)__float2int_rn(__fdiv_rn((float)c.x * s0, s1));
      c.y = (signed char)__float2int_rn(__fdiv_rn((float)c.y * s0, s1));
      c.z = (signed char)__float2int_rn(__fdiv_rn((float)c.z * s0, s1));
      c.w = (signed char)__float2int_rn(__fdiv_rn((float)c.w * s0, s1));
      reinterpret_cast<char4*>(codes)[i] = c;
    }
  }
  if (threadIdx.x == 0 && (w.from == 0 || now != was)) *scale = (uint16_t)now;

  // 1 / s may not be finite for a tiny s: both are scaled by 2^64 there
  const float s = bf16_bits(now);
  const float pre = s < 0x1p-64f ? 0x1p64f : 1.0f;
  const float inv = bad || s == 0.0f ? 0.0f : __frcp_rn(s * pre);
  const float mul = bad ? 0.0f : pre;
  auto code = [&](float f) {
    const float t = (f * mul) * inv;
    const float snapped = __fadd_rn(__fadd_rn(t, 6144.0f), -6144.0f);
    return __float_as_uint(__fadd_rn(snapped, 12582912.0f));
  };
  auto four = [&](uint32_t a, uint32_t b) {
    const uint32_t c0 = code(__uint_as_float(a << 16)), c1 = code(__uint_as_float(a & 0xffff0000u));
    const uint32_t c2 = code(__uint_as_float(b << 16)), c3 = code(__uint_as_float(b & 0xffff0000u));
    return __byte_perm(__byte_perm(c0, c1, 0x0040), __byte_perm(c2, c3, 0x0040), 0x5410);
  };
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    const int r = r0 + i * kRowsAt;
    if (r >= w.count) break;
    uint2 c = make_uint2(0, 0);
    if (!bad) c = make_uint2(four(in[i].x, in[i].y), four(in[i].z, in[i].w));
    *reinterpret_cast<uint2*>(codes + (size_t)(w.from + r) * D + chunk * 8) = c;
  }
}

// Rows of a cache back as bf16: bf16(c * s).
template <int D>
__global__ void __launch_bounds__(kAppendThreads)
    kv8_read_kernel(KvPages p, __nv_bfloat16* k, int ldk, __nv_bfloat16* v, int ldv)
{
  constexpr int kChunks = D / 16;
  pdl_wait();
  pdl_trigger();
  KvSpan w;
  if (!kv_span(p, (int)blockIdx.x, (int)blockIdx.y, &w)) return;
  const bool val = blockIdx.z != 0;
  __nv_bfloat16* x = val ? v : k;
  const int ld = val ? ldv : ldk;
  const int8_t* codes = (val ? p.v : p.k) + w.page * (size_t)(kPage * D) + (size_t)w.from * D;
  const float s = bf16_bits((val ? p.vs : p.ks)[w.page]);
  for (int i = (int)threadIdx.x; i < w.count * kChunks; i += kAppendThreads) {
    const uint4 c = reinterpret_cast<const uint4*>(codes)[i];
    const uint32_t words[4] = {c.x, c.y, c.z, c.w};
    uint32_t o[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const char4 b = *reinterpret_cast<const char4*>(&words[j]);
      o[2 * j] = pack_bf16((float)b.x * s, (float)b.y * s);
      o[2 * j + 1] = pack_bf16((float)b.z * s, (float)b.w * s);
    }
    uint4* dst = reinterpret_cast<uint4*>(x + (size_t)(w.row + i / kChunks) * ld +
                                          (size_t)blockIdx.y * D + (i % kChunks) * 16);
    dst[0] = make_uint4(o[0], o[1], o[2], o[3]);
    dst[1] = make_uint4(o[4], o[5], o[6], o[7]);
  }
}

// ---- attention over the cache ----------------------------------------------
//
// The new rows of a sequence (n tokens, the last n of its `length`) times the
// G query heads of a key/value head are rows token * G + head, in tiles of 16:
// one warp MMA's rows.  The work is the list of all (sequence, kv head, row
// tile, 8 KB stage of keys and values) in that order, and every warp of the
// grid takes an equal run of it, whatever the lengths: at most its first and
// its last tile are shared with other warps.  A tile that one warp has whole
// goes straight to o; the others leave (max, sum, O) in the workspace for
// kv8_merge_kernel.
//
// This reads 2 D bytes a token and key head and is bound by HBM as long as a
// code costs few instructions: int8 -> f16 is a byte permute into 1024 + u and
// one packed subtraction (exact), the products run on warp MMAs with f32 sums
// (m16n8k16), K's scale goes into the exponent's factor and V's into P.  Codes
// and P are f16 (P rounds at 2^-11); q, whose 8 bits f16 holds exactly, is
// brought near 2^8 by a power of two a row.
//
// Each warp streams its stages through a ring of its own with 16-byte
// asynchronous copies (no barrier between warps).  Shared memory is swizzled
// by 16-byte pieces so that the fragment reads below are free of conflicts:
// keys of one MMA column group for K, pairs of keys for V.

template <int D>
struct KvCfg {
  static constexpr int kTok = 4096 / D;                // tokens of a stage
  static constexpr int kStages = 3;
  static constexpr int kWarps = 4;
  static constexpr int kStageBytes = 8192;             // K, then V
  static constexpr int kWarpBytes = kStages * kStageBytes + kStages * 16;
  static constexpr int kSmem = kWarps * kWarpBytes;
  static constexpr int kNT = kTok / 8;                 // score column tiles
  static constexpr int kOT = D / 8;                    // output column tiles
};

constexpr int kTileRows = 16;
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
  float* part_o;                  // [workers][2][16][D]
  float* part_ml;                 // [workers][2][16][2]
  int* err;
};

// What one sequence asks for.
struct KvSeq {
  int row0, n, len;               // its new rows, its length
  int tiles, first, units;        // row tiles; first stage and stages of each
};

template <int D>
__device__ __forceinline__ KvSeq kv_seq(const KvAttn& p, int s)
{
  constexpr int T = KvCfg<D>::kTok;
  KvSeq q;
  q.row0 = clamp_int(p.cu[s], 0, p.rows);
  q.n = clamp_int(p.cu[s + 1], q.row0, p.rows) - q.row0;
  const int len = p.lengths[s], cap = p.table_ld * kPage;
  q.len = clamp_int(len, 0, cap);
  if (len != q.len) atomicCAS(p.err, 0, KERR_PLACE);
  q.tiles = (q.n * p.group + kTileRows - 1) / kTileRows;
  const int lo = key_low(q.len - q.n, p.window);
  q.first = lo / T;
  q.units = q.len > lo ? (q.len + T - 1) / T - q.first : 0;
  return q;
}

template <int D>
__device__ __forceinline__ u64 kv_work(const KvAttn& p, const KvSeq& q)
{
  return (u64)q.tiles * (u64)p.kv_heads * (u64)q.units;
}

// pre[t] = work of the sequences before thread t's (an equal run of them each);
// pre[N] = all of it.  Every thread of the block calls it.
template <int D, int N>
__device__ __forceinline__ void kv_plan(const KvAttn& p, u64* pre)
{
  __shared__ u64 s_warp[N / 32];
  const int each = (p.seqs + N - 1) / N;
  const int t = (int)threadIdx.x, lane = t & 31;
  u64 mine = 0;
  for (int s = t * each; s < min(p.seqs, (t + 1) * each); ++s)
    mine += kv_work<D>(p, kv_seq<D>(p, s));
  u64 sum = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const u64 o = __shfl_up_sync(0xffffffffu, sum, d);
    if (lane >= d) sum += o;
  }
  if (lane == 31) s_warp[t >> 5] = sum;
  __syncthreads();
  u64 before = 0;
#pragma unroll
  for (int w = 0; w < N / 32; ++w)
    if (w < (t >> 5)) before += s_warp[w];
  pre[t + 1] = before + sum;
  if (t == 0) pre[0] = 0;
  __syncthreads();
}

// The sequence that work item x falls into, and the work before it.
template <int D, int N>
__device__ __forceinline__ int kv_find(const KvAttn& p, const u64* pre, u64 x, u64* before)
{
  int lo = 0, hi = N;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (pre[mid] <= x) lo = mid;
    else hi = mid;
  }
  const int each = (p.seqs + N - 1) / N;
  int s = lo * each;
  u64 at = pre[lo];
  const int last = min(p.seqs, (lo + 1) * each) - 1;
  while (s < last) {
    const u64 w = kv_work<D>(p, kv_seq<D>(p, s));
    if (x < at + w) break;
    at += w;
    ++s;
  }
  *before = at;
  return s;
}

// A place in the list of work.
template <int D>
struct KvCursor {
  KvSeq q;
  int s, head, tile, unit;

  __device__ __forceinline__ void set(const KvAttn& p, int seq, u64 within)
  {
    s = seq;
    q = kv_seq<D>(p, s);
    const u64 per = (u64)q.tiles * (u64)q.units;
    head = (int)(within / per);
    const u64 r = within % per;
    tile = (int)(r / (u64)q.units);
    unit = (int)(r % (u64)q.units);
  }
  __device__ __forceinline__ void next(const KvAttn& p)
  {
    if (++unit < q.units) return;
    unit = 0;
    if (++tile < q.tiles) return;
    tile = 0;
    if (++head < p.kv_heads) return;
    head = 0;
    while (++s < p.seqs) {
      q = kv_seq<D>(p, s);
      if (kv_work<D>(p, q) != 0) return;
    }
  }
};

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

__device__ __forceinline__ uint4 lds128(uint32_t a)
{
  uint4 r;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "r"(a));
  return r;
}
__device__ __forceinline__ uint2 lds64(uint32_t a)
{
  uint2 r;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(r.x), "=r"(r.y) : "r"(a));
  return r;
}

// Bytes 0, 1 (hi = false) or 2, 3 of w, each 128 + c, as the f16 pair c.
__device__ __forceinline__ uint32_t f16_pair(uint32_t w, bool hi)
{
  const uint32_t u = __byte_perm(w, 0x64646464u, hi ? 0x4342 : 0x4140);   // 1024 + 128 + c
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

// Columns of the output that lane column c holds in the accumulators' order:
// value e of row half h (0: row g, 1: row g + 8) is O[row][kv_col(c, e)] with
// e = w * 32 + half * 16 + j at widths 128 and 256 (128 w + 32 c + e % 32) and
// e = half * 8 + j at 64 (16 c + e).
template <int D>
__device__ __forceinline__ float kv_acc(const float (&o)[D / 8][4], int h, int e)
{
  constexpr int J = D == 64 ? 8 : 16;                  // bytes of a lane's V piece
  const int w = e / (2 * J), half = (e / J) & 1, j = e % J;
  return o[w * J + j][h * 2 + half];
}

template <int D>
__global__ void __launch_bounds__(KvCfg<D>::kWarps * 32, 2)
    kv8_attention_kernel(const __grid_constant__ KvAttn p)
{
  using C = KvCfg<D>;
  constexpr int T = C::kTok, N = C::kWarps * 32;
  extern __shared__ __align__(128) uint8_t smem_raw[];
  __shared__ u64 s_pre[N + 1];
  const int warp = (int)threadIdx.x >> 5, lane = (int)threadIdx.x & 31;
  const int g = lane >> 2, cc = lane & 3;
  const uint32_t ring = smem_u32(smem_raw) + (uint32_t)(warp * C::kWarpBytes);
  float4* heads = reinterpret_cast<float4*>(smem_raw + warp * C::kWarpBytes +
                                            C::kStages * C::kStageBytes);
  pdl_wait();
  pdl_trigger();
  kv_plan<D, N>(p, s_pre);
  const u64 all = s_pre[N];
  const u64 workers = min((u64)p.workers, all);
  const u64 me = (u64)blockIdx.x * C::kWarps + warp;
  if (me >= workers) return;
  const u64 begin = work_bound(all, workers, me), end = work_bound(all, workers, me + 1);

  KvCursor<D> ld, at;
  u64 before;
  const int s0 = kv_find<D, N>(p, s_pre, begin, &before);
  at.set(p, s0, begin - before);
  ld = at;
  // pages and scales of 32 blocks of the loading cursor's sequence and head
  int c_s = -1, c_head = -1, c_group = -1, c_page = -1;
  float c_ks = 0.0f, c_vs = 0.0f;
  u64 loaded = begin;

  auto load = [&](int stage) {
    if (loaded < end) {
      const int tok = (ld.q.first + ld.unit) * T;
      const int block = tok / kPage, group = block & ~31;
      if (ld.s != c_s || ld.head != c_head || group != c_group) {
        c_s = ld.s;
        c_head = ld.head;
        c_group = group;
        c_page = -1;
        if ((group + lane) * kPage < ld.q.len)
          c_page = p.table[(size_t)ld.s * p.table_ld + group + lane];
        if (!page_ok(c_page, p.pages)) {
          if ((group + lane) * kPage < ld.q.len) atomicCAS(p.err, 0, KERR_PLACE);
          c_page = -1;
        }
        if (c_page >= 0) {
          c_ks = bf16_bits(p.ks[(size_t)c_page * p.kv_heads + ld.head]);
          c_vs = bf16_bits(p.vs[(size_t)c_page * p.kv_heads + ld.head]);
        }
      }
      const int page = __shfl_sync(0xffffffffu, c_page, block - group);
      const float ks = __shfl_sync(0xffffffffu, c_ks, block - group);
      const float vs = __shfl_sync(0xffffffffu, c_vs, block - group);
      if (lane == 0) heads[stage] = make_float4(ks, vs, page < 0 ? 0.0f : 1.0f, 0.0f);
      if (page >= 0) {
        const size_t off = ((size_t)page * p.kv_heads + ld.head) * (size_t)(kPage * D) +
                           (size_t)(tok % kPage) * D;
        const uint32_t dst = ring + (uint32_t)(stage * C::kStageBytes);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int x = i * 32 + lane, r = x / (D / 16), ch = x % (D / 16);
          cp_async16(dst + kv_place<D, false>(r, ch), p.k + off + (size_t)x * 16);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int x = i * 32 + lane, r = x / (D / 16), ch = x % (D / 16);
          cp_async16(dst + 4096u + kv_place<D, true>(r, ch), p.v + off + (size_t)x * 16);
        }
      }
      ++loaded;
      ld.next(p);
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < C::kStages - 1; ++i) load(i);

  uint32_t qf[D / 16][4];
  float o[C::kOT][4];
  float qs[2], m[2], l[2];
  float ref = 0.0f;                                    // the scale O is held in (0: none yet)
  int lo[2], hi[2], rr[2];
  bool fresh = true;
  int stage = 0;

  for (u64 x = begin; x < end; ++x) {
    if (fresh) {
      // a tile begins (or this worker's share of it): its queries
      fresh = false;
      ref = 0.0f;
#pragma unroll
      for (int t = 0; t < C::kOT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[t][e] = 0.0f;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = at.tile * kTileRows + g + 8 * h;
        const int tok = r / p.group, head = at.head * p.group + r % p.group;
        const bool valid = tok < at.q.n;
        // rows past the tile's last are computed and never stored
        rr[h] = valid ? r : -1;
        const int pos = at.q.len - at.q.n + tok;
        lo[h] = valid ? key_low(pos, p.window) : 0;
        hi[h] = valid ? key_high(pos, at.q.len, 1) : INT_MAX;
        m[h] = -INFINITY;
        l[h] = 0.0f;
        const __nv_bfloat16* q = p.q + (size_t)(at.q.row0 + tok) * p.ldq + (size_t)head * D;
        uint32_t most = 0;
        uint4 w[D / 64][2];
#pragma unroll
        for (int j = 0; j < D / 64; ++j)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            w[j][i] = make_uint4(0, 0, 0, 0);
            if (valid) w[j][i] = *reinterpret_cast<const uint4*>(q + j * 64 + cc * 16 + i * 8);
            const uint32_t a = __vmaxu2(w[j][i].x & 0x7fff7fffu, w[j][i].y & 0x7fff7fffu);
            const uint32_t b = __vmaxu2(w[j][i].z & 0x7fff7fffu, w[j][i].w & 0x7fff7fffu);
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
        qs[h] = p.c * __uint_as_float((uint32_t)(127 - 8 + ex) << 23);
#pragma unroll
        for (int j = 0; j < D / 64; ++j)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t words[4] = {w[j][i].x, w[j][i].y, w[j][i].z, w[j][i].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              // 8 bf16 of piece half i: k steps 2 i and 2 i + 1
              const float a = __uint_as_float(words[e] << 16) * up;
              const float b = __uint_as_float(words[e] & 0xffff0000u) * up;
              qf[j * 4 + i * 2 + (e >> 1)][(e & 1) * 2 + h] = pack_f16(a, b);
            }
          }
      }
    }

    cp_async_wait<C::kStages - 2>();
    __syncwarp();
    load((stage + C::kStages - 1) % C::kStages);
    const float4 head = heads[stage];
    const uint32_t kb = ring + (uint32_t)(stage * C::kStageBytes), vb = kb + 4096u;
    if (head.z != 0.0f) {
      const int j0 = (at.q.first + at.unit) * T;
      float sc[C::kNT][4];
#pragma unroll
      for (int t = 0; t < C::kNT; ++t) {
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[t][e] = 0.0f;
#pragma unroll
        for (int j = 0; j < D / 64; ++j) {
          const uint4 w = lds128(kb + kv_place<D, false>(t * 8 + g, j * 4 + cc));
          const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const uint32_t y = words[u] ^ 0x80808080u;
            const uint32_t* a = qf[j * 4 + u];
            mma_f16(sc[t], a[0], a[1], a[2], a[3], f16_pair(y, false), f16_pair(y, true));
          }
        }
      }
      // exponents of two: score * qs * K's scale, masked where a row does not look
      const float f0 = qs[0] * head.x, f1 = qs[1] * head.x;
      float mx0 = -INFINITY, mx1 = -INFINITY;
      const bool part = j0 + T > hi[0] || j0 + T > hi[1] || j0 < lo[0] || j0 < lo[1];
      const bool masked = __any_sync(0xffffffffu, part);
#pragma unroll
      for (int t = 0; t < C::kNT; ++t) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          sc[t][e] *= f0;
          sc[t][2 + e] *= f1;
          if (masked) {
            const int j = j0 + t * 8 + 2 * cc + e;
            if (j < lo[0] || j >= hi[0]) sc[t][e] = -INFINITY;
            if (j < lo[1] || j >= hi[1]) sc[t][2 + e] = -INFINITY;
          }
          mx0 = fmaxf(mx0, sc[t][e]);
          mx1 = fmaxf(mx1, sc[t][2 + e]);
        }
      }
      mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 1));
      mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 1));
      mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 2));
      mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 2));
      // O is held in units of `ref`, 1/32 of a V scale met before, and P carries
      // the page's scale over it.  ref moves when that leaves [1/2, 512]: P, at
      // most 2^kKvGrow, then stays inside f16's range and loses bits (below its
      // normal 2^-14) only 2^13 under the row's largest
      const float vs = head.y;
      float fo = 1.0f;
      if (vs > 0.0f && vs <= FLT_MAX && !(vs <= ref * 512.0f && vs >= ref * 0.5f)) {
        fo = ref * 32.0f / vs;
        ref = vs * 0.03125f;
      }
      const float ratio = ref > 0.0f ? vs / ref : vs;
      float f[2] = {fo, fo};
      if (mx0 > m[0] + kKvGrow) {
        const float d = fast_exp2(m[0] - mx0);
        m[0] = mx0;
        l[0] *= d;
        f[0] *= d;
      }
      if (mx1 > m[1] + kKvGrow) {
        const float d = fast_exp2(m[1] - mx1);
        m[1] = mx1;
        l[1] *= d;
        f[1] *= d;
      }
      if (__any_sync(0xffffffffu, f[0] != 1.0f || f[1] != 1.0f)) {
#pragma unroll
        for (int t = 0; t < C::kOT; ++t) {
          o[t][0] *= f[0];
          o[t][1] *= f[0];
          o[t][2] *= f[1];
          o[t][3] *= f[1];
        }
      }
      const float n0 = m[0] == -INFINITY ? 0.0f : m[0], n1 = m[1] == -INFINITY ? 0.0f : m[1];
      uint32_t pf[C::kNT][2];
#pragma unroll
      for (int t = 0; t < C::kNT; ++t) {
        float pr[4];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          pr[e] = fast_exp2(sc[t][e] - n0);
          pr[2 + e] = fast_exp2(sc[t][2 + e] - n1);
        }
        l[0] += pr[0] + pr[1];
        l[1] += pr[2] + pr[3];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float w = pr[e] * ratio;
          // a masked place stays 0 when the page's scale is not finite
          pr[e] = masked && pr[e] == 0.0f ? 0.0f : w;
        }
        pf[t][0] = pack_f16(pr[0], pr[1]);
        pf[t][1] = pack_f16(pr[2], pr[3]);
      }
#pragma unroll
      for (int s = 0; s < T / 16; ++s) {
        const int r = s * 16 + 2 * cc;
        const uint32_t a0 = pf[2 * s][0], a1 = pf[2 * s][1];
        const uint32_t a2 = pf[2 * s + 1][0], a3 = pf[2 * s + 1][1];
        // four output columns from one word of each of the lane's four keys
        auto four = [&](int base, uint32_t w0, uint32_t w1, uint32_t w8, uint32_t w9) {
          w0 ^= 0x80808080u;
          w1 ^= 0x80808080u;
          w8 ^= 0x80808080u;
          w9 ^= 0x80808080u;
          const uint32_t x0 = __byte_perm(w0, w1, 0x5140), x1 = __byte_perm(w0, w1, 0x7362);
          const uint32_t y0 = __byte_perm(w8, w9, 0x5140), y1 = __byte_perm(w8, w9, 0x7362);
          mma_f16(o[base + 0], a0, a1, a2, a3, f16_pair(x0, false), f16_pair(y0, false));
          mma_f16(o[base + 1], a0, a1, a2, a3, f16_pair(x0, true), f16_pair(y0, true));
          mma_f16(o[base + 2], a0, a1, a2, a3, f16_pair(x1, false), f16_pair(y1, false));
          mma_f16(o[base + 3], a0, a1, a2, a3, f16_pair(x1, true), f16_pair(y1, true));
        };
        if constexpr (D == 64) {
          const uint32_t sub = (uint32_t)(g & 1) * 8u;
          const uint2 w0 = lds64(vb + kv_place<D, true>(r, g >> 1) + sub);
          const uint2 w1 = lds64(vb + kv_place<D, true>(r + 1, g >> 1) + sub);
          const uint2 w8 = lds64(vb + kv_place<D, true>(r + 8, g >> 1) + sub);
          const uint2 w9 = lds64(vb + kv_place<D, true>(r + 9, g >> 1) + sub);
          four(0, w0.x, w1.x, w8.x, w9.x);
          four(4, w0.y, w1.y, w8.y, w9.y);
        } else {
#pragma unroll
          for (int w = 0; w < D / 128; ++w) {
            const uint4 w0 = lds128(vb + kv_place<D, true>(r, w * 8 + g));
            const uint4 w1 = lds128(vb + kv_place<D, true>(r + 1, w * 8 + g));
            const uint4 w8 = lds128(vb + kv_place<D, true>(r + 8, w * 8 + g));
            const uint4 w9 = lds128(vb + kv_place<D, true>(r + 9, w * 8 + g));
            four(w * 16 + 0, w0.x, w1.x, w8.x, w9.x);
            four(w * 16 + 4, w0.y, w1.y, w8.y, w9.y);
            four(w * 16 + 8, w0.z, w1.z, w8.z, w9.z);
            four(w * 16 + 12, w0.w, w1.w, w8.w, w9.w);
          }
        }
      }
    }
    stage = (stage + 1) % C::kStages;

    const bool tile_end = at.unit + 1 == at.q.units;
    if (tile_end || x + 1 == end) {
      const u64 seg = (u64)at.unit;                    // stages of the tile before this one
      const bool from_start = x - begin >= seg;        // this worker had the tile's first
      constexpr int E = D / 4;                         // values of a lane's row
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
        if (rr[h] < 0) continue;
        if (tile_end && from_start) {
          const int tok = rr[h] / p.group, head_q = at.head * p.group + rr[h] % p.group;
          __nv_bfloat16* dst = p.o + (size_t)(at.q.row0 + tok) * p.ldo + (size_t)head_q * D;
          const bool sees = hi[h] > lo[h];
          const float norm = (ref > 0.0f ? ref : 1.0f) / l[h];
#pragma unroll
          for (int e = 0; e < E; e += 8) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
              w[i] = sees ? pack_bf16(kv_acc<D>(o, h, e + 2 * i) * norm,
                                      kv_acc<D>(o, h, e + 2 * i + 1) * norm)
                          : 0u;
            const int col = D == 64 ? cc * 16 + e : (e / 32) * 128 + cc * 32 + e % 32;
            *reinterpret_cast<uint4*>(dst + col) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        } else {
          // its first tile goes to place 0, its last to 1 (0 where they are one)
          const int place = x - begin >= (u64)at.unit + 1 ? 1 : 0;
          const size_t site = (me * 2 + place) * kTileRows + (g + 8 * h);
          const float norm = ref > 0.0f ? ref : 1.0f;
          float* dst = p.part_o + site * D;
#pragma unroll
          for (int e = 0; e < E; e += 4) {
            const int col = D == 64 ? cc * 16 + e : (e / 32) * 128 + cc * 32 + e % 32;
            *reinterpret_cast<float4*>(dst + col) =
                make_float4(kv_acc<D>(o, h, e) * norm, kv_acc<D>(o, h, e + 1) * norm,
                            kv_acc<D>(o, h, e + 2) * norm, kv_acc<D>(o, h, e + 3) * norm);
          }
          if (cc == 0) *reinterpret_cast<float2*>(p.part_ml + site * 2) = make_float2(m[h], l[h]);
        }
      }
      fresh = true;
    }
    at.next(p);
  }
  cp_async_wait<0>();
}

// Joins the tiles that several workers share: with M the largest of their
// maxima, o = sum 2^(m_i - M) O_i / sum 2^(m_i - M) l_i.  Writes zeros for the
// rows of sequences without keys, which no worker has.  A block a (row tile,
// kv head); its warps share the parts of a row where there are many, and the
// rows where there are few.
constexpr int kMergeThreads = 256;

template <int D>
__global__ void __launch_bounds__(kMergeThreads) kv8_merge_kernel(const __grid_constant__ KvAttn p)
{
  constexpr int N = kMergeThreads, W = N / 32, E = D / 32;
  __shared__ u64 s_pre[N + 1];
  __shared__ float s_o[W][D];
  __shared__ float s_l[W];
  pdl_wait();
  pdl_trigger();
  const int warp = (int)threadIdx.x >> 5, lane = (int)threadIdx.x & 31;
  const int head = (int)blockIdx.y;
  const int slot = (int)blockIdx.x;
  // tiles of rows are slots of cu * group rows
  int lo = 0, hi = p.seqs;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (slot_base(clamp_int(p.cu[mid], 0, p.rows) * p.group, mid, kTileRows, 1) <= slot) lo = mid;
    else hi = mid;
  }
  const int s = lo;
  const KvSeq q = kv_seq<D>(p, s);
  const int tile = slot - slot_base(q.row0 * p.group, s, kTileRows, 1);
  if (tile < 0 || tile >= q.tiles) return;
  const int rows = min(kTileRows, q.n * p.group - tile * kTileRows);
  if (q.units == 0) {
    for (int i = (int)threadIdx.x; i < rows * D; i += N) {
      const int r = tile * kTileRows + i / D;
      p.o[(size_t)(q.row0 + r / p.group) * p.ldo + (size_t)(head * p.group + r % p.group) * D +
          i % D] = __float2bfloat16_rn(0.0f);
    }
    return;
  }
  kv_plan<D, N>(p, s_pre);
  const u64 all = s_pre[N];
  const u64 workers = min((u64)p.workers, all);
  // the work before this sequence
  const int each = (p.seqs + N - 1) / N;
  u64 at = s_pre[s / each];
  for (int i = s / each * each; i < s; ++i) at += kv_work<D>(p, kv_seq<D>(p, i));
  at += ((u64)head * q.tiles + tile) * (u64)q.units;
  const u64 first = work_owner(all, workers, at);
  const u64 last = work_owner(all, workers, at + q.units - 1);
  if (first == last) return;                           // written by its worker
  const int parts = (int)(last - first) + 1;
  const u64 place0 = work_bound(all, workers, first) < at ? 1 : 0;
  auto site = [&](int i, int r) {
    return ((first + i) * 2 + (i == 0 ? place0 : 0)) * kTileRows + r;
  };
  const bool few = parts <= W;                         // a warp a row
  for (int r0 = 0; r0 < rows; r0 += few ? W : 1) {
    const int r = few ? r0 + warp : r0;
    const bool active = r < rows;
    float M = -INFINITY;
    if (active)
      for (int i = lane; i < parts; i += 32) M = fmaxf(M, p.part_ml[site(i, r) * 2]);
    for (int w = 16; w > 0; w >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, w));
    float acc[E], l = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.0f;
    if (active) {
#pragma unroll 4
      for (int i = few ? 0 : warp; i < parts; i += few ? 1 : W) {
        const u64 at_i = site(i, r);
        const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + at_i * 2);
        // a part that saw nothing has sum 0 and O 0
        const float f = ml.x == -INFINITY ? (ml.y == 0.0f ? 0.0f : 1.0f) : fast_exp2(ml.x - M);
        l = fmaf(f, ml.y, l);
        const float* src = p.part_o + at_i * D;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = fmaf(f, src[e * 32 + lane], acc[e]);
      }
    }
    if (!few) {
#pragma unroll
      for (int e = 0; e < E; ++e) s_o[warp][e * 32 + lane] = acc[e];
      if (lane == 0) s_l[warp] = l;
      __syncthreads();
    }
    const int rt = tile * kTileRows + r;
    const int tok = rt / p.group, pos = q.len - q.n + tok;
    const bool sees = key_high(pos, q.len, 1) > key_low(pos, p.window);
    __nv_bfloat16* dst = p.o + (size_t)(q.row0 + tok) * p.ldo +
                         (size_t)(head * p.group + rt % p.group) * D;
    if (few) {
      if (active)
#pragma unroll
        for (int e = 0; e < E; ++e)
          dst[e * 32 + lane] = __float2bfloat16_rn(sees ? acc[e] / l : 0.0f);
    } else {
      for (int d = (int)threadIdx.x; d < D; d += N) {
        float a = 0.0f, b = 0.0f;
#pragma unroll
        for (int w = 0; w < W; ++w) {
          a += s_o[w][d];
          b += s_l[w];
        }
        dst[d] = __float2bfloat16_rn(sees ? a / b : 0.0f);
      }
      __syncthreads();
    }
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

dim3 kv_pages_grid(const Kv8Cache& c, const Kv8Rows& r)
{
  return dim3((unsigned)slot_count(r.rows, r.seqs, kPage, 2), (unsigned)c.kv_heads, 2);
}

template <int D>
int kv_attn_launch(const Kv8Attention& a, int num_sms, int* err, cudaStream_t s)
{
  using C = KvCfg<D>;
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
  const int slots = slot_count(p.rows * p.group, p.seqs, kTileRows, 1);
  // two blocks an SM, fewer where the longest sequences cannot fill them
  const long long units = (long long)slots * p.kv_heads * ((a.max_len + C::kTok - 1) / C::kTok + 1);
  const long long blocks = (units + C::kWarps - 1) / C::kWarps;
  const int grid = (int)(blocks < 2 * num_sms ? (blocks < 1 ? 1 : blocks) : 2 * num_sms);
  p.workers = grid * C::kWarps;
  p.part_o = a.workspace;
  p.part_ml = a.workspace + (size_t)p.workers * 2 * kTileRows * D;
  static std::atomic<unsigned long long> attr{0};
  if (!smem_limit_once(kv8_attention_kernel<D>, C::kSmem, attr)) return -1;
  launch_k(kv8_attention_kernel<D>, dim3((unsigned)grid), dim3(C::kWarps * 32), C::kSmem, s, 1, p);
  if (launched() != 0) return -1;
  launch_k(kv8_merge_kernel<D>, dim3((unsigned)slots, (unsigned)p.kv_heads), dim3(kMergeThreads), 0,
           s, 1, p);
  return launched();
}

}  // namespace

int launch_kv8_append(const Kv8Cache& c, const Kv8Rows& r, const __nv_bfloat16* k, int ldk,
                      const __nv_bfloat16* v, int ldv, int* err, cudaStream_t s)
{
  const KvPages p = kv_pages(c, r, err);
  const dim3 grid = kv_pages_grid(c, r);
  switch (c.head_dim) {
    case 64: launch_k(kv8_append_kernel<64>, grid, dim3(kAppendThreads), 0, s, 1, p, k, ldk, v, ldv); break;
    case 128: launch_k(kv8_append_kernel<128>, grid, dim3(kAppendThreads), 0, s, 1, p, k, ldk, v, ldv); break;
    case 256: launch_k(kv8_append_kernel<256>, grid, dim3(kAppendThreads), 0, s, 1, p, k, ldk, v, ldv); break;
    default: return -2;
  }
  return launched();
}

int launch_kv8_read(const Kv8Cache& c, const Kv8Rows& r, __nv_bfloat16* k, int ldk,
                    __nv_bfloat16* v, int ldv, int* err, cudaStream_t s)
{
  const KvPages p = kv_pages(c, r, err);
  const dim3 grid = kv_pages_grid(c, r);
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
  return (size_t)(2 * num_sms) * 4 * 2 * kTileRows * (size_t)(head_dim + 2) * sizeof(float);
}

int launch_kv8_attention(const Kv8Attention& a, int num_sms, int* err, cudaStream_t s)
{
  switch (a.cache.head_dim) {
    case 64: return kv_attn_launch<64>(a, num_sms, err, s);
    case 128: return kv_attn_launch<128>(a, num_sms, err, s);
    case 256: return kv_attn_launch<256>(a, num_sms, err, s);
    default: return -2;
  }
}

}  // namespace ltx
