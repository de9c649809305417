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
// A CTA holds two query tiles (head widths 64 and 128) or one (256: its O
// takes 256 of the 512 TMEM columns), the layout of attention_tc.cu:
//   warp 0      TMA: Q, then K and V tiles in the order the MMAs use them,
//               through one ring of equal slots
//   warp 1      MMA: S = Q K^T, O += P V with P read from TMEM
//   warps 4-..  softmax, eight warps a query tile, two for each TMEM lane
//               quarter (64 score columns each)
// With two tiles one's MMAs run under the other's softmax; with one tile the
// scores are double-buffered, so S of key tile j + 1 runs under softmax j.
// V is used as TMA lays it down, [key][64 dims] in 128-byte swizzled rows: the
// MN-major form of the MMA's B operand, no transposed copy.
//
// What P multiplies must not matter where P is 0, but 0 * NaN is NaN: a key
// tile may hold V rows that no row, or not this row, may see (the next
// sequence's, later tokens').  A row that ends up with a NaN is therefore
// computed again by repair_row from the keys it sees alone; a NaN that belongs
// there comes out the same.
//
// Every wait is bounded; a timeout sets the context's error word and the CTA
// drains and exits.
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
constexpr int kKeys = 128;        // keys of a tile
constexpr float kGrow = 8.0f;     // log2 of the largest P before O is rescaled

enum : int {
  PERR_PRODUCER = 0x65,
  PERR_MMA = 0x66,
  PERR_SOFTMAX = 0x67,
  PERR_DRAIN = 0x68,
};

template <int D>
struct PkCfg {
  static constexpr int kTiles = D == 256 ? 1 : 2;      // query tiles of a CTA
  static constexpr int kThreads = 128 + 256 * kTiles;
  static constexpr int kAtom = 128 * 128;              // 128 rows x 128 B (64 dims)
  static constexpr int kQTile = (D / 64) * kAtom;
  // One ring slot: a K or V tile, or half of one at width 256 (K: 128 dims
  // of 128 keys; V: all dims of 64 keys).
  static constexpr int kParts = D == 256 ? 2 : 1;
  static constexpr int kSlot = (D / 64) * kAtom / kParts;
  static constexpr int kSlots = D == 64 ? 8 : (D == 128 ? 4 : 5);
  static constexpr int kVKeys = kKeys / kParts;        // keys of a V slot
  // row maxima of the two half-row warps: [tile][parity][half][row] f32
  static constexpr int kMaxBytes = kTiles * 4 * kRows * 4;
  static constexpr int kSmem = kTiles * kQTile + kSlots * kSlot + kMaxBytes + 256;
  static constexpr uint32_t kOCol = 0;                 // O_t at t * D
  static constexpr uint32_t kSCol = kTiles * D;        // two score buffers
  static_assert(kSCol + 2 * kKeys <= 512, "TMEM columns");
  static_assert(kSmem <= 232448, "shared memory");
  static_assert((2 * kSlots + 8) * 8 + 8 <= 256, "barriers");
};

struct PkParams {
  const __nv_bfloat16 *q, *k, *v;
  __nv_bfloat16* o;
  int ldq, ldk, ldv, ldo;
  const int *cu_q, *cu_k;
  int seqs, rows, keys;     // rows of q and o, rows of k and v
  int kv_heads, group, tq;  // tq: tokens of a query tile
  int causal, window;
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

// Columns [col0, col0 + D / 2) of one output row from the keys [lo, hi) of its
// sequence alone (rows key0 + j of k and v), in f32, by one warp.
template <int D>
__device__ __noinline__ void repair_row(const PkParams& p, int row, int head, int kvh, int key0,
                                        int lo, int hi, int col0)
{
  constexpr int W = D / 64;                       // dims of a lane
  const int lane = (int)lane_id();
  const __nv_bfloat16* q = p.q + (size_t)row * p.ldq + (size_t)head * D;
  float m = -INFINITY, l = 0.0f, acc[W];
  for (int e = 0; e < W; ++e) acc[e] = 0.0f;
  for (int j0 = lo; j0 < hi; j0 += 32) {
    const int n = min(32, hi - j0);
    float s = -INFINITY;
    if (lane < n) {
      const __nv_bfloat16* k = p.k + (size_t)(key0 + j0 + lane) * p.ldk + (size_t)kvh * D;
      float dot = 0.0f;
      for (int d = 0; d < D; ++d) dot = fmaf(__bfloat162float(q[d]), __bfloat162float(k[d]), dot);
      s = dot * p.c;
    }
    float mx = s;
    for (int w = 16; w > 0; w >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
    const float m_new = fmaxf(m, mx);
    const float r = m_new == -INFINITY ? 0.0f : m_new;
    const float f = m == -INFINITY ? 0.0f : exp2f(m - r);
    const float pj = lane < n ? exp2f(s - r) : 0.0f;
    m = m_new;
    l = l * f + pj;                               // this lane's share
    for (int e = 0; e < W; ++e) acc[e] *= f;
    for (int i = 0; i < n; ++i) {
      const float pi = __shfl_sync(0xffffffffu, pj, i);
      const __nv_bfloat16* v = p.v + (size_t)(key0 + j0 + i) * p.ldv + (size_t)kvh * D + col0;
      for (int e = 0; e < W; ++e) acc[e] = fmaf(pi, __bfloat162float(v[lane * W + e]), acc[e]);
    }
  }
  for (int w = 16; w > 0; w >>= 1) l += __shfl_xor_sync(0xffffffffu, l, w);
  __nv_bfloat16* o = p.o + (size_t)row * p.ldo + (size_t)head * D + col0;
  for (int e = 0; e < W; ++e) o[lane * W + e] = __float2bfloat16_rn(acc[e] / l);
}

template <int D>
__global__ void __launch_bounds__(PkCfg<D>::kThreads, 1)
    pk_attention_kernel(const __grid_constant__ CUtensorMap tm_q,
                        const __grid_constant__ CUtensorMap tm_k,
                        const __grid_constant__ CUtensorMap tm_v,
                        const __grid_constant__ PkParams p)
{
  using C = PkCfg<D>;
  constexpr int T = C::kTiles, R = C::kSlots;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* s_q = smem_raw;                             // tile t at t * kQTile
  uint8_t* s_ring = s_q + T * C::kQTile;
  float (*s_mx)[2][2][kRows] =                         // [tile][parity][half][row]
      reinterpret_cast<float (*)[2][2][kRows]>(s_ring + R * C::kSlot);
  uint64_t* bars = reinterpret_cast<uint64_t*>(s_ring + R * C::kSlot + C::kMaxBytes);
  uint64_t* q_full = bars;
  uint64_t* full = q_full + 1;
  uint64_t* empty = full + R;
  uint64_t* s_full = empty + R;
  uint64_t* p_full = s_full + 2;
  uint64_t* o_done = p_full + 2;
  uint64_t* drain = o_done + 2;
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* s_abort = reinterpret_cast<volatile int*>(s_tmem + 1);
  const int warp = threadIdx.x >> 5;
  const uint32_t lane = threadIdx.x & 31;
  if ((smem_u32(smem_raw) & 1023u) != 0) {             // the swizzle's atom
    if (threadIdx.x == 0) atomicCAS(p.err, 0, PERR_DRAIN);
    return;
  }

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    for (int i = 0; i < R; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 8);
      mbar_init(&o_done[i], 1);
    }
    mbar_init(drain, 1);
    *s_abort = 0;
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  if (warp == 1) {
    tmem_alloc(s_tmem, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *s_tmem;
  pdl_wait();
  pdl_trigger();

  // the CTA's sequence, tokens and keys.  Slots run backwards, so that a
  // causal sequence's longest tiles start first.
  const int kvh = (int)(blockIdx.x % (unsigned)p.kv_heads);
  const int slots = slot_count(p.rows, p.seqs, T * p.tq, 1);
  const int slot = slots - 1 - (int)(blockIdx.x / (unsigned)p.kv_heads);
  const int seq = find_seq(p.cu_q, p.seqs, p.rows, T * p.tq, 1, slot);
  const int row0 = clamp_int(p.cu_q[seq], 0, p.rows);
  const int nq = clamp_int(p.cu_q[seq + 1], row0, p.rows) - row0;
  const int key0 = clamp_int(p.cu_k[seq], 0, p.keys);
  const int nk = clamp_int(p.cu_k[seq + 1], key0, p.keys) - key0;
  const int tok0 = max(0, slot - slot_base(row0, seq, T * p.tq, 1)) * (T * p.tq);
  // keys any of the rows sees: from the first row's low to the last one's high
  const int shift = nk - nq;
  const int jb = key_low(shift + tok0, p.window);
  int n_t[2] = {0, 0};                                 // key tiles of each query tile
#pragma unroll
  for (int t = 0; t < T; ++t) {
    const int a = tok0 + t * p.tq, b = min(a + p.tq, nq);
    if (b > a) {
      const int je = key_high(shift + b - 1, nk, p.causal);
      n_t[t] = je > jb ? (je - jb + kKeys - 1) / kKeys : 0;
    }
  }
  const int n = max(n_t[0], n_t[1]);

  if (warp == 0) {
    // ------------------------------------------------------------- TMA
    if (lane == 0 && n > 0) {
      uint32_t armed = 0, armed_par = 0;
      const int boxes = C::kTiles * (D / 64);
      mbar_arrive_expect_tx(q_full, (uint32_t)(boxes * p.group * p.tq * 128));
      for (int t = 0; t < T; ++t)
        for (int a = 0; a < D / 64; ++a)
          tma_load_3d(&tm_q, q_full, s_q + t * C::kQTile + a * C::kAtom, a * 64,
                      kvh * p.group, row0 + tok0 + t * p.tq);
      int used = 0;
      bool ok = true;
      // one slot: `v` selects V, part its half at width 256
      auto load = [&](bool v, int j) {
        for (int part = 0; ok && part < C::kParts; ++part, ++used) {
          const int st = used % R;
          const uint32_t ph = (uint32_t)(used / R) & 1u;
          ok = mbar_wait(&empty[st], ph ^ 1u, s_abort, p.err, PERR_PRODUCER);
          if (!ok) break;
          uint8_t* dst = s_ring + st * C::kSlot;
          const int key = key0 + jb + j * kKeys;
          mbar_arrive_expect_tx(&full[st], C::kSlot);
          if (v) {
            for (int a = 0; a < D / 64; ++a)
              tma_load_3d(&tm_v, &full[st], dst + a * C::kVKeys * 128, a * 64, kvh,
                          key + part * C::kVKeys);
          } else {
            constexpr int A = D / 64 / C::kParts;
            for (int a = 0; a < A; ++a)
              tma_load_3d(&tm_k, &full[st], dst + a * C::kAtom, (part * A + a) * 64, kvh, key);
          }
          armed |= 1u << st;
          armed_par = (armed_par & ~(1u << st)) | (ph << st);
        }
      };
      load(false, 0);
      for (int j = 0; ok && j < n; ++j) {
        if (T == 1 && j + 1 < n) load(false, j + 1);
        load(true, j);
        if (T == 2 && j + 1 < n) load(false, j + 1);
      }
      // Every load lands before the CTA may exit.
      volatile int no_abort = 0;
      mbar_wait(q_full, 0, &no_abort, p.err, PERR_DRAIN);
      for (int st = 0; st < R; ++st)
        if (armed & (1u << st))
          mbar_wait(&full[st], (armed_par >> st) & 1u, &no_abort, p.err, PERR_DRAIN);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------- MMA
    if (lane == 0 && n > 0) {
      constexpr uint32_t idesc_s = idesc_bf16(kRows, kKeys);
      constexpr uint32_t idesc_o = idesc_bf16_bmn(kRows, D);
      int used = 0;                                    // ring slots taken so far
      auto wait_slots = [&](int at) {
        for (int part = 0; part < C::kParts; ++part) {
          const int u = at + part;
          if (!mbar_wait(&full[u % R], (uint32_t)(u / R) & 1u, s_abort, p.err, PERR_MMA))
            return false;
        }
        tc_fence_after();
        return true;
      };
      auto free_slots = [&](int at) {
        for (int part = 0; part < C::kParts; ++part) umma_commit(&empty[(at + part) % R]);
      };
      // scores of key tile in slot(s) `at` for query tile t into buffer b
      auto issue_s = [&](int t, int b, int at) {
        const uint32_t sq = smem_u32(s_q + t * C::kQTile);
        const uint32_t d = tmem + C::kSCol + (uint32_t)b * kKeys;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          constexpr int A = D / 64 / C::kParts;        // 64-dim atoms of a slot
          const int a = kk >> 2;
          const uint32_t sk = smem_u32(s_ring + ((at + a / A) % R) * C::kSlot) +
                              (uint32_t)((a % A) * C::kAtom);
          umma_f16_ss(d, sdesc_k128_sw128(sq + (uint32_t)(a * C::kAtom)) + (uint64_t)(2 * (kk & 3)),
                      sdesc_k128_sw128(sk) + (uint64_t)(2 * (kk & 3)), idesc_s, kk > 0 ? 1u : 0u);
        }
        umma_commit(&s_full[b]);
      };
      auto issue_pv = [&](int t, int b, int at, bool first) {
        const uint32_t pa = tmem + C::kSCol + (uint32_t)b * kKeys;
#pragma unroll
        for (int kk = 0; kk < kKeys / 16; ++kk) {
          constexpr int KS = C::kVKeys / 16;           // k steps of a slot
          const uint32_t sv = smem_u32(s_ring + ((at + kk / KS) % R) * C::kSlot) +
                              (uint32_t)((kk % KS) * 16 * 128);
          umma_f16_ts(tmem + C::kOCol + (uint32_t)(t * D), pa + (uint32_t)(kk * 8),
                      sdesc_mn_sw128(sv, C::kVKeys * 128), idesc_o, !first || kk > 0 ? 1u : 0u);
        }
        umma_commit(&o_done[t]);
      };
      bool ok = mbar_wait(q_full, 0, s_abort, p.err, PERR_MMA) && wait_slots(0);
      if (T == 2) {
        if (ok) {
          for (int t = 0; t < T; ++t)
            if (n_t[t] > 0) issue_s(t, t, 0);
          free_slots(0);
        }
        used = C::kParts;
        for (int j = 0; ok && j < n; ++j) {
          const int av = used, ak = used + C::kParts;  // V_j, K_{j+1}
          const bool more = j + 1 < n;
          bool have_v = false, have_k = false;
          for (int t = 0; ok && t < T; ++t) {
            if (j >= n_t[t]) continue;
            // P V, then the tile's next S (in order: the S MMA overwrites the
            // buffer only after this P V has read P from it)
            ok = mbar_wait(&p_full[t], (uint32_t)j & 1u, s_abort, p.err, PERR_MMA) &&
                 (have_v || wait_slots(av));
            if (!ok) break;
            have_v = true;
            tc_fence_after();
            issue_pv(t, t, av, j == 0);
            if (j + 1 < n_t[t]) {
              ok = have_k || wait_slots(ak);
              if (!ok) break;
              have_k = true;
              issue_s(t, t, ak);
            }
          }
          if (!ok) break;
          free_slots(av);
          if (more) free_slots(ak);
          used = ak + (more ? C::kParts : 0);
        }
      } else {
        int ak[2] = {0, 0}, av = 0;
        if (ok) {
          issue_s(0, 0, 0);
          free_slots(0);
        }
        used = C::kParts;
        for (int j = 0; ok && j < n; ++j) {
          if (j + 1 < n) {
            ak[0] = used;
            used += C::kParts;
            ok = wait_slots(ak[0]);
            if (!ok) break;
            issue_s(0, (j + 1) & 1, ak[0]);
            free_slots(ak[0]);
          }
          av = used;
          used += C::kParts;
          ok = mbar_wait(&p_full[j & 1], (uint32_t)(j >> 1) & 1u, s_abort, p.err, PERR_MMA) &&
               wait_slots(av);
          if (!ok) break;
          issue_pv(0, j & 1, av, j == 0);
          free_slots(av);
        }
      }
      umma_commit(drain);
      volatile int no_abort = 0;
      mbar_wait(drain, 0, &no_abort, p.err, PERR_DRAIN);
    }
  } else if (warp >= 4) {
    // ---------------------------------------------------------- softmax
    // Within a tile the first four warps take score columns [0, 64), the next
    // four [64, 128) of the same rows.
    const int t = (warp - 4) >> 3;
    const int hh = ((warp - 4) >> 2) & 1;
    const int r = (warp & 3) * 32 + (int)lane;
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t ocol = tmem + lane_base + C::kOCol + (uint32_t)(t * D + hh * (D / 2));
    const float c = p.c;
    const int nt = n_t[t];
    // this thread's row: token and head, and the keys it sees
    const int tok = tok0 + t * p.tq + r / p.group;
    const bool valid_row = r < p.tq * p.group && tok < nq;
    const int lo = key_low(shift + tok, p.window);
    const int hi = valid_row ? key_high(shift + tok, nk, p.causal) : 0;
    // key tiles that every valid row of this query tile sees whole
    const int a_tok = tok0 + t * p.tq, b_tok = min(a_tok + p.tq, nq) - 1;
    const int all_lo = key_low(shift + b_tok, p.window);
    const int all_hi = key_high(shift + a_tok, nk, p.causal);
    float m_run = -INFINITY, l_run = 0.0f;
    bool ok = true;
    // Every warp of a tile takes the same nt + 1 named barriers, also after an
    // abort (which then only skips the TMEM work), so none is left waiting.
    for (int i = 0; i < nt; ++i) {
      const int sb = T == 2 ? t : (i & 1);
      const uint32_t ph = T == 2 ? (uint32_t)i & 1u : (uint32_t)(i >> 1) & 1u;
      const uint32_t scol = tmem + lane_base + C::kSCol + (uint32_t)(sb * kKeys);
      ok = __all_sync(0xffffffffu, ok && mbar_wait(&s_full[sb], ph, s_abort, p.err, PERR_SOFTMAX));
      uint32_t a[32], b[32];
      tc_fence_after();
      tmem_ld32(scol + (uint32_t)(hh * 64), a);
      tmem_ld32(scol + (uint32_t)(hh * 64 + 32), b);
      tmem_wait_ld();
      const int j0 = jb + i * kKeys;
      if (j0 < all_lo || j0 + kKeys > all_hi) {
        const int from = lo - j0 - hh * 64, to = hi - j0 - hh * 64;
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          if (e < from || e >= to) a[e] = 0xff800000u;             // -inf
          if (32 + e < from || 32 + e >= to) b[e] = 0xff800000u;
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
      // the row's max over both halves: exchange through shared memory (both
      // halves have their scores in registers after this barrier, so either
      // may then overwrite the TMEM columns with P)
      s_mx[t][i & 1][hh][r] = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
      named_bar_sync(1 + t, 256);
      if (!ok) continue;
      const float m_tile = fmaxf(s_mx[t][i & 1][0][r], s_mx[t][i & 1][1][r]) * c;
      // a row's first visible tile sets its maximum; later it moves only when
      // it grows by more than 2^kGrow (until then P stays below 2^kGrow)
      const bool need = m_tile > m_run + kGrow;
      const bool rescale = i > 0 && __any_sync(0xffffffffu, need);
      float f = 1.0f;
      if (need) {
        f = fast_exp2(m_run - m_tile);
        l_run *= f;
        m_run = m_tile;
      }
      const float nm = m_run == -INFINITY ? 0.0f : -m_run;
      const unsigned long long c2 = pair2(__float_as_uint(c), __float_as_uint(c));
      const unsigned long long nm2 = pair2(__float_as_uint(nm), __float_as_uint(nm));
      unsigned long long sa = 0ull, sb2 = 0ull;
      uint32_t pk[32];
      fa3_exp(a, b, c2, nm2, pk, sa, sb2);
      tmem_st32(scol + (uint32_t)(hh * 32), pk);
      const unsigned long long st2 = fadd2(sa, sb2);
      l_run += __uint_as_float((uint32_t)st2) + __uint_as_float((uint32_t)(st2 >> 32));
      if (rescale)
        ok = __all_sync(0xffffffffu, mbar_wait(&o_done[t], (uint32_t)(i - 1) & 1u, s_abort, p.err,
                                               PERR_SOFTMAX));
      if (rescale && ok) {
        tc_fence_after();
#pragma unroll
        for (int c4 = 0; c4 < D / 64; ++c4) {
          uint32_t v[32];
          tmem_ld32(ocol + (uint32_t)(c4 * 32), v);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) * f);
          tmem_st32(ocol + (uint32_t)(c4 * 32), v);
        }
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (ok && lane == 0) mbar_arrive(&p_full[sb]);
    }
    // the row's sum over both halves (parity slot nt & 1 is free now)
    s_mx[t][nt & 1][hh][r] = l_run;
    named_bar_sync(1 + t, 256);
    const float l_row = s_mx[t][nt & 1][0][r] + s_mx[t][nt & 1][1][r];
    if (ok && nt > 0)
      ok = __all_sync(0xffffffffu, mbar_wait(&o_done[t], (uint32_t)(nt - 1) & 1u, s_abort, p.err,
                                             PERR_SOFTMAX));
    if (ok) {
      tc_fence_after();
      const bool sees = hi > lo;
      const int row = row0 + tok;
      const int head = kvh * p.group + r % p.group;
      const float g = 1.0f / l_row;
      __nv_bfloat16* orow = p.o + (size_t)row * p.ldo + (size_t)head * D + hh * (D / 2);
      bool nan = false;
#pragma unroll
      for (int c4 = 0; c4 < D / 64; ++c4) {
        uint32_t v[32];
        if (nt > 0) {
          tmem_ld32(ocol + (uint32_t)(c4 * 32), v);
          tmem_wait_ld();
        }
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          const float x = nt > 0 && sees ? __uint_as_float(v[e]) * g : 0.0f;
          nan |= x != x;
          v[e] = __float_as_uint(x);
        }
        if (valid_row) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            uint4 w;
            w.x = pack_bf16(__uint_as_float(v[8 * e + 0]), __uint_as_float(v[8 * e + 1]));
            w.y = pack_bf16(__uint_as_float(v[8 * e + 2]), __uint_as_float(v[8 * e + 3]));
            w.z = pack_bf16(__uint_as_float(v[8 * e + 4]), __uint_as_float(v[8 * e + 5]));
            w.w = pack_bf16(__uint_as_float(v[8 * e + 6]), __uint_as_float(v[8 * e + 7]));
            *reinterpret_cast<uint4*>(orow + c4 * 32 + 8 * e) = w;
          }
        }
      }
      uint32_t bad = __ballot_sync(0xffffffffu, nan && valid_row);
      while (bad != 0) {
        const int src = __ffs((int)bad) - 1;
        bad &= bad - 1;
        repair_row<D>(p, __shfl_sync(0xffffffffu, row, src), __shfl_sync(0xffffffffu, head, src),
                      kvh, key0, __shfl_sync(0xffffffffu, lo, src),
                      __shfl_sync(0xffffffffu, hi, src), hh * (D / 2));
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
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

template <int D>
int pk_launch(const PackedAttention& a, int* err, cudaStream_t s)
{
  using C = PkCfg<D>;
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
  // no keys at all: every row is empty and nothing loads through mk and mv
  const bool none = a.keys == 0;
  if (!pk_encode(&mq, a.q, D, a.heads, a.rows, a.ldq, p.group, p.tq) ||
      !pk_encode(&mk, none ? a.q : a.k, D, a.kv_heads, none ? 1 : a.keys, a.ldk, 1, kKeys) ||
      !pk_encode(&mv, none ? a.q : a.v, D, a.kv_heads, none ? 1 : a.keys, a.ldv, 1, C::kVKeys))
    return -1;
  const long long grid =
      (long long)slot_count(a.rows, a.seqs, C::kTiles * p.tq, 1) * a.kv_heads;
  if (grid > INT_MAX) return -2;
  static std::atomic<unsigned long long> attr{0};
  if (!smem_limit_once(pk_attention_kernel<D>, C::kSmem, attr)) return -1;
  launch_k(pk_attention_kernel<D>, dim3((unsigned)grid), dim3(C::kThreads), C::kSmem, s, 1, mq, mk,
           mv, p);
  return launched();
}

}  // namespace

int launch_attention_packed(const PackedAttention& a, int* err, cudaStream_t s)
{
  switch (a.head_dim) {
    case 64: return pk_launch<64>(a, err, s);
    case 128: return pk_launch<128>(a, err, s);
    case 256: return pk_launch<256>(a, err, s);
    default: return -2;
  }
}

}  // namespace ltx
