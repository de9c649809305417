// ltx25-lm-ops.cc -- argument checks of the language-model operators.
#include "ltx25-lm-ops.h"

#include <climits>
#include <cmath>
#include <cstdint>

#include "../../include/ltx25_cuda.h"

namespace ltx25 {

namespace {

// Work slots are counted in 32 bits, up to two a sequence beside those of its rows.
constexpr int kMaxSeqs = 1 << 29;

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// heads, head width and the factor of the scores
int check_heads(const char* op, int heads, int kv_heads, int head_dim, int window, float scale,
                std::string* why)
{
  const std::string o(op);
  if (heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 || heads / kv_heads > 128) {
    *why = o + ": need heads a multiple of kv_heads, at most 128 heads a kv head";
    return LTX_E_SHAPE;
  }
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) {
    *why = o + ": need head_dim 64, 128 or 256";
    return LTX_E_SHAPE;
  }
  if (window < 0) {
    *why = o + ": need window >= 0 (0: no window)";
    return LTX_E_SHAPE;
  }
  // the kernels take it times log2 e
  if (!(scale > 0.0f) || !std::isfinite(scale * 1.4426950408889634f)) {
    *why = o + ": need a scale > 0, below 2e38";
    return LTX_E_SHAPE;
  }
  return LTX_OK;
}

// a bf16 operand of `rows` rows of `cols` elements
int check_rows(const char* op, const char* name, const void* p, int ld, int rows, long long cols,
               std::string* why)
{
  if (rows == 0) return LTX_OK;
  const std::string o = std::string(op) + ": " + name;
  if (p == nullptr) {
    *why = o + " is null";
    return LTX_E_NULL;
  }
  if (!aligned(p, 16) || ld % 8 != 0) {
    *why = o + " must be 16-byte aligned with a row stride % 8 == 0";
    return LTX_E_ALIGN;
  }
  if (ld < cols) {
    *why = o + ": need a row stride of at least heads * head_dim";
    return LTX_E_SHAPE;
  }
  return LTX_OK;
}

int check_ints(const char* op, const char* name, const int* p, std::string* why)
{
  const std::string o = std::string(op) + ": " + name;
  if (p == nullptr) {
    *why = o + " is null";
    return LTX_E_NULL;
  }
  if (!aligned(p, 4)) {
    *why = o + " must be 4-byte aligned";
    return LTX_E_ALIGN;
  }
  return LTX_OK;
}

// the cache's buffers, and the offsets, starts and table of its sequences
int check_cache(const char* op, const ltx::Kv8Cache& c, const ltx::Kv8Rows& r, std::string* why)
{
  const std::string o(op);
  if (c.kv_heads <= 0 || c.kv_heads > 65535 || c.pages < 0 ||
      (c.head_dim != 64 && c.head_dim != 128 && c.head_dim != 256)) {
    *why = o + ": need pages >= 0, kv_heads 1..65535, head_dim 64, 128 or 256";
    return LTX_E_SHAPE;
  }
  if (r.seqs < 0 || r.rows < 0 || r.seqs > kMaxSeqs || r.table_ld < 1 || r.table_ld > (1 << 24)) {
    *why = o + ": need seqs 0..2^29, rows >= 0, table columns 1..2^24";
    return LTX_E_SHAPE;
  }
  if (r.seqs == 0 || r.rows == 0) return LTX_OK;
  if (c.k == nullptr || c.v == nullptr || c.ks == nullptr || c.vs == nullptr) {
    *why = o + ": a cache buffer is null";
    return LTX_E_NULL;
  }
  if (!aligned(c.k, 16) || !aligned(c.v, 16) || !aligned(c.ks, 2) || !aligned(c.vs, 2)) {
    *why = o + ": cache codes must be 16-byte, scales 2-byte aligned";
    return LTX_E_ALIGN;
  }
  int rc;
  if ((rc = check_ints(op, "cu", r.cu, why)) != LTX_OK ||
      (rc = check_ints(op, "starts / lengths", r.starts, why)) != LTX_OK)
    return rc;
  return check_ints(op, "table", r.table, why);
}

}  // namespace

int check_kv8_rows(const char* op, const ltx::Kv8Cache& c, const ltx::Kv8Rows& r, const void* k,
                   int ldk, const void* v, int ldv, std::string* why)
{
  int rc = check_cache(op, c, r, why);
  if (rc != LTX_OK || r.seqs == 0) return rc;
  const long long cols = (long long)c.kv_heads * c.head_dim;
  if ((rc = check_rows(op, "k", k, ldk, r.rows, cols, why)) != LTX_OK) return rc;
  return check_rows(op, "v", v, ldv, r.rows, cols, why);
}

int check_kv8_attention(const ltx::Kv8Attention& a, size_t workspace_bytes, size_t need,
                        std::string* why)
{
  const char* op = "kv8_attention";
  int rc = check_heads(op, a.heads, a.cache.kv_heads, a.cache.head_dim, a.window, a.scale, why);
  if (rc != LTX_OK || (rc = check_cache(op, a.cache, a.rows, why)) != LTX_OK) return rc;
  if ((long long)a.rows.rows * a.heads > INT_MAX || a.max_len < 0) {
    *why = "kv8_attention: need rows * heads < 2^31 and max_len >= 0";
    return LTX_E_SHAPE;
  }
  if (a.rows.seqs == 0 || a.rows.rows == 0) return LTX_OK;
  const long long cols = (long long)a.heads * a.cache.head_dim;
  if ((rc = check_rows(op, "q", a.q, a.ldq, a.rows.rows, cols, why)) != LTX_OK ||
      (rc = check_rows(op, "o", a.o, a.ldo, a.rows.rows, cols, why)) != LTX_OK)
    return rc;
  if (a.workspace == nullptr) {
    *why = "kv8_attention: workspace is null";
    return LTX_E_NULL;
  }
  if (!aligned(a.workspace, 16)) {
    *why = "kv8_attention: workspace must be 16-byte aligned";
    return LTX_E_ALIGN;
  }
  if (workspace_bytes < need) {
    *why = "kv8_attention: need a workspace of " + std::to_string(need) + " bytes";
    return LTX_E_SHAPE;
  }
  return LTX_OK;
}

int check_attention_packed(const ltx::PackedAttention& a, std::string* why)
{
  const char* op = "attention_packed";
  int rc = check_heads(op, a.heads, a.kv_heads, a.head_dim, a.window, a.scale, why);
  if (rc != LTX_OK) return rc;
  if (a.seqs < 0 || a.rows < 0 || a.keys < 0 || a.seqs > kMaxSeqs) {
    *why = "attention_packed: need seqs 0..2^29, rows and keys >= 0";
    return LTX_E_SHAPE;
  }
  if (a.seqs == 0 || a.rows == 0) return LTX_OK;
  const long long qc = (long long)a.heads * a.head_dim, kc = (long long)a.kv_heads * a.head_dim;
  if ((rc = check_ints(op, "cu_q", a.cu_q, why)) != LTX_OK ||
      (rc = check_ints(op, "cu_k", a.cu_k, why)) != LTX_OK ||
      (rc = check_rows(op, "q", a.q, a.ldq, a.rows, qc, why)) != LTX_OK ||
      (rc = check_rows(op, "o", a.o, a.ldo, a.rows, qc, why)) != LTX_OK ||
      (rc = check_rows(op, "k", a.k, a.ldk, a.keys, kc, why)) != LTX_OK ||
      (rc = check_rows(op, "v", a.v, a.ldv, a.keys, kc, why)) != LTX_OK)
    return rc;
  return LTX_OK;
}

}  // namespace ltx25
