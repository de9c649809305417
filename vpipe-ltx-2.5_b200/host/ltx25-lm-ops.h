// ltx25-lm-ops.h -- argument checks of the language-model operators: what can be
// known of a call on the host, before anything is launched.
#pragma once

#include <string>

#include "../csrc/block_ops.h"

namespace ltx25 {

// LTX_OK, or the code and message the C ABI answers with.
int check_attention_packed(const ltx::PackedAttention& a, std::string* why);
int check_kv8_rows(const char* op, const ltx::Kv8Cache& c, const ltx::Kv8Rows& r, const void* k,
                   int ldk, const void* v, int ldv, std::string* why);
int check_kv8_attention(const ltx::Kv8Attention& a, size_t workspace_bytes, size_t need,
                        std::string* why);

}  // namespace ltx25
