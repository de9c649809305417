// ltx25-lm-ops.h -- argument checks of the language-model operators: what can be
// known of a call on the host, before anything is launched.
#pragma once

#include <string>

#include "../csrc/block_ops.h"

namespace ltx25 {

// LTX_OK, or the code and message the C ABI answers with.
int check_attention_packed(const ltx::PackedAttention& a, std::string* why);

}  // namespace ltx25
