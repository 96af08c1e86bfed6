// wx_text.h — shared by the text-side translation units (wx_text.cu, wx_text_attn.cu).
#pragma once
#include "wx_internal.h"

namespace wx {

constexpr int kRopeMaxPairs = 64;  // head_dim 128
constexpr int kKvBf16 = WX_KV_BF16, kKvInt8 = WX_KV_INT8, kKvE4m3 = WX_KV_E4M3;

// geometry, alignment and index-range checks of a cache descriptor
int check_kv_cache(wx_ctx* ctx, const wx_kv_cache* c);

}  // namespace wx
