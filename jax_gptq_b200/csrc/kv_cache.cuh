// The paged cache of 8-bit keys and values: layout and launch parameters shared by its kernels.
//
// A page holds P tokens (P = 64, 128 or 256) of every kv head, as codes in excess 128 (byte = code + 128, code in [-127, 127])
// of rows padded to DW = 64, 128 or 256 channels:
//   keys    k[page][head][token][DW]
//   values  v[page][head][token / 64][DW][64]      (64 tokens of a channel side by side: the order in which they are summed)
//   k_scale[page][head], v_scale[page][head]       fp32; value = (byte - 128) * scale
#pragma once
#include "common.cuh"

namespace jgq {

constexpr int KV_TILE = 64;                // tokens taken at a time; a page is one or more of them

inline int kv_width(int64_t head_dim) { return head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256; }
inline bool kv_page_ok(int page) { return page == 64 || page == 128 || page == 256; }

}  // namespace jgq
