// What tqk_attn.hip offers the library's other units.
#pragma once

#include "tqk_common.h"

// Tiles of the attention kernels start at multiples of this many keys.
constexpr int kMaxKeys = 64;

// Keys and values without the rows that no query sees.  A sequence's first
// visible tokens and the window of its queries are kept in whole tiles; the
// tiles between them are left out, and the later ones move down by the gap.
struct KeptRows {
  int sinks;  // rows of the first tiles
  int gap;    // rows left out after them
  // n keys, the last m of them queries; start: first visible token
  __host__ __device__ KeptRows(int n, int m, int start, int sink_end, int window) {
    const int first = n - m;  // the first query's position
    const int lo = window > 0 && window < n && first - window + 1 > start ? first - window + 1 : start;
    const int low = (lo > 0 ? lo : 0) / kMaxKeys * kMaxKeys;
    sinks = (sink_end + kMaxKeys - 1) / kMaxKeys * kMaxKeys;
    gap = low > sinks ? low - sinks : 0;
  }
  __host__ __device__ int row(int pos) const { return pos - (pos >= sinks ? gap : 0); }
};

// tqk_attention; compact: keys and values hold the kept rows only.  k_lo, where
// given (fp16): what the keys' rounding left, laid out as they are.
int tqk_run_attention(const tqk_attn_desc* d, const void* q, const void* k, const void* v, const int32_t* kv_lens,
                      const int32_t* q_lens, const int32_t* kv_starts, void* out, void* workspace,
                      size_t workspace_bytes, int compact, const void* k_lo, void* stream);
