// What the kernels that attend few rows over the codes of an fp16 cache share: their
// workgroup, runs of blocks, split plan and arguments.
#pragma once

#include "tqk_attend.h"
#include "tqk_wave.h"

// Division by a number that a launch has: by a product (2^32 / n, rounded up: exact while
// x n < 2^32) where the host knows that x stays below that.  The compiler's own are some
// 200 cycles each, ten of them in a row before the first block.
struct FewDiv {
  int n;
  uint32_t mul;  // 0: a division
  __device__ __forceinline__ int operator()(int x) const {
    return n == 1 ? x : mul ? (int)__umulhi((uint32_t)x, mul) : x / n;
  }
};
inline FewDiv few_div(long long n, long long most) {  // x from 0 to `most`
  return FewDiv{(int)n, n > 1 && (most + 1) * n <= (1LL << 32) ? (uint32_t)(0xFFFFFFFFu / (uint32_t)n + 1) : 0u};
}
// What tqk_attend_rows divides by.
struct FewDivs {
  FewDiv splits, heads, items;  // of the workgroups
  FewDiv heads_of;              // query heads of a kv head
  FewDiv group, blocks;         // tokens of a group, its blocks
  FewDiv waves;                 // of all splits
  float per_page;               // 1 / tokens of a page
  int group_pages;
};

// Arguments of the kernels behind tqk_attend_groups, tqk_attend_weights and
// tqk_attend_shared: a window, or a list of groups in its place, or the tokens from one
// on; partial results, and every coded block's maximum and sum, for launches that follow.
struct MoreArgs {
  tqk_cache_desc d;
  tqk_cache_ptrs p;
  const uint16_t* q;
  const int32_t* seq_lens;
  const int32_t* q_lens;
  void* out;
  float* part_acc;  // [split][row][D]
  float* part_ml;   // [split][row][2]: running maximum (log2 units) and sum
  long long rows;   // rows of all sequences and heads, and of the launch's queries
  long long q_stride[3];
  long long o_stride[3];
  int batch, q_len, max_len, window, sinks, out_type;
  int per_item;     // queries of a workgroup
  int q_items;      // workgroups a sequence's queries take
  int n_splits;
  const int32_t* groups;  // [sequence][kv head][query][n_list] by strides, or null
  long long g_stride[3];
  int n_list;
  int skip;          // first token that is seen (a multiple of G)
  int shared;        // tokens that every sequence begins with (a multiple of G; the prefix kernel's)
  int t0, t_len;     // the queries of this launch
  int split0;        // the launch's first split of the partial results
  int direct;        // one split, and its result is the output
  float* block_ml;   // [row][blocks][2]: maximum and sum of a coded block, or null
  int blocks;        // blocks of a row there
  FewDivs by;
};

// up to eight rows of a (sequence, kv head) a workgroup (tqk_attend_rows.h)
void tqk_launch_rows_64(const MoreArgs& a, unsigned groups, hipStream_t st);
void tqk_launch_rows_128(const MoreArgs& a, unsigned groups, hipStream_t st);
void tqk_launch_rows_256(const MoreArgs& a, unsigned groups, hipStream_t st);
// 128 rows of any sequences a workgroup, over shared tokens (tqk_attend_prefix.hip)
void tqk_launch_prefix(const MoreArgs& a, unsigned groups, hipStream_t st);

namespace {

typedef _Float16 h2_t __attribute__((ext_vector_type(2)));
constexpr int kFewWaves = 8, kFewThreads = 64 * kFewWaves;
constexpr float kFewLazy = 2.0f;  // log2 units: weights stay at most 4, norms at most TQK_MAX_VNORM: fp16
constexpr int kNoToken = 1 << 30;  // past every token (max_len is at most that)

// A run of blocks in two pieces, [0, n0) and [from, from + n - n0): the first
// tokens' and the window's.
struct BlockRuns {
  int n0, from, n;
  __device__ __forceinline__ int at(int i) const { return i < n0 ? i : i - n0 + from; }
};

// Splits: rounds of the workgroups that fit (one a CU) times a wave's run of
// blocks and the set-up, joining and rotation of about three blocks' time;
// another launch to join them, about two (`join`; 0 where it runs in any case).
[[maybe_unused]] int few_splits(long long pairs, long long blocks, double join) {
  const uint32_t slots = (uint32_t)device_cus(), most = pairs < (1 << 20) ? 64 : 1;
  double best = 1e30;
  int splits = 1;
  for (uint32_t s = 1; s <= most && (s == 1 || kFewWaves * (s - 1) < (uint64_t)blocks); ++s) {
    const uint32_t rounds = most > 1 ? ((uint32_t)pairs * s + slots - 1) / slots : 1;
    const uint32_t run = ((uint32_t)blocks + kFewWaves * s - 1) / (kFewWaves * s);
    const double cost = (double)rounds * (double)(run + 3) + (s > 1 ? join : 0.0);
    if (cost < best - 1e-9) {
      best = cost;
      splits = (int)s;
    }
  }
  return splits;
}

// x / n of uniform numbers that are mostly small
[[maybe_unused]] __device__ __forceinline__ int few_quotient(int x, int n) {
  if (x >= 1 << 22) return x / n;
  const int q = (int)((float)x * __builtin_amdgcn_rcpf((float)n)), r = x - q * n;  // (within one of it)
  return q + (r >= n) - (r < 0);
}

}  // namespace
