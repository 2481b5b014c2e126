// tree_common.cuh -- what a drafted token sees, shared by the tree-attention kernels.
#pragma once

#include "attn_common.cuh"

namespace g9 {

struct TreeArgs {
  G9AttnBatch p;
  const int32_t* mask;           // ancestor bits, `words` int32 a row
  int64_t mask_stride;           // int32 between rows
  int words;
  int G;                         // query heads per kv head
  float scale_log2;
  float cap_in, cap_out;         // soft-cap: scale / softcap and softcap * log2(e)
};

// drafts of sequence b: never more than the host bound the launch was planned with
__device__ __forceinline__ int tree_nq(const G9AttnBatch& p, int b) {
  const int n = seq_nq(p, b);
  return n < 0 ? 0 : (n < p.seq_q ? n : p.seq_q);
}

__device__ __forceinline__ const int32_t* tree_row(const TreeArgs& a, int b, int t) {
  const int64_t r = a.p.q_start ? (int64_t)a.p.q_start[b] + t : (int64_t)b * a.p.seq_q + t;
  return a.mask + r * a.mask_stride;
}

// Word w of a row, drafts j >= nq cleared.
__device__ __forceinline__ uint32_t tree_word(const int32_t* row, int w, int words, int nq) {
  if (w >= words) return 0;
  const int left = nq - 32 * w;
  if (left <= 0) return 0;
  const uint32_t x = (uint32_t)row[w];
  return left >= 32 ? x : x & ((1u << left) - 1u);
}

// First key inside a row's window (INT_MIN without one): a key's distance is
// counted along the row's own path, the drafts it selects behind its context.
// A path shorter than the window leaves some context in it; of a longer one the
// last `window` drafts stay, and the first of them is the row's first key.
__device__ __forceinline__ int tree_window_lo(const TreeArgs& a, const int32_t* row, int nq, int ctx) {
  if (a.p.window <= 0) return -0x7fffffff - 1;
  int seen = 0;
  for (int w = 0; 32 * w < nq; ++w) seen += __popc(tree_word(row, w, a.words, nq));
  int drop = seen - a.p.window;              // drafts past the window
  if (drop <= 0) {
    const int64_t lo = (int64_t)ctx + drop;
    return lo < -0x7fffffff ? -0x7fffffff : (int)lo;
  }
  int w = 0;
  uint32_t x = tree_word(row, 0, a.words, nq);
  for (; drop >= __popc(x); x = tree_word(row, ++w, a.words, nq)) drop -= __popc(x);
  for (; drop > 0; --drop) x &= x - 1;
  return ctx + 32 * w + __ffs(x) - 1;
}

}  // namespace g9
