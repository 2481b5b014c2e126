// tree_mask.cu -- ancestor bit rows and positions of drafted token trees.
//
// Sequence b drafted n_b tokens, query_start_loc[b] .. query_start_loc[b+1]-1;
// parents[t] is the index of token t's parent inside its sequence's drafts
// (< t's own index), negative for a token that follows the context directly.
//   bit j of row t  = 1 iff j = i(t) or draft j is an ancestor of token t
//   position[t]     = seq_lens[b] - n_b + depth(t)   (seq_lens counts the drafts)
//
// One thread per token walks its parent links.  The links only go down
// (a link that does not is reported and cut), so the words of the row come
// out in descending order and each is written once, without a zeroing pass.
// The walk is a chain of L1 loads, as long as the token is deep: the whole
// step is launch latency for trees a speculator drafts (3.4 us on the device
// for 16 drafts, 8.8 us cold for 256 sequences of up to 64).
#include "common.cuh"
#include "gfx906_fa_b200.h"

namespace g9 {

constexpr int kMaskThreads = 128;

__global__ void __launch_bounds__(kMaskThreads) tree_mask_kernel(const int32_t* parents, const int32_t* start,
                                                                 const int32_t* seq_lens, int num_seqs, int T,
                                                                 int words, int32_t* mask, int64_t* positions) {
  const int t = blockIdx.x * kMaskThreads + threadIdx.x;
  if (t >= T) return;
  int32_t* row = mask + (int64_t)t * words;
  int lo = 0, hi = num_seqs;                       // largest b with start[b] <= t
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (start[mid] <= t) lo = mid; else hi = mid;
  }
  const int a = start[lo], n = start[lo + 1] - a;
  const int i = t - a;
  if (a < 0 || i < 0 || i >= n) {                  // no sequence owns the row (padding)
    for (int w = 0; w < words; ++w) row[w] = 0;
    if (positions) positions[t] = 0;
    return;
  }
  int w = words - 1, depth = -1;
  uint32_t bits = 0;
  for (int j = i;;) {
    ++depth;
    const int jw = j >> 5;
    for (; w > jw; --w) {
      row[w] = (int32_t)bits;
      bits = 0;
    }
    if (jw < words) bits |= 1u << (j & 31);        // a row too narrow for its tree loses the high drafts
    const int up = parents[a + j];
    if (up < 0) break;
    if (up >= j) {                                 // not an earlier draft: a root
      raise_error(ERR_BAD_INDEX);
      break;
    }
    j = up;
  }
  for (; w >= 0; --w) {
    row[w] = (int32_t)bits;
    bits = 0;
  }
  if (positions) positions[t] = (int64_t)seq_lens[lo] - n + depth;
}

}  // namespace g9

G9_ERROR_ACCESSORS(tree_mask)

using namespace g9;

extern "C" cudaError_t gfx906_fa_tree_mask(const int32_t* parents, const int32_t* query_start_loc,
                                           const int32_t* seq_lens, int num_seqs, int num_tokens, int mask_words,
                                           int32_t* mask, int64_t* positions, cudaStream_t stream) {
  if (num_seqs < 0 || num_tokens < 0 || mask_words <= 0) return cudaErrorInvalidValue;
  if (num_tokens == 0) return cudaSuccess;
  if (num_seqs == 0 || !parents || !query_start_loc || !mask || (positions && !seq_lens)) return cudaErrorInvalidValue;
  tree_mask_kernel<<<(num_tokens + kMaskThreads - 1) / kMaskThreads, kMaskThreads, 0, stream>>>(
      parents, query_start_loc, seq_lens, num_seqs, num_tokens, mask_words, mask, positions);
  return cudaGetLastError();
}
