// kv_move.cu -- rows and pages of the KV cache moved inside the cache, every
// layer in one launch.
//
// move_kv: the accepted path of a draft tree is scattered over the slots its
// tokens were stored at; the rows move to the first slots after the context.
// Pairs come in groups (one per sequence) and move as if every row of a group
// were read before any is written, so a path may overlap its destination.  A
// CTA takes (group, layer, some kv heads), brings the group's rows into shared
// memory (every copy in flight at once), synchronises and writes them.  Few
// groups are spread over more CTAs by giving each fewer heads.  Groups must not
// share slots.
//
// copy_pages: whole pages, for a fork's last partly filled page or a swap.
//
// Both move bytes; L2 flushed before: 500 pages of 64 KB in 16 layers 166 us,
// 6.3 TB/s, HBM.  8 rows of 128 sequences in 32 layers (206 MB of 136- and 256-byte
// rows) 55 us, bound by the two round trips of a CTA; with page-transposed V
// (143 MB) 301 us, bound by its byte accesses, 16 apart.  Few rows: one launch and
// the same two round trips, 10 us.  Layer addresses travel as kernel parameters, so a call
// needs no device-side table.
#include <type_traits>

#include "common.cuh"
#include "gfx906_fa_b200.h"

namespace g9 {

constexpr int kMoveLayers = 64;                    // layers per launch: 1 KB of kernel parameters
constexpr int kMoveThreads = 256;
constexpr int kMoveSmem = 96 * 1024;

struct MoveArgs {
  uint8_t* k[kMoveLayers];
  uint8_t* v[kMoveLayers];
  const int64_t* src;
  const int64_t* dst;
  G9KvCache c;                                     // strides and mode; k / v above
  int per, heads;                                  // pairs in a group, kv heads a CTA takes
  int v_bytes, k_w, v_w;                           // bytes of a V row (0: none), access widths
};

template <int W>
__device__ __forceinline__ void move_bytes(uint8_t* dst, const uint8_t* src) {
  if constexpr (W == 16) *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(src);
  else if constexpr (W == 8) *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(src);
  else *reinterpret_cast<uint16_t*>(dst) = *reinterpret_cast<const uint16_t*>(src);
}

// Rows of BYTES bytes between the cache (row_at(row)) and `stage`; IN: cache
// to stage, by asynchronous copies where they are wide enough.
template <int W, int BYTES, bool IN, typename RowAt>
__device__ __forceinline__ void move_rows(uint8_t* stage, int rows, RowAt row_at) {
  constexpr int PER = BYTES / W;
  for (int i = threadIdx.x; i < rows * PER; i += kMoveThreads) {
    const int r = i / PER, o = (i - r * PER) * W;
    uint8_t* g = row_at(r);
    if (!g) continue;
    if (!IN) move_bytes<W>(g + o, stage + r * BYTES + o);
    else if (W >= 8) cp_async(stage + r * BYTES + o, g + o, W);
    else move_bytes<W>(stage + r * BYTES + o, g + o);
  }
}

template <int BYTES, bool IN, typename RowAt>
__device__ __forceinline__ void move_rows_w(uint8_t* stage, int rows, int w, RowAt row_at) {
  if (w == 16 && BYTES % 16 == 0) move_rows<16, BYTES, IN>(stage, rows, row_at);
  else if (w >= 8) move_rows<8, BYTES, IN>(stage, rows, row_at);
  else move_rows<2, BYTES, IN>(stage, rows, row_at);
}

__global__ void __launch_bounds__(kMoveThreads) move_kv_kernel(const __grid_constant__ MoveArgs a) {
  extern __shared__ __align__(16) uint8_t smem[];
  const int layer = blockIdx.y, h0 = blockIdx.z * a.heads;
  const int nh = min(a.heads, a.c.num_heads_kv - h0);
  const int rows = a.per * nh;
  constexpr int D = 128, RB = D / QK * QBLOCK;
  const int bs = a.c.block_size;
  // [source / destination][pair]: page and offset (page -1: skip the pair)
  int2* slot = reinterpret_cast<int2*>(smem);
  uint8_t* ks = smem + 16 * a.per;
  uint8_t* vs = ks + ((a.per * a.heads * RB + 15) & ~15);
  for (int i = threadIdx.x; i < a.per; i += kMoveThreads) {
    const int64_t s = a.src[(int64_t)blockIdx.x * a.per + i], d = a.dst[(int64_t)blockIdx.x * a.per + i];
    bool skip = s < 0 || d < 0 || s == d;
    const int64_t end = (int64_t)a.c.num_blocks * bs;
    if (!skip && (s >= end || d >= end)) {
      raise_error(ERR_BAD_INDEX);
      skip = true;
    }
    slot[i] = skip ? make_int2(-1, 0) : make_int2((int)(s / bs), (int)(s % bs));
    slot[a.per + i] = skip ? make_int2(-1, 0) : make_int2((int)(d / bs), (int)(d % bs));
  }
  __syncthreads();
  auto krow = [&](int r, int which) -> uint8_t* {
    const int p = r / nh, h = h0 + r - p * nh;
    const int2 s = slot[which * a.per + p];
    return s.x < 0 ? nullptr : a.k[layer] + s.x * a.c.k_page_stride + s.y * a.c.k_tok_stride + h * a.c.k_head_stride;
  };
  auto vrow = [&](int r, int which) -> uint8_t* {
    const int p = r / nh, h = h0 + r - p * nh;
    const int2 s = slot[which * a.per + p];
    return s.x < 0 ? nullptr : a.v[layer] + s.x * a.c.v_page_stride + s.y * a.c.v_tok_stride + h * a.c.v_head_stride;
  };
  // Page-transposed records: a token's scales and values, one element every
  // block_size.  Eight elements a thread in flight.
  auto vrec = [&](bool in) {
    constexpr int PER = D + D / QK, U = 8;
    for (int i0 = threadIdx.x; i0 < rows * PER; i0 += kMoveThreads * U) {
      uint8_t* at[U];
      uint16_t x[U];
      int st[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + u * kMoveThreads;
        const int r = i / PER, e = i - r * PER;
        at[u] = nullptr;
        st[u] = 0;
        if (i >= rows * PER) continue;
        const int p = r / nh, h = h0 + r - p * nh;
        const int2 s = slot[(in ? 0 : a.per) + p];
        if (s.x < 0) continue;
        const int off = s.y;
        uint8_t* rec = a.v[layer] + s.x * a.c.v_page_stride + h * a.c.v_head_stride;
        // elements 0..3: scales (two bytes), the rest: values
        at[u] = e < D / QK ? rec + 2 * ((int64_t)e * bs + off) : rec + 2 * (D / QK) * bs + (int64_t)(e - D / QK) * bs + off;
        st[u] = r * RB + (e < D / QK ? 2 * e : 2 * (D / QK) + e - D / QK) + (e < D / QK ? 1 << 30 : 0);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (!at[u]) continue;
        const bool wide = st[u] >> 30;
        const uint8_t* from = in ? at[u] : vs + (st[u] & 0x3fffffff);
        x[u] = wide ? *reinterpret_cast<const uint16_t*>(from) : *from;
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (!at[u]) continue;
        const bool wide = st[u] >> 30;
        uint8_t* to = in ? vs + (st[u] & 0x3fffffff) : at[u];
        if (wide) *reinterpret_cast<uint16_t*>(to) = x[u];
        else *to = (uint8_t)x[u];
      }
    }
  };
  auto vcopy = [&](auto in) {
    constexpr bool IN = decltype(in)::value;
    auto row = [&](int r) { return vrow(r, IN ? 0 : 1); };
    if (a.v_bytes == RB) move_rows_w<RB, IN>(vs, rows, a.v_w, row);
    else if (a.v_bytes) move_rows_w<2 * D, IN>(vs, rows, a.v_w, row);
  };
  move_rows_w<RB, true>(ks, rows, a.k_w, [&](int r) { return krow(r, 0); });
  if (a.c.v_mode == G9_V_Q8T) vrec(true);
  else vcopy(std::true_type());
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();
  move_rows_w<RB, false>(ks, rows, a.k_w, [&](int r) { return krow(r, 1); });
  if (a.c.v_mode == G9_V_Q8T) vrec(false);
  else vcopy(std::false_type());
}

// ---------------------------------------------------------------------------
struct PagesArgs {
  uint8_t* cache[kMoveLayers];
  const int64_t* src;
  const int64_t* dst;
  int64_t page_stride, page_bytes, num_blocks;
};

constexpr int kPageUnroll = 8;

// CTA (pair, layer, piece of the page): kPageUnroll vectors per thread in flight
template <int W>
__global__ void __launch_bounds__(kMoveThreads) copy_pages_kernel(const __grid_constant__ PagesArgs a) {
  const int64_t s = a.src[blockIdx.x], d = a.dst[blockIdx.x];
  if (s < 0 || d < 0 || s == d) return;
  if (s >= a.num_blocks || d >= a.num_blocks) {
    raise_error(ERR_BAD_PAGE);
    return;
  }
  using V = typename std::conditional<W == 16, uint4, uint16_t>::type;
  const V* from = reinterpret_cast<const V*>(a.cache[blockIdx.y] + s * a.page_stride);
  V* to = reinterpret_cast<V*>(a.cache[blockIdx.y] + d * a.page_stride);
  const int64_t n = a.page_bytes / W;
  const int64_t i0 = (int64_t)blockIdx.z * kMoveThreads * kPageUnroll + threadIdx.x;
  V x[kPageUnroll];
#pragma unroll
  for (int u = 0; u < kPageUnroll; ++u)
    if (i0 + u * kMoveThreads < n) x[u] = from[i0 + u * kMoveThreads];
#pragma unroll
  for (int u = 0; u < kPageUnroll; ++u)
    if (i0 + u * kMoveThreads < n) to[i0 + u * kMoveThreads] = x[u];
}

static int width_of(uintptr_t m) { return (m & 15) == 0 ? 16 : (m & 7) == 0 ? 8 : 2; }

}  // namespace g9

G9_ERROR_ACCESSORS(kv_move)

using namespace g9;

extern "C" cudaError_t gfx906_fa_move_kv(void* const* k_layers, void* const* v_layers, int num_layers,
                                         const G9KvCache* cache, const int64_t* src_slots, const int64_t* dst_slots,
                                         int num_groups, int group_size, cudaStream_t stream) {
  if (!cache || num_layers < 0 || num_groups < 0 || group_size < 0) return cudaErrorInvalidValue;
  const G9KvCache& c = *cache;
  if (c.block_size <= 0 || c.num_heads_kv <= 0 || c.num_blocks <= 0 || c.v_mode < 0 || c.v_mode > 3) return cudaErrorInvalidValue;
  if (num_layers == 0 || num_groups == 0 || group_size == 0) return cudaSuccess;
  if (!k_layers || !src_slots || !dst_slots || (c.v_mode != G9_V_NONE && !v_layers)) return cudaErrorInvalidValue;
  constexpr int D = 128, RB = D / QK * QBLOCK;
  uintptr_t km = (uintptr_t)c.k_page_stride | (uintptr_t)c.k_tok_stride | (uintptr_t)c.k_head_stride | 8;
  uintptr_t vm = (uintptr_t)c.v_page_stride | (uintptr_t)c.v_head_stride;
  if (c.v_mode != G9_V_Q8T) vm |= (uintptr_t)c.v_tok_stride;
  if (c.v_mode == G9_V_Q8) vm |= 8;                // 136-byte rows
  for (int i = 0; i < num_layers; ++i) {
    if (!k_layers[i] || (c.v_mode != G9_V_NONE && !v_layers[i])) return cudaErrorInvalidValue;
    km |= (uintptr_t)k_layers[i];
    if (c.v_mode != G9_V_NONE) vm |= (uintptr_t)v_layers[i];
  }
  if ((km & 1) || (c.v_mode != G9_V_NONE && (vm & 1))) return cudaErrorInvalidValue;
  MoveArgs a{};
  a.c = c; a.src = src_slots; a.dst = dst_slots; a.per = group_size;
  a.v_bytes = c.v_mode == G9_V_NONE ? 0 : c.v_mode == G9_V_COPY16 ? 2 * D : RB;
  a.k_w = width_of(km); a.v_w = width_of(vm);
  // as many kv heads a CTA as shared memory holds; a group's rows of one head must fit (in 64 bits: any group_size may be asked for)
  const int64_t head_bytes = (int64_t)group_size * (RB + a.v_bytes), left = kMoveSmem - 16 * (int64_t)group_size - 16;
  if (left < head_bytes) return cudaErrorInvalidValue;
  a.heads = (int)(left / head_bytes);
  if (a.heads > c.num_heads_kv) a.heads = c.num_heads_kv;
  // few groups: halve the heads of a CTA until every SM has four
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  while (a.heads > 1 && (int64_t)num_groups * num_layers * ((c.num_heads_kv + a.heads - 1) / a.heads) < 4 * (int64_t)sms)
    a.heads = (a.heads + 1) / 2;
  const int zs = (c.num_heads_kv + a.heads - 1) / a.heads;
  if (zs > 65535) return cudaErrorInvalidValue;
  const int smem = 16 * group_size + ((group_size * a.heads * RB + 15) & ~15) + group_size * a.heads * a.v_bytes;
  cudaError_t e = cudaFuncSetAttribute(move_kv_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMoveSmem);
  if (e != cudaSuccess) return e;
  for (int l0 = 0; l0 < num_layers; l0 += kMoveLayers) {
    const int n = num_layers - l0 < kMoveLayers ? num_layers - l0 : kMoveLayers;
    for (int i = 0; i < n; ++i) {
      a.k[i] = reinterpret_cast<uint8_t*>(k_layers[l0 + i]);
      a.v[i] = c.v_mode != G9_V_NONE ? reinterpret_cast<uint8_t*>(v_layers[l0 + i]) : nullptr;
    }
    move_kv_kernel<<<dim3(num_groups, n, zs), kMoveThreads, smem, stream>>>(a);
    if ((e = cudaGetLastError()) != cudaSuccess) return e;
  }
  return cudaSuccess;
}

extern "C" cudaError_t gfx906_fa_copy_pages(void* const* layers, int num_layers, int64_t num_blocks,
                                            int64_t page_stride, int64_t page_bytes, const int64_t* src_pages,
                                            const int64_t* dst_pages, int num_pairs, cudaStream_t stream) {
  if (num_layers < 0 || num_pairs < 0 || num_blocks < 0 || page_bytes < 0) return cudaErrorInvalidValue;
  if (num_layers == 0 || num_pairs == 0 || page_bytes == 0) return cudaSuccess;
  if (!layers || !src_pages || !dst_pages || (page_bytes & 1)) return cudaErrorInvalidValue;
  PagesArgs a{};
  a.src = src_pages; a.dst = dst_pages;
  a.page_stride = page_stride; a.page_bytes = page_bytes; a.num_blocks = num_blocks;
  uintptr_t m = (uintptr_t)page_stride | (uintptr_t)page_bytes;
  for (int i = 0; i < num_layers; ++i) {
    if (!layers[i]) return cudaErrorInvalidValue;
    m |= (uintptr_t)layers[i];
  }
  if (m & 1) return cudaErrorInvalidValue;
  const int w = (m & 15) == 0 ? 16 : 2;
  const int64_t piece = (int64_t)w * kMoveThreads * kPageUnroll;
  const int64_t pieces = (page_bytes + piece - 1) / piece;
  if (pieces > 65535) return cudaErrorInvalidValue;
  for (int l0 = 0; l0 < num_layers; l0 += kMoveLayers) {
    const int n = num_layers - l0 < kMoveLayers ? num_layers - l0 : kMoveLayers;
    for (int i = 0; i < n; ++i) a.cache[i] = reinterpret_cast<uint8_t*>(layers[l0 + i]);
    const dim3 grid(num_pairs, n, (unsigned)pieces);
    if (w == 16) copy_pages_kernel<16><<<grid, kMoveThreads, 0, stream>>>(a);
    else copy_pages_kernel<2><<<grid, kMoveThreads, 0, stream>>>(a);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}
