// tree_attn_rows.cu -- entry points of the draft-tree attention, and its
// kernel for caches the tensor-core kernels (tree_attn_tc.cuh) cannot read:
// pages that are not a multiple of 16 tokens, or rows off the 8-byte (Q8_0)
// or 16-byte (16-bit V, page-transposed V) boundaries that their copies need.
//
//   o_t = sum_k p_tk v_k,  p = softmax over the keys token t sees:
//   context keys k < ctx and the drafts its bit row selects, inside its window
//
// A warp per (token, query head): lane k of a 32-key step scores key k, the
// running maximum and sum are kept in fp32, and lane l accumulates output
// elements 4l .. 4l+3.  Every head and draft reads its keys anew: 4 sequences of
// 1K-4K tokens, 16 drafts, 48/8 heads take 3.9 ms, where the tensor-core kernel
// takes 46 us on a cache that it can read.
#include <algorithm>

#include "tree_attn_tc.cuh"

namespace g9 {

constexpr int kRowWarps = 8;

// elements 4*lane .. +3 of the V row of (page, offset, head)
__device__ __forceinline__ void load_v4(const G9AttnBatch& p, int phys, int off, int h, int lane, float v[4]) {
  const uint8_t* base = p.v_cache + (int64_t)phys * p.v_page_stride + (int64_t)h * p.v_head_stride;
  if (p.v_fmt == G9_VFMT_Q8T) {
    const int bs = p.block_size;
    const float d = half_bits_to_float(*reinterpret_cast<const uint16_t*>(base + 2 * ((int64_t)(lane >> 3) * bs + off)));
    const int8_t* q = reinterpret_cast<const int8_t*>(base + 2 * (128 / QK) * bs + off) + (int64_t)4 * lane * bs;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = (float)q[(int64_t)e * bs] * d;
    return;
  }
  const uint8_t* row = base + (int64_t)off * p.v_tok_stride;
  if (p.v_fmt == G9_VFMT_Q8) {
    const uint8_t* b = row + (lane >> 3) * QBLOCK;
    const float d = half_bits_to_float(*reinterpret_cast<const uint16_t*>(b));
    const int8_t* q = reinterpret_cast<const int8_t*>(b + 2 + 4 * (lane & 7));
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = (float)q[e] * d;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = load_one(row, 4 * lane + e, p.v_fmt == G9_VFMT_F16 ? DT_F16 : DT_BF16);
  }
}

__global__ void __launch_bounds__(kRowWarps * 32) tree_rows_kernel(const __grid_constant__ TreeArgs a, int row_blocks) {
  __shared__ float qs[kRowWarps][128];
  const G9AttnBatch& p = a.p;
  const int lane = lane_id(), warp = warp_id();
  const int b = blockIdx.x / row_blocks, h = blockIdx.y;
  const int r = (blockIdx.x % row_blocks) * kRowWarps + warp;
  const int nq = tree_nq(p, b);
  if (r >= nq * a.G) return;                       // whole warps; no barrier below is CTA-wide
  const int t = r / a.G, hq = h * a.G + r % a.G;
  const int L = seq_len_kv(p, b), ctx = L - nq;
  const int32_t* row = tree_row(a, b, t);
  const int lo = tree_window_lo(a, row, nq, ctx);
  const int64_t qo = q_offset(p, b, t, hq);
#pragma unroll
  for (int e = 0; e < 4; ++e) qs[warp][lane + 32 * e] = load_one(p.q, qo + lane + 32 * e, p.q_dtype);
  __syncwarp();
  float m = -INFINITY, l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
  const int first = lo > 0 ? min(lo, ctx < 0 ? 0 : ctx) & ~31 : 0;
  for (int k0 = first; k0 < L; k0 += 32) {
    const int k = k0 + lane;
    bool see = k < L;
    if (see) {
      if (k < ctx) see = true;
      else see = (tree_word(row, (k - ctx) >> 5, a.words, nq) >> ((k - ctx) & 31)) & 1;
      see = see && k >= lo;
    }
    int phys = -1;
    if (see) {
      phys = p.block_table[(int64_t)b * p.max_blocks + k / p.block_size];
      if (page_bad(p, phys)) {
        raise_error(ERR_BAD_PAGE);
        see = false;
      }
    }
    float s = -INFINITY;
    const int off = k % p.block_size;
    if (see) {
      const uint8_t* kr = p.k_cache + (int64_t)phys * p.k_page_stride + (int64_t)off * p.k_tok_stride +
                          (int64_t)h * p.k_head_stride;
      float dot = 0.f;
      for (int j = 0; j < 128 / QK; ++j) {
        const uint8_t* blk = kr + j * QBLOCK;
        const uint16_t* q16 = reinterpret_cast<const uint16_t*>(blk + 2);
        float part = 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const uint16_t w = q16[e];
          part += (float)(int8_t)(w & 0xff) * qs[warp][32 * j + 2 * e] + (float)(int8_t)(w >> 8) * qs[warp][32 * j + 2 * e + 1];
        }
        dot += part * half_bits_to_float(*reinterpret_cast<const uint16_t*>(blk));
      }
      s = p.softcap > 0.f ? softcap_log2(dot, a.cap_in, a.cap_out) : dot * a.scale_log2;
    }
    float top = s;
#pragma unroll
    for (int x = 16; x; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
    const uint32_t seen = __ballot_sync(0xffffffffu, see);
    if (!seen) continue;
    const float mn = fmaxf(m, top), ref = mn == -INFINITY ? 0.f : mn;
    const float w = see ? exp2f(s - ref) : 0.f;
    const float shrink = exp2f(m - ref);           // m = -inf: 0
    m = mn;
    float sum = w;
#pragma unroll
    for (int x = 16; x; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
    l = l * shrink + sum;
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] *= shrink;
    for (uint32_t left = seen; left; left &= left - 1) {
      const int j = __ffs(left) - 1;               // the same in every lane
      const float pj = __shfl_sync(0xffffffffu, w, j);
      float v[4];
      load_v4(p, __shfl_sync(0xffffffffu, phys, j), __shfl_sync(0xffffffffu, off, j), h, lane, v);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] += pj * v[e];
    }
  }
  const bool any = l > 0.f || l != l;              // NaN scores stay NaN
  if (p.sinks && any) l += exp2f(sink_log2(p, hq) - m);
  const float inv = (any ? 1.f / l : 0.f) * out_quant_factor(p);
  const int64_t oo = o_offset(p, b, t, hq) + 4 * lane;
  store_out2(p.out, p.out_dtype, oo, any ? acc[0] * inv : 0.f, any ? acc[1] * inv : 0.f);
  store_out2(p.out, p.out_dtype, oo + 2, any ? acc[2] * inv : 0.f, any ? acc[3] * inv : 0.f);
}

cudaError_t run_tree_rows(const TreeArgs& a, cudaStream_t stream) {
  const int blocks = (int)(((int64_t)a.p.seq_q * a.G + kRowWarps - 1) / kRowWarps);
  if ((int64_t)blocks * a.p.num_seqs > 0x7fffffff || a.p.num_heads_kv > 65535) return cudaErrorInvalidValue;
  tree_rows_kernel<<<dim3((unsigned)(blocks * a.p.num_seqs), a.p.num_heads_kv), kRowWarps * 32, 0, stream>>>(a, blocks);
  return cudaGetLastError();
}

}  // namespace g9

G9_ERROR_ACCESSORS(tree_rows)

using namespace g9;

// Shapes every kernel takes; out rows are written in pairs of elements.
static bool tree_batch_ok(const G9AttnBatch& p) {
  if (p.head_dim != 128 || p.num_heads_kv <= 0 || p.num_heads_q <= 0 || p.num_heads_q % p.num_heads_kv) return false;
  if (p.num_seqs < 0 || p.seq_q < 0 || p.block_size <= 0 || p.max_blocks < 0 || p.max_kv < 0) return false;
  if (p.q_dtype < 0 || p.q_dtype > 2 || p.out_dtype < 0 || p.out_dtype > 3 || p.v_fmt < 0 || p.v_fmt > 3) return false;
  if (p.out_dtype == G9_DT_FP8E4M3 && !p.out_scale) return false;
  if (p.q_abs || p.mask || (p.flags & G9_F_CAUSAL_END)) return false;
  if ((p.flags & G9_F_CU_SEQLENS) && !p.n_q && !p.q_start) return false;     // drafts are counted from q_start
  if (((uintptr_t)p.k_cache | (uintptr_t)p.k_page_stride | (uintptr_t)p.k_tok_stride | (uintptr_t)p.k_head_stride) & 1) return false;
  uintptr_t v = (uintptr_t)p.v_cache | (uintptr_t)p.v_page_stride | (uintptr_t)p.v_head_stride;
  if (p.v_fmt != G9_VFMT_Q8T) v |= (uintptr_t)p.v_tok_stride;
  const int64_t es = p.out_dtype == DT_F32 ? 4 : p.out_dtype == DT_FP8 ? 1 : 2;
  const uintptr_t o = (uintptr_t)p.out | (uintptr_t)(p.o_seq_stride * es) | (uintptr_t)(p.o_tok_stride * es) |
                      (uintptr_t)(p.o_head_stride * es);
  return !(v & 1) && o % (2 * es) == 0;
}

namespace g9 {
cudaError_t launch_tree_tc_v0(const TreeTcParams& pp, int nq, cudaStream_t stream);
cudaError_t launch_tree_tc_v1(const TreeTcParams& pp, int nq, cudaStream_t stream);
cudaError_t launch_tree_tc_v2(const TreeTcParams& pp, int nq, cudaStream_t stream);
cudaError_t launch_tree_tc_v3(const TreeTcParams& pp, int nq, cudaStream_t stream);
}  // namespace g9

namespace {

struct TreePlan {
  int nq = 0;                    // query tiles a CTA holds; 0: the row kernel
  int NG = 0, rc = 0;
  size_t cum = 0, po = 0, total = 0;
};

TreePlan plan_tree(const G9AttnBatch& p) {
  TreePlan pl;
  auto off = [](uintptr_t base, int64_t a, int64_t b, int64_t c, uintptr_t to) {
    return ((base | (uintptr_t)a | (uintptr_t)b | (uintptr_t)c) & (to - 1)) != 0;
  };
  if (p.block_size % 16 || p.max_blocks == 0) return pl;
  if (off((uintptr_t)p.k_cache, p.k_page_stride, p.k_tok_stride, p.k_head_stride, 8)) return pl;
  const uintptr_t va = p.v_fmt == G9_VFMT_Q8 ? 8 : 16;
  if (off((uintptr_t)p.v_cache, p.v_page_stride, p.v_fmt == G9_VFMT_Q8T ? 0 : p.v_tok_stride, p.v_head_stride, va)) return pl;
  // offsets inside a page are held in 32 bits, page strides in unsigned 32
  const int64_t vt = p.v_fmt == G9_VFMT_Q8T ? 0 : p.v_tok_stride;
  if (p.k_tok_stride < 0 || vt < 0 || p.block_size > 32768 || p.k_tok_stride * p.block_size > 0x3fffffff || vt * p.block_size > 0x3fffffff)
    return pl;
  if (p.k_page_stride < 0 || p.k_page_stride > 0xffffffffll || p.v_page_stride < 0 || p.v_page_stride > 0xffffffffll) return pl;
  const int64_t rows = (int64_t)p.seq_q * (p.num_heads_q / p.num_heads_kv);
  const int nq = rows > tt::BM ? 2 : 1;
  const int64_t groups = (rows + nq * tt::BM - 1) / (nq * tt::BM);
  const int64_t units = (int64_t)p.num_seqs * groups * ((int64_t)p.max_kv / tt::BN + 1);
  if (units > 0x3fffffff || (int64_t)p.num_seqs * groups * 8 > 0x7fffffff || p.num_heads_kv > 65535) return pl;
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  pl.nq = nq;
  pl.NG = (int)std::max<int64_t>(1, std::min<int64_t>(sms / p.num_heads_kv, units));
  pl.rc = (int)std::min<int64_t>(nq * tt::BM, (rows + 31) / 32 * 32);
  auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
  const size_t slots = (size_t)2 * pl.NG * p.num_heads_kv;
  pl.cum = up(((size_t)p.num_seqs + 1) * sizeof(int));
  pl.po = up(slots * tt::D * pl.rc * sizeof(float));
  pl.total = pl.cum + pl.po + up(slots * 2 * pl.rc * sizeof(float)) + 256;
  return pl;
}

}  // namespace

extern "C" size_t gfx906_fa_tree_attention_workspace_size(const G9AttnBatch* batch) {
  if (!batch || !tree_batch_ok(*batch) || batch->num_seqs == 0 || batch->seq_q == 0) return 0;
  return plan_tree(*batch).total;
}

extern "C" cudaError_t gfx906_fa_tree_attention(const G9AttnBatch* batch, const int32_t* tree_mask,
                                                int64_t mask_row_stride, int mask_words, void* workspace,
                                                size_t workspace_bytes, cudaStream_t stream) {
  if (!batch || !tree_batch_ok(*batch) || mask_words <= 0) return cudaErrorInvalidValue;
  if (batch->num_seqs == 0 || batch->seq_q == 0) return cudaSuccess;
  if (!tree_mask || !batch->q || !batch->out || !batch->k_cache || !batch->v_cache || !batch->block_table || !batch->kv_len)
    return cudaErrorInvalidValue;
  TreeArgs a{};
  a.p = *batch;
  a.mask = tree_mask;
  a.mask_stride = mask_row_stride;
  a.words = mask_words;
  a.G = batch->num_heads_q / batch->num_heads_kv;
  a.scale_log2 = batch->scale * kLog2e;
  if (batch->softcap > 0.f) {
    a.cap_in = batch->scale / batch->softcap;
    a.cap_out = batch->softcap * kLog2e;
  }
  const TreePlan pl = plan_tree(*batch);
  if (pl.nq == 0) return run_tree_rows(a, stream);
  if (!workspace || workspace_bytes < pl.total) return cudaErrorInvalidValue;
  TreeTcParams pp{};
  pp.a = a;
  pp.Hkv = batch->num_heads_kv;
  pp.NG = pl.NG;
  pp.rc = pl.rc;
  pp.kp = (uint32_t)batch->k_page_stride;
  pp.vp = (uint32_t)batch->v_page_stride;
  pp.kt = (int)batch->k_tok_stride;
  pp.vt = batch->v_fmt == G9_VFMT_Q8T ? 0 : (int)batch->v_tok_stride;
  pp.bs_log2 = -1;
  if ((batch->block_size & (batch->block_size - 1)) == 0)
    for (pp.bs_log2 = 0; (1 << pp.bs_log2) < batch->block_size;) ++pp.bs_log2;
  // Rows of odd heads start 8 bytes off a 16-byte boundary and take the 8 bytes before them along; those of even heads the 8
  // behind them, which the next head's row holds.
  pp.k_wide = (((uintptr_t)batch->k_cache | (uintptr_t)batch->k_page_stride | (uintptr_t)batch->k_tok_stride) & 15) == 0 &&
              batch->k_head_stride == q8_row_bytes(tt::D) && batch->num_heads_kv % 2 == 0;
  const int64_t es = batch->out_dtype == DT_F32 ? 4 : batch->out_dtype == DT_FP8 ? 1 : 2;
  pp.out_vec = (((uintptr_t)batch->out | (uintptr_t)(batch->o_seq_stride * es) | (uintptr_t)(batch->o_tok_stride * es) |
                 (uintptr_t)(batch->o_head_stride * es)) & 15) == 0;
  uint8_t* w = reinterpret_cast<uint8_t*>(((uintptr_t)workspace + 255) & ~(uintptr_t)255);
  pp.cum = reinterpret_cast<int*>(w);
  pp.po = reinterpret_cast<float*>(w + pl.cum);
  pp.pml = reinterpret_cast<float*>(w + pl.cum + pl.po);
  switch (batch->v_fmt) {
    case G9_VFMT_F16: return launch_tree_tc_v0(pp, pl.nq, stream);
    case G9_VFMT_BF16: return launch_tree_tc_v1(pp, pl.nq, stream);
    case G9_VFMT_Q8: return launch_tree_tc_v2(pp, pl.nq, stream);
    default: return launch_tree_tc_v3(pp, pl.nq, stream);
  }
}
