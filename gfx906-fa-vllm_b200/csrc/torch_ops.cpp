// torch_ops.cpp -- the `gfx906_fa` torch extension module.
//
// Same module name, function names, keyword arguments, output allocation and
// error behaviour as the reference's pybind module
// (extension/gfx906_fa.cpp:660-690): TORCH_CHECK on every argument (raising
// RuntimeError), outputs allocated with torch::empty on the input's device,
// every launch asynchronous on the current CUDA stream.  The work itself is
// done by the C ABI in libgfx906fa_b200.so (include/gfx906_fa_b200.h); this
// file only validates, allocates and forwards pointers.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include "gfx906_fa_b200.h"

namespace {

#define CHECK_CUDA(x) TORCH_CHECK((x).device().is_cuda(), #x " must be a CUDA tensor")
#define CHECK_CONTIG(x) TORCH_CHECK((x).is_contiguous(), #x " must be contiguous")

int dtype_code(const torch::Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case torch::kFloat16: return G9_DT_F16;
    case torch::kBFloat16: return G9_DT_BF16;
    case torch::kFloat32: return G9_DT_F32;
    default: TORCH_CHECK(false, name, " must be fp16, bf16 or fp32, got ", t.scalar_type());
  }
  return -1;
}

void check_status(cudaError_t e, const char* what) {
  TORCH_CHECK(e == cudaSuccess, what, " failed: ", cudaGetErrorString(e));
}

cudaStream_t cur_stream() { return at::cuda::getCurrentCUDAStream().stream(); }

// ---------------------------------------------------------------------------
// quantize_q8_0 (extension/gfx906_fa.cpp:273-309)
// ---------------------------------------------------------------------------
torch::Tensor quantize_q8_0(torch::Tensor k_fp16) {
  CHECK_CUDA(k_fp16);
  CHECK_CONTIG(k_fp16);
  TORCH_CHECK(k_fp16.dim() >= 1, "k_fp16 must have at least 1 dim");
  const int dt = dtype_code(k_fp16, "k_fp16");
  const int64_t D = k_fp16.size(-1);
  TORCH_CHECK(D % 32 == 0 && D > 0 && D <= 512, "last dim must be a multiple of 32 (<= 512)");
  const int64_t N = D ? k_fp16.numel() / D : 0;
  std::vector<int64_t> shape(k_fp16.sizes().begin(), k_fp16.sizes().end());
  shape.back() = (D / 32) * 34;
  auto out = torch::empty(shape, k_fp16.options().dtype(torch::kUInt8));
  c10::cuda::CUDAGuard g(k_fp16.device());
  check_status(gfx906_fa_quantize_q8_0(k_fp16.data_ptr(), dt, out.data_ptr<uint8_t>(), N, (int)D,
                                       cur_stream()),
               "launch_quantize_q8_0_dense");
  return out;
}

// ---------------------------------------------------------------------------
// reshape_and_cache_q8 (extension/gfx906_fa.cpp:322-374)
// ---------------------------------------------------------------------------
void reshape_and_cache_q8(torch::Tensor key, torch::Tensor slot_mapping, torch::Tensor k_cache_q8) {
  CHECK_CUDA(key);
  CHECK_CUDA(slot_mapping);
  CHECK_CUDA(k_cache_q8);
  const int kdt = dtype_code(key, "key");
  TORCH_CHECK(slot_mapping.dtype() == torch::kInt64, "slot_mapping must be int64");
  TORCH_CHECK(k_cache_q8.dtype() == torch::kUInt8, "k_cache_q8 must be uint8");
  TORCH_CHECK(key.dim() == 3, "key must be [num_tokens, Hkv, D]");
  TORCH_CHECK(k_cache_q8.dim() == 4, "k_cache_q8 must be [B, bs, Hkv, bytes]");
  TORCH_CHECK(key.stride(2) == 1, "key last dim must be contiguous");
  CHECK_CONTIG(slot_mapping);
  CHECK_CONTIG(k_cache_q8);
  const int T = key.size(0), Hkv = key.size(1), D = key.size(2);
  TORCH_CHECK(D % 32 == 0, "head_size must be multiple of 32");
  const int rb = (D / 32) * 34;
  const int bs = k_cache_q8.size(1);
  TORCH_CHECK(k_cache_q8.size(2) == Hkv, "k_cache_q8 Hkv mismatch: got ", k_cache_q8.size(2),
              " vs key Hkv=", Hkv);
  TORCH_CHECK(k_cache_q8.size(3) == rb, "k_cache_q8 last dim mismatch: got ", k_cache_q8.size(3),
              " expected ", rb);
  TORCH_CHECK(slot_mapping.size(0) == T, "slot_mapping length mismatch");
  c10::cuda::CUDAGuard g(key.device());
  check_status(gfx906_fa_store_kv(key.data_ptr(), kdt, key.stride(0), key.stride(1), nullptr, G9_DT_F16, 0, 0,
                                  slot_mapping.data_ptr<int64_t>(), k_cache_q8.data_ptr<uint8_t>(),
                                  (int64_t)bs * Hkv * rb, (int64_t)Hkv * rb, rb, nullptr, 0, 0, 0,
                                  G9_V_NONE, T, Hkv, D, bs, cur_stream()),
               "launch_reshape_and_cache_q8");
}

// ---------------------------------------------------------------------------
// gather_paged_kv_q8 (extension/gfx906_fa.cpp:393-498)
// ---------------------------------------------------------------------------
std::vector<torch::Tensor> gather_paged_kv_q8(torch::Tensor key_cache_q8, torch::Tensor value_cache,
                                              torch::Tensor block_table, torch::Tensor seq_lens,
                                              int64_t Sk, c10::optional<torch::Tensor> k_out_opt,
                                              c10::optional<torch::Tensor> v_out_opt) {
  CHECK_CUDA(key_cache_q8);
  CHECK_CUDA(value_cache);
  CHECK_CUDA(block_table);
  CHECK_CUDA(seq_lens);
  TORCH_CHECK(key_cache_q8.dtype() == torch::kUInt8, "key_cache_q8 must be uint8");
  TORCH_CHECK(value_cache.dtype() == torch::kFloat16 || value_cache.dtype() == torch::kBFloat16,
              "value_cache must be fp16 (or bf16)");
  TORCH_CHECK(seq_lens.dtype() == torch::kInt32, "seq_lens must be int32");
  TORCH_CHECK(key_cache_q8.dim() == 4, "key_cache_q8 must be 4D");
  TORCH_CHECK(value_cache.dim() == 4, "value_cache must be 4D");
  CHECK_CONTIG(key_cache_q8);
  CHECK_CONTIG(value_cache);
  const int NB = key_cache_q8.size(0), bs = key_cache_q8.size(1), Hkv = key_cache_q8.size(2);
  const int rb = key_cache_q8.size(3), D = value_cache.size(3);
  TORCH_CHECK(value_cache.size(0) == NB, "value_cache blocks mismatch");
  TORCH_CHECK(value_cache.size(1) == bs, "value_cache block_size mismatch");
  TORCH_CHECK(value_cache.size(2) == Hkv, "value_cache Hkv mismatch");
  TORCH_CHECK(D % 32 == 0, "D must be multiple of 32");
  TORCH_CHECK(rb == (D / 32) * 34, "bytes_per_row must equal (D/32)*34, got ", rb,
              " vs expected ", (D / 32) * 34);
  TORCH_CHECK(block_table.dtype() == torch::kInt32, "block_table must be int32 (caller should .to(torch.int32))");
  TORCH_CHECK(block_table.is_contiguous(), "block_table must be contiguous");
  TORCH_CHECK(seq_lens.is_contiguous(), "seq_lens must be contiguous");
  TORCH_CHECK(block_table.dim() == 2, "block_table must be [num_seqs, max_blocks]");
  const int B = block_table.size(0), MB = block_table.size(1);
  TORCH_CHECK(seq_lens.size(0) == B, "seq_lens vs block_table batch mismatch");
  TORCH_CHECK(Sk > 0 && (Sk % 32) == 0, "Sk must be positive multiple of 32, got ", Sk);
  auto use_or_alloc = [&](const c10::optional<torch::Tensor>& buf, at::TensorOptions opts,
                          int64_t last) -> torch::Tensor {
    if (buf.has_value()) {
      const auto& t = buf.value();
      if (t.dim() == 4 && t.size(0) == B && t.size(1) == Hkv && t.size(2) == Sk && t.size(3) == last &&
          t.dtype() == opts.dtype() && t.device() == opts.device() && t.is_contiguous())
        return t;
    }
    return torch::empty({(int64_t)B, (int64_t)Hkv, Sk, last}, opts);
  };
  auto k_out = use_or_alloc(k_out_opt, key_cache_q8.options(), rb);
  auto v_out = use_or_alloc(v_out_opt, value_cache.options(), D);
  c10::cuda::CUDAGuard g(key_cache_q8.device());
  check_status(gfx906_fa_gather_paged_kv_q8_checked(key_cache_q8.data_ptr<uint8_t>(), value_cache.data_ptr(),
                                         block_table.data_ptr<int32_t>(), seq_lens.data_ptr<int32_t>(),
                                         k_out.data_ptr<uint8_t>(), v_out.data_ptr(), B, Hkv, (int)Sk, D,
                                         rb, bs, MB, NB, (int64_t)bs * Hkv * rb, (int64_t)Hkv * rb, rb,
                                         (int64_t)bs * Hkv * D, (int64_t)Hkv * D, D, cur_stream()),
               "launch_gather_paged_kv_q8");
  return {k_out, v_out};
}

// ---------------------------------------------------------------------------
// store_kv: fused K (Q8_0) + V store by slot_mapping (new)
// ---------------------------------------------------------------------------
void store_kv(torch::Tensor key, torch::Tensor value, torch::Tensor slot_mapping, torch::Tensor k_cache,
              torch::Tensor v_cache, int64_t v_mode) {
  CHECK_CUDA(key);
  CHECK_CUDA(slot_mapping);
  CHECK_CUDA(k_cache);
  const int kdt = dtype_code(key, "key");
  TORCH_CHECK(key.dim() == 3 && key.stride(2) == 1, "key must be [T, Hkv, D] with contiguous D");
  TORCH_CHECK(slot_mapping.dtype() == torch::kInt64 && slot_mapping.dim() == 1, "slot_mapping must be int64 [T]");
  CHECK_CONTIG(slot_mapping);
  TORCH_CHECK(v_mode >= 0 && v_mode <= 3,
              "v_mode must be 0 (none), 1 (copy), 2 (q8_0 rows) or 3 (q8_0 page-transposed)");
  const int T = key.size(0), Hkv = key.size(1), D = key.size(2);
  TORCH_CHECK(slot_mapping.size(0) == T, "slot_mapping length mismatch");
  // k_cache / v_cache: 4-D [NB, bs, Hkv, row] views (any dtype) with byte strides
  TORCH_CHECK(k_cache.dim() == 4 && k_cache.size(2) == Hkv, "k_cache must be [NB, bs, Hkv, row]");
  const int bs = k_cache.size(1);
  const int64_t ke = k_cache.element_size();
  const void* vptr = nullptr;
  int vdt = G9_DT_F16;
  int64_t vts = 0, vhs = 0, vb0 = 0, vb1 = 0, vb2 = 0;
  uint8_t* vc = nullptr;
  if (v_mode != 0) {
    CHECK_CUDA(value);
    CHECK_CUDA(v_cache);
    vdt = dtype_code(value, "value");
    TORCH_CHECK(value.dim() == 3 && value.size(0) == T && value.size(1) == Hkv && value.size(2) == D &&
                    value.stride(2) == 1,
                "value must be [T, Hkv, D] with contiguous D");
    vptr = value.data_ptr();
    vts = value.stride(0);
    vhs = value.stride(1);
    const int64_t ve = v_cache.element_size();
    if (v_mode == G9_V_Q8T) {
      TORCH_CHECK(v_cache.dim() == 3 && v_cache.size(1) == Hkv && v_cache.dtype() == torch::kUInt8 &&
                      v_cache.size(2) == (int64_t)bs * (D / 32) * 34 && v_cache.stride(2) == 1,
                  "v_cache must be uint8 [NB, Hkv, block_size*(D/32)*34] page-transposed records");
      vb0 = v_cache.stride(0);
      vb2 = v_cache.stride(1);
    } else {
      TORCH_CHECK(v_cache.dim() == 4 && v_cache.size(1) == bs && v_cache.size(2) == Hkv,
                  "v_cache must be [NB, bs, Hkv, row]");
      vb0 = v_cache.stride(0) * ve;
      vb1 = v_cache.stride(1) * ve;
      vb2 = v_cache.stride(2) * ve;
    }
    vc = reinterpret_cast<uint8_t*>(v_cache.data_ptr());
  }
  c10::cuda::CUDAGuard g(key.device());
  check_status(gfx906_fa_store_kv(key.data_ptr(), kdt, key.stride(0), key.stride(1), vptr, vdt, vts, vhs,
                                  slot_mapping.data_ptr<int64_t>(), reinterpret_cast<uint8_t*>(k_cache.data_ptr()),
                                  k_cache.stride(0) * ke, k_cache.stride(1) * ke, k_cache.stride(2) * ke, vc, vb0,
                                  vb1, vb2, (int)v_mode, T, Hkv, D, bs, cur_stream()),
               "gfx906_fa_store_kv");
}

// ---------------------------------------------------------------------------
// rope_store_kv: fused RoPE (query and key rotated in place) + KV store (new)
// ---------------------------------------------------------------------------
void rope_store_kv(c10::optional<torch::Tensor> query, torch::Tensor key, torch::Tensor value,
                   torch::Tensor positions, torch::Tensor cos_sin_cache, bool is_neox, torch::Tensor slot_mapping,
                   torch::Tensor k_cache, torch::Tensor v_cache, int64_t v_mode) {
  CHECK_CUDA(key);
  CHECK_CUDA(positions);
  CHECK_CUDA(cos_sin_cache);
  CHECK_CUDA(slot_mapping);
  CHECK_CUDA(k_cache);
  const int kdt = dtype_code(key, "key");
  TORCH_CHECK(key.dim() == 3 && key.stride(2) == 1, "key must be [T, Hkv, D] with contiguous D");
  const int T = key.size(0), Hkv = key.size(1), D = key.size(2);
  TORCH_CHECK(D == 128, "head_size must be 128");
  TORCH_CHECK(positions.dtype() == torch::kInt64 && positions.dim() == 1 && positions.size(0) >= T &&
                  positions.is_contiguous(), "positions must be contiguous int64 [>= T]");
  TORCH_CHECK(slot_mapping.dtype() == torch::kInt64 && slot_mapping.dim() == 1 && slot_mapping.size(0) == T &&
                  slot_mapping.is_contiguous(), "slot_mapping must be contiguous int64 [T]");
  TORCH_CHECK(cos_sin_cache.dim() == 2 && cos_sin_cache.is_contiguous(), "cos_sin_cache must be [max_pos, rot_dim]");
  const int csdt = dtype_code(cos_sin_cache, "cos_sin_cache");
  const int rot = cos_sin_cache.size(1);
  TORCH_CHECK(rot == 32 || rot == 64 || rot == 128, "rot_dim must be 32, 64 or 128, got ", rot);
  TORCH_CHECK(v_mode >= 0 && v_mode <= 3, "v_mode must be 0..3");
  void* qptr = nullptr;
  int qdt = G9_DT_F16, Hq = 0;
  int64_t qts = 0, qhs = 0;
  if (query.has_value()) {
    auto q = query.value();
    CHECK_CUDA(q);
    TORCH_CHECK(q.dim() == 3 && q.size(0) >= T && q.size(2) == D && q.stride(2) == 1,
                "query must be [>= T, Hq, D] with contiguous D");
    qdt = dtype_code(q, "query");
    qptr = q.data_ptr();
    Hq = q.size(1);
    qts = q.stride(0);
    qhs = q.stride(1);
  }
  TORCH_CHECK(k_cache.dim() == 4 && k_cache.size(2) == Hkv, "k_cache must be [NB, bs, Hkv, row]");
  const int bs = k_cache.size(1);
  const int64_t ke = k_cache.element_size();
  const void* vptr = nullptr;
  int vdt = G9_DT_F16;
  int64_t vts = 0, vhs = 0, vb0 = 0, vb1 = 0, vb2 = 0;
  uint8_t* vc = nullptr;
  if (v_mode != 0) {
    CHECK_CUDA(value);
    CHECK_CUDA(v_cache);
    vdt = dtype_code(value, "value");
    TORCH_CHECK(value.dim() == 3 && value.size(0) == T && value.size(1) == Hkv && value.size(2) == D &&
                    value.stride(2) == 1, "value must be [T, Hkv, D] with contiguous D");
    vptr = value.data_ptr();
    vts = value.stride(0);
    vhs = value.stride(1);
    if (v_mode == G9_V_Q8T) {
      TORCH_CHECK(v_cache.dim() == 3 && v_cache.size(1) == Hkv && v_cache.dtype() == torch::kUInt8,
                  "v_cache must be uint8 [NB, Hkv, record]");
      vb0 = v_cache.stride(0);
      vb2 = v_cache.stride(1);
    } else {
      TORCH_CHECK(v_cache.dim() == 4 && v_cache.size(1) == bs && v_cache.size(2) == Hkv,
                  "v_cache must be [NB, bs, Hkv, row]");
      const int64_t ve = v_cache.element_size();
      vb0 = v_cache.stride(0) * ve;
      vb1 = v_cache.stride(1) * ve;
      vb2 = v_cache.stride(2) * ve;
    }
    vc = reinterpret_cast<uint8_t*>(v_cache.data_ptr());
  }
  c10::cuda::CUDAGuard g(key.device());
  check_status(gfx906_fa_rope_store_kv(qptr, qdt, qts, qhs, Hq, key.data_ptr(), kdt, key.stride(0), key.stride(1),
                                       vptr, vdt, vts, vhs, positions.data_ptr<int64_t>(), cos_sin_cache.data_ptr(),
                                       csdt, rot, is_neox ? 1 : 0, slot_mapping.data_ptr<int64_t>(),
                                       reinterpret_cast<uint8_t*>(k_cache.data_ptr()), k_cache.stride(0) * ke,
                                       k_cache.stride(1) * ke, k_cache.stride(2) * ke, vc, vb0, vb1, vb2,
                                       (int)v_mode, T, Hkv, D, bs, cur_stream()),
               "gfx906_fa_rope_store_kv");
}

// ---------------------------------------------------------------------------
// attention
// ---------------------------------------------------------------------------
G9AttnBatch batch_base(const torch::Tensor& key_cache_q8, const torch::Tensor& value_cache, int v_fmt,
                       const torch::Tensor& block_table, const torch::Tensor& kv_len) {
  G9AttnBatch b{};
  const int64_t ke = key_cache_q8.element_size();
  const int64_t ve = value_cache.element_size();
  b.k_cache = reinterpret_cast<const uint8_t*>(key_cache_q8.data_ptr());
  b.k_page_stride = key_cache_q8.stride(0) * ke;
  b.k_tok_stride = key_cache_q8.stride(1) * ke;
  b.k_head_stride = key_cache_q8.stride(2) * ke;
  b.v_cache = reinterpret_cast<const uint8_t*>(value_cache.data_ptr());
  if (v_fmt == G9_VFMT_Q8T) {           // [NB, Hkv, record] uint8
    b.v_page_stride = value_cache.stride(0);
    b.v_tok_stride = 0;
    b.v_head_stride = value_cache.stride(1);
  } else {
    b.v_page_stride = value_cache.stride(0) * ve;
    b.v_tok_stride = value_cache.stride(1) * ve;
    b.v_head_stride = value_cache.stride(2) * ve;
  }
  b.v_fmt = v_fmt;
  b.block_table = block_table.data_ptr<int32_t>();
  b.max_blocks = block_table.size(1);
  b.block_size = key_cache_q8.size(1);
  b.kv_len = kv_len.data_ptr<int32_t>();
  b.num_seqs = block_table.size(0);
  b.num_heads_kv = key_cache_q8.size(2);
  b.num_blocks = key_cache_q8.size(0);      // entries past the cache are flagged, never read
  return b;
}

// Optional score features (not in the reference ops): logit soft-cap,
// sliding window, per-query-head sinks.  `sinks_c` keeps a contiguous fp32
// copy alive for the launch.
void set_features(G9AttnBatch& b, int64_t Hq, double softcap, int64_t window, c10::optional<torch::Tensor>& sinks,
                  torch::Tensor& sinks_c, const torch::Tensor& like) {
  TORCH_CHECK(softcap >= 0.0, "softcap must be >= 0 (0 disables it)");
  TORCH_CHECK(window >= 0, "sliding_window must be >= 0 (0 disables it)");
  b.softcap = (float)softcap;
  b.window = (int)window;
  if (sinks.has_value()) {
    auto s = sinks.value();
    CHECK_CUDA(s);
    TORCH_CHECK(s.dim() == 1 && s.size(0) == Hq, "sinks must be [num_heads_q]");
    TORCH_CHECK(s.device() == like.device(), "sinks must be on the query's device");
    sinks_c = s.to(torch::kFloat32).contiguous();
    b.sinks = sinks_c.data_ptr<float>();
  }
}

// 4-D caches hold token rows; a 3-D uint8 [NB, Hkv, record] cache holds
// page-transposed Q8_0 records (G9_VFMT_Q8T).
int infer_v_fmt(const torch::Tensor& value_cache, int64_t D) {
  if (value_cache.dim() == 3) {
    TORCH_CHECK(value_cache.dtype() == torch::kUInt8, "a 3-D value_cache must be uint8 page-transposed Q8_0");
    return G9_VFMT_Q8T;
  }
  if (value_cache.dtype() == torch::kUInt8) {
    TORCH_CHECK(value_cache.size(3) == (D / 32) * 34, "Q8_0 value_cache last dim must be (D/32)*34");
    return G9_VFMT_Q8;
  }
  TORCH_CHECK(value_cache.size(3) == D, "value_cache D mismatch q D");
  if (value_cache.dtype() == torch::kFloat16) return G9_VFMT_F16;
  TORCH_CHECK(value_cache.dtype() == torch::kBFloat16, "value_cache must be fp16, bf16 or uint8 (Q8_0)");
  return G9_VFMT_BF16;
}

void check_paged(const torch::Tensor& key_cache_q8, const torch::Tensor& value_cache,
                 const torch::Tensor& block_table, const torch::Tensor& seq_lens, int64_t D, int64_t B) {
  CHECK_CUDA(key_cache_q8);
  CHECK_CUDA(value_cache);
  CHECK_CUDA(block_table);
  CHECK_CUDA(seq_lens);
  TORCH_CHECK(key_cache_q8.dtype() == torch::kUInt8, "key_cache_q8 must be uint8");
  TORCH_CHECK(block_table.dtype() == torch::kInt32, "block_table must be int32");
  TORCH_CHECK(seq_lens.dtype() == torch::kInt32, "seq_lens must be int32");
  TORCH_CHECK(key_cache_q8.dim() == 4, "key_cache_q8 must be [num_blocks, block_size, Hkv, bytes_per_row]");
  TORCH_CHECK(D == 128, "head_dim must be 128");
  TORCH_CHECK(key_cache_q8.size(3) == (D / 32) * 34, "bytes_per_row must equal (D/32)*34");
  TORCH_CHECK(value_cache.size(0) == key_cache_q8.size(0), "value_cache blocks mismatch");
  if (value_cache.dim() == 3) {
    TORCH_CHECK(value_cache.size(1) == key_cache_q8.size(2), "value_cache Hkv mismatch");
    TORCH_CHECK(value_cache.size(2) == key_cache_q8.size(1) * key_cache_q8.size(3) && value_cache.stride(2) == 1,
                "page-transposed value_cache must be [num_blocks, Hkv, block_size*(D/32)*34]");
  } else {
    TORCH_CHECK(value_cache.dim() == 4, "value_cache must be [num_blocks, block_size, Hkv, D]");
    TORCH_CHECK(value_cache.size(1) == key_cache_q8.size(1), "value_cache block_size mismatch");
    TORCH_CHECK(value_cache.size(2) == key_cache_q8.size(2), "value_cache Hkv mismatch");
    TORCH_CHECK(value_cache.stride(3) == 1, "cache rows must be contiguous");
  }
  TORCH_CHECK(key_cache_q8.stride(3) == 1, "cache rows must be contiguous");
  TORCH_CHECK(block_table.dim() == 2 && block_table.size(0) == B, "block_table[0] must equal batch");
  TORCH_CHECK(seq_lens.dim() == 1 && seq_lens.size(0) == B, "seq_lens must be [batch]");
  TORCH_CHECK(block_table.is_contiguous() && seq_lens.is_contiguous(), "block_table / seq_lens must be contiguous");
}

// Runs one batch through gfx906_fa_attention (decode and/or tensor-core
// prefill), workspace from the caching allocator.
void run_attention(G9AttnBatch& b, const torch::Tensor& like, const int* nq_host = nullptr,
                   const int* kv_host = nullptr) {
  const size_t ws = gfx906_fa_attention_workspace_size(&b, nq_host, kv_host);
  TORCH_CHECK(ws > 0, "attention: unsupported shape");
  auto wsbuf = torch::empty({(int64_t)ws}, like.options().dtype(torch::kUInt8));
  check_status(gfx906_fa_attention(&b, nq_host, kv_host, wsbuf.data_ptr(), ws, cur_stream()),
               "gfx906_fa_attention");
}

void set_mask_qabs(G9AttnBatch& b, int64_t B, int64_t Sq, int64_t min_cols, c10::optional<torch::Tensor>& mask,
                   c10::optional<torch::Tensor>& q_abs_offset, torch::Tensor& mask_c, torch::Tensor& qo_c) {
  TORCH_CHECK(!(mask.has_value() && q_abs_offset.has_value()),
              "q_abs_offset and mask are mutually exclusive (inline causal replaces mask)");
  if (mask.has_value()) {
    auto m = mask.value();
    CHECK_CUDA(m);
    TORCH_CHECK(m.dtype() == torch::kFloat16, "mask must be fp16");
    TORCH_CHECK(m.dim() == 3 && m.size(0) == B && m.size(1) == Sq, "mask must be [B, Sq, Skv_pad]");
    TORCH_CHECK(m.size(2) >= min_cols, "mask.size(2) must cover every key (", min_cols, ")");
    mask_c = m.contiguous();
    b.mask = mask_c.data_ptr();
    b.mask_seq_stride = mask_c.size(1) * mask_c.size(2);
    b.mask_tok_stride = mask_c.size(2);
  }
  if (q_abs_offset.has_value()) {
    auto qo = q_abs_offset.value();
    CHECK_CUDA(qo);
    TORCH_CHECK(qo.dtype() == torch::kInt32 && qo.dim() == 1 && qo.size(0) == B, "q_abs_offset must be int32 [B]");
    qo_c = qo.contiguous();
    b.q_abs = qo_c.data_ptr<int32_t>();
  }
}

// forward (extension/gfx906_fa.cpp:120-265): q [B, Hq, Sq, D], k_q8
// [B, Hkv, Skv, D/32*34], v [B, Hkv, Skv, D] -> fp32 [B, Hq, Sq, D].
// kv_max int32 [B], mask fp16 [B, Sq, >=Skv], q_abs_offset int32 [B].
torch::Tensor forward(torch::Tensor q, torch::Tensor k_q8, torch::Tensor v, double scale,
                      c10::optional<torch::Tensor> kv_max, c10::optional<torch::Tensor> mask,
                      c10::optional<torch::Tensor> q_abs_offset, double softcap, int64_t sliding_window,
                      c10::optional<torch::Tensor> sinks) {
  CHECK_CUDA(q);
  CHECK_CUDA(k_q8);
  CHECK_CUDA(v);
  CHECK_CONTIG(q);
  CHECK_CONTIG(k_q8);
  CHECK_CONTIG(v);
  const int qdt = dtype_code(q, "q");
  TORCH_CHECK(k_q8.dtype() == torch::kUInt8, "k_q8 must be uint8 (block_q8_0 bytes)");
  TORCH_CHECK(q.dim() == 4, "q must be 4D [B, Hq, Sq, D]");
  TORCH_CHECK(v.dim() == 4, "v_fp16 must be 4D [B, Hkv, Skv, D]");
  const int64_t B = q.size(0), Hq = q.size(1), Sq = q.size(2), D = q.size(3);
  const int64_t Hkv = v.size(1), Skv = v.size(2);
  TORCH_CHECK(v.size(0) == B, "v batch mismatch");
  TORCH_CHECK(D % 32 == 0, "head_dim must be multiple of 32");
  TORCH_CHECK(D == 128, "head_dim must be 128");
  TORCH_CHECK(k_q8.dim() == 4 && k_q8.size(0) == B && k_q8.size(1) == Hkv && k_q8.size(2) == Skv,
              "k_q8 first 3 dims must match [B, Hkv, Skv]");
  TORCH_CHECK(k_q8.size(3) == (D / 32) * 34, "k_q8 last dim = (D/32)*34 bytes");
  TORCH_CHECK(Hq % Hkv == 0, "heads_q must be divisible by heads_kv");
  const int vfmt = infer_v_fmt(v, D);
  auto out = torch::empty({B, Hq, Sq, D}, q.options().dtype(torch::kFloat32));
  if (B == 0 || Sq == 0) return out;
  c10::cuda::CUDAGuard g(q.device());
  const int64_t rb = (D / 32) * 34, vrow = v.size(3) * v.element_size();
  auto ids = torch::arange(B, q.options().dtype(torch::kInt32)).view({B, 1});
  torch::Tensor kvl;
  if (kv_max.has_value()) {
    auto kvm = kv_max.value();
    CHECK_CUDA(kvm);
    TORCH_CHECK(kvm.dtype() == torch::kInt32, "kv_max must be int32");
    TORCH_CHECK(kvm.dim() == 1 && kvm.size(0) == B, "kv_max must be 1D [B]");
    kvl = kvm.clamp(0, Skv).to(torch::kInt32).contiguous();
  } else {
    kvl = torch::full({B}, Skv, q.options().dtype(torch::kInt32));
  }
  G9AttnBatch b{};
  b.q = q.data_ptr();
  b.q_dtype = qdt;
  b.q_seq_stride = Hq * Sq * D;
  b.q_tok_stride = D;
  b.q_head_stride = Sq * D;
  b.seq_q = Sq;
  b.out = out.data_ptr();
  b.out_dtype = G9_DT_F32;
  b.o_seq_stride = Hq * Sq * D;
  b.o_tok_stride = D;
  b.o_head_stride = Sq * D;
  b.k_cache = k_q8.data_ptr<uint8_t>();
  b.k_page_stride = Hkv * Skv * rb;
  b.k_tok_stride = rb;
  b.k_head_stride = Skv * rb;
  b.v_cache = reinterpret_cast<const uint8_t*>(v.data_ptr());
  b.v_page_stride = Hkv * Skv * vrow;
  b.v_tok_stride = vrow;
  b.v_head_stride = Skv * vrow;
  b.v_fmt = vfmt;
  b.block_table = ids.data_ptr<int32_t>();
  b.max_blocks = 1;
  b.block_size = std::max<int64_t>(Skv, 1);
  b.kv_len = kvl.data_ptr<int32_t>();
  b.max_kv = Skv;
  b.num_seqs = B;
  b.num_heads_q = Hq;
  b.num_heads_kv = Hkv;
  b.head_dim = D;
  b.scale = (float)scale;
  torch::Tensor mask_c, qo_c, sinks_c;
  set_mask_qabs(b, B, Sq, Skv, mask, q_abs_offset, mask_c, qo_c);
  set_features(b, Hq, softcap, sliding_window, sinks, sinks_c, q);
  // contiguous [B, Hkv, Skv, row] tensors are not 16-token pages: the batch
  // goes to the tensor-core path, whose pack step reads any row layout
  run_attention(b, q);
  return out;
}

// forward_paged_direct (extension/gfx906_fa.cpp:516-658): q [B, Hq, Sq, D]
// (fp32 as in the reference; fp16 / bf16 also accepted) -> fp32 [B, Hq, Sq, D].
torch::Tensor forward_paged_direct(torch::Tensor q, torch::Tensor key_cache_q8, torch::Tensor value_cache,
                                   torch::Tensor block_table, torch::Tensor seq_lens, double scale,
                                   c10::optional<torch::Tensor> mask, c10::optional<torch::Tensor> q_abs_offset,
                                   double softcap, int64_t sliding_window, c10::optional<torch::Tensor> sinks) {
  CHECK_CUDA(q);
  CHECK_CONTIG(q);
  TORCH_CHECK(q.dim() == 4, "q must be 4D [B, Hq, Sq, D]");
  const int qdt = dtype_code(q, "q");
  const int64_t B = q.size(0), Hq = q.size(1), Sq = q.size(2), D = q.size(3);
  check_paged(key_cache_q8, value_cache, block_table, seq_lens, D, B);
  const int vfmt = infer_v_fmt(value_cache, D);
  TORCH_CHECK(key_cache_q8.size(1) == 16, "Only block_size=16 supported, got ", key_cache_q8.size(1));
  TORCH_CHECK(Hq % key_cache_q8.size(2) == 0, "heads_q must be divisible by heads_kv");
  auto out = torch::empty({B, Hq, Sq, D}, q.options().dtype(torch::kFloat32));
  if (B == 0 || Sq == 0) return out;
  c10::cuda::CUDAGuard g(q.device());
  G9AttnBatch b = batch_base(key_cache_q8, value_cache, vfmt, block_table, seq_lens);
  b.q = q.data_ptr();
  b.q_dtype = qdt;
  b.q_seq_stride = Hq * Sq * D;
  b.q_tok_stride = D;
  b.q_head_stride = Sq * D;
  b.seq_q = Sq;
  b.out = out.data_ptr();
  b.out_dtype = G9_DT_F32;
  b.o_seq_stride = Hq * Sq * D;
  b.o_tok_stride = D;
  b.o_head_stride = Sq * D;
  b.max_kv = b.max_blocks * b.block_size;
  b.num_heads_q = Hq;
  b.head_dim = D;
  b.scale = (float)scale;
  torch::Tensor mask_c, qo_c, sinks_c;
  set_mask_qabs(b, B, Sq, b.max_kv, mask, q_abs_offset, mask_c, qo_c);
  set_features(b, Hq, softcap, sliding_window, sinks, sinks_c, q);
  // Sequences of Sq*G rows above the decode kernel's cap take the prefill
  // kernel, whose staging grows with each sequence's visible keys: size it
  // from the actual lengths (one host read of seq_lens) rather than bounding
  // every sequence by max_blocks * block_size.
  if (Sq * (Hq / key_cache_q8.size(2)) > 24) {
    auto sl_host = seq_lens.to(torch::kCPU);
    std::vector<int> nqh(B, (int)Sq), kvh(B);
    for (int64_t i = 0; i < B; ++i)
      kvh[i] = std::max(0, std::min<int>(sl_host.data_ptr<int32_t>()[i], b.max_kv));
    run_attention(b, q, nqh.data(), kvh.data());
  } else {
    run_attention(b, q);
  }
  return out;
}

// paged_attention: vLLM-layout entry.  query [T, Hq, D] (fp16/bf16/fp32),
// caches as [NB, bs, Hkv, row] views (any strides with contiguous rows),
// query_start_loc int32 [B+1], seq_lens int32 [B].  Causal with
// q_abs = seq_len - n_q (vLLM's chunked-prefill convention).  Writes `out`
// [T, Hq, D] (allocated in the query dtype when not given).  Optional host
// lists give exact query lengths / context-length bounds for routing.
torch::Tensor paged_attention(torch::Tensor query, torch::Tensor key_cache_q8, torch::Tensor value_cache,
                              torch::Tensor block_table, torch::Tensor seq_lens, torch::Tensor query_start_loc,
                              int64_t max_query_len, int64_t max_seq_len, double scale,
                              c10::optional<torch::Tensor> out_opt,
                              c10::optional<std::vector<int64_t>> query_lens_host,
                              c10::optional<std::vector<int64_t>> seq_lens_host, double softcap,
                              int64_t sliding_window, c10::optional<torch::Tensor> sinks,
                              c10::optional<torch::Tensor> output_scale) {
  CHECK_CUDA(query);
  CHECK_CUDA(query_start_loc);
  TORCH_CHECK(query.dim() == 3 && query.stride(2) == 1, "query must be [T, Hq, D] with contiguous D");
  const int qdt = dtype_code(query, "query");
  const int64_t T = query.size(0), Hq = query.size(1), D = query.size(2);
  const int64_t B = block_table.size(0);
  check_paged(key_cache_q8, value_cache, block_table, seq_lens, D, B);
  TORCH_CHECK(query_start_loc.dtype() == torch::kInt32 && query_start_loc.dim() == 1 &&
                  query_start_loc.size(0) == B + 1 && query_start_loc.is_contiguous(),
              "query_start_loc must be int32 [B+1]");
  TORCH_CHECK(Hq % key_cache_q8.size(2) == 0, "heads_q must be divisible by heads_kv");
  const int vfmt = infer_v_fmt(value_cache, D);
  torch::Tensor out;
  if (out_opt.has_value()) {
    out = out_opt.value();
    CHECK_CUDA(out);
    TORCH_CHECK(out.dim() == 3 && out.size(0) >= T && out.size(1) == Hq && out.size(2) == D && out.stride(2) == 1,
                "out must be [>=T, Hq, D] with contiguous D");
    TORCH_CHECK(out.device() == query.device(), "out must be on the query's device");
  } else {
    out = torch::empty({T, Hq, D}, query.options());
  }
  if (B == 0 || T == 0) return out;
  c10::cuda::CUDAGuard g(query.device());
  G9AttnBatch b = batch_base(key_cache_q8, value_cache, vfmt, block_table, seq_lens);
  b.q = query.data_ptr();
  b.q_dtype = qdt;
  b.q_tok_stride = query.stride(0);
  b.q_head_stride = query.stride(1);
  // n_q and the causal offsets (q_abs = seq_len - n_q) are derived in the
  // kernels from query_start_loc and seq_lens: no extra launches
  b.q_start = query_start_loc.data_ptr<int32_t>();
  b.flags = G9_F_CU_SEQLENS | G9_F_CAUSAL_END;
  b.seq_q = (int)max_query_len;
  b.out = out.data_ptr();
  torch::Tensor oscale_c;
  if (out.scalar_type() == torch::kFloat8_e4m3fn) {
    // vLLM's static per-tensor fp8 output quantisation: out = e4m3(o / scale)
    TORCH_CHECK(output_scale.has_value(), "an fp8 (e4m3) out needs output_scale");
    oscale_c = output_scale.value().to(torch::kFloat32).reshape({-1}).contiguous();
    TORCH_CHECK(oscale_c.numel() == 1 && oscale_c.device() == query.device(),
                "output_scale must be one fp32 value on the query's device");
    b.out_dtype = G9_DT_FP8E4M3;
    b.out_scale = oscale_c.data_ptr<float>();
  } else {
    TORCH_CHECK(!output_scale.has_value(), "output_scale applies to an fp8 (e4m3) out only");
    b.out_dtype = dtype_code(out, "out");
  }
  b.o_tok_stride = out.stride(0);
  b.o_head_stride = out.stride(1);
  b.max_kv = (int)max_seq_len;
  b.num_heads_q = Hq;
  b.head_dim = D;
  b.scale = (float)scale;
  std::vector<int> nqh, kvh;
  if (query_lens_host.has_value()) {
    TORCH_CHECK((int64_t)query_lens_host->size() == B, "query_lens_host must have num_seqs entries");
    for (auto x : *query_lens_host) nqh.push_back((int)x);
  }
  if (seq_lens_host.has_value()) {
    TORCH_CHECK((int64_t)seq_lens_host->size() == B, "seq_lens_host must have num_seqs entries");
    for (auto x : *seq_lens_host) kvh.push_back((int)x);
  }
  torch::Tensor sinks_c;
  set_features(b, Hq, softcap, sliding_window, sinks, sinks_c, query);
  run_attention(b, query, nqh.empty() ? nullptr : nqh.data(), kvh.empty() ? nullptr : kvh.data());
  return out;
}

// ---------------------------------------------------------------------------
// draft-tree speculation (no reference counterpart)
// ---------------------------------------------------------------------------
#define CHECK_SAME(x, y) TORCH_CHECK((x).device() == (y).device(), #x " must be on the device of " #y)

// G9KvCache of one layer's views: K [NB, bs, Hkv, D/32*34] uint8 and V as
// [NB, bs, Hkv, D] 16-bit, [NB, bs, Hkv, D/32*34] uint8 or page-transposed
// [NB, Hkv, bs*D/32*34] uint8; any strides with contiguous rows.
G9KvCache kv_layout(const torch::Tensor& k, const torch::Tensor& v, bool with_v, int64_t D) {
  CHECK_CUDA(k);
  TORCH_CHECK(k.dim() == 4 && k.dtype() == torch::kUInt8 && k.size(3) == (D / 32) * 34 && k.stride(3) == 1,
              "k_cache must be uint8 [NB, bs, Hkv, (D/32)*34] with contiguous rows");
  TORCH_CHECK(k.size(1) > 0 && k.size(2) > 0, "k_cache must have tokens and heads");
  G9KvCache c{};
  c.k = k.data_ptr<uint8_t>();
  c.k_page_stride = k.stride(0);
  c.k_tok_stride = k.stride(1);
  c.k_head_stride = k.stride(2);
  c.num_blocks = k.size(0);
  c.block_size = k.size(1);
  c.num_heads_kv = k.size(2);
  c.v_mode = G9_V_NONE;
  if (!with_v) return c;
  CHECK_CUDA(v);
  CHECK_SAME(v, k);
  TORCH_CHECK(v.size(0) == k.size(0), "v_cache blocks mismatch");
  const int64_t e = v.element_size();
  if (v.dim() == 3) {
    TORCH_CHECK(v.dtype() == torch::kUInt8 && v.size(1) == k.size(2) && v.size(2) == k.size(1) * k.size(3) && v.stride(2) == 1,
                "a 3-D v_cache must be uint8 [NB, Hkv, block_size*(D/32)*34] page-transposed records");
    c.v_mode = G9_V_Q8T;
    c.v_head_stride = v.stride(1);
  } else {
    TORCH_CHECK(v.dim() == 4 && v.size(1) == k.size(1) && v.size(2) == k.size(2) && v.stride(3) == 1,
                "v_cache must be [NB, bs, Hkv, row] with contiguous rows");
    if (v.dtype() == torch::kUInt8) {
      TORCH_CHECK(v.size(3) == (D / 32) * 34, "Q8_0 v_cache last dim must be (D/32)*34");
      c.v_mode = G9_V_Q8;
    } else {
      TORCH_CHECK((v.dtype() == torch::kFloat16 || v.dtype() == torch::kBFloat16) && v.size(3) == D,
                  "v_cache must be fp16 or bf16 [NB, bs, Hkv, D], or uint8 (Q8_0)");
      c.v_mode = G9_V_COPY16;
    }
    c.v_tok_stride = v.stride(1) * e;
    c.v_head_stride = v.stride(2) * e;
  }
  c.v = reinterpret_cast<uint8_t*>(v.data_ptr());
  c.v_page_stride = v.stride(0) * e;
  return c;
}

void check_index(const torch::Tensor& x, const char* name, c10::ScalarType dt, int64_t n) {
  TORCH_CHECK(x.device().is_cuda() && x.scalar_type() == dt && x.dim() == 1 && x.is_contiguous(), name,
              " must be a contiguous 1-D ", dt, " CUDA tensor");
  TORCH_CHECK(n < 0 || x.size(0) == n, name, " must have ", n, " entries, got ", x.size(0));
  TORCH_CHECK(x.size(0) <= INT32_MAX, name, " must have at most ", INT32_MAX, " entries, got ", x.size(0));   // the C entries count in int
}

std::vector<torch::Tensor> tree_mask(torch::Tensor parents, torch::Tensor query_start_loc, torch::Tensor seq_lens,
                                     int64_t max_query_len) {
  check_index(parents, "parents", torch::kInt32, -1);
  check_index(query_start_loc, "query_start_loc", torch::kInt32, -1);
  const int64_t B = query_start_loc.size(0) - 1, T = parents.size(0);
  TORCH_CHECK(B >= 0, "query_start_loc must be [num_seqs + 1]");
  check_index(seq_lens, "seq_lens", torch::kInt32, B);
  CHECK_SAME(query_start_loc, parents);
  CHECK_SAME(seq_lens, parents);
  TORCH_CHECK(max_query_len > 0 && max_query_len < (int64_t)1 << 30, "max_query_len must be positive");
  TORCH_CHECK(T == 0 || B > 0, "tokens without a sequence");
  const int64_t words = (max_query_len + 31) / 32;
  c10::cuda::CUDAGuard g(parents.device());
  auto mask = torch::empty({T, words}, parents.options());
  auto positions = torch::empty({T}, parents.options().dtype(torch::kInt64));
  check_status(gfx906_fa_tree_mask(parents.data_ptr<int32_t>(), query_start_loc.data_ptr<int32_t>(),
                                   seq_lens.data_ptr<int32_t>(), (int)B, (int)T, (int)words, mask.data_ptr<int32_t>(),
                                   positions.data_ptr<int64_t>(), cur_stream()),
               "gfx906_fa_tree_mask");
  return {mask, positions};
}

void norm_rope_store_kv(c10::optional<torch::Tensor> query, torch::Tensor key, torch::Tensor value,
                        c10::optional<torch::Tensor> q_weight, c10::optional<torch::Tensor> k_weight, double eps,
                        torch::Tensor positions, torch::Tensor cos_sin_cache, bool is_neox, torch::Tensor slot_mapping,
                        torch::Tensor k_cache, torch::Tensor v_cache, int64_t v_mode,
                        c10::optional<torch::Tensor> query_out, c10::optional<torch::Tensor> key_out) {
  CHECK_CUDA(key);
  TORCH_CHECK(key.dim() == 3 && key.stride(2) == 1, "key must be [T, Hkv, D] with contiguous D");
  const int64_t T = key.size(0), Hkv = key.size(1), D = key.size(2);
  TORCH_CHECK(D == 128, "head_size must be 128");
  TORCH_CHECK(v_mode >= 0 && v_mode <= 3, "v_mode must be 0..3");
  const int kdt = dtype_code(key, "key");
  TORCH_CHECK(positions.device().is_cuda() && positions.dtype() == torch::kInt64 && positions.dim() == 1 &&
                  positions.size(0) >= T && positions.is_contiguous(), "positions must be contiguous int64 [>= T]");
  check_index(slot_mapping, "slot_mapping", torch::kInt64, T);
  CHECK_CUDA(cos_sin_cache);
  TORCH_CHECK(cos_sin_cache.dim() == 2 && cos_sin_cache.is_contiguous() && cos_sin_cache.size(0) > 0,
              "cos_sin_cache must be contiguous [max_pos, rot_dim]");
  const int64_t rot = cos_sin_cache.size(1);
  TORCH_CHECK(rot > 0 && rot <= D && rot % 16 == 0, "rot_dim must be a multiple of 16 up to 128, got ", rot);
  const int csdt = dtype_code(cos_sin_cache, "cos_sin_cache");
  G9KvCache c = kv_layout(k_cache, v_cache, v_mode != 0, D);
  TORCH_CHECK(c.v_mode == v_mode, "v_cache does not have the layout of v_mode ", v_mode);
  TORCH_CHECK(c.num_heads_kv == Hkv, "k_cache Hkv mismatch");
  int vdt = G9_DT_F16;
  if (v_mode != 0) {
    CHECK_CUDA(value);
    CHECK_SAME(value, key);
    vdt = dtype_code(value, "value");
    TORCH_CHECK(value.dim() == 3 && value.size(0) == T && value.size(1) == Hkv && value.size(2) == D && value.stride(2) == 1,
                "value must be [T, Hkv, D] with contiguous D");
    TORCH_CHECK(v_mode != 1 || value.dtype() == v_cache.dtype(), "value and v_cache must have the same type (v_mode 1)");
  }
  auto weight = [&](const c10::optional<torch::Tensor>& w, const char* name, int& dt) -> const void* {
    dt = G9_DT_F16;
    if (!w.has_value()) return nullptr;
    TORCH_CHECK(w->device() == key.device() && w->dim() == 1 && w->size(0) == D && w->is_contiguous(), name,
                " must be contiguous [D] on the key's device");
    dt = dtype_code(*w, name);
    return w->data_ptr();
  };
  int qwdt, kwdt;
  const void* qw = weight(q_weight, "q_weight", qwdt);
  const void* kw = weight(k_weight, "k_weight", kwdt);
  for (const auto* x : {&positions, &slot_mapping, &cos_sin_cache, &k_cache})
    TORCH_CHECK(x->device() == key.device(), "every tensor must be on the key's device");
  torch::Tensor q, qo;
  int qdt = G9_DT_F16;
  if (query.has_value()) {
    q = *query;
    CHECK_CUDA(q);
    CHECK_SAME(q, key);
    TORCH_CHECK(q.dim() == 3 && q.size(0) >= T && q.size(1) > 0 && q.size(2) == D && q.stride(2) == 1,
                "query must be [>= T, Hq, D] with contiguous D");
    qdt = dtype_code(q, "query");
    qo = query_out.value_or(q);
    CHECK_SAME(qo, key);
    TORCH_CHECK(qo.dim() == 3 && qo.size(0) >= T && qo.size(1) == q.size(1) && qo.size(2) == D && qo.stride(2) == 1 &&
                    qo.dtype() == q.dtype(), "query_out must be [>= T, Hq, D] of the query's type with contiguous D");
  }
  if (key_out.has_value()) {
    CHECK_SAME(*key_out, key);
    TORCH_CHECK(key_out->dim() == 3 && key_out->size(0) >= T && key_out->size(1) == Hkv && key_out->size(2) == D &&
                    key_out->stride(2) == 1 && key_out->dtype() == key.dtype(),
                "key_out must be [>= T, Hkv, D] of the key's type with contiguous D");
  }
  if (T == 0) return;
  const bool wq = query.has_value(), wk = key_out.has_value();
  c10::cuda::CUDAGuard g(key.device());
  check_status(gfx906_fa_norm_rope_store_kv(
                   wq ? q.data_ptr() : nullptr, qdt, wq ? q.stride(0) : 0, wq ? q.stride(1) : 0, wq ? (int)q.size(1) : 0,
                   key.data_ptr(), kdt, key.stride(0), key.stride(1), v_mode ? value.data_ptr() : nullptr, vdt,
                   v_mode ? value.stride(0) : 0, v_mode ? value.stride(1) : 0, qw, qwdt, kw, kwdt, (float)eps,
                   positions.data_ptr<int64_t>(), cos_sin_cache.data_ptr(), csdt, (int)rot, cos_sin_cache.size(0),
                   is_neox ? 1 : 0, slot_mapping.data_ptr<int64_t>(), &c, wq ? qo.data_ptr() : nullptr,
                   wq ? qo.stride(0) : 0, wq ? qo.stride(1) : 0, wk ? key_out->data_ptr() : nullptr,
                   wk ? key_out->stride(0) : 0, wk ? key_out->stride(1) : 0, (int)T, cur_stream()),
               "gfx906_fa_norm_rope_store_kv");
}

std::vector<torch::Tensor> read_kv(torch::Tensor k_cache, torch::Tensor v_cache, torch::Tensor slots, at::ScalarType dtype) {
  check_index(slots, "slots", torch::kInt64, -1);
  CHECK_SAME(slots, k_cache);
  const G9KvCache c = kv_layout(k_cache, v_cache, true, 128);
  const int64_t N = slots.size(0);
  auto k = torch::empty({N, c.num_heads_kv, 128}, k_cache.options().dtype(dtype));
  auto v = torch::empty_like(k);
  const int dt = dtype_code(k, "dtype");
  c10::cuda::CUDAGuard g(k_cache.device());
  check_status(gfx906_fa_read_kv(&c, c.v_mode == G9_V_COPY16 ? dtype_code(v_cache, "v_cache") : G9_DT_F16,
                                 slots.data_ptr<int64_t>(), (int)N, k.data_ptr(), v.data_ptr(), dt, cur_stream()),
               "gfx906_fa_read_kv");
  return {k, v};
}

void move_kv(const std::vector<torch::Tensor>& k_caches, const std::vector<torch::Tensor>& v_caches,
             torch::Tensor src_slots, torch::Tensor dst_slots, int64_t group_size) {
  const size_t L = k_caches.size();
  TORCH_CHECK(v_caches.size() == L || v_caches.empty(), "k_caches and v_caches must have one entry per layer");
  check_index(src_slots, "src_slots", torch::kInt64, -1);
  const int64_t N = src_slots.size(0);
  check_index(dst_slots, "dst_slots", torch::kInt64, N);
  CHECK_SAME(dst_slots, src_slots);
  TORCH_CHECK(group_size > 0 && N % group_size == 0, "src_slots must hold whole groups of group_size pairs");
  if (L == 0 || N == 0) return;
  const bool with_v = !v_caches.empty();
  const G9KvCache c = kv_layout(k_caches[0], with_v ? v_caches[0] : k_caches[0], with_v, 128);
  std::vector<void*> ks(L), vs(with_v ? L : 0);
  for (size_t i = 0; i < L; ++i) {
    TORCH_CHECK(k_caches[i].device() == src_slots.device() && k_caches[i].sizes() == k_caches[0].sizes() &&
                    k_caches[i].strides() == k_caches[0].strides() && k_caches[i].dtype() == k_caches[0].dtype(),
                "every layer's k_cache must have the layout of the first, on the slots' device");
    ks[i] = k_caches[i].data_ptr();
    if (!with_v) continue;
    TORCH_CHECK(v_caches[i].device() == src_slots.device() && v_caches[i].sizes() == v_caches[0].sizes() &&
                    v_caches[i].strides() == v_caches[0].strides() && v_caches[i].dtype() == v_caches[0].dtype(),
                "every layer's v_cache must have the layout of the first, on the slots' device");
    vs[i] = v_caches[i].data_ptr();
  }
  c10::cuda::CUDAGuard g(src_slots.device());
  check_status(gfx906_fa_move_kv(ks.data(), with_v ? vs.data() : nullptr, (int)L, &c, src_slots.data_ptr<int64_t>(),
                                 dst_slots.data_ptr<int64_t>(), (int)(N / group_size), (int)group_size, cur_stream()),
               "gfx906_fa_move_kv");
}

void copy_pages(const std::vector<torch::Tensor>& caches, torch::Tensor src_pages, torch::Tensor dst_pages) {
  check_index(src_pages, "src_pages", torch::kInt64, -1);
  check_index(dst_pages, "dst_pages", torch::kInt64, src_pages.size(0));
  CHECK_SAME(dst_pages, src_pages);
  if (caches.empty() || src_pages.size(0) == 0) return;
  const auto& f = caches[0];
  TORCH_CHECK(f.dim() >= 2 && f.size(0) > 0, "a cache must be [num_blocks, ...]");
  TORCH_CHECK(f[0].is_contiguous(), "a page must be contiguous");
  std::vector<void*> at(caches.size());
  for (size_t i = 0; i < caches.size(); ++i) {
    const auto& x = caches[i];
    TORCH_CHECK(x.device().is_cuda() && x.device() == src_pages.device() && x.sizes() == f.sizes() &&
                    x.strides() == f.strides() && x.dtype() == f.dtype(),
                "every layer's cache must have the layout of the first, on the pages' device");
    at[i] = x.data_ptr();
  }
  const int64_t e = f.element_size();
  c10::cuda::CUDAGuard g(src_pages.device());
  check_status(gfx906_fa_copy_pages(at.data(), (int)at.size(), f.size(0), f.stride(0) * e, f.numel() / f.size(0) * e,
                                    src_pages.data_ptr<int64_t>(), dst_pages.data_ptr<int64_t>(),
                                    (int)src_pages.size(0), cur_stream()),
               "gfx906_fa_copy_pages");
}

// tree_attention: paged_attention's layout; the last n_q cache rows of each
// sequence are its drafts, and tree_mask's bit rows say which of them a draft
// sees (tree_mask [T, words] int32, see gfx906_fa_tree_attention).
torch::Tensor tree_attention(torch::Tensor query, torch::Tensor key_cache_q8, torch::Tensor value_cache,
                             torch::Tensor block_table, torch::Tensor seq_lens, torch::Tensor query_start_loc,
                             torch::Tensor tree_mask, int64_t max_query_len, int64_t max_seq_len, double scale,
                             c10::optional<torch::Tensor> out_opt, double softcap, int64_t sliding_window,
                             c10::optional<torch::Tensor> sinks, c10::optional<torch::Tensor> output_scale) {
  CHECK_CUDA(query);
  TORCH_CHECK(query.dim() == 3 && query.stride(2) == 1, "query must be [T, Hq, D] with contiguous D");
  const int qdt = dtype_code(query, "query");
  const int64_t T = query.size(0), Hq = query.size(1), D = query.size(2), B = block_table.size(0);
  check_paged(key_cache_q8, value_cache, block_table, seq_lens, D, B);
  check_index(query_start_loc, "query_start_loc", torch::kInt32, B + 1);
  TORCH_CHECK(key_cache_q8.size(0) > 0 && key_cache_q8.size(1) > 0, "the cache has no pages");
  TORCH_CHECK(Hq > 0 && key_cache_q8.size(2) > 0 && Hq % key_cache_q8.size(2) == 0, "heads_q must be divisible by heads_kv");
  TORCH_CHECK(tree_mask.device().is_cuda() && tree_mask.dtype() == torch::kInt32 && tree_mask.dim() == 2 &&
                  tree_mask.size(0) >= T && (tree_mask.size(1) <= 1 || tree_mask.stride(1) == 1),
              "tree_mask must be int32 [>= T, words] with contiguous words");
  TORCH_CHECK(max_query_len >= 0 && tree_mask.size(1) * 32 >= max_query_len,
              "tree_mask rows must have a bit for every draft of the longest tree (", max_query_len, ")");
  TORCH_CHECK(max_seq_len >= 0 && max_seq_len <= INT32_MAX && max_query_len <= INT32_MAX, "lengths must fit 32 bits");
  for (const auto* x : {&key_cache_q8, &value_cache, &block_table, &seq_lens, &query_start_loc, &tree_mask})
    TORCH_CHECK(x->device() == query.device(), "every tensor must be on the query's device");
  const int vfmt = infer_v_fmt(value_cache, D);
  torch::Tensor out;
  if (out_opt.has_value()) {
    out = out_opt.value();
    TORCH_CHECK(out.dim() == 3 && out.size(0) >= T && out.size(1) == Hq && out.size(2) == D && out.stride(2) == 1,
                "out must be [>=T, Hq, D] with contiguous D");
    CHECK_SAME(out, query);
  } else {
    out = torch::empty({T, Hq, D}, query.options());
  }
  if (B == 0 || T == 0 || max_query_len == 0) return out;
  c10::cuda::CUDAGuard g(query.device());
  G9AttnBatch b = batch_base(key_cache_q8, value_cache, vfmt, block_table, seq_lens);
  b.q = query.data_ptr();
  b.q_dtype = qdt;
  b.q_tok_stride = query.stride(0);
  b.q_head_stride = query.stride(1);
  b.q_start = query_start_loc.data_ptr<int32_t>();
  b.flags = G9_F_CU_SEQLENS;
  b.seq_q = (int)std::min<int64_t>(max_query_len, T);
  b.out = out.data_ptr();
  torch::Tensor oscale_c, sinks_c;
  if (out.scalar_type() == torch::kFloat8_e4m3fn) {
    TORCH_CHECK(output_scale.has_value(), "an fp8 (e4m3) out needs output_scale");
    oscale_c = output_scale.value().to(torch::kFloat32).reshape({-1}).contiguous();
    TORCH_CHECK(oscale_c.numel() == 1 && oscale_c.device() == query.device(),
                "output_scale must be one fp32 value on the query's device");
    b.out_dtype = G9_DT_FP8E4M3;
    b.out_scale = oscale_c.data_ptr<float>();
  } else {
    TORCH_CHECK(!output_scale.has_value(), "output_scale applies to an fp8 (e4m3) out only");
    b.out_dtype = dtype_code(out, "out");
  }
  b.o_tok_stride = out.stride(0);
  b.o_head_stride = out.stride(1);
  b.max_kv = (int)max_seq_len;
  b.num_heads_q = Hq;
  b.head_dim = D;
  b.scale = (float)scale;
  set_features(b, Hq, softcap, sliding_window, sinks, sinks_c, query);
  const size_t ws = gfx906_fa_tree_attention_workspace_size(&b);
  torch::Tensor wsbuf;
  if (ws) wsbuf = torch::empty({(int64_t)ws}, query.options().dtype(torch::kUInt8));
  check_status(gfx906_fa_tree_attention(&b, tree_mask.data_ptr<int32_t>(), tree_mask.stride(0), (int)tree_mask.size(1),
                                        ws ? wsbuf.data_ptr() : nullptr, ws, cur_stream()),
               "gfx906_fa_tree_attention");
  return out;
}

unsigned int device_error(bool clear) {
  unsigned int v = 0;
  check_status(gfx906_fa_get_device_error(&v), "gfx906_fa_get_device_error");
  if (clear) check_status(gfx906_fa_clear_device_error(), "gfx906_fa_clear_device_error");
  return v;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.doc() = "gfx906_fa on sm_100a: paged Q8_0 KV store, page gather and flash attention";
  m.def("quantize_q8_0", &quantize_q8_0,
        "Quantize a tensor (last dim D) to block_q8_0 uint8 [..., D/32*34] on the device",
        py::arg("k_fp16"));
  m.def("reshape_and_cache_q8", &reshape_and_cache_q8,
        "Quantize new K tokens and scatter them into the paged Q8 cache by slot_mapping (in place)",
        py::arg("key"), py::arg("slot_mapping"), py::arg("k_cache_q8"));
  m.def("gather_paged_kv_q8", &gather_paged_kv_q8,
        "Paged K_q8 + paged V -> contiguous BHSD; returns [k_out, v_out]. V tail zeroed per seq_lens; "
        "K tail left unwritten. k_out/v_out reused when their shape matches exactly.",
        py::arg("key_cache_q8"), py::arg("value_cache"), py::arg("block_table"), py::arg("seq_lens"),
        py::arg("Sk"), py::arg("k_out") = c10::nullopt, py::arg("v_out") = c10::nullopt);
  m.def("store_kv", &store_kv,
        "Fused KV store by slot_mapping: K -> Q8_0, V copied (v_mode=1) or quantized (v_mode=2)",
        py::arg("key"), py::arg("value"), py::arg("slot_mapping"), py::arg("k_cache"), py::arg("v_cache"),
        py::arg("v_mode") = 1);
  m.def("rope_store_kv", &rope_store_kv,
        "Fused RoPE + KV store: query / key rotated in place (fp32, rounded once), K -> Q8_0, V per v_mode, "
        "by slot_mapping",
        py::arg("query"), py::arg("key"), py::arg("value"), py::arg("positions"), py::arg("cos_sin_cache"),
        py::arg("is_neox"), py::arg("slot_mapping"), py::arg("k_cache"), py::arg("v_cache"), py::arg("v_mode") = 1);
  m.def("forward", &forward, "FA forward (Q fp32/fp16/bf16, K q8_0, V fp16): fp32 [B, Hq, Sq, D]",
        py::arg("q"), py::arg("k_q8"), py::arg("v_fp16"), py::arg("scale"), py::arg("kv_max") = c10::nullopt,
        py::arg("mask") = c10::nullopt, py::arg("q_abs_offset") = c10::nullopt, py::arg("softcap") = 0.0,
        py::arg("sliding_window") = 0, py::arg("sinks") = c10::nullopt);
  m.def("forward_paged_direct", &forward_paged_direct,
        "Direct-paged flash attention (no gather): q [B, Hq, Sq, D] -> fp32 [B, Hq, Sq, D]",
        py::arg("q"), py::arg("key_cache_q8"), py::arg("value_cache"), py::arg("block_table"),
        py::arg("seq_lens"), py::arg("scale"), py::arg("mask") = c10::nullopt,
        py::arg("q_abs_offset") = c10::nullopt, py::arg("softcap") = 0.0, py::arg("sliding_window") = 0,
        py::arg("sinks") = c10::nullopt);
  m.def("paged_attention", &paged_attention,
        "Varlen causal paged attention in vLLM layout: query [T, Hq, D] -> out [T, Hq, D]",
        py::arg("query"), py::arg("key_cache_q8"), py::arg("value_cache"), py::arg("block_table"),
        py::arg("seq_lens"), py::arg("query_start_loc"), py::arg("max_query_len"), py::arg("max_seq_len"),
        py::arg("scale"), py::arg("out") = c10::nullopt, py::arg("query_lens_host") = c10::nullopt,
        py::arg("seq_lens_host") = c10::nullopt, py::arg("softcap") = 0.0, py::arg("sliding_window") = 0,
        py::arg("sinks") = c10::nullopt, py::arg("output_scale") = c10::nullopt);
  m.def("tree_mask", &tree_mask,
        "Ancestor bit rows int32 [T, ceil(max_query_len/32)] and positions int64 [T] of drafted token trees from their "
        "parent links",
        py::arg("parents"), py::arg("query_start_loc"), py::arg("seq_lens"), py::arg("max_query_len"));
  m.def("norm_rope_store_kv", &norm_rope_store_kv,
        "Per-head RMS norm + RoPE of query (into query_out, default in place) and key, K -> Q8_0, V per v_mode, by "
        "slot_mapping; the rotated key is written only to key_out",
        py::arg("query"), py::arg("key"), py::arg("value"), py::arg("q_weight"), py::arg("k_weight"), py::arg("eps"),
        py::arg("positions"), py::arg("cos_sin_cache"), py::arg("is_neox"), py::arg("slot_mapping"), py::arg("k_cache"),
        py::arg("v_cache"), py::arg("v_mode") = 1, py::arg("query_out") = c10::nullopt, py::arg("key_out") = c10::nullopt);
  m.def("read_kv", &read_kv, "Cache rows by slot as values: [k, v], each [N, Hkv, D] of dtype (slot < 0: zeros)",
        py::arg("k_cache"), py::arg("v_cache"), py::arg("slots"), py::arg("dtype"));
  m.def("move_kv", &move_kv,
        "Move cache rows src_slots -> dst_slots in every layer, whole groups of group_size pairs at once",
        py::arg("k_caches"), py::arg("v_caches"), py::arg("src_slots"), py::arg("dst_slots"), py::arg("group_size"));
  m.def("copy_pages", &copy_pages, "Copy whole pages src_pages -> dst_pages in every layer", py::arg("caches"),
        py::arg("src_pages"), py::arg("dst_pages"));
  m.def("tree_attention", &tree_attention,
        "Attention of drafted token trees over the paged cache: query [T, Hq, D] -> out [T, Hq, D]",
        py::arg("query"), py::arg("key_cache_q8"), py::arg("value_cache"), py::arg("block_table"), py::arg("seq_lens"),
        py::arg("query_start_loc"), py::arg("tree_mask"), py::arg("max_query_len"), py::arg("max_seq_len"),
        py::arg("scale"), py::arg("out") = c10::nullopt, py::arg("softcap") = 0.0, py::arg("sliding_window") = 0,
        py::arg("sinks") = c10::nullopt, py::arg("output_scale") = c10::nullopt);
  m.def("device_error", &device_error, "Read (and optionally clear) the library's device error word",
        py::arg("clear") = false);
}
