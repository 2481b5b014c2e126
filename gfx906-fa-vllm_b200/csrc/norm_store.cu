// norm_store.cu -- per-head RMS norm + rotation of queries and keys with the
// Q8_0 store of keys and values in the same pass, and the reader of stored
// rows (head size 128).
//
//   y = x * rsqrt(mean(x^2) + eps) * w          over the 128 elements of a head
//   rotated pairs (a, b) of the first rot_dim elements:
//     a' = a cos - b sin,  b' = b cos + a sin   (angles by the token's position)
//   one rounding to the tensor's type; a key is quantised from that rounding
//
// Half a warp holds a row, 8 elements a lane, so every row is one 16-byte
// load per lane, the mean of squares four shuffles and a Q8_0 block's maximum
// two.  All arithmetic is fp32.  Queries and keys are read and written once,
// where separate norm, rotation and store passes move them three times.
// 16384 tokens of 48 + 8 heads (505 MB, L2 flushed before): 147 us, 3.4 TB/s; with
// token-row Q8_0 V 145 us, 16-bit V (521 MB) 141 us, 3.7 TB/s.  Bound by what 24
// warps an SM keep in flight between their dependent loads (position, angles,
// rows), with half the issue slots taken: 127 instructions a pair of query rows.
#include <cstdlib>

#include "common.cuh"
#include "gfx906_fa_b200.h"
#include "q8_quant.cuh"
#include "tcgen05.cuh"

namespace g9 {

struct NormStoreArgs {
  const void* q; const void* k; const void* v;
  void* q_out; void* k_out;                        // k_out may be null
  int q_dt, k_dt, v_dt;
  int64_t q_tok, q_head, k_tok, k_head, v_tok, v_head;      // elements
  int64_t qo_tok, qo_head, ko_tok, ko_head;
  int q_vec, k_vec, v_vec, qo_vec, ko_vec;         // 1: rows start on 16-byte boundaries
  const void* q_w; const void* k_w;                // null: no norm
  int qw_dt, kw_dt;
  float eps;
  const int64_t* positions;
  const void* cos_sin;                             // [max_pos, rot]: cos of pair j at j, sin at rot/2 + j
  int cs_dt, rot, neox, cs_vec;
  int64_t max_pos;
  const int64_t* slots;
  G9KvCache c;
  int bs_log2;                                     // of the page size, -1: not a power of two
  int k_w8, v_w8, v_w16, v_rec16;                  // cache rows: 8-byte (K, Q8_0 V), 16-byte (16-bit V), records 16-byte aligned
  int T, Hq, Hkv, rows;                            // rows of a token: Hq + Hkv + (V stored ? Hkv : 0)
  int rpw;                                         // rows of a token a half-warp takes
};

namespace ns {
constexpr int D = 128;
constexpr int WARPS = 8;
constexpr int BATCH = 4;                           // rows in flight per half-warp
constexpr int RB = D / QK * QBLOCK;
}  // namespace ns

__device__ __forceinline__ float half_of(uint16_t x) { return __half2float(__ushort_as_half(x)); }

// page of a slot; a power-of-two page size spares the 64-bit division (log2 < 0: it is none)
__device__ __forceinline__ int64_t slot_page(int64_t slot, int bs, int log2) { return log2 >= 0 ? slot >> log2 : slot / bs; }

// 8 consecutive elements of a row as loaded; fp32 rows take two registers quads
struct Raw8 { uint4 a, b; };

__device__ __forceinline__ Raw8 load_raw8(const void* p, int64_t i, int dt, bool vec) {
  Raw8 r;
  r.b = make_uint4(0, 0, 0, 0);
  if (dt == DT_F32) {
    const float* f = reinterpret_cast<const float*>(p) + i;
    if (vec) {
      r.a = reinterpret_cast<const uint4*>(f)[0];
      r.b = reinterpret_cast<const uint4*>(f)[1];
    } else {
      const uint32_t* u = reinterpret_cast<const uint32_t*>(f);
      r.a = make_uint4(u[0], u[1], u[2], u[3]);
      r.b = make_uint4(u[4], u[5], u[6], u[7]);
    }
  } else {
    const uint16_t* h = reinterpret_cast<const uint16_t*>(p) + i;
    if (vec) r.a = *reinterpret_cast<const uint4*>(h);
    else
      r.a = make_uint4(h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16, h[4] | (uint32_t)h[5] << 16,
                       h[6] | (uint32_t)h[7] << 16);
  }
  return r;
}

__device__ __forceinline__ void widen8(const Raw8& r, int dt, float v[8]) {
  const uint32_t w[8] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w};
  if (dt == DT_F32) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(w[e]);
  } else if (dt == DT_BF16) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[2 * e] = __uint_as_float(w[e] << 16);
      v[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&w[e]));
      v[2 * e] = x.x;
      v[2 * e + 1] = x.y;
    }
  }
}

// rounds v to dt (in place, back as fp32) and returns the packed 16-bit words (16-bit dt)
__device__ __forceinline__ uint4 round8(float v[8], int dt) {
  uint32_t w[4] = {0, 0, 0, 0};
  if (dt == DT_F16) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const __half2 h = __floats2half2_rn(v[2 * e], v[2 * e + 1]);
      w[e] = *reinterpret_cast<const uint32_t*>(&h);
      const float2 x = __half22float2(h);
      v[2 * e] = x.x;
      v[2 * e + 1] = x.y;
    }
  } else if (dt == DT_BF16) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * e], v[2 * e + 1]);
      w[e] = *reinterpret_cast<const uint32_t*>(&h);
      v[2 * e] = __uint_as_float(w[e] << 16);
      v[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// v already rounded to dt, `packed` its 16-bit words
__device__ __forceinline__ void store8(void* p, int64_t i, int dt, bool vec, const float v[8], uint4 packed) {
  if (dt == DT_F32) {
    float* f = reinterpret_cast<float*>(p) + i;
    if (vec) {
      reinterpret_cast<float4*>(f)[0] = make_float4(v[0], v[1], v[2], v[3]);
      reinterpret_cast<float4*>(f)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = v[e];
    }
  } else {
    uint16_t* h = reinterpret_cast<uint16_t*>(p) + i;
    if (vec) {
      *reinterpret_cast<uint4*>(h) = packed;
    } else {
      const uint32_t w[4] = {packed.x, packed.y, packed.z, packed.w};
#pragma unroll
      for (int e = 0; e < 8; ++e) h[e] = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
    }
  }
}

// Q8_0 of the 8 elements of this lane (a block is 4 neighbouring lanes): the
// quantiser's arithmetic, element for element (IEEE division and reciprocal,
// round half to even, clamp).
__device__ __forceinline__ uint2 quant8(const float v[8], uint16_t& scale) {
  float amax = fabsf(v[0]);
#pragma unroll
  for (int e = 1; e < 8; ++e) amax = fmaxf(amax, fabsf(v[e]));
  amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
  amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
  const float d = amax / 127.0f;
  const float id = d > 0.0f ? __frcp_rn(d) : 0.0f;
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    int qi = __float2int_rn(v[e] * id);
    qi = max(-128, min(127, qi));
    w[e >> 2] |= (uint32_t)(qi & 0xff) << (8 * (e & 3));
  }
  scale = __half_as_ushort(__float2half_rn(d));
  return make_uint2(w[0], w[1]);
}

// The same for elements that are fp16 or bf16 values.
__device__ __forceinline__ uint2 quant8_16bit(const float v[8], uint16_t& scale) {
  float amax = fabsf(v[0]);
#pragma unroll
  for (int e = 1; e < 8; ++e) amax = fmaxf(amax, fabsf(v[e]));
  amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
  amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
  float id;
  scale = __half_as_ushort(__float2half_rn(q8_scale_16bit(amax, id)));
  return make_uint2(q8_quants4(v[0], v[1], v[2], v[3], id), q8_quants4(v[4], v[5], v[6], v[7], id));
}

// cos / sin of this lane's 8 elements.  NeoX: element e pairs with e +- rot/2;
// otherwise 2j with 2j + 1, four pairs a lane.
struct Angles { float c[8] = {}, s[8] = {}; };

__device__ __forceinline__ void load_angles(const NormStoreArgs& a, int64_t pos, int hl, Angles& g) {
  const int half = a.rot >> 1, e0 = 8 * hl;
  if (e0 >= a.rot) return;
  const int64_t base = pos * a.rot;
  const int j0 = a.neox ? (e0 < half ? e0 : e0 - half) : e0 >> 1;
  if (a.neox) {
    widen8(load_raw8(a.cos_sin, base + j0, a.cs_dt, a.cs_vec), a.cs_dt, g.c);
    widen8(load_raw8(a.cos_sin, base + half + j0, a.cs_dt, a.cs_vec), a.cs_dt, g.s);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      g.c[e] = load_one(a.cos_sin, base + j0 + e, a.cs_dt);
      g.s[e] = load_one(a.cos_sin, base + half + j0 + e, a.cs_dt);
    }
  }
}

__device__ __forceinline__ void rotate8(const NormStoreArgs& a, const Angles& g, int hl, float v[8]) {
  const int e0 = 8 * hl;
  if (a.neox) {
    const int lanes = a.rot >> 4;                  // lanes per half of the rotated part
    const bool lower = hl < lanes;
    // the partner's lane; lanes past the rotated part read themselves
    const int peer = e0 >= a.rot ? hl : lower ? hl + lanes : hl - lanes;
    const int src = (threadIdx.x & 16) | peer;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float p = __shfl_sync(0xffffffffu, v[e], src);
      if (e0 < a.rot)
        v[e] = lower ? __fsub_rn(__fmul_rn(v[e], g.c[e]), __fmul_rn(p, g.s[e]))
                     : __fadd_rn(__fmul_rn(v[e], g.c[e]), __fmul_rn(p, g.s[e]));
    }
  } else if (e0 < a.rot) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float x = v[2 * e], y = v[2 * e + 1];
      v[2 * e] = __fsub_rn(__fmul_rn(x, g.c[e]), __fmul_rn(y, g.s[e]));
      v[2 * e + 1] = __fadd_rn(__fmul_rn(y, g.c[e]), __fmul_rn(x, g.s[e]));
    }
  }
}

__device__ __forceinline__ void norm8(float v[8], const float w[8], float eps) {
  float ss = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) ss += v[e] * v[e];
#pragma unroll
  for (int x = 1; x < 16; x <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, x);
  const float r = rsqrtf(ss * (1.0f / ns::D) + eps);
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = v[e] * r * w[e];
}

// Q8_0 row from the lanes' blocks: staged so that it leaves as 8-byte words
__device__ __forceinline__ void write_q8_row(uint8_t* dst, uint2 w, uint16_t scale, int hl, bool live, bool w8,
                                             uint8_t* stage) {
  uint16_t* o = reinterpret_cast<uint16_t*>(stage + (hl >> 2) * QBLOCK + 2 + 8 * (hl & 3));
  o[0] = (uint16_t)w.x; o[1] = (uint16_t)(w.x >> 16);
  o[2] = (uint16_t)w.y; o[3] = (uint16_t)(w.y >> 16);
  if ((hl & 3) == 0) *reinterpret_cast<uint16_t*>(stage + (hl >> 2) * QBLOCK) = scale;
  __syncwarp();
  if (live) {
    if (w8) {
      reinterpret_cast<uint64_t*>(dst)[hl] = reinterpret_cast<const uint64_t*>(stage)[hl];
      if (hl == 0) reinterpret_cast<uint64_t*>(dst)[16] = reinterpret_cast<const uint64_t*>(stage)[16];
    } else {
      for (int i = hl; i < ns::RB / 2; i += 16)
        reinterpret_cast<uint16_t*>(dst)[i] = reinterpret_cast<const uint16_t*>(stage)[i];
    }
  }
  __syncwarp();
}

__global__ void __launch_bounds__(ns::WARPS * 32) norm_store_kernel(const __grid_constant__ NormStoreArgs a) {
  using namespace ns;
  __shared__ __align__(16) uint8_t stage_all[WARPS * 2][RB];
  const int lane = lane_id(), hl = lane & 15;
  uint8_t* stage = stage_all[warp_id() * 2 + (lane >> 4)];
  const int chunks = (a.rows + a.rpw - 1) / a.rpw;
  const int64_t items = (int64_t)a.T * chunks;
  // both halves of a warp make the same trips: the shuffles and barriers below are warp-wide
  for (int64_t i0 = ((int64_t)blockIdx.x * WARPS + warp_id()) * 2; i0 < items;
       i0 += (int64_t)gridDim.x * WARPS * 2) {
    const int64_t it = i0 + (lane >> 4);
    const bool on = it < items;
    const int t = on ? (int)(it / chunks) : 0;
    const int r0 = on ? (int)(it % chunks) * a.rpw : 0;
    const int nr = on ? min(a.rpw, a.rows - r0) : 0;
    int64_t pos = a.positions[t];
    const int64_t slot = a.slots[t];
    if (pos < 0 || pos >= a.max_pos) {
      raise_error(ERR_BAD_INDEX);
      pos = 0;
    }
    const int64_t blk = slot_page(slot, a.c.block_size, a.bs_log2);
    const int off = (int)(slot - blk * a.c.block_size);
    bool stored = on && slot >= 0;
    if (stored && a.c.num_blocks > 0 && blk >= a.c.num_blocks) {
      raise_error(ERR_BAD_INDEX);
      stored = false;
    }
    Angles g;
    load_angles(a, pos, hl, g);
    for (int b = 0; b < a.rpw; b += BATCH) {
      Raw8 raw[BATCH];
#pragma unroll
      for (int x = 0; x < BATCH; ++x) {
        const int r = r0 + b + x;
        if (b + x >= a.rpw) break;
        raw[x].a = raw[x].b = make_uint4(0, 0, 0, 0);
        if (b + x < nr) {
          if (r < a.Hq) raw[x] = load_raw8(a.q, (int64_t)t * a.q_tok + (int64_t)r * a.q_head + 8 * hl, a.q_dt, a.q_vec);
          else if (r < a.Hq + a.Hkv)
            raw[x] = load_raw8(a.k, (int64_t)t * a.k_tok + (int64_t)(r - a.Hq) * a.k_head + 8 * hl, a.k_dt, a.k_vec);
          else
            raw[x] = load_raw8(a.v, (int64_t)t * a.v_tok + (int64_t)(r - a.Hq - a.Hkv) * a.v_head + 8 * hl, a.v_dt, a.v_vec);
        }
      }
#pragma unroll
      for (int x = 0; x < BATCH; ++x) {
        const int r = r0 + b + x;
        if (b + x >= a.rpw) break;                 // the same for the whole grid
        const bool live = b + x < nr;
        const bool isq = r < a.Hq, isv = r >= a.Hq + a.Hkv;
        const int dt = isq ? a.q_dt : isv ? a.v_dt : a.k_dt;
        float v[8];
        widen8(raw[x], dt, v);
        // every lane takes the shuffles; their results are used by live query and key rows only
        const void* wp = isq ? a.q_w : a.k_w;
        float w[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (wp) widen8(load_raw8(wp, 8 * hl, isq ? a.qw_dt : a.kw_dt, false), isq ? a.qw_dt : a.kw_dt, w);
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = v[e];
        norm8(y, w, a.eps);
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = wp ? y[e] : v[e];
        rotate8(a, g, hl, y);
        if (!isv) {
          const uint4 packed = round8(y, dt);
          if (live) {
            if (isq)
              store8(a.q_out, (int64_t)t * a.qo_tok + (int64_t)r * a.qo_head + 8 * hl, dt, a.qo_vec, y, packed);
            else if (a.k_out)
              store8(a.k_out, (int64_t)t * a.ko_tok + (int64_t)(r - a.Hq) * a.ko_head + 8 * hl, dt, a.ko_vec, y, packed);
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = y[e];
        }
        // ---- cache rows -------------------------------------------------------
        const bool q8 = !isq && (!isv || a.c.v_mode != G9_V_COPY16);
        if (!__any_sync(0xffffffffu, live && !isq && stored)) continue;
        uint16_t scale;
        const uint2 qw = quant8(v, scale);
        const int h = isv ? r - a.Hq - a.Hkv : r - a.Hq;
        const bool put = live && stored && !isq;
        const bool rows8 = q8 && !(isv && a.c.v_mode == G9_V_Q8T);
        uint8_t* dst = nullptr;
        if (put)
          dst = isv ? a.c.v + blk * a.c.v_page_stride + off * a.c.v_tok_stride + h * a.c.v_head_stride
                    : a.c.k + blk * a.c.k_page_stride + off * a.c.k_tok_stride + h * a.c.k_head_stride;
        write_q8_row(dst, qw, scale, hl, put && rows8, isv ? a.v_w8 : a.k_w8, stage);
        if (put && isv && a.c.v_mode == G9_V_COPY16) {
          store8(dst, 8 * hl, a.v_dt, a.v_w16, v, raw[x].a);
        } else if (put && isv && a.c.v_mode == G9_V_Q8T) {
          uint8_t* rec = a.c.v + blk * a.c.v_page_stride + h * a.c.v_head_stride;
          const int bs = a.c.block_size;
          if ((hl & 3) == 0) *reinterpret_cast<uint16_t*>(rec + 2 * ((int64_t)(hl >> 2) * bs + off)) = scale;
          uint8_t* o = rec + 2 * (D / QK) * bs + (int64_t)8 * hl * bs + off;
#pragma unroll
          for (int e = 0; e < 8; ++e) o[(int64_t)e * bs] = (uint8_t)((e < 4 ? qw.x : qw.y) >> (8 * (e & 3)));
        }
      }
    }
  }
}

// ---------------------------------------------------------------------------
// 16-bit tensors of one type on 16-byte rows, 8-byte cache rows: what a model
// serves.  Three CTAs an SM at 80 registers: with two, 16384 tokens and their read
// back took 1.18 times as long; four spill (0.98 times there, but 1.28 times at
// 2111 tokens).  Queries, keys and values are separate warp items, so that no warp
// carries another operand's code: a query item is QR rows of a token (their
// angles loaded once), a key item its kv heads, a value item a run of slots
// (page-transposed) or a token's heads.
// ---------------------------------------------------------------------------
struct FastItems {
  int qr, pq, pk, pv;            // query rows an item; items a token of queries, keys and (rows) values
  uint32_t nq, nk, nv;           // items, below 2^31 in all
};

// The tokens of a value item.  Page-transposed V is written by runs: tokens
// whose slots follow one another inside an aligned group of 16, at most 16.  A
// warp looks at 16 tokens and takes the runs that start among them; a run of
// all 16 slots leaves as 16-byte stores (one per dim), where single tokens cost
// a byte store per element.  Returns a bit per token i = 0..31 that continues the run of token i - 1.
__device__ __forceinline__ uint32_t run_bits(const int64_t* slots, int t0, int T, int64_t end, int64_t& mine) {
  const int t = t0 + lane_id();
  mine = t < T ? slots[t] : -1;
  const int64_t before = t > 0 && t <= T ? slots[t - 1] : -1;
  const bool ok = mine >= 0 && mine < end;
  if (mine >= end) raise_error(ERR_BAD_INDEX);
  if (!ok) mine = -1;
  return __ballot_sync(0xffffffffu, ok && before >= 0 && mine == before + 1 && (mine & 15) != 0);
}

template <int DT>
__device__ __forceinline__ void widen16(uint4 r, float v[8]) {
  Raw8 x;
  x.a = r;
  widen8(x, DT, v);
}

// 4 x 4 bytes: word i of w holds byte i of each result word
__device__ __forceinline__ void transpose4(uint32_t w[4]) {
  const uint32_t a = __byte_perm(w[0], w[1], 0x5140), b = __byte_perm(w[2], w[3], 0x5140);
  const uint32_t c = __byte_perm(w[0], w[1], 0x7362), d = __byte_perm(w[2], w[3], 0x7362);
  w[0] = __byte_perm(a, b, 0x5410);
  w[1] = __byte_perm(a, b, 0x7632);
  w[2] = __byte_perm(c, d, 0x5410);
  w[3] = __byte_perm(c, d, 0x7632);
}

// A half-warp's angles and weight as packed pairs of fp32 (f32x2 arithmetic: one
// instruction, two elements).  s carries the sign of its term; lanes past the rotated part keep their values.
struct Pairs { uint64_t c[4], s[4], w[4]; };

__device__ __forceinline__ void make_pairs(const NormStoreArgs& a, const Angles& g, const float w[8], int hl, Pairs& o) {
  const bool lower = hl < (a.rot >> 4);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    o.w[e] = f2pack(w[2 * e], w[2 * e + 1]);
    if (a.neox) {
      o.c[e] = f2pack(g.c[2 * e], g.c[2 * e + 1]);
      o.s[e] = lower ? f2pack(-g.s[2 * e], -g.s[2 * e + 1]) : f2pack(g.s[2 * e], g.s[2 * e + 1]);
    } else {                                         // pair (x, y): x' = x c - y s, y' = y c + x s
      o.c[e] = f2pack(g.c[e], g.c[e]);
      o.s[e] = f2pack(-g.s[e], g.s[e]);
    }
  }
}

// Norm and rotation of the row held as 8 elements a lane; the arithmetic of
// norm8 and rotate8, product by product.  FULL: every element is rotated.
template <bool NEOX, bool FULL>
__device__ __forceinline__ void norm_rope_row(const NormStoreArgs& a, const Pairs& g, bool norm, int hl, int src, float v[8]) {
  uint64_t x[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = f2pack(v[2 * e], v[2 * e + 1]);
  if (norm) {
    uint64_t ss2 = f2mul(x[0], x[0]);
#pragma unroll
    for (int e = 1; e < 4; ++e) ss2 = f2fma(x[e], x[e], ss2);
    float s0, s1;
    f2unpack(ss2, s0, s1);
    float ss = s0 + s1;
#pragma unroll
    for (int k = 1; k < 16; k <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, k);
    const float r = rsqrtf(ss * (1.0f / ns::D) + a.eps);
    const uint64_t r2 = f2pack(r, r);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = f2mul(f2mul(x[e], r2), g.w[e]);
  }
  uint64_t y[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float lo, hi;
    f2unpack(x[e], lo, hi);
    uint64_t p;                                      // the partners
    if (NEOX) p = f2pack(__shfl_sync(0xffffffffu, lo, src), __shfl_sync(0xffffffffu, hi, src));
    else p = f2pack(hi, lo);
    y[e] = f2add(f2mul(x[e], g.c[e]), f2mul(p, g.s[e]));
  }
  const bool in = FULL || 8 * hl < a.rot;
#pragma unroll
  for (int e = 0; e < 4; ++e) f2unpack(in ? y[e] : x[e], v[2 * e], v[2 * e + 1]);
}

template <int DT, bool NEOX, bool FULL>
__global__ void __launch_bounds__(ns::WARPS * 32, 3) norm_store_fast_kernel(const __grid_constant__ NormStoreArgs a,
                                                                         const __grid_constant__ FastItems f) {
  using namespace ns;
  __shared__ __align__(16) uint8_t stage_all[WARPS][16 * 128 + 128];
  uint8_t* stage = stage_all[warp_id()];
  const int lane = lane_id(), hl = lane & 15, half = lane >> 4;
  const uint32_t total = f.nq + f.nk + f.nv, stride = gridDim.x * WARPS;
  for (uint32_t it = blockIdx.x * WARPS + warp_id(); it < total; it += stride) {
    if (it < f.nq + f.nk) {
      const bool isq = it < f.nq;
      const uint32_t i = isq ? it : it - f.nq, parts = isq ? f.pq : f.pk;
      const int t = (int)(i / parts), H = isq ? a.Hq : a.Hkv;
      const int per = isq ? f.qr : 8;                    // rows of this item: per / 2 a half-warp
      const int r0 = (int)(i - t * parts) * per;
      const int rows = min(per, H - r0);
      int64_t pos = a.positions[t];
      if (pos < 0 || pos >= a.max_pos) {
        raise_error(ERR_BAD_INDEX);
        pos = 0;
      }
      const uint16_t* src = reinterpret_cast<const uint16_t*>(isq ? a.q : a.k) + (int64_t)t * (isq ? a.q_tok : a.k_tok) + 8 * hl;
      const int64_t hs = isq ? a.q_head : a.k_head;        // below 2^24
      // this half-warp's rows are `step` apart; a row past the last is read at the last one's place
      const int step = (int)(2 * hs);
      const uint16_t* sp = src + (int64_t)(r0 + half) * hs;
      uint4 raw[4];
#pragma unroll
      for (int x = 0; x < 4; ++x)
        raw[x] = *reinterpret_cast<const uint4*>(2 * x + half < rows ? sp + x * step : src + (int64_t)(r0 + rows - 1) * hs);
      Angles angles;
      load_angles(a, pos, hl, angles);
      const void* wp = isq ? a.q_w : a.k_w;
      float w[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (wp) widen8(load_raw8(wp, 8 * hl, isq ? a.qw_dt : a.kw_dt, false), isq ? a.qw_dt : a.kw_dt, w);
      Pairs g;
      make_pairs(a, angles, w, hl, g);
      // the lane that holds this one's partners; lanes past the rotated part read themselves
      const int lanes = a.rot >> 4, peer = hl >= 2 * lanes ? hl : hl < lanes ? hl + lanes : hl - lanes;
      const int from = (lane & 16) | peer;
      if (isq) {
        uint16_t* dp = reinterpret_cast<uint16_t*>(a.q_out) + (int64_t)t * a.qo_tok + (int64_t)(r0 + half) * a.qo_head + 8 * hl;
        const int dstep = (int)(2 * a.qo_head);
#pragma unroll 1
        for (int left = rows - half; left > -half; left -= 8) {        // rows from this half's next one on
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            if (left + half <= 2 * x) break;             // the same for both halves
            float v[8];
            widen16<DT>(raw[x], v);
            // the row eight further on takes its place, in flight while the others are worked on
            if (left > 8 + 2 * x) raw[x] = *reinterpret_cast<const uint4*>(sp + (x + 4) * step);
            norm_rope_row<NEOX, FULL>(a, g, wp != nullptr, hl, from, v);
            const uint4 packed = round8(v, DT);
            if (left > 2 * x) *reinterpret_cast<uint4*>(dp + x * dstep) = packed;
          }
          sp += 4 * step;
          dp += 4 * dstep;
        }
      } else {
        const int64_t slot = a.slots[t];
        const int64_t blk = slot_page(slot, a.c.block_size, a.bs_log2);
        const int off = (int)(slot - blk * a.c.block_size);
        bool stored = slot >= 0;
        if (stored && a.c.num_blocks > 0 && blk >= a.c.num_blocks) {
          raise_error(ERR_BAD_INDEX);
          stored = false;
        }
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          if (2 * x >= rows) break;
          const int r = 2 * x + half;
          float v[8];
          widen16<DT>(raw[x], v);
          norm_rope_row<NEOX, FULL>(a, g, wp != nullptr, hl, from, v);
          const uint4 packed = round8(v, DT);
          if (a.k_out && r < rows)
            *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(a.k_out) + (int64_t)t * a.ko_tok + (int64_t)(r0 + r) * a.ko_head + 8 * hl) = packed;
          if (!stored) continue;                         // the same for the warp
          uint16_t scale;
          const uint2 q = quant8_16bit(v, scale);
          uint8_t* dst = a.c.k + blk * a.c.k_page_stride + off * a.c.k_tok_stride + (int64_t)(r0 + r) * a.c.k_head_stride;
          write_q8_row(dst, q, scale, hl, r < rows, true, stage + half * RB);
        }
      }
      continue;
    }
    const uint32_t i = it - f.nq - f.nk;
    if (a.c.v_mode != G9_V_Q8T) {
      // token rows: eight kv heads of a token
      const int t = (int)(i / (uint32_t)f.pv), r0 = (int)(i - t * f.pv) * 8, rows = min(8, a.Hkv - r0);
      const uint16_t* src = reinterpret_cast<const uint16_t*>(a.v) + (int64_t)t * a.v_tok + 8 * hl;
      uint4 raw[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) raw[x] = *reinterpret_cast<const uint4*>(src + (int64_t)(r0 + min(2 * x + half, rows - 1)) * a.v_head);
      const int64_t slot = a.slots[t];
      const int64_t blk = slot_page(slot, a.c.block_size, a.bs_log2);
      const int off = (int)(slot - blk * a.c.block_size);
      if (slot < 0) continue;
      if (a.c.num_blocks > 0 && blk >= a.c.num_blocks) {
        raise_error(ERR_BAD_INDEX);
        continue;
      }
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        if (2 * x >= rows) break;
        const int r = 2 * x + half;
        uint8_t* dst = a.c.v + blk * a.c.v_page_stride + off * a.c.v_tok_stride + (int64_t)(r0 + r) * a.c.v_head_stride;
        if (a.c.v_mode == G9_V_COPY16) {
          if (r < rows) *reinterpret_cast<uint4*>(dst + 16 * hl) = raw[x];
        } else {
          float v[8];
          widen16<DT>(raw[x], v);
          uint16_t scale;
          const uint2 q = quant8_16bit(v, scale);
          write_q8_row(dst, q, scale, hl, r < rows, true, stage + half * RB);
        }
      }
      continue;
    }
    // ---- page-transposed V: (16 tokens, kv head) ----------------------------------
    const int h = (int)(i % (uint32_t)a.Hkv);
    const int t0 = (int)(i / (uint32_t)a.Hkv) * 16;
    const int bs = a.c.block_size;
    int64_t mine;
    const uint32_t cont = run_bits(a.slots, t0, a.T, a.c.num_blocks > 0 ? (int64_t)a.c.num_blocks * bs : INT64_MAX, mine);
    const uint32_t live = __ballot_sync(0xffffffffu, mine >= 0);
    for (uint32_t heads = live & ~cont & 0xffffu; heads; heads &= heads - 1) {
      const int i0 = __ffs(heads) - 1;                   // the run's first token
      const int n = 1 + (i0 == 31 ? 0 : __ffs(~(cont >> (i0 + 1))) - 1);         // cont has a zero above bit 31 - i0
      const int64_t slot = __shfl_sync(0xffffffffu, mine, i0);
      const int64_t blk = slot_page(slot, bs, a.bs_log2);
      const int off = (int)(slot - blk * bs), sub = off & 15;
      const uint16_t* src = reinterpret_cast<const uint16_t*>(a.v) + (int64_t)(t0 + i0) * a.v_tok + (int64_t)h * a.v_head + 8 * hl;
      uint16_t* scales = reinterpret_cast<uint16_t*>(stage + 16 * 128);          // [block][16]
      // quantised rows into [slot % 16][dim], two tokens a step, four steps' loads in flight
      for (int b = 0; b < n; b += 8) {
        uint4 raw[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) raw[x] = *reinterpret_cast<const uint4*>(src + (int64_t)min(b + 2 * x + half, n - 1) * a.v_tok);
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          if (b + 2 * x >= n) break;
          const int k = b + 2 * x + half;
          float v[8];
          widen16<DT>(raw[x], v);
          uint16_t scale;
          const uint2 q = quant8_16bit(v, scale);
          if (k < n) {
            *reinterpret_cast<uint2*>(stage + (sub + k) * 128 + 8 * hl) = q;
            if ((hl & 3) == 0) scales[(hl >> 2) * 16 + sub + k] = scale;
          }
        }
      }
      __syncwarp();
      uint8_t* rec = a.c.v + blk * a.c.v_page_stride + (int64_t)h * a.c.v_head_stride;
      uint8_t* sdst = rec + 2 * (off - sub);
      uint8_t* vdst = rec + 2 * (D / QK) * bs + (off - sub);
      // lane: dims 4 * lane .. + 3, 16 tokens each
      uint32_t y[4][4];
#pragma unroll
      for (int k4 = 0; k4 < 4; ++k4) {
        uint32_t x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = *reinterpret_cast<const uint32_t*>(stage + (4 * k4 + e) * 128 + 4 * lane);
        transpose4(x);
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e][k4] = x[e];
      }
      if (n == 16 && a.v_rec16) {
        if (lane < 8) *reinterpret_cast<uint4*>(sdst + 2 * (lane >> 1) * bs + 16 * (lane & 1)) =
            *reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(scales) + 16 * lane);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          *reinterpret_cast<uint4*>(vdst + (int64_t)(4 * lane + e) * bs) = make_uint4(y[e][0], y[e][1], y[e][2], y[e][3]);
      } else {
        for (int x = lane; x < 4 * n; x += 32) {
          const int blkq = x / n, k = sub + x - blkq * n;
          *reinterpret_cast<uint16_t*>(sdst + 2 * (blkq * bs + k)) = scales[blkq * 16 + k];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int k = 0; k < 16; ++k)
            if (k >= sub && k < sub + n) vdst[(int64_t)(4 * lane + e) * bs + k] = (uint8_t)(y[e][k >> 2] >> (8 * (k & 3)));
      }
      __syncwarp();
    }
  }
}

// ---------------------------------------------------------------------------
// read_kv: rows of the cache by slot, as 16- or 32-bit values
// ---------------------------------------------------------------------------
constexpr int RR = 4;

struct ReadArgs {
  G9KvCache c;
  const int64_t* slots;
  int bs_log2, N, Hkv, out_dt, v_src;                       // v_src: DT_F16 / DT_BF16 of 16-bit V rows
  int k_w8, v_w8, v_w16, v_rec16;                  // rows on 8- and 16-byte boundaries, records on 16
  uint32_t rows;                                   // rows the row items cover: N * Hkv keys, then as many values unless they go by runs
  uint32_t nrows, nruns;                           // row items (2 * RR rows a warp); run items follow
  void* k_out; void* v_out;                        // [N, Hkv, 128]; v_out may be null
};

// elements 8 * hl .. + 7 of a Q8_0 row as loaded, and their scale
struct Q8Lane { uint64_t lo, hi; uint16_t d; };

__device__ __forceinline__ Q8Lane q8_load(const uint8_t* row, int hl, bool w8) {
  const int blk = hl >> 2, o = blk * QBLOCK + 2 + 8 * (hl & 3);
  Q8Lane x;
  x.d = *reinterpret_cast<const uint16_t*>(row + blk * QBLOCK);
  if (w8) {
    // the 8 values start 2, 4, 6 or 0 bytes into an aligned word: that word and the next, which block 3 does not need
    const uint64_t* p = reinterpret_cast<const uint64_t*>(row + (o & ~7));
    x.lo = p[0];
    x.hi = p[blk < 3];
  } else {
    const uint16_t* q = reinterpret_cast<const uint16_t*>(row + o);
    x.lo = (uint64_t)q[0] | (uint64_t)q[1] << 16 | (uint64_t)q[2] << 32 | (uint64_t)q[3] << 48;
    x.hi = 0;
  }
  return x;
}

__device__ __forceinline__ void q8_values(const Q8Lane& x, int hl, bool w8, float v[8]) {
  const int blk = hl >> 2, sh = w8 ? ((blk * QBLOCK + 2) & 7) * 8 : 0;
  const uint64_t q = sh ? x.lo >> sh | x.hi << (64 - sh) : x.lo;
  const float d = half_of(x.d);
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = (float)(int8_t)(q >> (8 * e)) * d;
}

// 16384 rows of 8 heads (L2 flushed before): 43 us for 103 MB with page-transposed V, 58 us for 118 MB with 16-bit V, 59 us
// for 103 MB with token-row Q8_0 V: latency, nothing of an item is asked for before the one before it is done.  Row items: half a warp reads RR rows.  Run items: page-transposed V by
// runs of slots (run_bits): a lane takes 4 dims x 16 tokens as four 16-byte
// loads, whatever part of the 16 the run covers.
__global__ void __launch_bounds__(ns::WARPS * 32) read_kv_kernel(const __grid_constant__ ReadArgs a) {
  using namespace ns;
  const int lane = lane_id(), hl = lane & 15;
  const int bs = a.c.block_size;
  const int64_t end = a.c.num_blocks > 0 ? (int64_t)a.c.num_blocks * bs : INT64_MAX;
  const uint32_t total = a.nrows + a.nruns, krows = (uint32_t)a.N * a.Hkv, stride = gridDim.x * WARPS;
  for (uint32_t it = blockIdx.x * WARPS + warp_id(); it < total; it += stride) {
    if (it < a.nrows) {
      // RR rows a half-warp: their slots, then their cache rows, loaded together
      uint32_t r[RR];
      int64_t slot[RR];
      bool isv[RR];
#pragma unroll
      for (int k = 0; k < RR; ++k) {
        const uint32_t y = (it * RR + k) * 2 + (lane >> 4);
        isv[k] = y >= krows;
        r[k] = y >= a.rows ? krows : isv[k] ? y - krows : y;           // past the last row: no row
        slot[k] = r[k] < krows ? a.slots[r[k] / (uint32_t)a.Hkv] : -1;
      }
      Q8Lane q[RR];
      Raw8 w[RR];
#pragma unroll
      for (int k = 0; k < RR; ++k) {
        q[k].lo = q[k].hi = 0;
        q[k].d = 0;
        w[k].a = w[k].b = make_uint4(0, 0, 0, 0);
        if (slot[k] >= end) {
          raise_error(ERR_BAD_INDEX);
          slot[k] = -1;
        }
        if (slot[k] < 0) continue;
        const int h = (int)(r[k] % (uint32_t)a.Hkv);
        const int64_t blk = slot_page(slot[k], bs, a.bs_log2);
        const int off = (int)(slot[k] - blk * bs);
        if (!isv[k]) {
          q[k] = q8_load(a.c.k + blk * a.c.k_page_stride + off * a.c.k_tok_stride + h * a.c.k_head_stride, hl, a.k_w8);
        } else if (a.c.v_mode == G9_V_Q8T) {             // records off 16-byte boundaries
          const uint8_t* rec = a.c.v + blk * a.c.v_page_stride + h * a.c.v_head_stride;
          q[k].d = *reinterpret_cast<const uint16_t*>(rec + 2 * ((int64_t)(hl >> 2) * bs + off));
          const uint8_t* x = rec + 2 * (D / QK) * bs + (int64_t)8 * hl * bs + off;
#pragma unroll
          for (int e = 0; e < 8; ++e) q[k].lo |= (uint64_t)x[(int64_t)e * bs] << (8 * e);
        } else {
          const uint8_t* row = a.c.v + blk * a.c.v_page_stride + off * a.c.v_tok_stride + h * a.c.v_head_stride;
          if (a.c.v_mode == G9_V_Q8) q[k] = q8_load(row, hl, a.v_w8);
          else w[k] = load_raw8(row, 8 * hl, a.v_src, a.v_w16);
        }
      }
#pragma unroll
      for (int k = 0; k < RR; ++k) {
        if (r[k] >= krows) continue;
        float v[8];
        if (isv[k] && a.c.v_mode == G9_V_COPY16) widen8(w[k], a.v_src, v);
        else q8_values(q[k], hl, isv[k] ? a.c.v_mode == G9_V_Q8 && a.v_w8 : a.k_w8, v);
        const uint4 packed = round8(v, a.out_dt);
        store8(isv[k] ? a.v_out : a.k_out, (int64_t)r[k] * D + 8 * hl, a.out_dt, true, v, packed);
      }
      continue;
    }
    const uint32_t i = it - a.nrows;
    const int h = (int)(i % (uint32_t)a.Hkv);
    const int t0 = (int)(i / (uint32_t)a.Hkv) * 16;
    int64_t mine;
    const uint32_t cont = run_bits(a.slots, t0, a.N, end, mine);
    const uint32_t live = __ballot_sync(0xffffffffu, mine >= 0);
    for (uint32_t heads = ~(live & cont) & 0xffffu; heads; heads &= heads - 1) {
      const int i0 = __ffs(heads) - 1;
      if (t0 + i0 >= a.N) break;
      const int n = 1 + __ffs(~(cont >> (i0 + 1))) - 1;
      const int64_t slot = __shfl_sync(0xffffffffu, mine, i0);
      uint4 q[4];
      uint4 s[2];
#pragma unroll
      for (int e = 0; e < 4; ++e) q[e] = make_uint4(0, 0, 0, 0);
      s[0] = s[1] = make_uint4(0, 0, 0, 0);
      int sub = 0;
      if (slot >= 0) {
        const int64_t blk = slot_page(slot, bs, a.bs_log2);
        const int off = (int)(slot - blk * bs);
        sub = off & 15;
        const uint8_t* rec = a.c.v + blk * a.c.v_page_stride + (int64_t)h * a.c.v_head_stride;
        const uint4* sp = reinterpret_cast<const uint4*>(rec + 2 * ((int64_t)(lane >> 3) * bs + off - sub));
        s[0] = sp[0];
        s[1] = sp[1];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          q[e] = *reinterpret_cast<const uint4*>(rec + 2 * (D / QK) * bs + (int64_t)(4 * lane + e) * bs + off - sub);
      }
      const uint32_t sw[8] = {s[0].x, s[0].y, s[0].z, s[0].w, s[1].x, s[1].y, s[1].z, s[1].w};
#pragma unroll
      for (int k4 = 0; k4 < 4; ++k4) {
        uint32_t x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = k4 == 0 ? q[e].x : k4 == 1 ? q[e].y : k4 == 2 ? q[e].z : q[e].w;
        transpose4(x);                                   // x[k]: token 4 * k4 + k, this lane's 4 dims
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int tok = 4 * k4 + k;
          if (tok < sub || tok >= sub + n) continue;
          const float d = half_of((uint16_t)(sw[tok >> 1] >> (16 * (tok & 1))));
          float v[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = (float)(int8_t)(x[k] >> (8 * e)) * d;
          const int64_t at = ((int64_t)(t0 + i0 + tok - sub) * a.Hkv + h) * D + 4 * lane;
          if (a.out_dt == DT_F32) {
            *reinterpret_cast<float4*>(reinterpret_cast<float*>(a.v_out) + at) = make_float4(v[0], v[1], v[2], v[3]);
          } else {
            uint2 o;
            if (a.out_dt == DT_F16) {
              const __half2 x0 = __floats2half2_rn(v[0], v[1]), x1 = __floats2half2_rn(v[2], v[3]);
              o = make_uint2(*reinterpret_cast<const uint32_t*>(&x0), *reinterpret_cast<const uint32_t*>(&x1));
            } else {
              const __nv_bfloat162 x0 = __floats2bfloat162_rn(v[0], v[1]), x1 = __floats2bfloat162_rn(v[2], v[3]);
              o = make_uint2(*reinterpret_cast<const uint32_t*>(&x0), *reinterpret_cast<const uint32_t*>(&x1));
            }
            *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(a.v_out) + at) = o;
          }
        }
      }
    }
  }
}

static int ns_sms() {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms;
}

static bool rows16(const void* base, int dt, int64_t s0, int64_t s1) {
  const int64_t per = dt == DT_F32 ? 4 : 8;        // elements in 16 bytes
  return (uintptr_t)base % 16 == 0 && s0 % per == 0 && s1 % per == 0;
}

// 2-byte aligned Q8_0 rows (scales are 16-bit words), 16-bit V rows likewise
static bool cache_ok(const G9KvCache& c) {
  if (!c.k || c.block_size <= 0 || c.num_heads_kv <= 0 || c.num_blocks < 0 || c.v_mode < 0 || c.v_mode > 3) return false;
  if (((uintptr_t)c.k | (uintptr_t)c.k_page_stride | (uintptr_t)c.k_tok_stride | (uintptr_t)c.k_head_stride) & 1) return false;
  if (c.v_mode == G9_V_NONE) return true;
  uintptr_t m = (uintptr_t)c.v | (uintptr_t)c.v_page_stride | (uintptr_t)c.v_head_stride;
  if (c.v_mode != G9_V_Q8T) m |= (uintptr_t)c.v_tok_stride;
  return c.v && !(m & 1);
}

static int log2_or(int x) {
  if (x & (x - 1)) return -1;
  int n = 0;
  while ((1 << n) < x) ++n;
  return n;
}

static bool aligned(uintptr_t base, int64_t a, int64_t b, int64_t c, uintptr_t to) {
  return ((base | (uintptr_t)a | (uintptr_t)b | (uintptr_t)c) & (to - 1)) == 0;
}

}  // namespace g9

G9_ERROR_ACCESSORS(norm_store)

using namespace g9;

extern "C" cudaError_t gfx906_fa_norm_rope_store_kv(
    const void* query, int query_dtype, int64_t query_token_stride, int64_t query_head_stride, int num_heads_q,
    const void* key, int key_dtype, int64_t key_token_stride, int64_t key_head_stride, const void* value,
    int value_dtype, int64_t value_token_stride, int64_t value_head_stride, const void* q_weight, int q_weight_dtype,
    const void* k_weight, int k_weight_dtype, float eps, const int64_t* positions, const void* cos_sin_cache,
    int cos_sin_dtype, int rot_dim, int64_t max_position, int is_neox, const int64_t* slot_mapping,
    const G9KvCache* cache, void* query_out, int64_t query_out_token_stride, int64_t query_out_head_stride,
    void* key_out, int64_t key_out_token_stride, int64_t key_out_head_stride, int num_tokens, cudaStream_t stream) {
  if (!cache || num_tokens < 0 || !cache_ok(*cache)) return cudaErrorInvalidValue;
  if (!key || !positions || !cos_sin_cache || !slot_mapping || max_position <= 0) return cudaErrorInvalidValue;
  if (rot_dim <= 0 || rot_dim > 128 || rot_dim % 16) return cudaErrorInvalidValue;
  auto dt_ok = [](int d) { return d >= 0 && d <= 2; };
  if (!dt_ok(key_dtype) || !dt_ok(cos_sin_dtype) || !dt_ok(q_weight_dtype) || !dt_ok(k_weight_dtype)) return cudaErrorInvalidValue;
  if (query && (num_heads_q <= 0 || !dt_ok(query_dtype) || !query_out)) return cudaErrorInvalidValue;
  if (cache->v_mode != G9_V_NONE && (!value || !dt_ok(value_dtype))) return cudaErrorInvalidValue;
  if (cache->v_mode == G9_V_COPY16 && value_dtype == G9_DT_F32) return cudaErrorInvalidValue;
  if (num_tokens == 0) return cudaSuccess;
  NormStoreArgs a{};
  a.q = query; a.q_dt = query_dtype; a.q_tok = query_token_stride; a.q_head = query_head_stride;
  a.k = key; a.k_dt = key_dtype; a.k_tok = key_token_stride; a.k_head = key_head_stride;
  a.v = value; a.v_dt = value_dtype; a.v_tok = value_token_stride; a.v_head = value_head_stride;
  a.q_out = query_out; a.qo_tok = query_out_token_stride; a.qo_head = query_out_head_stride;
  a.k_out = key_out; a.ko_tok = key_out_token_stride; a.ko_head = key_out_head_stride;
  a.q_vec = rows16(query, query_dtype, query_token_stride, query_head_stride);
  a.k_vec = rows16(key, key_dtype, key_token_stride, key_head_stride);
  a.v_vec = rows16(value, value_dtype, value_token_stride, value_head_stride);
  a.qo_vec = rows16(query_out, query_dtype, query_out_token_stride, query_out_head_stride);
  a.ko_vec = rows16(key_out, key_dtype, key_out_token_stride, key_out_head_stride);
  a.q_w = q_weight; a.qw_dt = q_weight_dtype; a.k_w = k_weight; a.kw_dt = k_weight_dtype; a.eps = eps;
  a.positions = positions; a.cos_sin = cos_sin_cache; a.cs_dt = cos_sin_dtype; a.rot = rot_dim; a.neox = is_neox ? 1 : 0;
  a.max_pos = max_position;
  a.cs_vec = rows16(cos_sin_cache, cos_sin_dtype, rot_dim, rot_dim / 2);
  a.slots = slot_mapping;
  a.c = *cache;
  a.k_w8 = aligned((uintptr_t)cache->k, cache->k_page_stride, cache->k_tok_stride, cache->k_head_stride, 8);
  a.v_w8 = aligned((uintptr_t)cache->v, cache->v_page_stride, cache->v_tok_stride, cache->v_head_stride, 8);
  a.v_w16 = aligned((uintptr_t)cache->v, cache->v_page_stride, cache->v_tok_stride, cache->v_head_stride, 16);
  a.bs_log2 = log2_or(cache->block_size);
  a.T = num_tokens; a.Hq = query ? num_heads_q : 0; a.Hkv = cache->num_heads_kv;
  a.rows = a.Hq + a.Hkv + (cache->v_mode != G9_V_NONE ? a.Hkv : 0);
  a.v_rec16 = cache->block_size % 16 == 0 &&
              aligned((uintptr_t)cache->v, cache->v_page_stride, cache->v_head_stride, 0, 16);
  const int sms = ns_sms();
  const bool withv = cache->v_mode != G9_V_NONE;
  const bool fast = key_dtype != G9_DT_F32 && (!query || query_dtype == key_dtype) && (!withv || value_dtype == key_dtype) &&
                    a.k_vec && (!query || (a.q_vec && a.qo_vec)) && (!key_out || a.ko_vec) && (!withv || a.v_vec) && a.k_w8 &&
                    (cache->v_mode != G9_V_Q8 || a.v_w8) && (cache->v_mode != G9_V_COPY16 || a.v_w16) &&
                    (cache->v_mode != G9_V_Q8T || cache->block_size % 16 == 0) &&
                    (int64_t)num_tokens * (a.Hq + 3 * (int64_t)a.Hkv) < 0x3fffffff &&    // 32-bit item numbers
                    std::abs(a.q_head) < (1 << 24) && std::abs(a.k_head) < (1 << 24) && std::abs(a.qo_head) < (1 << 24);
  if (fast) {
    FastItems f{};
    // Few tokens: 8 query rows a warp, so that more SMs have work.  Many: a token's queries, which share its angles and the
    // weights (16384 tokens of 48 + 8 heads, the call and its read back: 16 rows an item take 1.06 times as long).
    f.qr = (int64_t)num_tokens * a.Hq < (int64_t)sms * ns::WARPS * 32 ? 8 : (a.Hq + 7) / 8 * 8;
    f.pq = (a.Hq + f.qr - 1) / f.qr;
    f.pk = (a.Hkv + 7) / 8;
    f.pv = (a.Hkv + 7) / 8;
    f.nq = num_tokens * f.pq;
    f.nk = num_tokens * f.pk;
    f.nv = !withv ? 0 : cache->v_mode == G9_V_Q8T ? (num_tokens + 15) / 16 * a.Hkv : num_tokens * f.pv;
    const int64_t want = (int64_t)(f.nq + f.nk + f.nv + ns::WARPS - 1) / ns::WARPS, cap = (int64_t)sms * 32;
    const int grid = (int)(want < cap ? want : cap);
    auto launch = [&](auto kern) {
      kern<<<grid, ns::WARPS * 32, 0, stream>>>(a, f);
      return cudaGetLastError();
    };
    const bool full = rot_dim == 128;
    if (key_dtype == G9_DT_F16) {
      if (a.neox) return full ? launch(norm_store_fast_kernel<DT_F16, true, true>) : launch(norm_store_fast_kernel<DT_F16, true, false>);
      return full ? launch(norm_store_fast_kernel<DT_F16, false, true>) : launch(norm_store_fast_kernel<DT_F16, false, false>);
    }
    if (a.neox) return full ? launch(norm_store_fast_kernel<DT_BF16, true, true>) : launch(norm_store_fast_kernel<DT_BF16, true, false>);
    return full ? launch(norm_store_fast_kernel<DT_BF16, false, true>) : launch(norm_store_fast_kernel<DT_BF16, false, false>);
  }
  // other types, alignments and page sizes; a half-warp a row when rows are few, else BATCH rows share a token's angles
  a.rpw = (int64_t)num_tokens * a.rows < (int64_t)sms * ns::WARPS * 2 * ns::BATCH ? 1 : ns::BATCH;
  const int64_t items = (int64_t)num_tokens * ((a.rows + a.rpw - 1) / a.rpw);
  const int64_t want = (items + ns::WARPS * 2 - 1) / (ns::WARPS * 2);
  norm_store_kernel<<<(int)(want < (int64_t)sms * 16 ? want : (int64_t)sms * 16), ns::WARPS * 32, 0, stream>>>(a);
  return cudaGetLastError();
}

extern "C" cudaError_t gfx906_fa_read_kv(const G9KvCache* cache, int value_dtype, const int64_t* slots, int num_rows,
                                         void* key_out, void* value_out, int out_dtype, cudaStream_t stream) {
  if (!cache || num_rows < 0 || !cache_ok(*cache) || out_dtype < 0 || out_dtype > 2) return cudaErrorInvalidValue;
  if (num_rows == 0) return cudaSuccess;
  if (!slots || !key_out || (uintptr_t)key_out % 16 || (uintptr_t)value_out % 16) return cudaErrorInvalidValue;
  if (value_out && cache->v_mode == G9_V_NONE) return cudaErrorInvalidValue;
  if (value_out && cache->v_mode == G9_V_COPY16 && value_dtype != G9_DT_F16 && value_dtype != G9_DT_BF16)
    return cudaErrorInvalidValue;
  ReadArgs a{};
  a.c = *cache;
  a.bs_log2 = log2_or(cache->block_size);
  a.slots = slots; a.N = num_rows; a.Hkv = cache->num_heads_kv; a.out_dt = out_dtype; a.v_src = value_dtype;
  a.k_out = key_out; a.v_out = value_out;
  a.k_w8 = aligned((uintptr_t)cache->k, cache->k_page_stride, cache->k_tok_stride, cache->k_head_stride, 8);
  a.v_w8 = aligned((uintptr_t)cache->v, cache->v_page_stride, cache->v_tok_stride, cache->v_head_stride, 8);
  a.v_w16 = aligned((uintptr_t)cache->v, cache->v_page_stride, cache->v_tok_stride, cache->v_head_stride, 16);
  a.v_rec16 = cache->block_size % 16 == 0 && aligned((uintptr_t)cache->v, cache->v_page_stride, cache->v_head_stride, 0, 16);
  const int64_t rows = (int64_t)num_rows * a.Hkv;
  if (rows >= 0x3fffffff) return cudaErrorInvalidValue;                // 32-bit row numbers
  const bool runs = value_out && cache->v_mode == G9_V_Q8T && a.v_rec16;
  a.rows = (uint32_t)(rows * (value_out && !runs ? 2 : 1));
  a.nrows = (a.rows + 2 * RR - 1) / (2 * RR);
  a.nruns = runs ? (uint32_t)((num_rows + 15) / 16) * a.Hkv : 0;
  const int64_t want = (int64_t)(a.nrows + a.nruns + ns::WARPS - 1) / ns::WARPS, cap = (int64_t)ns_sms() * 32;
  read_kv_kernel<<<(int)(want < cap ? want : cap), ns::WARPS * 32, 0, stream>>>(a);
  return cudaGetLastError();
}
