// tree_attn_tc.cuh -- attention of drafted token trees on 5th-generation
// tensor cores, straight from the paged Q8_0 cache.
//
//   S = Q K^T,  P = 2^(S - m) on the keys a row sees,  O += P V,  out = O / l
//
// The rows of one kv head of one sequence are its drafts times the GQA group
// (row = t * G + g): 16 drafts at GQA 6 are 96 rows, so one pass over the cache
// carries 512 * 96 FLOP for the 272 bytes of a key and its Q8_0 value.  That is 180 FLOP a
// byte, near the balance of HBM and tensor cores: a warp-level MMA would be
// bound by its own rate, a dequantised staging copy by traffic, and what
// this kernel has to fit beside both is dequantisation and softmax.
//
// Work: the key tiles (128 keys) of all (sequence, row group) items laid end
// to end are cut into NG equal ranges; CTA (g, h) computes range g for kv head
// h, so the heads of a group walk the same pages at the same time (a K page
// holds all heads' 136-byte rows, which share memory lines) and every CTA gets
// the same number of tiles whatever the lengths.  An item cut by a range border
// leaves partial rows that tree_combine_kernel joins.
//
// CTA:
//   warps 0-7    two softmax streams, a thread a row (row = TMEM lane).  A thread of a stream's
//                last warp also issues its tcgen05.mma: the stream has nothing else to do until its
//                next scores are there, so no warp is spent on it.
//   warps 8-     loaders, groups of four warps that take key tiles in turn: they load cache rows
//                and convert them, K to [key][d], V to [d][key] (page-transposed Q8_0) or [key][d]
//                (token rows).  A warp owns 32 keys of its tiles, so loading and converting need no
//                barrier between warps.  NQ = 1 has two groups (16 warps of 128 registers): one
//                warp a scheduler leaves it idle through its latencies and instruction fetches.
//                NQ = 2, whose softmax is twice the work per key, has one (12 warps of 168).
// One query tile (NQ = 1): the streams take alternate key tiles of the same
// rows, each with its own running maximum, sum and accumulator, so that one
// stream's softmax runs under the other's MMAs; they are joined through TMEM at
// the end.  NQ = 2 (more than 128 rows): the streams take one row tile each and share
// every converted key tile.
// Tensor memory: S0 S1 O0 O1, 128 columns each; P_i over the first half of S_i.
// bf16 V stays bf16, whose range fp16 does not have; its MMA wants P in bf16 too, which keeps 8 bits
// of a weight where fp16 keeps 11 (rows of few keys show it), so P is the sum of two bf16 terms (16 bits), multiplied
// one after the other; they take all of S_i.  Against fp16 values (and their pass over every V tile): 32 sequences of
// 1K-32K tokens 681 -> 724 us, 8 of 4K-16K with up to 60 drafts 290 -> 288 us.
// Every mbarrier wait is bounded.
//
// 32 sequences of 1K-32K tokens, 16 drafts, 48/8 heads, Q8_0 V (1.19 GB): 496 us
// for a call by itself, 2.4 TB/s, 307 TFLOP/s; 500-535 us in a row of them.  Token-row Q8_0 V 532 us, fp16
// V (1.7 GB) 628 us; 64/8 heads 499 us, 128/8 heads 853 us; a soft-cap 941 us (another pass over the scores, and its tanh);
// a window of 1024 keys 83 us.  A stream's chain of softmax, PV and
// next scores takes 6300 cycles for two tiles, the loaders 6200, so neither the
// tensor core (1000 busy cycles a tile) nor HBM (1500) is the bound.  8 sequences
// of 4K-16K, up to 60 drafts, fp16 V: 235-245 us, 390 TFLOP/s, the softmax of two row tiles.
#pragma once

#include "tcgen05.cuh"
#include "tree_common.cuh"

namespace g9 {

namespace tt {
constexpr int D = 128;
constexpr int BM = 128;
constexpr int BN = 128;
constexpr int ST = 2;                        // K and V stages
constexpr int TILE = BM * D * 2;             // 32 KB
constexpr int PITCH = 144;                   // raw Q8_0 rows: 136 bytes, up to 8 before or behind them
constexpr int RAW = 32 * PITCH;              // a warp's 32 raw rows
constexpr int loader_groups(int nq) { return nq == 1 ? 2 : 1; }
constexpr int threads(int nq) { return 256 + 128 * loader_groups(nq); }
constexpr float kRescale = 8.0f;             // log2 units

constexpr int smem_raw_off(int nq) { return (2 * ST + nq) * TILE; }
constexpr int smem_stat_off(int nq) { return smem_raw_off(nq) + 4 * loader_groups(nq) * RAW; }
constexpr int smem_scale_off(int nq) { return smem_stat_off(nq) + (nq == 1 ? 2 * 2 * BM * 4 : 0); }
constexpr int smem_bar_off(int nq) { return smem_scale_off(nq) + 4 * loader_groups(nq) * 256; }
constexpr int smem_bytes(int nq) { return smem_bar_off(nq) + 512; }
static_assert(smem_bytes(1) <= 232448 && smem_bytes(2) <= 232448, "shared memory");
}  // namespace tt

struct TreeTcParams {
  TreeArgs a;
  int Hkv, NG;
  int rc;                        // rows of a partial block (a multiple of 32)
  int bs_log2;                   // of the page size, -1: not a power of two
  uint32_t kp, vp;               // byte strides of a page and of a token in 32 bits: one multiply an address
  int kt, vt;
  int k_wide;                    // K rows may be copied as 16-byte pieces (even head counts)
  int out_vec;                   // output rows may be written 16 bytes at a time
  int* cum;                      // [num_seqs + 1] first unit of each sequence
  float* po;                     // [2 * NG][Hkv][128][rc] partial O
  float* pml;                    // [2 * NG][Hkv][2][rc] partial maximum and sum
};

// Units of a sequence: row groups x key tiles, at least one tile per row group
// (a group that sees no key still writes its zeros).
struct TreeShape { int nq, L, ctx, R, groups, j0, tiles; };

template <int NQ>
__device__ __forceinline__ TreeShape tree_shape(const TreeArgs& a, int b) {
  TreeShape s;
  s.nq = tree_nq(a.p, b);
  s.L = seq_len_kv(a.p, b);
  s.ctx = s.L - s.nq;
  s.R = s.nq * a.G;
  s.groups = (s.R + NQ * tt::BM - 1) / (NQ * tt::BM);
  // first context key any row's window can hold (a row sees at least no draft: depth -1)
  const int lo = a.p.window > 0 && s.ctx > a.p.window ? s.ctx - a.p.window : 0;
  s.j0 = lo / tt::BN;
  s.tiles = max(1, (s.L + tt::BN - 1) / tt::BN - s.j0);
  return s;
}

// First unit of CTA group g: never more groups than units, so that every
// group below the last has one.
__device__ __forceinline__ int range_start(int total, int NG, int g) {
  const int ng = min(NG, total);
  return g >= ng ? total : (int)((int64_t)g * total / ng);
}

// A run of key tiles of one (sequence, row group) item inside a CTA's range.
struct TreeSeg {
  int b, row0, rows;             // first packed row, rows of the group
  int j, n;                      // first key tile, tiles
  int part;                      // -1: the whole item; 0: continues an item; 1: starts one that goes on
  int nq, L, ctx;
};

template <int NQ>
struct TreeWalk {
  int u, end, b, base;
  __device__ __forceinline__ bool next(const TreeArgs& a, TreeSeg& s) {
    while (u < end && b < a.p.num_seqs) {
      const TreeShape x = tree_shape<NQ>(a, b);
      const int off = u - base;
      if (off >= x.groups * x.tiles) {
        base += x.groups * x.tiles;
        ++b;
        continue;
      }
      const int rg = off / x.tiles, j = off - rg * x.tiles;
      // rows spread evenly over the sequence's groups, whole warps of 32
      const int per = ((x.R + x.groups - 1) / x.groups + 31) & ~31;
      s.b = b;
      s.row0 = rg * per;
      s.rows = max(0, min(per, x.R - s.row0));
      s.j = x.j0 + j;
      s.n = min(x.tiles - j, end - u);
      s.part = j > 0 ? 0 : (s.n < x.tiles ? 1 : -1);
      s.nq = x.nq;
      s.L = x.L;
      s.ctx = x.ctx;
      u += s.n;
      return true;
    }
    return false;
  }
};

// Rows a tile of 128 keys starting at k0 must check key by key.
__device__ __forceinline__ bool tree_checked(const TreeArgs& a, const TreeSeg& s, int k0) {
  if (k0 + tt::BN > s.ctx) return true;
  // the nearest window start: a row that sees all nq drafts
  return a.p.window > 0 && k0 < s.ctx + s.nq - a.p.window;
}

// Visibility of keys base .. base + 31 for one row.
__device__ __forceinline__ uint32_t low_bits(int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u; }

__device__ __forceinline__ uint32_t tree_sees(const int32_t* row, int words, int nq, int ctx, int lo, int base) {
  uint32_t v = low_bits(ctx - base);
  const int j = base - ctx;                  // draft index of the first key
  if (j > -32 && j < nq) {
    if (j < 0) v |= tree_word(row, 0, words, nq) << -j;
    else v |= __funnelshift_r(tree_word(row, j >> 5, words, nq), tree_word(row, (j >> 5) + 1, words, nq), j & 31);
  }
  if (lo > base) v &= ~low_bits(lo - base);
  return v;
}

// K-major or MN-major 128-byte-swizzled operand.  MN-major: rows of 64
// elements along N are 128 bytes, 8-row groups along K 1024 bytes apart, the
// two 64-element halves of N `half` bytes apart.
__device__ __forceinline__ uint64_t sw128_desc_mn(uint32_t saddr, uint32_t half) {
  uint64_t d = 0;
  d |= (uint64_t)((saddr >> 4) & 0x3FFF);
  d |= (uint64_t)((half >> 4) & 0x3FFF) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}

// int8 x 4 (packed) -> two fp16x2 times scale, one rounding: scales differ by 32-element block, so they cannot be applied to a
// score that is one product over 128 elements, and a second term for what rounding leaves would double a K tile's shared
// memory, of which 16 to 27 KB are left.  2^-12 of each element; with fp16 output the whole error is 4e-4 where fp32 operands leave 2e-4.
__device__ __forceinline__ void dequant4(uint32_t x, __half2 s01, __half2 s23, uint32_t& lo, uint32_t& hi) {
  x ^= 0x80808080u;
  const uint32_t a = __byte_perm(x, 0x64646464u, 0x5140), b = __byte_perm(x, 0x64646464u, 0x5342);
  const __half2 bias = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));   // 1152
  const __half2 p = __hmul2(__hsub2(*reinterpret_cast<const __half2*>(&a), bias), s01);
  const __half2 q = __hmul2(__hsub2(*reinterpret_cast<const __half2*>(&b), bias), s23);
  lo = *reinterpret_cast<const uint32_t*>(&p);
  hi = *reinterpret_cast<const uint32_t*>(&q);
}

// exponent bits of a 16-bit value: all ones where it is not finite
constexpr uint32_t exponent16(bool bf16) { return bf16 ? 0x7f80u : 0x7c00u; }

// Clears the halves of w whose bit in `dead` is set and those that are not
// finite (E: the type's exponent bits); returns 1 if a live one was not finite.
template <uint32_t E>
__device__ __forceinline__ int clean2(uint32_t& w, bool dead0, bool dead1) {
  int hit = 0;
  if (dead0) w &= 0xffff0000u;
  else if ((w & E) == E) { w &= 0xffff0000u; hit = 1; }
  if (dead1) w &= 0x0000ffffu;
  else if ((w & (E << 16)) == (E << 16)) { w &= 0x0000ffffu; hit = 1; }
  return hit;
}

// Rare: a tile whose keys are checked held a value that is not finite.  The
// converters cleared it, so that rows which do not see the key stay clean;
// here is what a row that sees such keys has lost of elements d0 .. d0 + 31: bits
// of those that met +infinity (x) and -infinity (y), both for not a number.
static __device__ __noinline__ uint2 tree_lost(const TreeArgs& a, const TreeSeg& s, int h, const int32_t* row, int lo, int d0) {
  const G9AttnBatch& p = a.p;
  uint2 lost = make_uint2(0u, 0u);
  for (int j = s.j; j < s.j + s.n; ++j) {
    bool checked = tree_checked(a, s, j * tt::BN);         // or a page of it is not there
    for (int k = j * tt::BN; !checked && k < min(s.L, (j + 1) * tt::BN); k += 16)
      checked = page_bad(p, p.block_table[(int64_t)s.b * p.max_blocks + k / p.block_size]);
    if (!checked) continue;
    for (int k = j * tt::BN; k < min(s.L, (j + 1) * tt::BN); ++k) {
      if (!(tree_sees(row, a.words, s.nq, s.ctx, lo, k) & 1u)) continue;
      const int phys = p.block_table[(int64_t)s.b * p.max_blocks + k / p.block_size];
      if (page_bad(p, phys)) continue;
      const int off = k % p.block_size, bs = p.block_size;
      const uint8_t* base = p.v_cache + (int64_t)phys * p.v_page_stride + (int64_t)h * p.v_head_stride;
      const uint32_t E = exponent16(p.v_fmt == G9_VFMT_BF16);
      for (int i = 0; i < 32; ++i) {
        const int d = d0 + i;
        uint16_t v;
        if (p.v_fmt == G9_VFMT_F16 || p.v_fmt == G9_VFMT_BF16) {
          v = reinterpret_cast<const uint16_t*>(base + (int64_t)off * p.v_tok_stride)[d];
        } else {
          const uint8_t *sc, *q;
          if (p.v_fmt == G9_VFMT_Q8T) {
            sc = base + 2 * ((int64_t)(d / QK) * bs + off);
            q = base + 2 * (tt::D / QK) * bs + (int64_t)d * bs + off;
          } else {
            sc = base + (int64_t)off * p.v_tok_stride + d / QK * QBLOCK;
            q = sc + 2 + d % QK;
          }
          v = __half_as_ushort(__hmul(__short2half_rn((short)*reinterpret_cast<const int8_t*>(q)), *reinterpret_cast<const __half*>(sc)));
        }
        if ((v & E) != E) continue;
        const bool nan = (v & ~E & 0x7fffu) != 0;
        if (nan || !(v >> 15)) lost.x |= 1u << i;
        if (nan || v >> 15) lost.y |= 1u << i;
      }
    }
  }
  return lost;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async8(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
// loads that stay where they are written, ahead of the work that hides them
__device__ __forceinline__ uint32_t ldg4_early(const void* p) {
  uint32_t v;
  asm volatile("ld.global.L1::no_allocate.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ uint4 ldg16_early(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
  return v;
}

__device__ __forceinline__ void sts128(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
// 16 raw Q8_0 token rows (PITCH bytes apart, starting 8 * ODD bytes into them)
// -> rows row0 .. row0 + 15 of an operand tile [row][128] fp16 (two 64-element
// halves, 128-byte swizzle).  Lane (f, row) converts blocks 2f and 2f + 1: the
// 68 bytes from 68 f on, read as five aligned 16-byte words.  Eight lanes in
// a run hold eight rows of one half: their stores and loads spread over all banks.
template <int ODD>
__device__ __forceinline__ void convert_rows(const uint8_t* raw, uint8_t* tile, int row0) {
  const int lane = lane_id(), f = lane >> 4, row = row0 + (lane & 15);
  const uint4* src = reinterpret_cast<const uint4*>(raw + (lane & 15) * tt::PITCH + 64 * f);
  uint32_t w[20];
#pragma unroll
  for (int i = 0; i < 5; ++i) {
    const uint4 x = src[i];
    w[4 * i] = x.x; w[4 * i + 1] = x.y; w[4 * i + 2] = x.z; w[4 * i + 3] = x.w;
  }
  uint32_t y[17];                            // the 68 bytes: they start a word later for f = 1
#pragma unroll
  for (int i = 0; i < 17; ++i) y[i] = f ? w[i + 2 * ODD + 1] : w[i + 2 * ODD];
  const uint32_t s0 = (y[0] & 0xffffu) * 0x10001u, s1 = (y[8] >> 16) * 0x10001u;
  uint8_t* dst = tile + f * (tt::TILE / 2) + row * 128;
  const int sw = row & 7;
#pragma unroll
  for (int c = 0; c < 8; ++c) {              // 8 elements
    uint32_t o[4];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int i = 2 * (c & 3) + e;
      // the first block's values start in mid-word, the second's on a word
      const uint32_t q = c < 4 ? __byte_perm(y[i], y[i + 1], 0x5432) : y[9 + i];
      const __half2 s = *reinterpret_cast<const __half2*>(c < 4 ? &s0 : &s1);
      dequant4(q, s, s, o[2 * e], o[2 * e + 1]);
    }
    *reinterpret_cast<uint4*>(dst + ((c ^ sw) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
  }
}

// ===========================================================================
template <int NQ, int VF>
__global__ void __launch_bounds__(tt::threads(NQ), 1) tree_tc_kernel(const __grid_constant__ TreeTcParams pp) {
  using namespace tt;
  constexpr int NT = threads(NQ), GROUPS = loader_groups(NQ);
  constexpr bool BF = VF == G9_VFMT_BF16, DIRECT = VF == G9_VFMT_F16 || BF;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t sbase = smem_u32(smem);
  const uint32_t sK = sbase, sV = sK + ST * TILE, sQ = sV + ST * TILE;
  float* stat = reinterpret_cast<float*>(smem + smem_stat_off(NQ));          // [stream][m, l][row]
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + smem_bar_off(NQ));
  uint64_t *kfull = bars, *kempty = bars + 2, *vfull = bars + 4, *vempty = bars + 6, *qfull = bars + 8, *bs_ = bars + 10,
           *bp = bars + 12, *bo = bars + 14, *bx = bars + 16, *by = bars + 17, *bpv = bars + 18, *vraw = bars + 20;
  int* misc = reinterpret_cast<int*>(bars + 28);     // 0: tensor memory, 1: abort, 2: a value was not finite, 4: b, 5: base, 8..23: scan
  uint32_t* tilebad = reinterpret_cast<uint32_t*>(misc + 24);                // [8], a byte per 32 keys

  const TreeArgs& a = pp.a;
  const G9AttnBatch& p = a.p;
  const int warp = warp_id(), lane = lane_id(), tid = threadIdx.x;
  const int g = blockIdx.x / pp.Hkv, h = blockIdx.x - g * pp.Hkv;

  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      // a tile is free when every stream that reads it is done: one (NQ = 1) or both
      mbar_init(&kfull[i], 4); mbar_init(&kempty[i], NQ);
      mbar_init(&vfull[i], 4); mbar_init(&vempty[i], NQ);
      mbar_init(&bs_[i], 1); mbar_init(&bp[i], 128); mbar_init(&bo[i], 1); mbar_init(&bpv[i], 1);
      mbar_init(&qfull[i], NQ == 1 ? 256 : 128);
    }
    for (int i = 0; i < 4 * GROUPS; ++i) mbar_init(&vraw[i], 32);
    mbar_init(bx, 256); mbar_init(by, 256);
    misc[1] = misc[2] = 0;
    fence_barrier_init();
  }
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&misc[0])));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  // Launched while the kernel before it in the stream finishes: nothing above reads or writes global memory.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");
  // ---- this CTA's range of units ----------------------------------------------
  // Prefix sums of the sequences' units, NT sequences at a time; the sequence
  // that holds the range's first unit is found once the total is known, which
  // for up to NT sequences is the same pass.
  int total = 0;
  const bool one_chunk = p.num_seqs <= NT;
  for (int pass = one_chunk ? 1 : 0; pass < 2; ++pass) {
    int base = 0;
    for (int b0 = 0; b0 < p.num_seqs; b0 += NT) {
      const int b = b0 + tid;
      int n = 0;
      if (b < p.num_seqs) {
        const TreeShape s = tree_shape<NQ>(a, b);
        n = s.groups * s.tiles;
      }
      int inc = n;
#pragma unroll
      for (int x = 1; x < 32; x <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, inc, x);
        if (lane >= x) inc += o;
      }
      if (!one_chunk) __syncthreads();
      if (lane == 31) misc[8 + warp] = inc;
      __syncthreads();
      int before = 0, all = 0;
#pragma unroll
      for (int w = 0; w < NT / 32; ++w) {
        const int x = misc[8 + w];
        if (w < warp) before += x;
        all += x;
      }
      if (one_chunk) total = all;
      const int first = base + before + inc - n;
      if (pass == 1 && b < p.num_seqs) {
        const int u0 = range_start(total, pp.NG, g);
        if (blockIdx.x == 0) pp.cum[b] = first;
        if (u0 >= first && u0 < first + n) {
          misc[4] = b;
          misc[5] = first;
        }
      }
      base += all;
    }
    total = base;
  }
  if (blockIdx.x == 0 && tid == 0) pp.cum[p.num_seqs] = total;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = (uint32_t)misc[0];
  TreeWalk<NQ> walk{};
  walk.u = range_start(total, pp.NG, g);
  walk.end = range_start(total, pp.NG, g + 1);
  const int N = walk.end - walk.u;           // key tiles of this CTA
  walk.b = N > 0 ? misc[4] : 0;
  walk.base = N > 0 ? misc[5] : 0;
  volatile int* abort_flag = &misc[1];

  if (warp >= 8) {
    // ======================= cache rows: load and convert ========================
    const int lw = warp - 8, w = lw & 3;     // this warp's 32 keys of a tile
    const int bsz = p.block_size;
    uint8_t* raw = smem + smem_raw_off(NQ) + lw * RAW;
    uint32_t* vscale = reinterpret_cast<uint32_t*>(smem + smem_scale_off(NQ) + lw * 256);
    const int odd = pp.k_wide && (h & 1);    // the row starts 8 bytes into its first 16-byte piece
    const uint8_t* kbase = p.k_cache + (int64_t)h * p.k_head_stride - 8 * odd;
    const uint8_t* vbase = p.v_cache + (int64_t)h * p.v_head_stride;
    int koff[9];                             // this lane's pieces of 32 rows: nine of 16 bytes a row
#pragma unroll
    for (int i = 0; i < 9; ++i) {
      const int y = i * 32 + lane, r = y / 9;
      koff[i] = (r & 15) * pp.kt + (y - r * 9) * 16;
    }
    // of a page-transposed record: this lane's scale word and its dims' values
    const int vs_off = 2 * (lane >> 3) * bsz + 4 * (lane & 7), vq_off = 2 * (D / QK) * bsz + lane * bsz;
    TreeSeg s;
    s.n = 0;
    int pos = lw >> 2;                       // the next tile's place in the segment
    const int32_t* bt = p.block_table;       // and the segment's row of the table
    // This warp's share of a tile: pages and in-page offsets of its two 16-key groups (page -1: none), keys inside the
    // sequence | checked << 8.
    struct Share { int ph0, ph1, of0, of1, info; };
    Share cur{-1, -1, 0, 0, 0}, nxt = cur;
    bool ok = true;
    // Asks for the next tile's pages; nothing here waits for them.  No branch around a load that is meant to stay in
    // flight: joining its result with another value waits for it.
    auto lookup = [&]() {
      while (pos >= s.n) {
        pos -= s.n;
        if (!walk.next(a, s)) return;
        bt = p.block_table + (int64_t)s.b * p.max_blocks;
      }
      const int k = (s.j + pos) * BN + 32 * w;
      int pg0, pg1;
      if (pp.bs_log2 >= 0) {
        pg0 = k >> pp.bs_log2;
        pg1 = (k + 16) >> pp.bs_log2;
      } else {
        pg0 = k / bsz;
        pg1 = (k + 16) / bsz;
      }
      nxt.ph0 = bt[min(pg0, p.max_blocks - 1)];
      nxt.ph1 = bt[min(pg1, p.max_blocks - 1)];
      nxt.of0 = k - pg0 * bsz;
      nxt.of1 = k + 16 - pg1 * bsz;
      nxt.info = max(0, min(32, s.L - k)) | (tree_checked(a, s, k - 32 * w) ? 256 : 0);
      pos += GROUPS;
    };
    // what the last lookup brought; t: its tile
    auto settle = [&](int t) {
      cur = nxt;
      const int valid = cur.info & 0xff;
      uint32_t bad = 0;                      // keys on a page that is not there
      if (valid > 0 && page_bad(p, cur.ph0)) bad = 1;
      if (valid > 16 && page_bad(p, cur.ph1)) bad |= 2;
      if (valid <= 16 || bad) {              // not every tile
        if (valid == 0 || (bad & 1)) { cur.ph0 = -1; cur.of0 = 0; }
        if (valid <= 16 || (bad & 2)) { cur.ph1 = -1; cur.of1 = 0; }
        if (bad) {
          cur.info |= 256;
          if (lane == 0) raise_error(ERR_BAD_PAGE);
        }
      }
      if (lane == 0) reinterpret_cast<uint8_t*>(&tilebad[t & 7])[w] = (uint8_t)bad;
    };
    // 32 token rows of 136 bytes into the raw slot.  A page that is not there: page 0's bytes, whose scores are masked
    // and whose values are cleared.
    auto load_rows = [&](const uint8_t* base, uint32_t page_stride, int tok_stride, bool wide) {
      const uint8_t* s0 = base + (uint64_t)(uint32_t)max(cur.ph0, 0) * page_stride + cur.of0 * tok_stride;
      const uint8_t* s1 = base + (uint64_t)(uint32_t)max(cur.ph1, 0) * page_stride + cur.of1 * tok_stride;
      const uint32_t dst = smem_u32(raw) + lane * 16;
      if (wide) {
        // pieces 0..143 are the first group's rows
#pragma unroll
        for (int i = 0; i < 9; ++i) cp_async16(dst + i * 512, (i < 4 || (i == 4 && lane < 16) ? s0 : s1) + koff[i]);
      } else {
#pragma unroll 2
        for (int y = lane; y < 544; y += 32) {
          const int r = y / 17, c = y - r * 17;
          cp_async8(smem_u32(raw) + r * PITCH + c * 8, (r < 16 ? s0 : s1) + (r & 15) * tok_stride + c * 8);
        }
      }
    };
    // K rows of the settled tile
    auto load_k = [&]() {
      load_rows(kbase, pp.kp, pp.kt, pp.k_wide);
      cp_async_commit();
    };
    auto wait_empty = [&](uint64_t* bar, int t) {
      if (t >= ST && !mbar_wait(&bar[t & 1], ((t >> 1) - 1) & 1)) ok = false;
      ok = __all_sync(0xffffffffu, ok);
      return ok;
    };
    auto convert = [&](uint8_t* tile, int shift) {
#pragma unroll 1
      for (int grp = 0; grp < 2; ++grp) {
        if (shift) convert_rows<1>(raw + grp * 16 * PITCH, tile, 32 * w + 16 * grp);
        else convert_rows<0>(raw + grp * 16 * PITCH, tile, 32 * w + 16 * grp);
      }
      fence_proxy_async();                   // the tensor core reads what this thread wrote
      __syncwarp();
    };
    if ((lw >> 2) < N) {
      lookup();
      settle(lw >> 2);
      load_k();
    }
#pragma unroll 1
    for (int t = lw >> 2; ok && t < N; t += GROUPS) {
      // `cur` is tile t; its K rows are on their way
      const Share me = cur;
      const int valid = me.info & 0xff;      // keys of this warp inside the sequence
      const bool checked = (me.info & 256) != 0;
      const bool more = t + GROUPS < N;
      uint8_t* vtile = smem + (ST + (t & 1)) * TILE;
      uint4 q[2][4];
      uint32_t sc[2];
      if constexpr (VF == G9_VFMT_Q8T) {
        // Page-transposed records go through registers: a lane's 16 bytes are 16 keys of one dim.
        // Scale word `lane`: keys 2 * (lane % 8), + 1 of block lane / 8.
#pragma unroll
        for (int grp = 0; grp < 2; ++grp) {
          const int ph = grp ? me.ph1 : me.ph0, at = grp ? me.of1 : me.of0;
          const uint8_t* rec = vbase + (uint64_t)(uint32_t)max(ph, 0) * pp.vp;
          sc[grp] = ldg4_early(rec + vs_off + 2 * at);
          const uint8_t* val = rec + vq_off + at;
#pragma unroll
          for (int i = 0; i < 4; ++i) q[grp][i] = ldg16_early(val + i * 32 * bsz);
        }
      } else if constexpr (DIRECT) {
        // 16-bit rows go straight into the operand tile; rows of a page that is not there are zeroed
        if (!wait_empty(vempty, t)) break;
        const int c = lane & 15;
#pragma unroll
        for (int grp = 0; grp < 2; ++grp) {
          const int ph = grp ? me.ph1 : me.ph0, at = grp ? me.of1 : me.of0;
          const uint8_t* src = vbase + (uint64_t)(uint32_t)ph * pp.vp + at * pp.vt + 16 * c;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int r = 2 * i + (lane >> 4), key = 32 * w + 16 * grp + r;
            uint8_t* to = vtile + (c >> 3) * (TILE / 2) + key * 128 + (((c & 7) ^ (key & 7)) << 4);
            if (ph >= 0) cp_async16(smem_u32(to), src + r * pp.vt);
            else *reinterpret_cast<uint4*>(to) = make_uint4(0, 0, 0, 0);
          }
        }
        cp_async_arrive_noinc(&vraw[lw]);
        cp_async_commit();
      }
      if (more) lookup();
      // ---- K ------------------------------------------------------------------------
      cp_async_wait<DIRECT ? 1 : 0>();
      __syncwarp();
      if (!wait_empty(kempty, t)) break;
      convert(smem + (t & 1) * TILE, odd);
      if (lane == 0) mbar_arrive(&kfull[t & 1]);
      if (VF == G9_VFMT_Q8) {                // token-row V takes the slot in turn
        load_rows(vbase, pp.vp, pp.vt, false);
        cp_async_commit();
      } else if (more) {
        settle(t + GROUPS);
        load_k();
      }
      // ---- V ------------------------------------------------------------------------
      int hit = 0;
      if constexpr (VF == G9_VFMT_Q8T) {
        if (!wait_empty(vempty, t)) break;
        vscale[lane] = me.ph0 < 0 ? 0u : sc[0];
        vscale[32 + lane] = me.ph1 < 0 ? 0u : sc[1];
        __syncwarp();
        uint8_t* to = vtile + (w >> 1) * (TILE / 2);       // this warp's half tile
        const int c0 = (w & 1) * 4;                        // and its first 8-key chunk there
#pragma unroll
        for (int grp = 0; grp < 2; ++grp) {
          const int c = c0 + 2 * grp;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int d = lane + 32 * i;
            const uint4 s0 = *reinterpret_cast<const uint4*>(&vscale[32 * grp + 8 * i]);
            const uint4 s4 = *reinterpret_cast<const uint4*>(&vscale[32 * grp + 8 * i + 4]);
            const uint32_t qs[4] = {q[grp][i].x, q[grp][i].y, q[grp][i].z, q[grp][i].w};
            const uint32_t s8[8] = {s0.x, s0.y, s0.z, s0.w, s4.x, s4.y, s4.z, s4.w};
            uint32_t o[8];
#pragma unroll
            for (int e = 0; e < 4; ++e)
              dequant4(qs[e], *reinterpret_cast<const __half2*>(&s8[2 * e]), *reinterpret_cast<const __half2*>(&s8[2 * e + 1]),
                       o[2 * e], o[2 * e + 1]);
            *reinterpret_cast<uint4*>(to + d * 128 + ((c ^ (d & 7)) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
            *reinterpret_cast<uint4*>(to + d * 128 + (((c + 1) ^ (d & 7)) << 4)) = make_uint4(o[4], o[5], o[6], o[7]);
          }
        }
        if (checked) {
          // again over what this lane wrote: keys past the sequence, values that are not finite
#pragma unroll 1
          for (int i = 0; i < 16; ++i) {
            const int d = lane + 32 * (i & 3), nv = valid - 8 * (i >> 2);
            uint4* x = reinterpret_cast<uint4*>(to + d * 128 + (((c0 + (i >> 2)) ^ (d & 7)) << 4));
            const uint4 x4 = *x;
            uint32_t o[4] = {x4.x, x4.y, x4.z, x4.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) hit |= clean2<exponent16(false)>(o[e], 2 * e >= nv, 2 * e + 1 >= nv);
            *x = make_uint4(o[0], o[1], o[2], o[3]);
          }
        }
      } else {
        if constexpr (DIRECT) {
          if (!mbar_wait(&vraw[lw], (t / GROUPS) & 1)) ok = false;
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
        } else {
          cp_async_wait<0>();
          __syncwarp();
          if (!wait_empty(vempty, t)) break;
          convert(vtile, 0);
          if (more) {
            settle(t + GROUPS);
            load_k();
          }
        }
        if (checked) {
          const int key = 32 * w + lane;
          const bool dead = lane >= valid;
#pragma unroll 2
          for (int c = 0; c < 16; ++c) {
            uint4* x = reinterpret_cast<uint4*>(vtile + (c >> 3) * (TILE / 2) + key * 128 + (((c & 7) ^ (key & 7)) << 4));
            const uint4 x4 = *x;
            uint32_t o[4] = {x4.x, x4.y, x4.z, x4.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) hit |= clean2<exponent16(BF)>(o[e], dead, dead);
            *x = make_uint4(o[0], o[1], o[2], o[3]);
          }
        }
      }
      if (hit) misc[2] = 1;
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(&vfull[t & 1]);
    }
    cp_async_wait<0>();
    ok = __all_sync(0xffffffffu, ok);
    if (!ok) *abort_flag = 1;
  } else {
    // ======================= softmax streams =====================================
    const int wi = warp >> 2;          // stream
    const int r = (warp & 3) * 32 + lane;    // row of the tile = TMEM lane
    const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + wi * 128 + lane_off, tO = tmem + 256 + wi * 128 + lane_off;
    const bool general = p.softcap > 0.f || !(p.scale > 0.f);
    const bool leader = (tid & 127) == 96;   // issues the stream's MMAs; its warp has no rows of its own below 97 of them
    constexpr uint32_t kS = (1u << 4) | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(BM >> 4) << 24);
    // V by token rows: N-major; bf16 V: both operands bf16
    constexpr uint32_t kPV = kS | (VF == G9_VFMT_Q8T ? 0u : 1u << 16) | (BF ? 1u << 7 | 1u << 10 : 0u);
    const uint32_t qs = sQ + (NQ == 2 ? wi * TILE : 0);
    // Descriptors are advanced from one base each: the start address counts 16-byte units in the low bits.
    auto issue_s = [&](int n) {              // S = Q K(n)^T
      const uint64_t qd = sw128_desc(qs), kd = sw128_desc(sK + (n & 1) * TILE);
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        const uint32_t off = ((kk >> 2) * (TILE / 2) + (kk & 3) * 32) >> 4;
        tc_mma_ss(tmem + wi * 128, qd + off, kd + off, kS, kk > 0);
      }
      tc_commit(&bs_[wi]);
      tc_commit(&kempty[n & 1]);
    };
    auto issue_pv = [&](int n, bool first) { // O += P V(n)
      const uint32_t vs = sV + (n & 1) * TILE;
      const uint64_t vd = VF == G9_VFMT_Q8T ? sw128_desc(vs) : sw128_desc_mn(vs, TILE / 2);
#pragma unroll
      for (int kk = 0; kk < BN / 16; ++kk) {
        const uint32_t off = (VF == G9_VFMT_Q8T ? (kk >> 2) * (TILE / 2) + (kk & 3) * 32 : kk * 2048) >> 4;
        const uint32_t pa = tmem + wi * 128 + (BF ? (kk >> 2) * 64 + (kk & 3) * 8 : kk * 8);
        tc_mma_ts(tmem + 256 + wi * 128, pa, vd + off, kPV, (!first || kk > 0) ? 1u : 0u);
        if (BF) tc_mma_ts(tmem + 256 + wi * 128, pa + 32, vd + off, kPV, 1u);
      }
      tc_commit(&bpv[wi]);
      tc_commit(&vempty[n & 1]);
    };
    constexpr int STEP = NQ == 1 ? 2 : 1;    // tiles between a stream's own
    int n0 = 0, ns = 0, cs = 0, cq = 0;      // tiles, segments, steps and Q tiles of this stream so far
    bool alive = true;
    TreeSeg s;
    while (alive && walk.next(a, s)) {
      const int rl = (NQ == 2 ? wi * BM : 0) + r;        // row of the group
      const bool warp_live = (NQ == 2 ? wi * BM : 0) + (warp & 3) * 32 < s.rows;
      const bool row_live = rl < s.rows;
      const int rg = s.row0 + (row_live ? rl : 0), t = rg / a.G, hq = h * a.G + rg - t * a.G;
      const int32_t* bits = tree_row(a, s.b, t);
      const int lo = row_live ? tree_window_lo(a, bits, s.nq, s.ctx) : 0;
      float m = -INFINITY, l = 0.f;          // log2 units
      const bool stream_on = NQ == 1 || wi == 0 || s.rows > BM;
      const int j0 = NQ == 1 ? wi : 0;
      // ---- Q rows of this stream's tile (NQ = 1: half the columns each) -------------
      // The previous segment's MMAs are done: every thread has waited for them.
      if (stream_on || NQ == 1) {
        constexpr int COLS = NQ == 1 ? 8 : 16;           // 16-byte pieces of a row
        const int c0 = NQ == 1 ? 8 * wi : 0;
#pragma unroll 4
        for (int it = tid & 127; it < BM * COLS; it += 128) {
          const int qr = it / COLS, c = c0 + it % COLS;
          const int gr = (NQ == 2 ? wi * BM : 0) + qr;
          uint32_t v[4] = {0, 0, 0, 0};
          if (gr < s.rows) {
            const int x = s.row0 + gr, xt = x / a.G;
            const int64_t at = q_offset(p, s.b, xt, h * a.G + x - xt * a.G) + 8 * c;
#pragma unroll
            for (int e = 0; e < 4; ++e)
              v[e] = pack_half2(load_one(p.q, at + 2 * e, p.q_dtype), load_one(p.q, at + 2 * e + 1, p.q_dtype));
          }
          sts128(qs + (c >> 3) * (TILE / 2) + qr * 128 + (((c & 7) ^ (qr & 7)) << 4), v[0], v[1], v[2], v[3]);
        }
        fence_proxy_async();
        mbar_arrive(&qfull[NQ == 1 ? 0 : wi]);
      }
      if (leader) {
        if (stream_on && j0 < s.n) {
          alive = mbar_wait(&qfull[NQ == 1 ? 0 : wi], (NQ == 1 ? ns : cq) & 1) && mbar_wait(&kfull[(n0 + j0) & 1], ((n0 + j0) >> 1) & 1);
          if (alive) {
            tc_fence_after();
            issue_s(n0 + j0);
          }
        } else {
          mbar_arrive(&bo[wi]);              // nothing to multiply
          if (NQ == 2)                       // pass this stream's share of every tile on
            for (int j = 0; alive && j < s.n; ++j) {
              alive = mbar_wait(&kfull[(n0 + j) & 1], ((n0 + j) >> 1) & 1);
              mbar_arrive(&kempty[(n0 + j) & 1]);
              alive = alive && mbar_wait(&vfull[(n0 + j) & 1], ((n0 + j) >> 1) & 1);
              mbar_arrive(&vempty[(n0 + j) & 1]);
            }
        }
      }
      if (NQ == 2 && stream_on) ++cq;
      // after a step's weights are in place: PV of this tile, then the scores of the stream's next one
      auto multiply = [&](int j) {
        if (!leader) return;
        const int n = n0 + j;
        alive = mbar_wait(&bp[wi], (cs - 1) & 1) && mbar_wait(&vfull[n & 1], (n >> 1) & 1);
        if (!alive) return;
        tc_fence_after();
        issue_pv(n, j == j0);
        if (j + STEP < s.n) {
          // the next scores overwrite the weights that this PV reads (only MMAs of one accumulator are sure to run in order)
          alive = mbar_wait(&kfull[(n + STEP) & 1], ((n + STEP) >> 1) & 1) && mbar_wait(&bpv[wi], (cs - 1) & 1);
          if (!alive) return;
          tc_fence_after();
          issue_s(n + STEP);
        } else {
          tc_commit(&bo[wi]);
        }
      };
      for (int j = j0; stream_on && j < s.n; j += STEP) {
        if (alive && !mbar_wait(&bs_[wi], cs & 1)) alive = false;
        alive = __all_sync(0xffffffffu, alive);
        if (!alive) break;
        ++cs;
        tc_fence_after();
        if (warp_live) {
        const int k0 = (s.j + j) * BN;
        const uint32_t bad = tilebad[(n0 + j) & 7];
        const bool checked = bad || tree_checked(a, s, k0);
        // Scores that a cap or the mask changes are written back first, in small loops: code that most tiles skip must
        // not stand between the instructions that every tile runs (the kernel was bound by instruction fetch).
        if (general) {
#pragma unroll 1
          for (int c = 0; c < 16; ++c) {
            uint32_t x[8];
            tmem_ld8(tS + c * 8, x);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float y = __uint_as_float(x[e]);
              x[e] = __float_as_uint(p.softcap > 0.f ? softcap_log2(y, a.cap_in, a.cap_out) : y * a.scale_log2);
            }
            __syncwarp();                    // tanhf branches by lane; tensor-memory accesses are the whole warp's
            tmem_st8(tS + c * 8, x);
          }
          tmem_wait_st();
        }
        if (checked) {
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            uint32_t x[32];
            tmem_ld32(tS + c * 32, x);
            tmem_wait_ld();
            uint32_t v = row_live ? tree_sees(bits, a.words, s.nq, s.ctx, lo, k0 + 32 * c) : 0u;
            const uint32_t bc = bad >> (8 * c);
            if (bc & 1) v &= 0xffff0000u;
            if (bc & 2) v &= 0x0000ffffu;
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (!(v >> e & 1u)) x[e] = 0xff800000u;
            __syncwarp();                    // the bit rows were read by lane
            tmem_st32(tS + c * 32, x);
          }
          tmem_wait_st();
        }
        // 64 scores at a time, each half against the running maximum as it is then
#pragma unroll 1
        for (int hf = 0; hf < 2; ++hf) {
          uint32_t x[2][32];
          tmem_ld32(tS + hf * 64, x[0]);
          tmem_ld32(tS + hf * 64 + 32, x[1]);
          tmem_wait_ld();
          float mx = -INFINITY;
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float m0 = __uint_as_float(x[c][0]), m1 = __uint_as_float(x[c][1]);
#pragma unroll
            for (int e = 2; e < 30; e += 4) {
              m0 = fmax3(m0, __uint_as_float(x[c][e]), __uint_as_float(x[c][e + 1]));
              m1 = fmax3(m1, __uint_as_float(x[c][e + 2]), __uint_as_float(x[c][e + 3]));
            }
            mx = fmax3(mx, fmax3(m0, m1, __uint_as_float(x[c][30])), __uint_as_float(x[c][31]));
          }
          if (!general) mx *= a.scale_log2;  // scale > 0: the maximum commutes with it
          float alpha = 1.f;
          bool rescale = false;
          if (mx != -INFINITY && (m == -INFINITY || mx > m + kRescale)) {
            // A whole number: weights already written are scaled by a power of two, which rounds none of them a second
            // time, at the price of weights up to 2 times smaller (fp16 keeps 2^-24 of the largest).
            mx = ceilf(mx);
            if (m != -INFINITY) {
              alpha = fast_exp2(m - mx);
              l *= alpha;
              rescale = true;
            }
            m = mx;
          }
          if (__any_sync(0xffffffffu, rescale)) {
            // earlier tiles' PV are in O (the scores were issued after them); this tile's first half is still P
            if (j != j0) {
#pragma unroll 1
              for (int c = 0; c < 8; ++c) {
                uint32_t o[16];
                tmem_ld16(tO + c * 16, o);
                tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
                tmem_st16(tO + c * 16, o);
              }
            }
            if (hf) {
#pragma unroll 1
              for (int c = 0; c < (BF ? 8 : 4); ++c) {
                uint32_t o[8];
                tmem_wait_st();
                tmem_ld8(tS + c * 8, o);
                tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                  if constexpr (BF) {        // either term
                    o[e] = pack_bf162(__uint_as_float(o[e] << 16) * alpha, __uint_as_float(o[e] & 0xffff0000u) * alpha);
                  } else {
                    const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&o[e]));
                    o[e] = pack_half2(y.x * alpha, y.y * alpha);
                  }
                }
                tmem_st8(tS + c * 8, o);
              }
            }
          }
          const float mu = m == -INFINITY ? 0.f : m;
          const float sc = general ? 1.f : a.scale_log2;
          const uint64_t sc2 = f2pack(sc, sc), nmu2 = f2pack(-mu, -mu);
          uint64_t ls2[2] = {0ull, 0ull};
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t pk[8], lo[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const uint64_t y2 = f2fma(f2pack(__uint_as_float(x[c >> 1][(c & 1) * 16 + 2 * e]),
                                               __uint_as_float(x[c >> 1][(c & 1) * 16 + 2 * e + 1])), sc2, nmu2);
              float y0, y1;
              f2unpack(y2, y0, y1);
              y0 = fast_exp2(y0);
              y1 = fast_exp2(y1);
              ls2[e & 1] = f2add(ls2[e & 1], f2pack(y0, y1));
              if constexpr (BF) {
                // Upper halves, and what is left of y * (1 + 2^-23): never 0 where y is not, so that an infinite value
                // meets two weights of one sign and stays infinite
                const uint32_t b0 = __float_as_uint(y0), b1 = __float_as_uint(y1);
                pk[e] = __byte_perm(b0, b1, 0x7632);
                constexpr uint32_t H = 0xffff0000u, S = 0x80000000u;
                float l0, l1;
                f2unpack(f2fma(f2pack(y0, y1), f2pack(1.f + 0x1p-23f, 1.f + 0x1p-23f),
                               f2pack(__uint_as_float((b0 & H) | S), __uint_as_float((b1 & H) | S))), l0, l1);
                lo[e] = pack_bf162(l0, l1);
              } else {
                pk[e] = pack_half2(y0, y1);
              }
            }
            // 64 weights take 32 columns, two bf16 terms 64: columns whose scores this row has read
            tmem_st8(tS + hf * (BF ? 64 : 32) + c * 8, pk);
            if constexpr (BF) tmem_st8(tS + hf * 64 + 32 + c * 8, lo);
          }
          float a0, a1, b0, b1;
          f2unpack(ls2[0], a0, a1);
          f2unpack(ls2[1], b0, b1);
          l += (a0 + a1) + (b0 + b1);
        }
        tmem_wait_st();
        }                                    // rows past the group keep whatever S holds: O's rows are apart
        tc_fence_before();
        mbar_arrive(&bp[wi]);
        multiply(j);
      }
      // ---- the segment's rows ------------------------------------------------------
      if (l != l && m == -INFINITY) m = 0.f; // only NaN scores: the row is one too
      float w0 = 1.f, w1 = 0.f;              // weights of this stream's and the other stream's O
      bool use0 = m != -INFINITY, use1 = false;
      if constexpr (NQ == 1) {
        stat[(wi * 2) * BM + r] = m;
        stat[(wi * 2 + 1) * BM + r] = l;
        mbar_arrive(bx);
        if (alive && !mbar_wait(bx, ns & 1)) alive = false;
      }
      if (!alive || !mbar_wait(&bo[0], ns & 1) || !mbar_wait(&bo[1], ns & 1)) alive = false;
      alive = __all_sync(0xffffffffu, alive);
      if (!alive) break;
      tc_fence_after();
      if constexpr (NQ == 1) {
        const float m1 = stat[((wi ^ 1) * 2) * BM + r], l1 = stat[((wi ^ 1) * 2 + 1) * BM + r];
        const float top = fmaxf(m, m1);
        use1 = m1 != -INFINITY;
        w0 = use0 ? fast_exp2(m - top) : 0.f;
        w1 = use1 ? fast_exp2(m1 - top) : 0.f;
        l = (use0 ? l * w0 : 0.f) + (use1 ? l1 * w1 : 0.f);
        m = top;
      }
      if (warp_live && stream_on) {
        const bool whole = s.part < 0;
        const bool any = l > 0.f || l != l;
        float fin = 1.f;
        if (whole) {
          if (p.sinks && any) l += fast_exp2(sink_log2(p, hq) - m);
          fin = (any ? 1.f / l : 0.f) * out_quant_factor(p);
        }
        // the streams of one row tile (NQ = 1) write half the columns each
        const int c0 = NQ == 1 ? 2 * wi : 0, c1 = NQ == 1 ? c0 + 2 : 4;
        const uint32_t tOther = tmem + 256 + (wi ^ 1) * 128 + lane_off;
        const int64_t slot = ((int64_t)(2 * g + (s.part > 0 ? 1 : 0)) * pp.Hkv + h);
        const int64_t ob = row_live ? o_offset(p, s.b, t, hq) : 0;
#pragma unroll 1
        for (int c = c0; c < c1; ++c) {
          uint2 lost = make_uint2(0u, 0u);
          if (row_live && misc[2]) lost = tree_lost(a, s, h, bits, lo, c * 32);
          __syncwarp();                      // rows past the group skip the stores below
          uint32_t o[32];
          tmem_ld32(tO + c * 32, o);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = use0 ? __float_as_uint(__uint_as_float(o[e]) * w0) : 0u;
          if (NQ == 1) {
            uint32_t q[32];
            tmem_ld32(tOther + c * 32, q);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (use1) o[e] = __float_as_uint(__uint_as_float(o[e]) + __uint_as_float(q[e]) * w1);
          }
          if (!row_live) continue;
          if (lost.x | lost.y) {
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              float x = __uint_as_float(o[e]);
              if (lost.x >> e & 1u) x += INFINITY;
              if (lost.y >> e & 1u) x -= INFINITY;
              o[e] = __float_as_uint(x);
            }
          }
          if (!whole) {
            float* dst = pp.po + (slot * D + c * 32) * pp.rc + rl;
#pragma unroll
            for (int e = 0; e < 32; ++e) dst[(int64_t)e * pp.rc] = __uint_as_float(o[e]);
            continue;
          }
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = any ? __float_as_uint(__uint_as_float(o[e]) * fin) : 0u;
          if (pp.out_vec && p.out_dtype != DT_FP8) {
            uint8_t* dst = reinterpret_cast<uint8_t*>(p.out) + (ob + c * 32) * (p.out_dtype == DT_F32 ? 4 : 2);
            if (p.out_dtype == DT_F32) {
#pragma unroll
              for (int e = 0; e < 8; ++e)
                reinterpret_cast<uint4*>(dst)[e] = make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
            } else {
              uint32_t y[16];
#pragma unroll
              for (int e = 0; e < 16; ++e)
                y[e] = p.out_dtype == DT_F16 ? pack_half2(__uint_as_float(o[2 * e]), __uint_as_float(o[2 * e + 1]))
                                             : pack_bf162(__uint_as_float(o[2 * e]), __uint_as_float(o[2 * e + 1]));
#pragma unroll
              for (int e = 0; e < 4; ++e)
                reinterpret_cast<uint4*>(dst)[e] = make_uint4(y[4 * e], y[4 * e + 1], y[4 * e + 2], y[4 * e + 3]);
            }
          } else {
#pragma unroll
            for (int e = 0; e < 32; e += 2)
              store_out2(p.out, p.out_dtype, ob + c * 32 + e, __uint_as_float(o[e]), __uint_as_float(o[e + 1]));
          }
        }
        if (!whole && row_live && (NQ == 2 || wi == 0)) {
          pp.pml[slot * 2 * pp.rc + rl] = m;
          pp.pml[(slot * 2 + 1) * pp.rc + rl] = l;
        }
      }
      if constexpr (NQ == 1) {
        // the other stream has read this one's O before the next segment writes it
        tc_fence_before();
        mbar_arrive(by);
        if (!mbar_wait(by, ns & 1)) alive = false;
        alive = __all_sync(0xffffffffu, alive);
        tc_fence_after();
      }
      n0 += s.n;
      ++ns;
    }
    if (!alive) *abort_flag = 1;
  }
  tc_fence_before();
  __syncthreads();
  if (tid == 0 && misc[1]) raise_error(ERR_WAIT_TIMEOUT);
  if (warp == 8) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
  }
}

// ---------------------------------------------------------------------------
// Joins the partial rows of items that a range border cut: CTA (32 rows of an
// item, kv head).  out = sum_s 2^(m_s - M) O_s / sum_s 2^(m_s - M) l_s.
// ---------------------------------------------------------------------------
template <int NQ>
__global__ void __launch_bounds__(256) tree_combine_kernel(const __grid_constant__ TreeTcParams pp, int row_blocks, int max_groups) {
  using namespace tt;
  __shared__ float rows[32][D + 1];
  const TreeArgs& a = pp.a;
  const G9AttnBatch& p = a.p;
  const int rb = blockIdx.x % row_blocks;
  const int rg = (blockIdx.x / row_blocks) % max_groups, b = blockIdx.x / row_blocks / max_groups;
  const int h = blockIdx.y;
  asm volatile("griddepcontrol.wait;" ::: "memory");       // queued behind the attention kernel's start, runs after its end
  const TreeShape x = tree_shape<NQ>(a, b);
  if (rg >= x.groups) return;
  const int per = ((x.R + x.groups - 1) / x.groups + 31) & ~31;
  const int nrows = max(0, min(per, x.R - rg * per));
  if (rb * 32 >= nrows) return;
  const int64_t T = pp.cum[p.num_seqs];
  const int64_t u0 = (int64_t)pp.cum[b] + (int64_t)rg * x.tiles, u1 = u0 + x.tiles;
  const int64_t ng = min((int64_t)pp.NG, T);
  const int gf = (int)(((u0 + 1) * ng - 1) / T), gl = (int)((u1 * ng - 1) / T);
  if (gf == gl) return;                      // written by the CTA that held all of it
  const int lane = lane_id(), warp = warp_id();
  const int r = rb * 32 + lane;
  const bool live = r < nrows;
  // The group that starts the item writes slot 2g + 1, the ones that go on 2g.
  // Four partials at a time: their statistics are loaded together, then their
  // rows, so that a long item costs a few memory round trips and not one a partial.
  constexpr int U = 4;
  float M = -INFINITY, l = 0.f, acc[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) acc[e] = 0.f;
  const int rr0 = live ? r : 0;
  for (int g0 = gf; g0 <= gl; g0 += U) {
    float ms[U], ls[U], v[U][16];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int g = min(g0 + k, gl);
      const int64_t slot = (int64_t)(2 * g + (g == gf ? 1 : 0)) * pp.Hkv + h;
      ms[k] = pp.pml[slot * 2 * pp.rc + rr0];
      ls[k] = pp.pml[(slot * 2 + 1) * pp.rc + rr0];
      const float* src = pp.po + (slot * D + warp * 16) * pp.rc + rr0;
#pragma unroll
      for (int e = 0; e < 16; ++e) v[k][e] = src[(int64_t)e * pp.rc];
    }
    float top = M;
#pragma unroll
    for (int k = 0; k < U; ++k) {
      if (g0 + k > gl) ms[k] = -INFINITY;
      top = fmaxf(top, ms[k]);
    }
    if (top == -INFINITY) continue;
    const float shrink = M == -INFINITY ? 0.f : exp2f(M - top);
    M = top;
    l = shrink == 1.f ? l : l * shrink;
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[e] *= shrink;
#pragma unroll
    for (int k = 0; k < U; ++k) {
      if (ms[k] == -INFINITY) continue;      // nothing seen: its O is zero, or was not written
      const float w = exp2f(ms[k] - top);
      l += w * ls[k];                        // not a number stays so
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[e] += w * v[k][e];
    }
  }
  const int row = rg * per + r, t = live ? row / a.G : 0;
  const int hq = h * a.G + (live ? row - t * a.G : 0);
  const bool any = l > 0.f || l != l;
  if (p.sinks && any) l += exp2f(sink_log2(p, hq) - M);
  const float fin = (any ? 1.f / l : 0.f) * out_quant_factor(p);
#pragma unroll
  for (int e = 0; e < 16; ++e) rows[lane][warp * 16 + e] = any ? acc[e] * fin : 0.f;
  __syncthreads();
  for (int i = warp; i < 32; i += 8) {
    const int rr = rg * per + rb * 32 + i;
    if (rb * 32 + i >= nrows) break;
    const int tt_ = rr / a.G;
    const int64_t ob = o_offset(p, b, tt_, h * a.G + rr - tt_ * a.G);
    store_out2(p.out, p.out_dtype, ob + 2 * lane, rows[i][2 * lane], rows[i][2 * lane + 1]);
    store_out2(p.out, p.out_dtype, ob + 64 + 2 * lane, rows[i][64 + 2 * lane], rows[i][64 + 2 * lane + 1]);
  }
}

template <int NQ, int VF>
cudaError_t launch_tree_tc_t(const TreeTcParams& pp, cudaStream_t stream) {
  using namespace tt;
  auto kern = tree_tc_kernel<NQ, VF>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes(NQ));
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(pp.NG * pp.Hkv);
  cfg.blockDim = dim3(threads(NQ));
  cfg.dynamicSmemBytes = smem_bytes(NQ);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if ((e = cudaLaunchKernelEx(&cfg, kern, pp)) != cudaSuccess) return e;
  if (pp.NG == 1) return cudaSuccess;        // nothing is cut
  const int rows = pp.a.p.seq_q * pp.a.G, groups = (rows + NQ * BM - 1) / (NQ * BM), blocks = pp.rc / 32;
  cfg.gridDim = dim3((unsigned)(pp.a.p.num_seqs * groups * blocks), pp.Hkv);
  cfg.blockDim = dim3(256);
  cfg.dynamicSmemBytes = 0;
  return cudaLaunchKernelEx(&cfg, tree_combine_kernel<NQ>, pp, blocks, groups);
}

}  // namespace g9
