// q8_quant.cuh -- Q8_0 quantisation of fp16 and bf16 values without the
// division routine and the float -> int conversions.  Bytes equal to the
// general form's (IEEE amax / 127 and 1 / d, round half to even, clamp) for
// every finite maximum: test_store_gpu.py::test_fast_store_every_16bit_absmax
// (the KV store) and test_tree_quant_gpu.py::test_every_16bit_maximum
// (norm_rope_store_kv) run all of them against the oracle.
#pragma once

#include "common.cuh"

namespace g9 {

// Scale of a block, amax / 127, and its reciprocal (0 for a scale of 0).
// amax / 127 correctly rounded: y = amax * fl(1/127), then one
// residual-correction step of the reciprocal product (Markstein's method:
// r = amax - y*127 exactly by FMA, y' = y + r*fl(1/127)).  Exact for every
// finite fp16 and bf16 value, which are all the values amax takes here.
__device__ __forceinline__ float q8_scale_16bit(float amax, float& inv) {
  constexpr float kInv127 = 1.0f / 127.0f;
  const float y = __fmul_rn(amax, kInv127);
  const float d = fmaf(fmaf(-y, 127.0f, amax), kInv127, y);
  inv = d > 0.0f ? __frcp_rn(d) : 0.0f;
  return d;
}

// rint(v * inv) clamped to [-128, 127], four elements packed, without the
// (quarter-rate) float -> int conversion: the product is rounded to fp32,
// adding 1.5 * 2^23 rounds it to an integer with ties to even (exactly rintf
// for |x| < 2^22) and leaves it in the low mantissa bits; the clamp is
// applied to the sum, and the int8 is its low byte.  When the scale underflows
// so far that its reciprocal is infinite, a zero element gives 0 * inf = NaN:
// it becomes 0, as a float -> int conversion makes it; +-inf products clamp.
__device__ __forceinline__ uint32_t q8_quants4(float v0, float v1, float v2, float v3, float inv) {
  constexpr float kMagic = 12582912.0f;
  const float v[4] = {v0, v1, v2, v3};
  uint32_t b[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float r = __fadd_rn(__fmul_rn(v[e], inv), kMagic);
    r = r == r ? r : kMagic;
    r = fminf(fmaxf(r, kMagic - 128.0f), kMagic + 127.0f);
    b[e] = __float_as_uint(r);
  }
  return __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
}

}  // namespace g9
