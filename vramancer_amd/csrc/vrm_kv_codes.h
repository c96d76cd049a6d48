// The int8 and e4m3 codes of the quantized pools (vrm_kv_quant.hip has their
// definition), shared by the writers.
#pragma once
#include "vrm_common.h"

namespace vrm {
namespace {

__device__ __forceinline__ int8_t int8_code(float x, float scale) {
  if (!(scale > 0.f)) return 0;
  float r = rintf(__fdiv_rn(x, scale));
  r = fminf(fmaxf(r, -127.f), 127.f);
  return (int8_t)(int)r;
}

__device__ __forceinline__ uint8_t fp8_code(float x, float scale) {
  if (!(scale > 0.f)) return 0;
  return vrm_e4m3::encode(__fdiv_rn(x, scale));
}

// x / s correctly rounded, from y = 1 / s correctly rounded: two residual
// corrections, the first of which brings the quotient within one ulp, where
// the second is exact (Markstein 1990).  Holds while the residuals stay
// normal: fast_scale below; for a smaller quotient (|x| < 2^-10 s at its
// smallest scale) both forms round to code 0 all the same.
__device__ __forceinline__ float div_by(float x, float s, float y) {
  float q = __fmul_rn(x, y);
  q = fmaf(fmaf(-q, s, x), y, q);
  return fmaf(fmaf(-q, s, x), y, q);
}
__device__ __forceinline__ bool fast_scale(float s) { return s > 0x1p-80f && s < 0x1p100f; }

// Four int8 codes, little end first: |q| <= 127 after the clamp, so adding
// 1.5 * 2^23 leaves the integer nearest to q (ties to even) in the low byte.
__device__ __forceinline__ uint32_t int8_codes4(const float* x, float s, float y) {
  uint32_t c[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float q = fminf(fmaxf(div_by(x[i], s, y), -127.f), 127.f);
    c[i] = __float_as_uint(__fadd_rn(q, 12582912.f));
  }
  const uint32_t lo = __builtin_amdgcn_perm(c[1], c[0], 0x0c0c0400u);
  const uint32_t hi = __builtin_amdgcn_perm(c[3], c[2], 0x04000c0cu);
  return lo | hi;
}

__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return a | (b << 8) | (c << 16) | (d << 24);
}

// Codes of 8 elements, little end first.  v_cvt_pk_fp8_f32 gives
// vrm_e4m3::encode's code for every float up to 464 in magnitude (all of them
// compared) but not for NaN, whose codes are the only ones with seven low bits
// set: those lanes take the general path.
template <bool FP8>
__device__ __forceinline__ void codes8(const float (&x)[8], float scale, uint32_t& lo, uint32_t& hi) {
  bool slow = !fast_scale(scale);
  if (!slow) {
    const float y = __fdiv_rn(1.f, scale);
    if constexpr (FP8) {
      float q[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) q[i] = copysignf(div_by(x[i], scale, y), x[i]);  // -0 stays -0
      int a = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
      a = __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], a, true);
      int b = __builtin_amdgcn_cvt_pk_fp8_f32(q[4], q[5], 0, false);
      b = __builtin_amdgcn_cvt_pk_fp8_f32(q[6], q[7], b, true);
      lo = (uint32_t)a;
      hi = (uint32_t)b;
      slow = ((((~lo & 0x7f7f7f7fu) - 0x01010101u) | ((~hi & 0x7f7f7f7fu) - 0x01010101u)) & 0x80808080u) != 0;
    } else {
      lo = int8_codes4(x, scale, y);
      hi = int8_codes4(x + 4, scale, y);
    }
  }
  if (slow) {
    uint32_t c[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = FP8 ? fp8_code(x[i], scale) : (uint8_t)int8_code(x[i], scale);
    lo = pack4(c[0], c[1], c[2], c[3]);
    hi = pack4(c[4], c[5], c[6], c[7]);
  }
}

}  // namespace
}  // namespace vrm
