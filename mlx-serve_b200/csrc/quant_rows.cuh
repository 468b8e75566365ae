// The affine quantiser of 16 values a thread, shared by the kernels that quantise rows (whole tensors, cache pages).
#pragma once
#include "common.cuh"

namespace qb {

constexpr int kRowVals = 16;    // values per thread: the group's parameters (four divisions) are worked out once per 16

// rint(x / s) clamped to [0, bins], exactly as the division rounds: away from the ties the product with 1 / s decides, near
// them (within 2^-10, far more than its error for quotients up to 256) and where anything is not finite the division does.
__device__ __forceinline__ uint32_t code_of(float x, float bias, float s, float rs, float bins) {
  const float n = __fsub_rn(x, bias);
  const float t = fmaf(n, rs, 12582912.f);          // 1.5 * 2^23 + rint(n / s): the low bits are the integer
  const float r = fmaf(n, rs, 12582912.f - t);      // what the rounding left
  float c = t - 12582912.f;
  if (!(fabsf(r) < 0.5f - 9.765625e-4f)) c = rintf(__fdiv_rn(n, s));
  return (uint32_t)fminf(fmaxf(c, 0.0f), bins);
}

__device__ __forceinline__ __nv_bfloat162 as_bf162(uint32_t v) { return *(const __nv_bfloat162*)&v; }
__device__ __forceinline__ uint32_t bits_of(__nv_bfloat162 v) { return *(const uint32_t*)&v; }

// 16 values (bf16 pairs) of a group that `tpg` neighbouring lanes (2, 4 or 8) share -> their packed words and the group's parameters, by
// the affine rule of mlx_quantize as the reference restates it (tests/dsv4_imatrix.py:169-183, codes :264).  Whole warps call it.
// Bound by instructions.  Minimum and maximum are taken on the pairs as they are.  The codes are rint(x / s) with the quotient rounded
// as a division rounds it: bf16 values lie so coarsely that one in 400 is a tie, so nothing is left to chance.  With y = 1 / s rounded
// to nearest, q + (n - q s) y is the correctly rounded n / s wherever q is within one step of it (Markstein's theorem), as it is after
// one such step; two quotients go through an instruction.  A code is the low byte of its quotient + 1.5 * 2^23.
template <int BITS>
__device__ __forceinline__ void quantize16(const uint32_t (&raw)[8], int tpg, uint32_t (&w)[BITS / 2], float& scale, float& bias) {
  __nv_bfloat162 lo = as_bf162(raw[0]), hi = lo;
#pragma unroll
  for (int k = 1; k < 8; ++k) { lo = __hmin2(lo, as_bf162(raw[k])); hi = __hmax2(hi, as_bf162(raw[k])); }
  for (int off = tpg >> 1; off > 0; off >>= 1) {
    lo = __hmin2(lo, as_bf162(__shfl_xor_sync(0xffffffffu, bits_of(lo), off)));
    hi = __hmax2(hi, as_bf162(__shfl_xor_sync(0xffffffffu, bits_of(hi), off)));
  }
  const float xmin = fminf(bf16lo(bits_of(lo)), bf16hi(bits_of(lo))), xmax = fmaxf(bf16lo(bits_of(hi)), bf16hi(bits_of(hi)));
  const float n_bins = (float)((1 << BITS) - 1);
  const bool mask = fabsf(xmin) > fabsf(xmax);
  scale = fmaxf(__fdiv_rn(__fsub_rn(xmax, xmin), n_bins), 1e-7f);
  scale = mask ? scale : -scale;
  const float edge = mask ? xmin : xmax;
  const float q0 = rintf(__fdiv_rn(edge, scale));
  bias = 0.0f;
  if (q0 != 0.0f) { scale = __fdiv_rn(edge, q0); bias = edge; }
  const float rs = __fdiv_rn(1.0f, scale), magic = 12582912.f;          // 1.5 * 2^23 + n: the low bits are n
  uint32_t c[16];
  if (fabsf(scale) < 1e36f && fabsf(scale) > 1e-18f) {                  // (with y and the remainders in the normal range)
    const uint64_t bias2 = two(-bias, -bias), y2 = two(rs, rs), s2 = two(-scale, -scale), magic2 = two(magic, magic);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint64_t n = add2(two(bf16lo(raw[k]), bf16hi(raw[k])), bias2);
      uint64_t q = mul2(n, y2);
      q = fma2(fma2(q, s2, n), y2, q);
      q = fma2(fma2(q, s2, n), y2, q);
      float t0, t1;
      untwo(add2(q, magic2), t0, t1);
      c[2 * k] = __float_as_uint(fminf(fmaxf(t0, magic), magic + n_bins));
      c[2 * k + 1] = __float_as_uint(fminf(fmaxf(t1, magic), magic + n_bins));
    }
  } else {
#pragma unroll
    for (int k = 0; k < 16; ++k) c[k] = code_of((k & 1) ? bf16hi(raw[k >> 1]) : bf16lo(raw[k >> 1]), bias, scale, rs, n_bins);
  }
  if constexpr (BITS == 8) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      w[k] = __byte_perm(__byte_perm(c[4 * k], c[4 * k + 1], 0x0040), __byte_perm(c[4 * k + 2], c[4 * k + 3], 0x0040), 0x5410);
  } else {
    uint32_t e[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) e[k] = c[2 * k] + (c[2 * k + 1] << 4);  // (the low byte is the two codes)
#pragma unroll
    for (int k = 0; k < 2; ++k)
      w[k] = __byte_perm(__byte_perm(e[4 * k], e[4 * k + 1], 0x0040), __byte_perm(e[4 * k + 2], e[4 * k + 3], 0x0040), 0x5410);
  }
}

}  // namespace qb
