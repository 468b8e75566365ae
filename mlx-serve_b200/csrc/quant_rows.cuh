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

__device__ __forceinline__ void unpack8_bf16(const uint4& raw, float* v) {
  const uint32_t q[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) { v[2 * j] = bf16lo(q[j]); v[2 * j + 1] = bf16hi(q[j]); }
}

// 16 values of a group that `tpg` neighbouring lanes (2, 4 or 8) share -> their packed words and the group's parameters, by the
// affine rule of mlx_quantize as the reference restates it (tests/dsv4_imatrix.py:169-183, codes :264).  Whole warps call it.
template <int BITS>
__device__ __forceinline__ void quantize16(const float (&v)[kRowVals], int tpg, uint32_t (&w)[BITS / 2], float& scale, float& bias) {
  float xmin = v[0], xmax = v[0];
#pragma unroll
  for (int k = 1; k < kRowVals; ++k) { xmin = fminf(xmin, v[k]); xmax = fmaxf(xmax, v[k]); }
  for (int off = tpg >> 1; off > 0; off >>= 1) {
    xmin = fminf(xmin, __shfl_xor_sync(0xffffffffu, xmin, off));
    xmax = fmaxf(xmax, __shfl_xor_sync(0xffffffffu, xmax, off));
  }
  const float n_bins = (float)((1 << BITS) - 1);
  const bool mask = fabsf(xmin) > fabsf(xmax);
  scale = fmaxf(__fdiv_rn(__fsub_rn(xmax, xmin), n_bins), 1e-7f);
  scale = mask ? scale : -scale;
  const float edge = mask ? xmin : xmax;
  const float q0 = rintf(__fdiv_rn(edge, scale));
  bias = 0.0f;
  if (q0 != 0.0f) { scale = __fdiv_rn(edge, q0); bias = edge; }
  const float rs = __fdiv_rn(1.0f, scale);
#pragma unroll
  for (int k = 0; k < BITS / 2; ++k) w[k] = 0u;
#pragma unroll
  for (int k = 0; k < kRowVals; ++k) w[k * BITS / 32] |= code_of(v[k], bias, scale, rs, n_bins) << (k * BITS % 32);
}

}  // namespace qb
