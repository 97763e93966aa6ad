// amf_int4_asym.h - the group quantizer of AMF_FMT_INT4_ASYM_G32, shared by the
// page codec (amf_int4.hip) and the kernels that write and read single tokens of
// a pool (amf_kv_step.hip, amf_paged_rows.hip).
#pragma once

#include "amf_kernel_util.h"

namespace amf {

constexpr float kAsymLevels = 15.0f;

// Nibble n (0..7) of a dword, as fp32.
__device__ __forceinline__ float nib(uint32_t w, int n) {
  return (float)__builtin_amdgcn_ubfe(w, 4 * n, 4);
}

// Group quantizer: min / max over 32 values, then
// scale = max(mx - mn, 1e-8) / 15 and q = clamp(rint((x - mn) / scale), 0, 15).
struct AsymParams {
  float mn, scale, rscale;
};

__device__ __forceinline__ AsymParams asym_params(const float* x) {
  float mn = x[0], mx = x[0];
#pragma unroll
  for (int n = 1; n < 32; ++n) {
    mn = fminf(mn, x[n]);
    mx = fmaxf(mx, x[n]);
  }
  AsymParams p;
  p.mn = mn;
  p.scale = fmaxf(mx - mn, 1e-8f) / kAsymLevels;
  p.rscale = 1.0f / p.scale;
  return p;
}

// Code n of eight into w, in order.  The wave-per-page save pushes it
// (push_code), which needs fewer operations; with a workgroup per page the
// compiler then holds so many chains at once that waves are lost (32 layers x
// 500 pages of 4 x 128: 145 us against 133).
template <int TEAM>
__device__ __forceinline__ uint32_t asym_insert(uint32_t w, int n, float x,
                                                const AsymParams& p) {
  if constexpr (TEAM == 64)
    return push_code(w, div_rn_code(x - p.mn, p.scale, p.rscale), 0.0f, kAsymLevels, 0.0f);
  float q = __builtin_rintf(div_rn(x - p.mn, p.scale, p.rscale));
  q = fminf(fmaxf(q, 0.0f), kAsymLevels);
  return w | (uint32_t)q << (4 * n);
}

__device__ __forceinline__ uint32_t asym_param_word(const AsymParams& p) {
  uint32_t s = __builtin_bit_cast(uint16_t, (_Float16)p.scale);
  uint32_t z = __builtin_bit_cast(uint16_t, (_Float16)p.mn);
  return s | (z << 16);
}

__device__ __forceinline__ float param_scale(uint32_t w) {
  return (float)__builtin_bit_cast(_Float16, (uint16_t)(w & 0xFFFFu));
}
__device__ __forceinline__ float param_zero(uint32_t w) {
  return (float)__builtin_bit_cast(_Float16, (uint16_t)(w >> 16));
}

}  // namespace amf
