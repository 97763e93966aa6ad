// amf_paged.h - what the operators over vLLM's paged K/V caches share: the
// block tables, block-wide scans and the element types of a cache.
#pragma once

#include "amf_internal.h"
#include "amf_kernel_util.h"

namespace amf {

// Sum of v over the lanes before this one in the wave; *total gets the wave's sum.
__device__ __forceinline__ int64_t wave_exclusive(int64_t v, int64_t* total) {
  const int lane = threadIdx.x & 63;
  int64_t x = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t y = __shfl_up(x, o);
    if (lane >= o) x += y;
  }
  *total = __shfl(x, 63);
  return x - v;
}

// The same over a workgroup of NT threads; tmp holds NT / 64 values.  Starts
// and ends with a barrier.
template <int NT>
__device__ __forceinline__ int64_t block_exclusive(int64_t v, int64_t* tmp, int64_t* total) {
  int64_t wsum;
  int64_t x = wave_exclusive(v, &wsum);
  const int wave = threadIdx.x >> 6;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) tmp[wave] = wsum;
  __syncthreads();
  int64_t all = 0;
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) {
    if (w == wave) x += all;
    all += tmp[w];
  }
  *total = all;
  __syncthreads();
  return x;
}

// Bytes of a cache element, AMF_DTYPE_E4M3 among the types; 0 for others.
inline int kv_elem_bytes(int32_t dtype) {
  return dtype == AMF_DTYPE_E4M3 ? 1 : cache_elem_bytes(dtype);
}

// One cache element as fp32.
template <int DT>
__device__ __forceinline__ float kv_elem(const uint8_t* p) {
  if constexpr (DT == AMF_DTYPE_F32) {
    return *reinterpret_cast<const float*>(p);
  } else if constexpr (DT == AMF_DTYPE_BF16) {
    return bf16_to_f32(*reinterpret_cast<const uint16_t*>(p));
  } else if constexpr (DT == AMF_DTYPE_F16) {
    return (float)*reinterpret_cast<const _Float16*>(p);
  } else {
    return __builtin_amdgcn_cvt_f32_fp8((int)*p, 0);
  }
}

}  // namespace amf
