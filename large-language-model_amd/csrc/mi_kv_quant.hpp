// mi_kv_quant.hpp -- the numbers of a K/V cache of 8 or 4 bits on the device (mi_kv_quant.hip, mi_paged_quant.hip):
// gfx950 converts two of them at a time and multiplies by the group's power of two on the way.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "mi_gemm_device.hpp"

namespace mig {

constexpr int KV_GROUP = 32;  // components that share a scale byte

// The power of two of a scale byte.  255 gives infinity, which the conversions below take for NaN, of any code; 0 gives 0,
// which leaves codes of 0 zeros and any others finite.
__device__ __forceinline__ float kv_power(uint32_t scale_byte) { return __uint_as_float(scale_byte << 23); }

// Codes 2i, 2i+1 of a dword of codes times s, as two bf16: exact for every scale byte that is written.
template <int BITS, int I>
__device__ __forceinline__ uint32_t kv_pair(uint32_t codes, float s) {
#if defined(__HIP_DEVICE_COMPILE__)
  if constexpr (BITS == 4) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, s, I));
  else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, s, I != 0));
#else
  return codes;
#endif
}

// Eight components from 4 (e2m1) or 8 (e4m3) bytes of codes.
template <int BITS>
__device__ __forceinline__ u32x4_t kv_eight(const uint32_t* codes, float s) {
  if constexpr (BITS == 4)
    return u32x4_t{kv_pair<4, 0>(codes[0], s), kv_pair<4, 1>(codes[0], s), kv_pair<4, 2>(codes[0], s),
                   kv_pair<4, 3>(codes[0], s)};
  else
    return u32x4_t{kv_pair<8, 0>(codes[0], s), kv_pair<8, 1>(codes[0], s), kv_pair<8, 0>(codes[1], s),
                   kv_pair<8, 1>(codes[1], s)};
}

}  // namespace mig
