// mi_rope.hpp -- pieces of the rotation that its kernels share (mi_rope.hip, mi_kv_quant.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <math.h>

#include "mi_gemm_device.hpp"
#include "mi_paged.hpp"

namespace mig {

template <typename T, int VEC>
struct RopeVec {
  float v[VEC];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (sizeof(T) == 4) {
      if constexpr (VEC == 4) {
        const f32x4_t x = *(const f32x4_t*)p;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = x[e];
      } else {
        v[0] = *(const float*)p;
      }
    } else if constexpr (VEC == 1) {
      v[0] = bf16_bits_to_f32(*(const uint16_t*)p);
    } else {
      uint32_t w[VEC / 2];
      if constexpr (VEC == 8) *(u32x4_t*)w = *(const u32x4_t*)p;
      else *(u32x2_t*)w = *(const u32x2_t*)p;
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[e] = (e & 1) ? __uint_as_float(w[e / 2] & 0xffff0000u) : bf16_bits_to_f32(w[e / 2]);
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (sizeof(T) == 4) {
      if constexpr (VEC == 4) *(f32x4_t*)p = f32x4_t{v[0], v[1], v[2], v[3]};
      else *(float*)p = v[0];
    } else if constexpr (VEC == 1) {
      *(uint16_t*)p = (uint16_t)f32_to_bf16_rne(v[0]);
    } else {
      uint32_t w[VEC / 2];
#pragma unroll
      for (int e = 0; e < VEC / 2; ++e) w[e] = pack_bf16x2(v[2 * e], v[2 * e + 1]);
      if constexpr (VEC == 8) *(u32x4_t*)p = *(const u32x4_t*)w;
      else *(u32x2_t*)p = *(const u32x2_t*)w;
    }
  }
};

// Turns the pairs of two vectors by cosines c and sines s: (a[e], b[e]) or, interleaved, the neighbours in the two
// taken as one run of 2 VEC components.
template <int VEC>
__device__ __forceinline__ void rope_turn(float (&a)[VEC], float (&b)[VEC], const float* c, const float* s,
                                          bool interleaved) {
  if (interleaved) {
    float x[2 * VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) x[e] = a[e], x[VEC + e] = b[e];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const float x0 = x[2 * e], x1 = x[2 * e + 1];
      x[2 * e] = x0 * c[e] - x1 * s[e];
      x[2 * e + 1] = x1 * c[e] + x0 * s[e];
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) a[e] = x[e], b[e] = x[VEC + e];
  } else {
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const float x0 = a[e], x1 = b[e];
      a[e] = x0 * c[e] - x1 * s[e];
      b[e] = x1 * c[e] + x0 * s[e];
    }
  }
}

// Checks the rotary of an entry point; MI_OK or an error with its text.
inline int check_rotary(const mi_rotary* r, int64_t head_dim) {
  if (r->rot_dim < 2 || r->rot_dim % 2 || r->rot_dim > head_dim)
    return host_fail(MI_ERR_SHAPE, "rot_dim=%lld: an even number from 2 to head_dim=%lld is needed",
                     (long long)r->rot_dim, (long long)head_dim);
  if (!r->inv_freq) return host_fail(MI_ERR_NULL, "inv_freq is NULL");
  if (((uintptr_t)r->inv_freq | (uintptr_t)r->positions) & 3)
    return host_fail(MI_ERR_UNSUPPORTED, "inv_freq and positions must be aligned to their element size");
  if (!isfinite(r->scale)) return host_fail(MI_ERR_UNSUPPORTED, "scale must be finite");
  if (r->interleaved != 0 && r->interleaved != 1)
    return host_fail(MI_ERR_SHAPE, "interleaved=%d is not 0 or 1", r->interleaved);
  return MI_OK;
}

}  // namespace mig
