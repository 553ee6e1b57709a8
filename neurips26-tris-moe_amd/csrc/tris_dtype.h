// 16-bit activations (fp16 or bf16, by a compile-time or a wave-uniform run-time flag) <-> fp32, eight at a time.
#pragma once

#include "tris_common.h"

namespace tris {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

// bits of a pair of fp32 values as bf16, round to nearest even (v_cvt_pk_bf16_f32)
__device__ __forceinline__ uint32_t pack_bf16_rne(float lo, float hi) {
  const bf16x2 v = {static_cast<__bf16>(lo), static_cast<__bf16>(hi)};
  return __builtin_bit_cast(uint32_t, v);
}
__device__ __forceinline__ uint32_t pack_f16_rne(float lo, float hi) {
  return static_cast<uint32_t>(f2h_bits(lo)) | (static_cast<uint32_t>(f2h_bits(hi)) << 16);
}

__device__ __forceinline__ float load1(const void* p, int64_t i, int32_t type) {
  if (type == TRIS_DTYPE_F32) return static_cast<const float*>(p)[i];
  const uint16_t b = static_cast<const uint16_t*>(p)[i];
  return type == TRIS_DTYPE_BF16 ? __uint_as_float(static_cast<uint32_t>(b) << 16) : h2f(b);
}
__device__ __forceinline__ void store1(void* p, int64_t i, float v, int32_t type) {
  static_cast<uint16_t*>(p)[i] =
      static_cast<uint16_t>(type == TRIS_DTYPE_BF16 ? pack_bf16_rne(v, 0.0f) : f2h_bits(v));
}

__device__ __forceinline__ void widen8(const uint4 w, bool bf16, float v[8]) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
  if (bf16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(u[i] << 16);
      v[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = h2f(static_cast<uint16_t>(u[i]));
      v[2 * i + 1] = h2f(static_cast<uint16_t>(u[i] >> 16));
    }
  }
}
__device__ __forceinline__ uint4 narrow8(const float v[8], bool bf16) {
  uint32_t u[4];
  if (bf16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = pack_bf16_rne(v[2 * i], v[2 * i + 1]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = pack_f16_rne(v[2 * i], v[2 * i + 1]);
  }
  return make_uint4(u[0], u[1], u[2], u[3]);
}

inline bool is_16bit(int32_t type) { return type == TRIS_DTYPE_F16 || type == TRIS_DTYPE_BF16; }
inline bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

}  // namespace tris
