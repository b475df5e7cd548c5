// What the cache's kernels and the attention over it share: the types' conversions and the cache's checks.
#pragma once
#include <hip/hip_fp16.h>

#include "dsv_common.h"

namespace dsv {

// A (token, head) whose largest magnitude lies below it is stored as zeros: the reciprocals stay finite.
constexpr float KV_TINY = 7.888609052210118e-31f;  // 2^-100

int check_cache(const char* what, const dsv_kv_cache* c);

template <int V>
struct Int {
  static constexpr int value = V;
};

__device__ __forceinline__ int64_t load_index(const void* p, int i64, int64_t i) {
  return i64 ? reinterpret_cast<const int64_t*>(p)[i] : (int64_t) reinterpret_cast<const int32_t*>(p)[i];
}

// r / d for r < 2^31.
struct FastDiv {
  uint32_t d, mul, shift;
  __device__ __forceinline__ uint32_t div(uint32_t r) const { return (uint32_t)(((uint64_t)r * mul) >> shift); }
};
inline FastDiv fast_div(uint32_t d) {
  FastDiv f;
  int log = 0;
  while ((1ull << log) < d) ++log;
  f.d = d;
  f.shift = 31 + log;
  f.mul = (uint32_t)(((1ull << f.shift) + d - 1) / d);
  return f;
}

// 16 bits of an activation as float32.
template <int XT>
__device__ __forceinline__ float act_to_f32(uint32_t bits) {
  if constexpr (XT == DSV_BF16)
    return bf16_bits_to_f32(bits);
  else
    return (float)__builtin_bit_cast(_Float16, (uint16_t)bits);
}

// Two float32 as activations, rounded to nearest even, the first in the low half (one instruction).
template <int XT>
__device__ __forceinline__ uint32_t pack_act(float lo, float hi) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  const f32x2 v = {lo, hi};
  if constexpr (XT == DSV_BF16) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
  } else {
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2));
  }
}

// Four float32 within the codes' range as codes, rounded to nearest even.
__device__ __forceinline__ uint32_t pack_e4m3(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}
__device__ __forceinline__ uint32_t pack_i8(float a, float b, float c, float d) {
  auto code = [](float x) { return (uint32_t)(int)__builtin_rintf(x) & 0xffu; };
  return code(a) | (code(b) << 8) | (code(c) << 16) | (code(d) << 24);
}

// Four codes as float32.
template <int CT>
__device__ __forceinline__ void unpack_codes(uint32_t w, float* f) {
  if constexpr (CT == DSV_E4M3) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    f[0] = lo.x;
    f[1] = lo.y;
    f[2] = hi.x;
    f[3] = hi.y;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = (float)(int8_t)(w >> (8 * i));
  }
}

}  // namespace dsv
