// Element types of the token operators (rms_norm.hip, linear.hip, cross_attention.hip): loads,
// stores and conversions of fp16, bf16, fp32 and e4m3 (OCP, largest value 448).
#pragma once
#include "common.h"
#include "internal.h"

namespace sengine {

typedef _Float16 half4_t __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x4_t __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef float float16_t __attribute__((ext_vector_type(16)));

struct E4m3 {  // a byte; arithmetic goes through the conversions below
  uint8_t bits;
};

struct E4m3Wide {  // the same bytes, multiplied as the fp16 values they stand for
  uint8_t bits;
};

inline int type_bytes(int code) {
  return code == SENGINE_ENC_F32 ? 4 : code == SENGINE_ENC_E4M3 ? 1 : 2;
}

// Whether one launch can have so many workgroups: its threads count to 2^32 - 1.
inline bool launchable(int64_t wgs, int threads) { return wgs <= 0xffffffffll / threads; }

// One element of a run-time type (a vector of coefficients read once per column).
__device__ __forceinline__ float load_as_float(const void* p, int code, int64_t i) {
  if (code == SENGINE_ENC_F32) return static_cast<const float*>(p)[i];
  if (code == SENGINE_ENC_F16) return (float)static_cast<const _Float16*>(p)[i];
  return (float)static_cast<const __bf16*>(p)[i];
}

// N consecutive values of T as floats: one load of N * sizeof(T) bytes, which the address is
// aligned to.
template <class T, int N>
__device__ __forceinline__ void load_floats(const T* p, float (&v)[N]) {
  if constexpr (N == 1) {
    v[0] = (float)*p;
  } else {
    typedef T vec_t __attribute__((ext_vector_type(N)));
    const vec_t x = *reinterpret_cast<const vec_t*>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (float)x[i];
  }
}

// Their nearest values of T (ties to even), stored the same way.
template <class T, int N>
__device__ __forceinline__ void store_floats(T* p, const float (&v)[N]) {
  if constexpr (N == 1) {
    *p = (T)v[0];
  } else {
    typedef T vec_t __attribute__((ext_vector_type(N)));
    vec_t x;
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = (T)v[i];
    *reinterpret_cast<vec_t*>(p) = x;
  }
}

// The same for e4m3 (N = 1 or a multiple of 4): the conversion instruction rounds to nearest even
// and keeps NaN; the caller keeps |v| <= 448.
template <int N>
__device__ __forceinline__ void store_floats(E4m3* p, const float (&v)[N]) {
  if constexpr (N == 1) {
    p->bits = (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[0], 0, false);
  } else {
    static_assert(N % 4 == 0, "whole words");
    typedef uint32_t vec_t __attribute__((ext_vector_type(N / 4)));
    uint32_t w[N / 4];
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      int x = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i], v[4 * i + 1], 0, false);
      w[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i + 2], v[4 * i + 3], x, true);
    }
    if constexpr (N == 4) {
      *reinterpret_cast<uint32_t*>(p) = w[0];
    } else {
      vec_t x;
#pragma unroll
      for (int i = 0; i < N / 4; ++i) x[i] = w[i];
      *reinterpret_cast<vec_t*>(p) = x;
    }
  }
}

}  // namespace sengine
