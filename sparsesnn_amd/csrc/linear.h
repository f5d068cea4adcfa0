// Parameters and epilogue shared by the linear kernels (linear.hip).
#pragma once
#include "token_types.h"

namespace sengine {

struct LinearParams {
  const uint8_t* x;   // (M, K) rows x_stride bytes apart
  const uint8_t* w;   // (N, K) rows w_stride bytes apart
  const float* x_scale;  // M, or null
  const float* w_scale;  // N, or null
  const void* bias;      // N of bias_type, or null
  const void* res;       // (M, N) of out_type, rows res_stride elements apart, or null
  void* out;             // (M, N) of out_type, rows out_stride elements apart
  int64_t M, x_stride, w_stride, res_stride, out_stride;
  int N, K;
  int kbytes;            // K in bytes
  int act, out_type, bias_type;
  int vec;               // out and res rows begin at multiples of four elements
};

// gelu(z) = z * Phi(z), Phi by erf; gelu_tanh(z) = z * sigmoid(2 sqrt(2/pi) (z + 0.044715 z^3)),
// which is the tanh form rewritten; silu(z) = z * sigmoid(z).
__device__ __forceinline__ float activate(float z, int act) {
  switch (act) {
    case SENGINE_ACT_RELU:
      return z < 0.f ? 0.f : z;  // a NaN stays
    case SENGINE_ACT_GELU:
      return 0.5f * z * (1.f + erff(z * 0.70710678118654752f));
    case SENGINE_ACT_GELU_TANH: {
      const float u = 1.5957691216057308f * (z + 0.044715f * z * z * z);
      return z / (1.f + __expf(-u));
    }
    case SENGINE_ACT_SILU:
      return z / (1.f + __expf(-z));
    default:
      return z;
  }
}

// Four consecutive output columns n..n+3 of row m, from the fp32 sums of the reduction: scales,
// bias, activation and residual in fp32, one rounding at the store.
__device__ __forceinline__ void linear_store4(const LinearParams& p, int64_t m, int n, float4_t acc) {
  if (m >= p.M || n >= p.N) return;
  float v[4];
  const int cnt = p.N - n < 4 ? p.N - n : 4;
  const float sx = p.x_scale ? p.x_scale[m] : 1.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[i] = acc[i];
    const int c = i < cnt ? n + i : n;
    if (p.x_scale) v[i] *= sx;
    if (p.w_scale) v[i] *= p.w_scale[c];
    if (p.bias) v[i] += load_as_float(p.bias, p.bias_type, c);
    v[i] = activate(v[i], p.act);
  }
  const int64_t o = m * p.out_stride + n, r = m * p.res_stride + n;
  if (p.vec && cnt == 4) {
    if (p.out_type == SENGINE_ENC_F32) {
      if (p.res) {
        float t[4];
        load_floats<float, 4>(static_cast<const float*>(p.res) + r, t);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] += t[i];
      }
      store_floats<float, 4>(static_cast<float*>(p.out) + o, v);
    } else if (p.out_type == SENGINE_ENC_F16) {
      if (p.res) {
        float t[4];
        load_floats<_Float16, 4>(static_cast<const _Float16*>(p.res) + r, t);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] += t[i];
      }
      store_floats<_Float16, 4>(static_cast<_Float16*>(p.out) + o, v);
    } else {
      if (p.res) {
        float t[4];
        load_floats<__bf16, 4>(static_cast<const __bf16*>(p.res) + r, t);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] += t[i];
      }
      store_floats<__bf16, 4>(static_cast<__bf16*>(p.out) + o, v);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (i < cnt) {
      if (p.res) v[i] += load_as_float(p.res, p.out_type, r + i);
      if (p.out_type == SENGINE_ENC_F32)
        static_cast<float*>(p.out)[o + i] = v[i];
      else if (p.out_type == SENGINE_ENC_F16)
        static_cast<_Float16*>(p.out)[o + i] = (_Float16)v[i];
      else
        static_cast<__bf16*>(p.out)[o + i] = (__bf16)v[i];
    }
  }
}

// Eight e4m3 codes as fp16: exact, every e4m3 value is one.
__device__ __forceinline__ half8_t widen_e4m3(uint32_t lo, uint32_t hi) {
  typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
  const half2_t a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, false);
  const half2_t b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, true);
  const half2_t c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, false);
  const half2_t d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, true);
  return half8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// 16 operand rows x 16 operand rows over one 128-byte step of the reduction: 64 values of 16 bits
// (two 16x16x32 instructions) or 128 of 8 bits (one 16x16x128).  Lane l of `a` and of `b` holds the
// same bytes of rows l % 16, in whatever order the reduction's values lie over the lanes: the sum does
// not depend on it as long as both have the same.  D: lane l, value i is row 4 (l / 16) + i of a and
// row l % 16 of b.
//
// The 8-bit instruction does not keep all of a 32-bit sum: its result was measured up to 2^-12 of the
// sum of the magnitudes off, 1.4e-5 of the result on normally distributed operands (the 16x16x32 8-bit
// form is the same; the 16-bit ones are within 2^-21).  That is a tenth of an fp16 output's rounding, so
// 16-bit outputs take it; an fp32 output is computed from the codes widened to fp16 (E4m3Wide), at half
// the rate, with sums of 32 bits.
typedef int int8v_t __attribute__((ext_vector_type(8)));
template <class T>
__device__ __forceinline__ float4_t mma_128b(u32x4_t a0, u32x4_t a1, u32x4_t b0, u32x4_t b1, float4_t c) {
  if constexpr (__is_same(T, _Float16)) {
    c = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a0), __builtin_bit_cast(half8_t, b0), c, 0,
                                               0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a1), __builtin_bit_cast(half8_t, b1), c,
                                                  0, 0, 0);
  } else if constexpr (__is_same(T, __bf16)) {
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a0), __builtin_bit_cast(bf16x8_t, b0), c,
                                                0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a1), __builtin_bit_cast(bf16x8_t, b1),
                                                   c, 0, 0, 0);
  } else if constexpr (__is_same(T, E4m3)) {
    const u32x8_t a = __builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7);
    const u32x8_t b = __builtin_shufflevector(b0, b1, 0, 1, 2, 3, 4, 5, 6, 7);
    // both block scales 2^0 (exponent byte 127), both operands e4m3 (format 0)
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(__builtin_bit_cast(int8v_t, a),
                                                            __builtin_bit_cast(int8v_t, b), c, 0, 0, 0, 0x7f7f7f7f, 0,
                                                            0x7f7f7f7f);
  } else {
    c = __builtin_amdgcn_mfma_f32_16x16x32_f16(widen_e4m3(a0[0], a0[1]), widen_e4m3(b0[0], b0[1]), c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x32_f16(widen_e4m3(a0[2], a0[3]), widen_e4m3(b0[2], b0[3]), c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x32_f16(widen_e4m3(a1[0], a1[1]), widen_e4m3(b1[0], b1[1]), c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(widen_e4m3(a1[2], a1[3]), widen_e4m3(b1[2], b1[3]), c, 0, 0, 0);
  }
}

}  // namespace sengine
