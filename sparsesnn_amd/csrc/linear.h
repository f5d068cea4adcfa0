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
  float* partial;        // sums of the reduction's parts (linear_tile.h), or null
  int part_steps;        // 128-byte steps a part
  int vec;               // N is a multiple of 8, out and res rows begin at multiples of 16 bytes
};

// Where the 128-byte step after the one at k begins, and whether there is one (rows go up to 2^31 - 1 bytes, past which
// a step at 2^31 lies: unsigned), and whether the row has all of its 16-byte piece at k, which lies inside it.
__host__ __device__ inline bool has_step(uint32_t k, int kbytes) { return k < (uint32_t)kbytes; }
__host__ __device__ inline uint32_t next_step(uint32_t k) { return k + 128; }
__host__ __device__ inline bool whole_piece(int k, int kbytes) { return kbytes - k >= 16; }

template <int V>
struct Int {
  static constexpr int value = V;
};

// z * sigmoid(t), t given as u = t / ln 2: z / (1 + 2^-u).
__device__ __forceinline__ float times_sigmoid2(float z, float u) {
  return z * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-u));
}

// gelu(z) = z * Phi(z), written as z * sigmoid(z * P(z^2)): P is the logit of Phi over z, an even
// function, as a polynomial of degree 6 in z^2 (weighted least squares towards the least largest error
// over |z| <= 6, in base 2).  Phi is off by at most 2.7 units of 2^-24, and P keeps growing beyond.
// Ten full-rate operations, an exponential and a reciprocal.
// gelu_tanh(z) = z * sigmoid(2 sqrt(2/pi) (z + 0.044715 z^3)), the tanh form rewritten;
// silu(z) = z * sigmoid(z).
template <int ACT>
__device__ __forceinline__ float activate(float z) {
  if constexpr (ACT == SENGINE_ACT_RELU) {
    return z < 0.f ? 0.f : z;  // a NaN stays
  } else if constexpr (ACT == SENGINE_ACT_GELU) {
    const float t = z * z;
    float p = 5.067260833158116e-09f;
    p = __builtin_fmaf(p, t, -3.816321054728178e-07f);
    p = __builtin_fmaf(p, t, 1.1439842637628317e-05f);
    p = __builtin_fmaf(p, t, -0.00015957998402882367f);
    p = __builtin_fmaf(p, t, -9.404912998434156e-05f);
    p = __builtin_fmaf(p, t, 0.10483512282371521f);
    p = __builtin_fmaf(p, t, 2.3022093772888184f);
    return times_sigmoid2(z, z * p);
  } else if constexpr (ACT == SENGINE_ACT_GELU_TANH) {
    // 2 sqrt(2/pi) / ln 2 and 0.044715 times it
    return times_sigmoid2(z, z * __builtin_fmaf(z * z, 0.10294324f, 2.3022082f));
  } else if constexpr (ACT == SENGINE_ACT_SILU) {
    return times_sigmoid2(z, z * 1.4426950408889634f);
  } else {
    return z;
  }
}

// f(Int<ACT>) for the run-time activation.
template <class F>
__device__ __forceinline__ void by_activation(int act, F f) {
  switch (act) {
    case SENGINE_ACT_RELU:
      f(Int<SENGINE_ACT_RELU>{});
      break;
    case SENGINE_ACT_GELU:
      f(Int<SENGINE_ACT_GELU>{});
      break;
    case SENGINE_ACT_GELU_TANH:
      f(Int<SENGINE_ACT_GELU_TANH>{});
      break;
    case SENGINE_ACT_SILU:
      f(Int<SENGINE_ACT_SILU>{});
      break;
    default:
      f(Int<SENGINE_ACT_NONE>{});
      break;
  }
}

// NV neighbouring values of type O as they lie in memory.
template <class O, int NV>
struct Raw {
  typedef O vec_t __attribute__((ext_vector_type(NV), aligned(NV * sizeof(O) < 16 ? NV * sizeof(O) : 16)));
  typedef O any_t __attribute__((ext_vector_type(NV), aligned(sizeof(O))));  // the same at any element
  vec_t v;
};

// NV columns from n on of NR rows m, m + STEP, ... of the residual.  They are not used before linear_finish, so
// that all rows' loads are in flight together.  VEC: N is a multiple of 8 and the rows of out and residual begin at
// multiples of 16 bytes; otherwise the same accesses begin at any element, and only a row's last columns go one by
// one (93982 x 377 x 144 bf16 with GELU and a residual: 71 us, all one by one 145).
template <class O, bool VEC, int NR, int STEP, int NV>
__device__ __forceinline__ void linear_residual(const LinearParams& p, int64_t m, int n, Raw<O, NV> (&r)[NR]) {
  if (!p.res || n >= p.N) return;
#pragma unroll
  for (int u = 0; u < NR; ++u) {
    const int64_t row = m + STEP * u < p.M ? m + STEP * u : p.M - 1;
    const O* at = static_cast<const O*>(p.res) + row * p.res_stride + n;
    if constexpr (VEC) {
      r[u].v = *reinterpret_cast<const typename Raw<O, NV>::vec_t*>(at);
    } else if (n + NV <= p.N) {
      r[u].v = *reinterpret_cast<const typename Raw<O, NV>::any_t*>(at);
    } else {
#pragma unroll
      for (int e = 0; e < NV; ++e)
        if (n + e < p.N) r[u].v[e] = at[e];
    }
  }
}

// The coefficients of NV columns and NR rows STEP apart; only 8-bit operands and widened 4-bit weights have scales.
// Tile kernels load them before their products, so that the epilogue does not wait for them.
template <class T, int NV>
struct Columns {
  static constexpr bool kScaled = Operand<T>::kScaled;
  float w[kScaled ? NV : 1], bias[NV];
  __device__ __forceinline__ void load(const LinearParams& p, int n) {
#pragma unroll
    for (int e = 0; e < NV; ++e) {
      const int at = n + e < p.N ? n + e : p.N - 1;
      if constexpr (kScaled) w[e] = p.w_scale ? p.w_scale[at] : 1.f;
      bias[e] = p.bias ? load_as_float(p.bias, p.bias_type, at) : 0.f;
    }
  }
};
template <class T, int NR, int STEP>
struct RowScales {
  static constexpr bool kScaled = Operand<T>::kScaled;
  float x[kScaled ? NR : 1];
  __device__ __forceinline__ void load(const LinearParams& p, int64_t m) {
    if constexpr (kScaled) {
#pragma unroll
      for (int u = 0; u < NR; ++u) {
        const int64_t row = m + STEP * u < p.M ? m + STEP * u : p.M - 1;
        x[u] = p.x_scale ? p.x_scale[row] : 1.f;
      }
    }
  }
};

// The same rows and columns finished from their sums: scales, bias, activation and residual in fp32, one rounding.
template <class T, class O, bool VEC, int NR, int STEP, int NV>
__device__ __forceinline__ void linear_finish(const LinearParams& p, int64_t m, int n, float (&v)[NR][NV],
                                              const Columns<T, NV>& c, const RowScales<T, NR, STEP>& rs,
                                              const Raw<O, NV> (&r)[NR]) {
#pragma unroll
  for (int u = 0; u < NR; ++u) {
    if constexpr (Columns<T, NV>::kScaled) {
#pragma unroll
      for (int e = 0; e < NV; ++e) v[u][e] *= rs.x[u] * c.w[e];
    }
#pragma unroll
    for (int e = 0; e < NV; ++e) v[u][e] += c.bias[e];
  }
  if (p.act != SENGINE_ACT_NONE) {
    by_activation(p.act, [&](auto act) {
#pragma unroll
      for (int u = 0; u < NR; ++u)
#pragma unroll
        for (int e = 0; e < NV; ++e) v[u][e] = activate<decltype(act)::value>(v[u][e]);
    });
  }
  if (n >= p.N) return;
  if (p.res) {
#pragma unroll
    for (int u = 0; u < NR; ++u)
#pragma unroll
      for (int e = 0; e < NV; ++e) v[u][e] += (float)r[u].v[e];
  }
#pragma unroll
  for (int u = 0; u < NR; ++u) {
    if (m + STEP * u >= p.M) continue;
    O* at = static_cast<O*>(p.out) + (m + STEP * u) * p.out_stride + n;
    typename Raw<O, NV>::vec_t x;
#pragma unroll
    for (int e = 0; e < NV; ++e) x[e] = (O)v[u][e];
    if constexpr (VEC) {
      *reinterpret_cast<typename Raw<O, NV>::vec_t*>(at) = x;
    } else if (n + NV <= p.N) {
      *reinterpret_cast<typename Raw<O, NV>::any_t*>(at) = x;
    } else {
#pragma unroll
      for (int e = 0; e < NV; ++e)
        if (n + e < p.N) at[e] = x[e];
    }
  }
}

// f(O(), Int<VEC>) for the output's type and layout.
template <class F>
__device__ __forceinline__ void by_output(const LinearParams& p, F f) {
  if (p.vec) {
    if (p.out_type == SENGINE_ENC_F32)
      f(0.f, Int<1>{});
    else if (p.out_type == SENGINE_ENC_F16)
      f((_Float16)0.f, Int<1>{});
    else
      f((__bf16)0.f, Int<1>{});
  } else {
    if (p.out_type == SENGINE_ENC_F32)
      f(0.f, Int<0>{});
    else if (p.out_type == SENGINE_ENC_F16)
      f((_Float16)0.f, Int<0>{});
    else
      f((__bf16)0.f, Int<0>{});
  }
}

// The epilogue of TM x TN fragments: value e of fragment acc[i][j] is row m + 16 j, column
// n + 32 (i / 2) + 4 (i % 2) + e, so that a lane has 8 neighbouring columns of a row.  c and rs are those
// columns' and rows' coefficients.
template <class T, int TM, int TN>
__device__ __forceinline__ void linear_epilogue(const LinearParams& p, int64_t m, int n, float4_t (&acc)[TN][TM],
                                                const Columns<T, 8> (&c)[TN / 2], const RowScales<T, TM, 16>& rs) {
  by_output(p, [&](auto o, auto vec) {
    using O = decltype(o);
    constexpr bool VEC = decltype(vec)::value;
    Raw<O, 8> res[2][TM];  // those of the next columns are in flight while these are finished
    linear_residual<O, VEC, TM, 16, 8>(p, m, n, res[0]);
#pragma unroll
    for (int i = 0; i < TN / 2; ++i) {
      if (i + 1 < TN / 2) linear_residual<O, VEC, TM, 16, 8>(p, m, n + 32 * (i + 1), res[(i + 1) % 2]);
      float v[TM][8];
#pragma unroll
      for (int j = 0; j < TM; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) v[j][e] = acc[2 * i + e / 4][j][e % 4];
      linear_finish<T, O, VEC, TM, 16, 8>(p, m, n + 32 * i, v, c[i], rs, res[i % 2]);
      __builtin_amdgcn_sched_barrier(0);
    }
  });
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
// form is the same; the 16-bit ones are within 2^-21).  For products of random signs that is a tenth of an
// fp16 output's rounding, so 16-bit outputs take it.  A sum that cancels loses more of its own bits, up to
// 2^-12 of the magnitudes that went into it.  An fp32 output is computed from the codes widened to fp16
// (E4m3Wide), at half the rate, with sums of 32 bits.
typedef int int8v_t __attribute__((ext_vector_type(8)));

// One 64-byte half of that step, for the types whose instruction takes it.
template <class T>
__device__ __forceinline__ float4_t mma_64b(u32x4_t a, u32x4_t b, float4_t c) {
  if constexpr (__is_same(typename Operand<T>::type, _Float16)) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0,
                                                  0, 0);
  } else if constexpr (__is_same(typename Operand<T>::type, __bf16)) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c,
                                                   0, 0, 0);
  } else {
    c = __builtin_amdgcn_mfma_f32_16x16x32_f16(widen_e4m3(a[0], a[1]), widen_e4m3(b[0], b[1]), c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(widen_e4m3(a[2], a[3]), widen_e4m3(b[2], b[3]), c, 0, 0, 0);
  }
}

template <class T>
__device__ __forceinline__ float4_t mma_128b(u32x4_t a0, u32x4_t a1, u32x4_t b0, u32x4_t b1, float4_t c) {
  if constexpr (__is_same(T, E4m3)) {
    const u32x8_t a = __builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7);
    const u32x8_t b = __builtin_shufflevector(b0, b1, 0, 1, 2, 3, 4, 5, 6, 7);
    // both block scales 2^0 (exponent byte 127), both operands e4m3 (format 0)
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(__builtin_bit_cast(int8v_t, a),
                                                            __builtin_bit_cast(int8v_t, b), c, 0, 0, 0, 0x7f7f7f7f, 0,
                                                            0x7f7f7f7f);
  } else {
    return mma_64b<T>(a1, b1, mma_64b<T>(a0, b0, c));
  }
}

// The linear operator on 16-bit operands of which the weight's rows have fp32 scales (w_scale), and the scratch memory
// that it takes parts in (linear.hip).  p is filled as by the entry.
hipError_t launch_linear_scaled(const LinearParams& p, bool fp16, float* workspace, size_t bytes, hipStream_t stream);
size_t linear_scaled_workspace(const LinearParams& p);

}  // namespace sengine
