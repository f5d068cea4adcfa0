// Matrix product of token rows with a weight in 4 bits, everything after it in the epilogue:
//   y[m, n] = act(r[n] sum_k x[m, k] s[n, k / group] c[n, k] + b[n]) + res[m, n]
// c: e2m1 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives), two a byte, the lower first; s: e4m3, one a group of
// 32, 64 or 128 values of a row; r: fp32, one a row.  x is fp16 or bf16.  Codes are fp16 and bf16 values, and so is
// s * c (six significant bits; its exponents are within fp16's), so that nothing of the weight is rounded on any route.
// Sums and epilogue are fp32 and y is rounded once.
#include "linear_rows.h"

namespace sengine {

struct E2m1Params {
  LinearParams lin;      // x, weight's codes (w, w_stride in bytes), w_scale = r, bias, residual, output
  const uint8_t* scale;  // s, rows scale_stride bytes apart
  int64_t scale_stride;
  int groups;            // scales of a row
};

// Eight codes of a dword as T, times a power of two.
template <class T>
__device__ __forceinline__ u32x4_t widen_e2m1(uint32_t v, float power) {
  u32x4_t r;
  if constexpr (__is_same(T, _Float16)) {
    r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(v, power, 0));
    r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(v, power, 1));
    r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(v, power, 2));
    r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(v, power, 3));
  } else {
    r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(v, power, 0));
    r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(v, power, 1));
    r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(v, power, 2));
    r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(v, power, 3));
  }
  return r;
}

// A group's scale s as power * rest, |rest| in 1..2.  bf16 codes take the power along: a bf16 value times a code alone may
// pass the range where it times code and scale does not.  fp16 values have no such products, and a power of 1.  (s = 0 and
// NaN: rest is 0 and NaN.)  8 x 8192 x 8192 takes 14.6 us with it, 14.4 without.
template <class T>
__device__ __forceinline__ void split_scale(float s, float& power, float& rest) {
  power = 1.f, rest = s;
  if constexpr (__is_same(T, __bf16)) {
    const uint32_t e = __builtin_bit_cast(uint32_t, s) & 0x7f800000u;
    power = __builtin_bit_cast(float, e);
    rest = s * __builtin_bit_cast(float, (254u << 23) - e);
  }
}

// Four dwords a lane, lane group g (of 16) with dwords 4 g .. 4 g + 3 of a row's 16: afterwards with dwords g, 4 + g,
// 8 + g, 12 + g.  Halves of 32 lanes change places, then neighbouring groups.
__device__ __forceinline__ void across_groups(u32x4_t& v) {
  typedef uint32_t u2 __attribute__((ext_vector_type(2)));
  const u2 a = __builtin_amdgcn_permlane32_swap(v[0], v[2], false, false);
  const u2 b = __builtin_amdgcn_permlane32_swap(v[1], v[3], false, false);
  const u2 c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
  const u2 d = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
  v = u32x4_t{c[0], c[1], d[0], d[1]};
}

// Few token rows: the time is that of reading the codes once.  Workgroup = 16 NT weight rows and up to 16 MT token rows; its
// W waves share the reduction, each a range of its segments of 128 values.  A segment of a row is 64 bytes, 16 a lane and as
// they lie in memory; four lane swaps later lane group g has the eight values 32 m + 8 g .. that it holds in matrix
// instruction m, whose 32 values belong to one group: its sums are multiplied by the group's scale in fp32 (G instructions
// share a scale).  x comes from the caches for every workgroup anew: with NT = 2 half as often.
//
// Measured, bf16 and groups of 32, us a call among others: 8 x 8192 x 8192 14.7 (36 MB of codes and scales: 2.4 TB/s; NT = 1
// 18.5), 1 x 13.8, 32 x 23.6 (37), 64 x 39 (67); 1 x 4096 x 4096 10.0 (NT = 2 9.9: the host's time), 64 x 1024 x 4096 18.6
// (21).  8 x 8192 x 8192 with waves that take segments in turn, not ranges: 20; the loads of codes and scales alone take 10,
// with x 11, with the widening and the products of what they bring 15.
template <class T, int MT, int NT, int G, int W, int U, int XB>
__global__ __launch_bounds__(64 * W, NT == 2 ? 2 : 3) void linear_e2m1_kernel(E2m1Params p) {
  constexpr int NG = 4 / G;  // scales of a segment
  __shared__ float4_t part[W][MT * NT][64];
  const LinearParams& q = p.lin;
  const int lane = (int)threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int g = lane >> 4, r = lane & 15;
  const int ntn = (q.N + 16 * NT - 1) / (16 * NT);
  const int n0 = (int)(blockIdx.x % ntn) * (16 * NT);
  const int64_t m0 = (int64_t)(blockIdx.x / ntn) * (16 * MT);
  // rows past the end repeat the last one; what they give is not stored
  const uint8_t *wp[NT], *sp[NT], *xp[MT];
  float4_t acc[MT][NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    const int wr = n0 + 16 * i + r < q.N ? n0 + 16 * i + r : q.N - 1;
    wp[i] = q.w + (int64_t)wr * q.w_stride + g * 16;
    sp[i] = p.scale + (int64_t)wr * p.scale_stride;
  }
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    const int64_t m = m0 + 16 * t + r < q.M ? m0 + 16 * t + r : q.M - 1;
    xp[t] = q.x + m * q.x_stride + g * 16;
#pragma unroll
    for (int i = 0; i < NT; ++i) acc[t][i] = float4_t{0.f, 0.f, 0.f, 0.f};
  }
  // This wave's whole segments: neighbouring ones, so that a row's lines are its own.
  const int full = q.K / 128, per = (full + W - 1) / W;
  const int first = wave * per < full ? wave * per : full;
  const int mine = full - first < per ? full - first : per;
  const auto load16 = [](const uint8_t* a) {
    u32x4_t v;
    __builtin_memcpy(&v, a, 16);
    return v;
  };
  struct Batch {  // U segments: their codes and scales
    u32x4_t w[NT][U];
    uint32_t s[NT][U * NG / 4 > 0 ? U * NG / 4 : 1];
  };
  static_assert(U * NG % 4 == 0, "whole words of scales");
  const auto load = [&](Batch& b, int j) {  // segments j .. of the wave's
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const int64_t k = first + j;
      if (j + U <= mine) {
#pragma unroll
        for (int u = 0; u < U; ++u) b.w[i][u] = load16(wp[i] + (k + u) * 64);
        __builtin_memcpy(b.s[i], sp[i] + k * NG, U * NG);
      } else {
        uint8_t* const s = reinterpret_cast<uint8_t*>(b.s[i]);
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (j + u >= mine) break;
          b.w[i][u] = load16(wp[i] + (k + u) * 64);
          __builtin_memcpy(s + u * NG, sp[i] + (k + u) * NG, NG);
        }
      }
    }
  };
  const auto load_x = [&](u32x4_t (&v)[MT][4], int64_t k) {
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int m = 0; m < 4; ++m) v[t][m] = load16(xp[t] + k * 256 + m * 64);
  };
  const auto multiply = [&](int i, u32x4_t w, uint32_t scales, int at, const u32x4_t (&x)[MT][4]) {
    across_groups(w);
    scales >>= 8 * at;
    const float s[4] = {__builtin_amdgcn_cvt_f32_fp8(scales, 0), __builtin_amdgcn_cvt_f32_fp8(scales, 1),
                        __builtin_amdgcn_cvt_f32_fp8(scales, 2), __builtin_amdgcn_cvt_f32_fp8(scales, 3)};
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      float power, rest;
      split_scale<T>(s[n], power, rest);
      float4_t sum[MT];
#pragma unroll
      for (int t = 0; t < MT; ++t) sum[t] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int m = n * G; m < (n + 1) * G; ++m) {
        const u32x4_t b = widen_e2m1<T>(w[m], power);
#pragma unroll
        for (int t = 0; t < MT; ++t) sum[t] = mma_64b<T>(x[t][m], b, sum[t]);
      }
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[t][i][e] = __builtin_fmaf(sum[t][e], rest, acc[t][i][e]);
    }
  };
  // Codes and scales are on their way U to 2 U segments ahead of their use, x, which the caches hold, up to one.
  u32x4_t x[XB][MT][4];
  const auto use = [&](const Batch& b, int j) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (j + u >= mine) break;
      const int64_t k = first + j + u;
      if (XB == 1)
        load_x(x[0], k);
      else if (j + u + 1 < mine)
        load_x(x[(u + 1) % XB], k + 1);
#pragma unroll
      for (int i = 0; i < NT; ++i) multiply(i, b.w[i][u], b.s[i][u * NG / 4], u * NG % 4, x[u % XB]);
    }
  };
  if (mine > 0) {
    Batch b0, b1;
    load(b0, 0);
    if (XB == 2) load_x(x[0], first);
    for (int j = 0; j < mine; j += 2 * U) {
      load(b1, j + U);
      use(b0, j);
      load(b0, j + 2 * U);
      use(b1, j + U);
    }
  }
  if (q.K % 128 != 0 && wave == W - 1) {  // the reduction's tail: zeros past its end
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int m = 0; m < 4; ++m) x[0][t][m] = fetch_piece(xp[t], full * 256 + m * 64, q.kbytes - g * 16);
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      uint32_t scales = 0;
      for (int n = 0; n < NG && full * NG + n < p.groups; ++n) scales |= (uint32_t)sp[i][full * NG + n] << (8 * n);
      multiply(i, fetch_piece(wp[i], full * 64, q.K / 2 - g * 16), scales, 0, x[0]);
    }
  }
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int i = 0; i < NT; ++i) part[wave][t * NT + i][lane] = acc[t][i];
  __syncthreads();
  // A wave finishes 16 token rows of 16 columns: a lane one of them, columns 4 (lane % 4) ..  The sums lie as the matrix
  // instruction leaves them: value e of lane l is token 4 (l / 16) + e, column l % 16.
  if (wave >= MT * NT) return;
  const int row = lane >> 2, col = n0 + 16 * (wave % NT) + 4 * (lane & 3);
  const int64_t m = m0 + 16 * (wave / NT) + row;
  by_output(q, [&](auto o, auto vec) {
    using O = decltype(o);
    constexpr bool VEC = decltype(vec)::value;
    Raw<O, 4> res[1];
    linear_residual<O, VEC, 1, 1, 4>(q, m, col, res);
    Columns<F16Rows, 4> c;
    RowScales<F16Rows, 1, 1> rs;
    c.load(q, col);
    rs.load(q, m);
    float v[1][4] = {{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int w = 0; w < W; ++w)
#pragma unroll
      for (int e = 0; e < 4; ++e) v[0][e] += part[w][wave][16 * (row >> 2) + 4 * (lane & 3) + e][row & 3];
    linear_finish<F16Rows, O, VEC, 1, 1, 4>(q, m, col, v, c, rs, res);
  });
}

// s * c as 16-bit values (4096 x 8192 in 19 us, 4.2 TB/s), eight a thread, rows of `width` of them (K rounded up to 8, zeros behind K).
template <class T>
__global__ __launch_bounds__(256) void widen_e2m1_kernel(E2m1Params p, T* out, int width, int shift) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int per_row = width / 8;
  const int64_t n = i / per_row;
  if (n >= p.lin.N) return;
  const int k = (int)(i - n * per_row) * 8;
  const uint8_t* at = p.lin.w + n * p.lin.w_stride + k / 2;
  uint32_t codes = 0;
  if (p.lin.K - k >= 8) {
    __builtin_memcpy(&codes, at, 4);
  } else {
    for (int b = 0; b < (p.lin.K - k) / 2; ++b) codes |= (uint32_t)at[b] << (8 * b);
  }
  const float s = __builtin_amdgcn_cvt_f32_fp8((uint32_t)p.scale[n * p.scale_stride + (k >> shift)], 0);
  typedef T vec_t __attribute__((ext_vector_type(8)));
  vec_t v = __builtin_bit_cast(vec_t, widen_e2m1<T>(codes, 1.f));
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = (T)((float)v[e] * s);
  *reinterpret_cast<vec_t*>(out + n * width + k) = v;
}

// Whether a call with scratch memory widens the weight there and multiplies it as a 16-bit one: where the kernel above would
// take more than a round of 32 columns and 64 token rows a CU.  Measured (bf16, us; widened and not): 128 x 8192 x 8192 64 and
// 76, 256 x 4096 x 4096 32 and 41, 4000 x 384 x 384 14 and 18; 128 x 4096 x 4096 30 and 22, 1000 x 384 x 384 14 and 10; 70 x
// 8192 x 8192 56 to 60 and 56.  Rows of x that are no whole pieces of 16 bytes (or lie backwards or far apart) keep linear's
// tiles off, and the weight's way through memory pays from three times 64 rows on: 70 x 8192 x 8190 134 and 98, 128 rows 133
// and 117 (of 8192 values 8196 apart 125 and 56, 8199 apart 127 and 148), 256 rows 142 and 230, 256 x 4096 x 4094 68 and 69,
// 4000 x 384 x 390 18 and 31.
static bool widens(const LinearParams& p) {
  const bool whole = ((uintptr_t)p.x | (uintptr_t)p.kbytes | (uintptr_t)p.x_stride) % 16 == 0 && p.x_stride >= 0 &&
                     p.x_stride < 1 << 22;
  return p.M > (whole ? 64 : 128) && ((int64_t)p.N + 31) / 32 * ((p.M + 63) / 64) > 256;
}

static LinearParams widened(const E2m1Params& p, const void* weight) {
  LinearParams q = p.lin;
  q.w = static_cast<const uint8_t*>(weight);
  q.w_stride = ((int64_t)q.K + 7) / 8 * 16;
  return q;
}
static size_t widened_bytes(const LinearParams& p) { return (((size_t)p.K + 7) / 8 * 16 * p.N + 255) / 256 * 256; }

template <class T, int MT, int NT, int G, int W, int U, int XB>
static hipError_t run_rows(const E2m1Params& p, hipStream_t stream) {
  const int64_t wgs = ((int64_t)p.lin.N + 16 * NT - 1) / (16 * NT) * ((p.lin.M + 16 * MT - 1) / (16 * MT));
  if (!launchable(wgs, 64 * W)) return hipErrorInvalidConfiguration;
  linear_e2m1_kernel<T, MT, NT, G, W, U, XB><<<dim3((unsigned)wgs), dim3(64 * W), 0, stream>>>(p);
  return hipGetLastError();
}

template <class T, int MT, int G>
static hipError_t by_columns(const E2m1Params& p, hipStream_t stream) {
  // 32 weight rows a workgroup where that leaves one for every CU
  const int64_t wide = ((int64_t)p.lin.N + 31) / 32 * ((p.lin.M + 16 * MT - 1) / (16 * MT));
  if (wide >= 256) return run_rows<T, MT, 2, G, 8, 4, MT == 1 ? 2 : 1>(p, stream);
  return run_rows<T, MT, 1, G, 8, 4, MT == 1 ? 2 : 1>(p, stream);
}

template <class T, int G>
static hipError_t by_rows(const E2m1Params& p, hipStream_t stream) {
  if (p.lin.M <= 16) return by_columns<T, 1, G>(p, stream);
  if (p.lin.M <= 32) return by_columns<T, 2, G>(p, stream);
  return by_columns<T, 4, G>(p, stream);
}

template <class T>
static hipError_t run(const E2m1Params& p, int group, uint8_t* workspace, size_t bytes, hipStream_t stream) {
  if (widens(p.lin) && p.lin.K > 0 && workspace && bytes >= widened_bytes(p.lin)) {
    const int width = (p.lin.K + 7) / 8 * 8;
    const int64_t wgs = ((int64_t)p.lin.N * (width / 8) + 255) / 256;
    if (!launchable(wgs, 256)) return hipErrorInvalidConfiguration;
    widen_e2m1_kernel<T><<<dim3((unsigned)wgs), dim3(256), 0, stream>>>(
        p, reinterpret_cast<T*>(workspace), width, group == 32 ? 5 : group == 64 ? 6 : 7);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const size_t at = widened_bytes(p.lin);
    return launch_linear_scaled(widened(p, workspace), __is_same(T, _Float16),
                                reinterpret_cast<float*>(workspace + at), bytes - at, stream);
  }
  if (group == 32) return by_rows<T, 1>(p, stream);
  if (group == 64) return by_rows<T, 2>(p, stream);
  return by_rows<T, 4>(p, stream);
}

// Sizes that the kernels' counts hold, as linear's: a row of x and of the widened weight in 31 bits of bytes.
static bool sizes_fit(const sengine_linear_e2m1_desc* d) {
  return d->K <= 0x3ffffff0 && d->N <= 0x7fffff00 && d->M <= 64ll * 0x7fffffff &&
         (d->M + 15) / 16 * (((int64_t)d->N + 15) / 16) <= 0x7fffffff;
}

}  // namespace sengine

using namespace sengine;

extern "C" int sengine_amd_linear_e2m1_ws(const sengine_linear_e2m1_desc* d, const void* x, const void* weight,
                                          const void* group_scale, const float* row_scale, const void* bias,
                                          const void* residual, void* out, void* workspace, size_t workspace_bytes,
                                          hipStream_t stream) {
  if (!d) return set_error(-1, "linear_e2m1: null descriptor");
  if (d->M < 0 || d->N < 1 || d->K < 0 || d->K % 2)
    return set_error(-2, "linear_e2m1: needs M >= 0, N >= 1 and an even K >= 0");
  if (d->group != 32 && d->group != 64 && d->group != 128)
    return set_error(-2, "linear_e2m1: groups of 32, 64 or 128 values");
  if (d->in_type != SENGINE_ENC_F16 && d->in_type != SENGINE_ENC_BF16)
    return set_error(-2, "linear_e2m1: x must be fp16 or bf16");
  const auto real = [](int t) { return t == SENGINE_ENC_F16 || t == SENGINE_ENC_BF16 || t == SENGINE_ENC_F32; };
  if (!real(d->out_type)) return set_error(-2, "linear_e2m1: the output must be fp16, bf16 or fp32");
  if (bias && !real(d->bias_type)) return set_error(-2, "linear_e2m1: the bias must be fp16, bf16 or fp32");
  if (d->activation < SENGINE_ACT_NONE || d->activation > SENGINE_ACT_SILU)
    return set_error(-2, "linear_e2m1: unknown activation");
  if (!sizes_fit(d)) return set_error(-2, "linear_e2m1: sizes too large");
  if (d->M == 0) return 0;
  if (!out || (d->K > 0 && (!x || !weight || !group_scale)))
    return set_error(-1, "linear_e2m1: null x, weight, group_scale or out");
  if (d->M > 1 && d->out_stride < d->N) return set_error(-2, "linear_e2m1: output rows overlap");
  if ((uintptr_t)workspace % 16) return set_error(-2, "linear_e2m1: the workspace must be aligned to 16 bytes");
  const int o = type_bytes(d->out_type);
  E2m1Params p{};
  LinearParams& q = p.lin;
  q.x = static_cast<const uint8_t*>(x);
  q.w = static_cast<const uint8_t*>(weight);
  q.w_scale = row_scale;
  q.bias = bias;
  q.res = residual;
  q.out = out;
  q.M = d->M;
  q.x_stride = d->x_stride * 2;
  q.w_stride = d->weight_stride;
  q.res_stride = d->residual_stride;
  q.out_stride = d->out_stride;
  q.N = d->N;
  q.K = d->K;
  q.kbytes = d->K * 2;
  q.act = d->activation;
  q.out_type = d->out_type;
  q.bias_type = d->bias_type;
  const auto fits = [&](const void* a, int64_t stride) {
    return !a || ((uintptr_t)a % 16 == 0 && (stride * o % 16 == 0 || d->M == 1));
  };
  q.vec = d->N % 8 == 0 && fits(out, d->out_stride) && fits(residual, d->residual_stride);
  p.scale = static_cast<const uint8_t*>(group_scale);
  p.scale_stride = d->scale_stride;
  p.groups = (d->K + d->group - 1) / d->group;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  return (int)(d->in_type == SENGINE_ENC_F16 ? run<_Float16>(p, d->group, ws, workspace_bytes, stream)
                                             : run<__bf16>(p, d->group, ws, workspace_bytes, stream));
}

extern "C" int sengine_amd_linear_e2m1(const sengine_linear_e2m1_desc* d, const void* x, const void* weight,
                                       const void* group_scale, const float* row_scale, const void* bias,
                                       const void* residual, void* out, hipStream_t stream) {
  return sengine_amd_linear_e2m1_ws(d, x, weight, group_scale, row_scale, bias, residual, out, nullptr, 0, stream);
}

extern "C" int sengine_amd_linear_e2m1_workspace(const sengine_linear_e2m1_desc* d, size_t* bytes) {
  if (!d || !bytes) return set_error(-1, "linear_e2m1_workspace: null argument");
  *bytes = 0;
  if (d->N < 1 || d->K < 1 || !sizes_fit(d)) return 0;  // refused by the entry, or no weight
  E2m1Params p{};  // x unknown: taken to begin at a multiple of 16 bytes
  p.lin.M = d->M;
  p.lin.N = d->N;
  p.lin.K = d->K;
  p.lin.kbytes = d->K * 2;
  p.lin.x_stride = d->x_stride * 2;
  if (widens(p.lin)) *bytes = widened_bytes(p.lin) + linear_scaled_workspace(widened(p, nullptr));
  return 0;
}
