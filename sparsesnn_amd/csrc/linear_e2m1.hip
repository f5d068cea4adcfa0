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

// Eight codes of a dword as T.
template <class T>
__device__ __forceinline__ u32x4_t widen_e2m1(uint32_t v) {
  u32x4_t r;
  if constexpr (__is_same(T, _Float16)) {
    r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(v, 1.f, 0));
    r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(v, 1.f, 1));
    r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(v, 1.f, 2));
    r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(v, 1.f, 3));
  } else {
    r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(v, 1.f, 0));
    r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(v, 1.f, 1));
    r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(v, 1.f, 2));
    r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(v, 1.f, 3));
  }
  return r;
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

// Few token rows: the time is that of reading the codes once.  Workgroup = 16 weight rows and up to 16 MT token rows;
// its W waves share the reduction, wave w taking the segments of 128 values w, w + W, ..  A segment of a row is 64
// bytes, 16 a lane and as they lie in memory; four lane swaps later lane group g has the eight values 32 m + 8 g ..
// that it holds in matrix instruction m, whose 32 values belong to one group: its sums are multiplied by the group's
// scale in fp32 (G instructions share a scale).
template <class T, int MT, int G, int W, int U>
__global__ __launch_bounds__(64 * W) void linear_e2m1_kernel(E2m1Params p) {
  constexpr int NG = 4 / G;  // scales of a segment
  __shared__ float4_t part[W][MT][64];
  const LinearParams& q = p.lin;
  const int lane = (int)threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int g = lane >> 4, r = lane & 15;
  const int ntn = (q.N + 15) / 16;
  const int n0 = (int)(blockIdx.x % ntn) * 16;
  const int64_t m0 = (int64_t)(blockIdx.x / ntn) * (16 * MT);
  // rows past the end repeat the last one; what they give is not stored
  const int wr = n0 + r < q.N ? n0 + r : q.N - 1;
  const uint8_t* wp = q.w + (int64_t)wr * q.w_stride + g * 16;
  const uint8_t* sp = p.scale + (int64_t)wr * p.scale_stride;
  const uint8_t* xp[MT];
  float4_t acc[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    const int64_t m = m0 + 16 * t + r < q.M ? m0 + 16 * t + r : q.M - 1;
    xp[t] = q.x + m * q.x_stride + g * 16;
    acc[t] = float4_t{0.f, 0.f, 0.f, 0.f};
  }
  struct Batch {
    u32x4_t w[U], x[U][MT][4];
    uint32_t s[U];
  };
  const int full = q.K / 128;
  const auto load16 = [](const uint8_t* a) {
    u32x4_t v;
    __builtin_memcpy(&v, a, 16);
    return v;
  };
  const auto load = [&](Batch& b, int s) {  // the whole segments among s, s + W, ..
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t k = s + u * W;
      if (k >= full) break;
      b.w[u] = load16(wp + k * 64);
      if constexpr (NG == 4) {
        __builtin_memcpy(&b.s[u], sp + k * 4, 4);
      } else if constexpr (NG == 2) {
        uint16_t two;
        __builtin_memcpy(&two, sp + k * 2, 2);
        b.s[u] = two;
      } else {
        b.s[u] = sp[k];
      }
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int m = 0; m < 4; ++m) b.x[u][t][m] = load16(xp[t] + k * 256 + m * 64);
    }
  };
  const auto multiply = [&](u32x4_t w, uint32_t scales, const u32x4_t (&x)[MT][4]) {
    across_groups(w);
    const float s[4] = {__builtin_amdgcn_cvt_f32_fp8(scales, 0), __builtin_amdgcn_cvt_f32_fp8(scales, 1),
                        __builtin_amdgcn_cvt_f32_fp8(scales, 2), __builtin_amdgcn_cvt_f32_fp8(scales, 3)};
#pragma unroll
    for (int i = 0; i < NG; ++i) {
      float4_t sum[MT];
#pragma unroll
      for (int t = 0; t < MT; ++t) sum[t] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int m = i * G; m < (i + 1) * G; ++m) {
        const u32x4_t b = widen_e2m1<T>(w[m]);
#pragma unroll
        for (int t = 0; t < MT; ++t) sum[t] = mma_64b<T>(x[t][m], b, sum[t]);
      }
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[t][e] = __builtin_fmaf(sum[t][e], s[i], acc[t][e]);
    }
  };
  const auto use = [&](const Batch& b, int s) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (s + u * W < full) multiply(b.w[u], b.s[u], b.x[u]);
  };
  if (wave < full) {
    Batch b0, b1;
    load(b0, wave);
    for (int s = wave; s < full; s += 2 * U * W) {
      load(b1, s + U * W);
      use(b0, s);
      load(b0, s + 2 * U * W);
      use(b1, s + U * W);
    }
  }
  if (q.K % 128 != 0 && wave == full % W) {  // the reduction's tail: zeros past its end
    const u32x4_t w = fetch_piece(wp, full * 64, q.K / 2 - g * 16);
    uint32_t scales = 0;
    for (int i = 0; i < NG && full * NG + i < p.groups; ++i) scales |= (uint32_t)sp[full * NG + i] << (8 * i);
    u32x4_t x[MT][4];
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int m = 0; m < 4; ++m) x[t][m] = fetch_piece(xp[t], full * 256 + m * 64, q.kbytes - g * 16);
    multiply(w, scales, x);
  }
#pragma unroll
  for (int t = 0; t < MT; ++t) part[wave][t][lane] = acc[t];
  __syncthreads();
  // Wave t finishes token rows 16 t ..: a lane one of them, columns 4 (lane % 4) ..  The sums lie as the matrix
  // instruction leaves them: value e of lane l is token 4 (l / 16) + e, column l % 16.
  if (wave >= MT) return;
  const int row = lane >> 2, col = n0 + 4 * (lane & 3);
  const int64_t m = m0 + 16 * wave + row;
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

// s * c as 16-bit values, eight a thread, rows of `width` of them (K rounded up to 8, zeros behind K).
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
  vec_t v = __builtin_bit_cast(vec_t, widen_e2m1<T>(codes));
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = (T)((float)v[e] * s);
  *reinterpret_cast<vec_t*>(out + n * width + k) = v;
}

constexpr int64_t kE2m1Rows = 64;  // most token rows of the kernel above where there is scratch memory

static LinearParams widened(const E2m1Params& p, const void* weight) {
  LinearParams q = p.lin;
  q.w = static_cast<const uint8_t*>(weight);
  q.w_stride = ((int64_t)q.K + 7) / 8 * 16;
  return q;
}
static size_t widened_bytes(const LinearParams& p) { return (((size_t)p.K + 7) / 8 * 16 * p.N + 255) / 256 * 256; }

template <class T, int MT, int G, int W, int U>
static hipError_t run_rows(const E2m1Params& p, hipStream_t stream) {
  const int64_t wgs = ((int64_t)p.lin.N + 15) / 16 * ((p.lin.M + 16 * MT - 1) / (16 * MT));
  if (!launchable(wgs, 64 * W)) return hipErrorInvalidConfiguration;
  linear_e2m1_kernel<T, MT, G, W, U><<<dim3((unsigned)wgs), dim3(64 * W), 0, stream>>>(p);
  return hipGetLastError();
}

template <class T, int G>
static hipError_t by_rows(const E2m1Params& p, hipStream_t stream) {
  if (p.lin.M <= 16) return run_rows<T, 1, G, 8, 4>(p, stream);
  if (p.lin.M <= 32) return run_rows<T, 2, G, 8, 2>(p, stream);
  return run_rows<T, 4, G, 8, 1>(p, stream);
}

template <class T>
static hipError_t run(const E2m1Params& p, int group, uint8_t* workspace, size_t bytes, hipStream_t stream) {
  if (p.lin.M > kE2m1Rows && p.lin.K > 0 && workspace && bytes >= widened_bytes(p.lin)) {
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
  if (d->M <= kE2m1Rows || d->N < 1 || d->K < 1 || !sizes_fit(d)) return 0;  // no need, or refused by the entry
  E2m1Params p{};
  p.lin.M = d->M;
  p.lin.N = d->N;
  p.lin.K = d->K;
  p.lin.kbytes = d->K * 2;
  p.lin.x_stride = d->x_stride * 2;
  *bytes = widened_bytes(p.lin) + linear_scaled_workspace(widened(p, nullptr));
  return 0;
}
