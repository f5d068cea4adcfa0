// Root-mean-square norm of token rows with the residual's addition:
//   s = x + r              (stored, rounded once, as the new stream when the caller wants it)
//   y = s / sqrt(mean(s^2) + eps) * w
// y is stored in x's type, or as e4m3 codes q with one fp32 scale c a row, y ~ q * c:
//   c = max |y| / 448, at least 2^-126 (1 for a row of zeros), q = e4m3(y / c).
// s, the sum of squares and y are fp32; y is rounded once, when it is stored.
//
// Bandwidth bound: x and r are read once and y and s written once, because a row stays in
// registers: L lanes hold a row, NV pieces of VEC elements each, and the sum of squares and the
// largest |y| are reduced over those L lanes (in the order of a butterfly, the same every time).
// 401408 x 384 fp16 with a residual to e4m3: 197 us, 5.5 TB/s (a copy of 2 GB reaches 4.9); 4 x 384: 3.0 us.  With a
// residual, fp32 100000 x 384: 108 us (5.7 TB/s), to e4m3 91; fp16 16384 x 16384: 360 (6.0), fp32 8192 x 32768: 798
// (5.4).  Narrow rows leave lanes idle: fp16 400000 x 64: 45 (4.5 TB/s), x 8: 28 (0.9).
#include "token_types.h"

namespace sengine {

struct RmsParams {
  const void* x;
  const void* res;     // or null
  const void* w;       // or null
  void* out;
  void* stream;        // s in x's type, or null
  float* scale;        // e4m3 output
  int64_t rows, x_stride, res_stride, out_stride, stream_stride;  // strides in elements
  int D, w_type;
  float eps;
};

// Sum / largest over L lanes.  The largest |y| is taken over the bit patterns: those of
// non-negative floats order as the floats do, with infinity and NaN on top, so a NaN survives.
template <int L>
struct RowReduce {
  static __device__ __forceinline__ float sum(float v, float* lds) {
#pragma unroll
    for (int o = (L < 64 ? L : 64) / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    if constexpr (L > 64) {
      if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
      __syncthreads();
      v = lds[0];
#pragma unroll
      for (int i = 1; i < L / 64; ++i) v += lds[i];
      __syncthreads();
    }
    return v;
  }
  static __device__ __forceinline__ uint32_t largest(uint32_t v, float* lds) {
#pragma unroll
    for (int o = (L < 64 ? L : 64) / 2; o > 0; o >>= 1) {
      const uint32_t u = __shfl_xor(v, o, 64);
      v = u > v ? u : v;
    }
    if constexpr (L > 64) {
      uint32_t* l = reinterpret_cast<uint32_t*>(lds);
      if ((threadIdx.x & 63) == 0) l[threadIdx.x >> 6] = v;
      __syncthreads();
      v = l[0];
#pragma unroll
      for (int i = 1; i < L / 64; ++i) v = l[i] > v ? l[i] : v;
      __syncthreads();
    }
    return v;
  }
};

// N values at p as floats, of which `left` are there; zeros beyond.  WHOLE: all are, at a multiple of their size;
// otherwise a whole piece is still one access, of whatever alignment.
template <bool WHOLE, class T, int N>
__device__ __forceinline__ void load_piece(const T* p, int left, float (&v)[N]) {
  if constexpr (WHOLE) {
    load_floats<T, N>(p, v);
  } else if (left >= N) {
    typedef T vec_t __attribute__((ext_vector_type(N), aligned(sizeof(T))));
    const vec_t x = *reinterpret_cast<const vec_t*>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (float)x[i];
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = i < left ? (float)p[i] : 0.f;
  }
}

template <bool WHOLE, class T, int N>
__device__ __forceinline__ void store_piece(T* p, int left, const float (&v)[N]) {
  if constexpr (WHOLE) {
    store_floats(p, v);
  } else {
    alignas(16) T x[N];
    store_floats(x, v);
    if (left >= N) {
      __builtin_memcpy(p, x, sizeof(x));
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (i < left) p[i] = x[i];
    }
  }
}

template <class T, class OUT, int L, int NV, int VEC, bool WHOLE>
__global__ __launch_bounds__(L < 256 ? 256 : L) void rms_norm_kernel(RmsParams p) {
  constexpr int NTH = L < 256 ? 256 : L;
  __shared__ float lds[L > 64 ? L / 64 : 1];
  const int64_t row = (int64_t)blockIdx.x * (NTH / L) + threadIdx.x / L;
  if (L <= 64 && row >= p.rows) return;  // L > 64: one row a workgroup, the grid has p.rows of them
  const int lane = (int)threadIdx.x % L;
  const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
  const T* res = static_cast<const T*>(p.res) + row * p.res_stride;
  float v[NV][VEC];
  float ss = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int at = (j * L + lane) * VEC;
    if (at < p.D) {
      load_piece<WHOLE>(x + at, p.D - at, v[j]);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[j][i] = 0.f;
    }
  }
  if (p.res) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int at = (j * L + lane) * VEC;
      if (at < p.D) {
        float r[VEC];
        load_piece<WHOLE>(res + at, p.D - at, r);
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[j][i] += r[i];
      }
    }
  }
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < VEC; ++i) ss = __builtin_fmaf(v[j][i], v[j][i], ss);
  ss = RowReduce<L>::sum(ss, lds);
  if (p.stream) {
    T* st = static_cast<T*>(p.stream) + row * p.stream_stride;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int at = (j * L + lane) * VEC;
      if (at < p.D) store_piece<WHOLE>(st + at, p.D - at, v[j]);
    }
  }
  const float rstd = 1.0f / sqrtf(ss / (float)p.D + p.eps);
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int at = (j * L + lane) * VEC;
    if (at < p.D) {
      float w[VEC];
      if (!p.w) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) w[i] = 1.f;
      } else if (p.w_type == SENGINE_ENC_F32) {
        load_piece<WHOLE>(static_cast<const float*>(p.w) + at, p.D - at, w);
      } else {
        load_piece<WHOLE>(static_cast<const T*>(p.w) + at, p.D - at, w);
      }
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        v[j][i] = v[j][i] * rstd * w[i];
        const uint32_t b = __builtin_bit_cast(uint32_t, v[j][i]) & 0x7fffffffu;
        top = b > top ? b : top;
      }
    }
  }
  if constexpr (__is_same(OUT, E4m3)) {
    top = RowReduce<L>::largest(top, lds);
    // a quotient below the normal numbers has lost bits, or all of them: codes of the smallest normal scale instead
    constexpr float kLeast = 1.17549435e-38f;
    const float quotient = __builtin_bit_cast(float, top) / 448.f;
    const float c = top == 0 ? 1.f : quotient < kLeast ? kLeast : quotient;  // a NaN stays
    if (lane == 0) p.scale[row] = c;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[j][i] = v[j][i] / c;
  }
  OUT* out = static_cast<OUT*>(p.out) + row * p.out_stride;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int at = (j * L + lane) * VEC;
    if (at < p.D) store_piece<WHOLE>(out + at, p.D - at, v[j]);
  }
}

// A launch holds fewer than 2^32 threads: 2^28 rows of 16 lanes and more go in several.
constexpr int64_t kRmsThreads = 1ll << 31;  // of a launch

template <class T, class OUT, int L, int NV, bool WHOLE>
static hipError_t run(RmsParams p, hipStream_t stream) {
  constexpr int NTH = L < 256 ? 256 : L, VEC = 16 / (int)sizeof(T);
  constexpr int64_t kMost = kRmsThreads / L;  // rows of a launch
  const int64_t rows = p.rows;
  for (int64_t first = 0; first < rows; first += kMost) {
    p.rows = rows - first < kMost ? rows - first : kMost;
    const int64_t wgs = (p.rows + NTH / L - 1) / (NTH / L);
    rms_norm_kernel<T, OUT, L, NV, VEC, WHOLE><<<dim3((unsigned)wgs), dim3(NTH), 0, stream>>>(p);
    const hipError_t rc = hipGetLastError();
    if (rc != hipSuccess) return rc;
    p.x = static_cast<const T*>(p.x) + kMost * p.x_stride;
    if (p.res) p.res = static_cast<const T*>(p.res) + kMost * p.res_stride;
    if (p.stream) p.stream = static_cast<T*>(p.stream) + kMost * p.stream_stride;
    p.out = static_cast<OUT*>(p.out) + kMost * p.out_stride;
    if (p.scale) p.scale += kMost;
  }
  return hipSuccess;
}

// Lanes per row by the pieces of 16 bytes a row has: 16 lanes for up to 64 pieces (four rows a wave: a 384-wide
// 16-bit row is 48 pieces, 3 a lane with none idle), a wave up to 256, then a workgroup.
template <class T, class OUT, bool WHOLE>
static hipError_t by_width(const RmsParams& p, hipStream_t stream) {
  constexpr int VEC = 16 / (int)sizeof(T);
  const int n = (p.D + VEC - 1) / VEC;
  if (n <= 16) return run<T, OUT, 16, 1, WHOLE>(p, stream);
  if (n <= 32) return run<T, OUT, 16, 2, WHOLE>(p, stream);
  if (n <= 48) return run<T, OUT, 16, 3, WHOLE>(p, stream);
  if (n <= 64) return run<T, OUT, 16, 4, WHOLE>(p, stream);
  if (n <= 128) return run<T, OUT, 64, 2, WHOLE>(p, stream);
  if (n <= 192) return run<T, OUT, 64, 3, WHOLE>(p, stream);
  if (n <= 256) return run<T, OUT, 64, 4, WHOLE>(p, stream);
  if (n <= 512) return run<T, OUT, 256, 2, WHOLE>(p, stream);
  if (n <= 1024) return run<T, OUT, 256, 4, WHOLE>(p, stream);
  if (n <= 4096) return run<T, OUT, 1024, 4, WHOLE>(p, stream);
  if constexpr (VEC == 4) return run<T, OUT, 1024, 8, WHOLE>(p, stream);
  return hipErrorInvalidValue;  // not reached: D <= kRmsMaxD
}

constexpr int kRmsMaxD = 32768;

// Whole aligned pieces where every row of every array begins at a multiple of its piece and D is whole pieces.
// Otherwise (bf16, 43984 x 1445 with a residual: 118 us, element by element 358) a row's pieces begin anywhere and
// its last may be short.
template <class T, class OUT>
static hipError_t by_alignment(const RmsParams& p, hipStream_t stream) {
  constexpr int VEC = 16 / (int)sizeof(T);
  const auto fits = [&](const void* a, int64_t stride, size_t bytes) {
    return !a || ((uintptr_t)a % (bytes * VEC) == 0 && (stride % VEC == 0 || p.rows == 1));
  };
  const size_t e = sizeof(T);
  if (p.D % VEC == 0 && fits(p.x, p.x_stride, e) && fits(p.res, p.res_stride, e) &&
      fits(p.stream, p.stream_stride, e) && fits(p.out, p.out_stride, sizeof(OUT)) &&
      fits(p.w, 0, 16 / VEC))
    return by_width<T, OUT, true>(p, stream);
  return by_width<T, OUT, false>(p, stream);
}

template <class T>
static hipError_t by_output(const RmsParams& p, int out_type, hipStream_t stream) {
  return out_type == SENGINE_ENC_E4M3 ? by_alignment<T, E4m3>(p, stream) : by_alignment<T, T>(p, stream);
}

}  // namespace sengine

using namespace sengine;

extern "C" int sengine_amd_rms_norm(const sengine_rms_norm_desc* d, const void* x, const void* residual,
                                    const void* weight, void* out, void* stream_out, float* scale,
                                    hipStream_t stream) {
  if (!d) return set_error(-1, "rms_norm: null descriptor");
  if (d->rows < 0 || d->D < 1 || d->D > kRmsMaxD)
    return set_error(-2, "rms_norm: needs rows >= 0 and 1 <= D <= 32768");
  if (d->rows > 0x7fffffffll) return set_error(-2, "rms_norm: more than 2^31 - 1 rows");
  if (d->in_type != SENGINE_ENC_F16 && d->in_type != SENGINE_ENC_BF16 && d->in_type != SENGINE_ENC_F32)
    return set_error(-2, "rms_norm: x must be fp16, bf16 or fp32");
  if (d->out_type != d->in_type && d->out_type != SENGINE_ENC_E4M3)
    return set_error(-2, "rms_norm: the output has x's type or e4m3");
  if (weight && d->weight_type != d->in_type && d->weight_type != SENGINE_ENC_F32)
    return set_error(-2, "rms_norm: the weight has x's type or fp32");
  if (!(d->eps >= 0.f)) return set_error(-2, "rms_norm: eps must be >= 0");
  if (d->rows == 0) return 0;
  if (!x || !out) return set_error(-1, "rms_norm: null x or out");
  if (d->out_type == SENGINE_ENC_E4M3 && !scale) return set_error(-1, "rms_norm: e4m3 output needs scale");
  if (d->rows > 1 && (d->out_stride < d->D || (stream_out && d->stream_stride < d->D)))
    return set_error(-2, "rms_norm: output rows overlap");
  const RmsParams p{x,           residual,      weight,           out,  stream_out,     scale,  d->rows, d->x_stride,
                    d->residual_stride, d->out_stride, d->stream_stride, d->D, d->weight_type, d->eps};
  hipError_t e;
  if (d->in_type == SENGINE_ENC_F16)
    e = by_output<_Float16>(p, d->out_type, stream);
  else if (d->in_type == SENGINE_ENC_BF16)
    e = by_output<__bf16>(p, d->out_type, stream);
  else
    e = by_output<float>(p, d->out_type, stream);
  return (int)e;
}
