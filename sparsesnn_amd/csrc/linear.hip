// Matrix product of token rows with a weight in nn.Linear's layout, everything after it in the
// epilogue:
//   y[m, n] = act(cx[m] cw[n] sum_k x[m, k] w[n, k] + b[n]) + r[m, n]
// x and w are both fp16, both bf16 (cx = cw = 1) or both e4m3 with fp32 scales per row.  The sum and
// the epilogue are fp32 and y is rounded once.
#include "linear.h"

namespace sengine {

// Any strides, any alignment, any K.  Workgroup = 64 rows x 64 columns, four waves of 32 x 32; per
// 128 bytes of the reduction both operands' rows go through registers into LDS: whole 16-byte pieces
// by one load of whatever alignment, the row's last piece byte by byte, zeros beyond.
constexpr int kLinStep = 128;        // bytes of the reduction a step
constexpr int kLinPitch = 128 + 16;  // LDS row: 16 bytes more, so that 16 rows' pieces spread over the banks

template <class T>
__global__ __launch_bounds__(256) void linear_any_kernel(LinearParams p) {
  __shared__ __attribute__((aligned(16))) uint8_t sX[64 * kLinPitch], sW[64 * kLinPitch];
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int ntn = (p.N + 63) / 64;
  const int64_t m0 = (int64_t)(blockIdx.x / ntn) * 64;
  const int n0 = (int)(blockIdx.x % ntn) * 64;
  const int wm = (wave >> 1) * 32, wn = (wave & 1) * 32;
  float4_t acc[2][2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) acc[i][j] = float4_t{0.f, 0.f, 0.f, 0.f};

  const int row = tid >> 3, piece = (tid & 7) * 16;  // rows row and row + 32 of each operand
  const auto fetch = [&](const uint8_t* base, bool valid, int k) {
    u32x4_t v = u32x4_t{0, 0, 0, 0};
    if (!valid || k >= p.kbytes) return v;
    if (k + 16 <= p.kbytes) {
      __builtin_memcpy(&v, base + k, 16);
      return v;
    }
    uint32_t w[4] = {0, 0, 0, 0};
    for (int i = 0; k + i < p.kbytes; ++i) w[i >> 2] |= (uint32_t)base[k + i] << (8 * (i & 3));
    return u32x4_t{w[0], w[1], w[2], w[3]};
  };
  for (int k = 0; k < p.kbytes; k += kLinStep) {
    u32x4_t xv[2], wv[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = row + 32 * h;
      xv[h] = fetch(p.x + (m0 + r) * p.x_stride, m0 + r < p.M, k + piece);
      wv[h] = fetch(p.w + (int64_t)(n0 + r) * p.w_stride, n0 + r < p.N, k + piece);
    }
    __syncthreads();  // the previous step's reads are done
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      *reinterpret_cast<u32x4_t*>(sX + (row + 32 * h) * kLinPitch + piece) = xv[h];
      *reinterpret_cast<u32x4_t*>(sW + (row + 32 * h) * kLinPitch + piece) = wv[h];
    }
    __syncthreads();
    u32x4_t a[2][2], b[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int at = 64 * h + (lane >> 4) * 16;
        a[i][h] = *reinterpret_cast<const u32x4_t*>(sW + (wn + 16 * i + (lane & 15)) * kLinPitch + at);
        b[i][h] = *reinterpret_cast<const u32x4_t*>(sX + (wm + 16 * i + (lane & 15)) * kLinPitch + at);
      }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) acc[i][j] = mma_128b<T>(a[i][0], a[i][1], b[j][0], b[j][1], acc[i][j]);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
      linear_store4(p, m0 + wm + 16 * j + (lane & 15), n0 + wn + 16 * i + 4 * (lane >> 4), acc[i][j]);
}

template <class T>
static hipError_t run(const LinearParams& p, hipStream_t stream) {
  const int64_t wgs = (p.M + 63) / 64 * ((p.N + 63) / 64);
  if (wgs > 0x7fffffffll) return hipErrorInvalidValue;
  linear_any_kernel<T><<<dim3((unsigned)wgs), dim3(256), 0, stream>>>(p);
  return hipGetLastError();
}

}  // namespace sengine

using namespace sengine;

extern "C" int sengine_amd_linear(const sengine_linear_desc* d, const void* x, const void* weight,
                                  const float* x_scale, const float* weight_scale, const void* bias,
                                  const void* residual, void* out, hipStream_t stream) {
  if (!d) return set_error(-1, "linear: null descriptor");
  if (d->M < 0 || d->N < 1 || d->K < 0) return set_error(-2, "linear: needs M >= 0, N >= 1, K >= 0");
  const bool e4m3 = d->in_type == SENGINE_ENC_E4M3;
  if (d->in_type != SENGINE_ENC_F16 && d->in_type != SENGINE_ENC_BF16 && !e4m3)
    return set_error(-2, "linear: x and weight must be fp16, bf16 or e4m3");
  const auto real = [](int t) { return t == SENGINE_ENC_F16 || t == SENGINE_ENC_BF16 || t == SENGINE_ENC_F32; };
  if (!real(d->out_type)) return set_error(-2, "linear: the output must be fp16, bf16 or fp32");
  if (bias && !real(d->bias_type)) return set_error(-2, "linear: the bias must be fp16, bf16 or fp32");
  if (d->activation < SENGINE_ACT_NONE || d->activation > SENGINE_ACT_SILU)
    return set_error(-2, "linear: unknown activation");
  if (!e4m3 && (x_scale || weight_scale)) return set_error(-2, "linear: scales go with e4m3 operands only");
  const int64_t mtiles = (d->M + 63) / 64, ntiles = ((int64_t)d->N + 63) / 64;
  if (d->K > 0x3fffffff || mtiles * ntiles > 0x7fffffffll) return set_error(-2, "linear: sizes too large");
  if (d->M == 0) return 0;
  if (!out || (d->K > 0 && (!x || !weight))) return set_error(-1, "linear: null x, weight or out");
  if (d->M > 1 && d->out_stride < d->N) return set_error(-2, "linear: output rows overlap");
  const int e = type_bytes(d->in_type), o = type_bytes(d->out_type);
  LinearParams p{};
  p.x = static_cast<const uint8_t*>(x);
  p.w = static_cast<const uint8_t*>(weight);
  p.x_scale = x_scale;
  p.w_scale = weight_scale;
  p.bias = bias;
  p.res = residual;
  p.out = out;
  p.M = d->M;
  p.x_stride = d->x_stride * e;
  p.w_stride = d->weight_stride * e;
  p.res_stride = d->residual_stride;
  p.out_stride = d->out_stride;
  p.N = d->N;
  p.K = d->K;
  p.kbytes = d->K * e;
  p.act = d->activation;
  p.out_type = d->out_type;
  p.bias_type = d->bias_type;
  const auto fits = [&](const void* a, int64_t stride) {
    return !a || ((uintptr_t)a % (4 * o) == 0 && (stride % 4 == 0 || d->M == 1));
  };
  p.vec = fits(out, d->out_stride) && fits(residual, d->residual_stride);
  hipError_t rc;
  if (e4m3)
    rc = d->out_type == SENGINE_ENC_F32 ? run<E4m3Wide>(p, stream) : run<E4m3>(p, stream);
  else if (d->in_type == SENGINE_ENC_F16)
    rc = run<_Float16>(p, stream);
  else
    rc = run<__bf16>(p, stream);
  return (int)rc;
}
