// Matrix product of token rows with a weight in nn.Linear's layout, everything after it in the
// epilogue:
//   y[m, n] = act(cx[m] cw[n] sum_k x[m, k] w[n, k] + b[n]) + r[m, n]
// x and w are both fp16, both bf16 (cx = cw = 1) or both e4m3 with fp32 scales per row.  The sum and
// the epilogue are fp32 and y is rounded once.
#include "linear_rows.h"
#include "linear_tile.h"

namespace sengine {

// Any strides, any alignment, any K: 8192 x 4096 x 8191 bf16 1410 us (8192 wide 424), since nothing is in flight during
// the products and the tile is 64 x 64; one operand whose rows are no whole pieces brings a call here.  Workgroup =
// 64 rows x 64 columns, four waves of 32 x 32; per 128 bytes of the reduction both operands' rows go through registers
// into LDS: whole 16-byte pieces by one load of whatever alignment, the row's last piece byte by byte, zeros beyond.
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
  for (uint32_t at = 0; has_step(at, p.kbytes); at = next_step(at)) {
    const int k = (int)at;
    u32x4_t xv[2], wv[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = row + 32 * h;
      xv[h] = fetch_piece(p.x + (m0 + r) * p.x_stride, k + piece, m0 + r < p.M ? p.kbytes : 0);
      wv[h] = fetch_piece(p.w + (int64_t)(n0 + r) * p.w_stride, k + piece, n0 + r < p.N ? p.kbytes : 0);
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
        // the epilogue's columns: fragment i's row 4 g + e is weight row 8 g + 4 i + e
        const int wr = wn + 8 * ((lane >> 2) & 3) + 4 * i + (lane & 3);
        a[i][h] = *reinterpret_cast<const u32x4_t*>(sW + wr * kLinPitch + at);
        b[i][h] = *reinterpret_cast<const u32x4_t*>(sX + (wm + 16 * i + (lane & 15)) * kLinPitch + at);
      }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) acc[i][j] = mma_128b<T>(a[i][0], a[i][1], b[j][0], b[j][1], acc[i][j]);
  }
  Columns<T, 8> cols[1];
  RowScales<T, 2, 16> rscales;
  cols[0].load(p, n0 + wn + 8 * (lane >> 4));
  rscales.load(p, m0 + wm + (lane & 15));
  linear_epilogue<T, 2, 2>(p, m0 + wm + (lane & 15), n0 + wn + 8 * (lane >> 4), acc, cols, rscales);
}

template <class T, int BM, int BN, int WM, int WN, int S, int WGS>
static hipError_t run_tile(const LinearParams& p, int parts, hipStream_t stream) {
  const int64_t ntm = (p.M + BM - 1) / BM, ntn = (p.N + BN - 1) / BN;
  if (!launchable(ntm * ntn, 64 * WM * WN)) return hipErrorInvalidConfiguration;
  linear_tile_kernel<T, BM, BN, WM, WN, S, WGS>
      <<<dim3((unsigned)(ntm * ntn), (unsigned)parts), dim3(64 * WM * WN), 0, stream>>>(p, (int)ntm, (int)ntn);
  return hipGetLastError();
}

// Which kernel, and in how many parts.  Measured (bf16, us a call among others, the kernels as they stand here):
//   up to 16 token rows     4 x 1536 x 384: rows 8.6 (64 x 64 tiles: 8.6; the kernels alone 3.2 and 4.8), 1 x 512 x
//                           8192: 11.3 (tiles in parts: 12.5; alone 11.5 and 8.4).  Few columns of a long reduction
//                           are where the rule is not the faster side any more: 16 x 512 x 8192: 16.7 (12.8)
//   256 x 256 tiles, if there is one for every CU and 8 steps: 4096 x 4096 x 512: 26 (128: 28), x 4096: 104 (120);
//                           with 6 steps, x 384 and GELU on 100352 x 1536: 253 (216)
//   128 x 128 tiles, if there is one for every CU: 2048 x 2048 x 1024: 15 (64: 19); 3001 x 1000 x 1552: 23 (24);
//                           1024 x 1024 x 1024: 10.6 (7.9)
//   64 x 64 tiles otherwise, in parts of 12 steps or more up to two workgroups a CU, where the reduction has 48
//                           steps: 32 x 4096 x 8192: 17.6 (in one: 33), x 512: 12.5 (30); 64 x 512 x 2048: 14.6 (10)
enum { kLinAny, kLinRows, kLin64, kLin128, kLin256 };
struct LinearPlan {
  int kernel, parts, part_steps;
};

static int64_t tiles_of(const LinearParams& p, int b) { return (p.M + b - 1) / b * (((int64_t)p.N + b - 1) / b); }

// Sizes that the kernels' counts hold: a row in 31 bits of bytes, a column in 31 bits up to the end of its tile, the
// 64 x 64 tiles in 31 bits.
static bool sizes_fit(const sengine_linear_desc* d) {
  return d->K <= 0x3fffffff && d->N <= 0x7fffff00 && d->M <= 64ll * 0x7fffffff &&
         (d->M + 63) / 64 * (((int64_t)d->N + 63) / 64) <= 0x7fffffff;
}

static LinearPlan plan(const LinearParams& p, bool wide) {
  constexpr int kCUs = 256;
  const int steps = p.kbytes / kLinStep + (p.kbytes % kLinStep != 0);
  if (p.M <= 16) return {kLinRows, 1, 0};
  // LDS copies: whole 16-byte pieces, offsets inside a tile in 31 bits and from its first row on (rows may lie
  // backwards in memory: the other kernels take any stride)
  const auto near = [](int64_t stride) { return stride >= 0 && stride < 1 << 22; };
  const bool copies = p.kbytes % 16 == 0 && p.x_stride % 16 == 0 && p.w_stride % 16 == 0 &&
                      (uintptr_t)p.x % 16 == 0 && (uintptr_t)p.w % 16 == 0 && p.kbytes < (1 << 29) &&
                      near(p.x_stride) && near(p.w_stride);
  if (!copies) return {kLinAny, 1, 0};
  if (!wide && tiles_of(p, 256) >= kCUs && steps >= 8) return {kLin256, 1, 0};
  if (tiles_of(p, 128) >= kCUs) return {kLin128, 1, 0};
  const int64_t most = 2 * kCUs / tiles_of(p, 64);
  const int parts = (int)(most < steps / 12 ? most : steps / 12);
  if (steps < 48 || parts < 2) return {kLin64, 1, 0};
  const int part_steps = (steps + parts - 1) / parts;
  return {kLin64, (steps + part_steps - 1) / part_steps, part_steps};
}

template <class T>
static hipError_t run(LinearParams p, float* workspace, size_t bytes, hipStream_t stream) {
  const LinearPlan q = plan(p, __is_same(T, E4m3Wide));
  switch (q.kernel) {
    case kLinRows:
      if (!launchable((p.N + 15) / 16, 512)) return hipErrorInvalidConfiguration;
      linear_rows_kernel<T, 8, 4><<<dim3((unsigned)((p.N + 15) / 16)), dim3(512), 0, stream>>>(p);
      return hipGetLastError();
    case kLin64: {
      const int64_t tiles = tiles_of(p, 64);
      if (q.parts > 1 && workspace && bytes >= (size_t)(q.parts * tiles) * 64 * 64 * 4) {
        p.partial = workspace;
        p.part_steps = q.part_steps;
        const hipError_t rc = run_tile<T, 64, 64, 2, 2, 3, 3>(p, q.parts, stream);
        if (rc != hipSuccess) return rc;
        linear_join_kernel<T>
            <<<dim3((unsigned)(tiles * 8)), dim3(64), 0, stream>>>(p, (p.N + 63) / 64, (int)tiles, q.parts);
        return hipGetLastError();
      }
      return run_tile<T, 64, 64, 2, 2, 3, 3>(p, 1, stream);
    }
    case kLin128:
      return run_tile<T, 128, 128, 2, 2, 2, 2>(p, 1, stream);
    case kLin256:
      if constexpr (!__is_same(T, E4m3Wide)) return run_tile<T, 256, 256, 2, 2, 2, 1>(p, 1, stream);
      [[fallthrough]];
    default:
      if (!launchable(tiles_of(p, 64), 256)) return hipErrorInvalidConfiguration;
      linear_any_kernel<T><<<dim3((unsigned)tiles_of(p, 64)), dim3(256), 0, stream>>>(p);
      return hipGetLastError();
  }
}

}  // namespace sengine

using namespace sengine;

extern "C" int sengine_amd_linear_ws(const sengine_linear_desc* d, const void* x, const void* weight,
                                     const float* x_scale, const float* weight_scale, const void* bias,
                                     const void* residual, void* out, void* workspace, size_t workspace_bytes,
                                     hipStream_t stream) {
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
  if (!sizes_fit(d)) return set_error(-2, "linear: sizes too large");
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
    return !a || ((uintptr_t)a % 16 == 0 && (stride * o % 16 == 0 || d->M == 1));
  };
  p.vec = d->N % 8 == 0 && fits(out, d->out_stride) && fits(residual, d->residual_stride);
  if ((uintptr_t)workspace % 16) return set_error(-2, "linear: the workspace must be aligned to 16 bytes");
  float* ws = static_cast<float*>(workspace);
  hipError_t rc;
  if (e4m3)
    rc = d->out_type == SENGINE_ENC_F32 ? run<E4m3Wide>(p, ws, workspace_bytes, stream)
                                        : run<E4m3>(p, ws, workspace_bytes, stream);
  else if (d->in_type == SENGINE_ENC_F16)
    rc = run<_Float16>(p, ws, workspace_bytes, stream);
  else
    rc = run<__bf16>(p, ws, workspace_bytes, stream);
  return (int)rc;
}

extern "C" int sengine_amd_linear(const sengine_linear_desc* d, const void* x, const void* weight,
                                  const float* x_scale, const float* weight_scale, const void* bias,
                                  const void* residual, void* out, hipStream_t stream) {
  return sengine_amd_linear_ws(d, x, weight, x_scale, weight_scale, bias, residual, out, nullptr, 0, stream);
}

extern "C" int sengine_amd_linear_workspace(const sengine_linear_desc* d, size_t* bytes) {
  if (!d || !bytes) return set_error(-1, "linear_workspace: null argument");
  *bytes = 0;
  if (d->M < 1 || d->N < 1 || d->K < 1 || !sizes_fit(d)) return 0;  // nothing to do, or refused by the entry
  const int e = type_bytes(d->in_type);
  LinearParams p{};
  p.M = d->M;
  p.N = d->N;
  p.kbytes = d->K * e;
  p.x_stride = d->x_stride * e;
  p.w_stride = d->weight_stride * e;
  const LinearPlan q = plan(p, d->in_type == SENGINE_ENC_E4M3 && d->out_type == SENGINE_ENC_F32);
  if (q.parts > 1) *bytes = (size_t)(q.parts * tiles_of(p, 64)) * 64 * 64 * 4;
  return 0;
}
