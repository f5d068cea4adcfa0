// The linear operator for few token rows (linear.hip): the time is that of reading the weight once.
//
// Workgroup = 16 weight rows and up to 16 token rows; its W waves share the reduction, wave w taking the
// 128-byte steps w, w + W, ...  Operands go from memory straight into the matrix instructions' registers
// (a step of 16 weight rows is two loads a lane, whatever their alignment), U steps ahead of their use, and
// the waves' sums are joined in LDS.  4 x 1536 x 384 fp16: 3.9 us; 1 x 512 x 8192: 11.5 and 16 rows of it 16.5, on
// 32 workgroups; with 17 rows or more the token rows' reads take longer than the tiles' copies (32 x 4096 x 8192: 27 us,
// in tiles 18).
#pragma once
#include "linear.h"

namespace sengine {

// 16 bytes at base + k of a row of kbytes bytes: zeros past its end.
__device__ __forceinline__ u32x4_t fetch_piece(const uint8_t* base, int k, int kbytes) {
  u32x4_t v = u32x4_t{0, 0, 0, 0};
  if (k >= kbytes) return v;
  if (whole_piece(k, kbytes)) {
    __builtin_memcpy(&v, base + k, 16);
    return v;
  }
  uint32_t w[4] = {0, 0, 0, 0};
  for (int i = 0; k + i < kbytes; ++i) w[i >> 2] |= (uint32_t)base[k + i] << (8 * (i & 3));
  return u32x4_t{w[0], w[1], w[2], w[3]};
}

template <class T, int W, int U>
__global__ __launch_bounds__(64 * W) void linear_rows_kernel(LinearParams p) {
  __shared__ float4_t part[W][64];
  const int lane = (int)threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int g = lane >> 4, r = lane & 15;
  const int n0 = (int)blockIdx.x * 16;
  // rows past the end repeat the last one; what they give is not stored
  const int wr = n0 + r < p.N ? n0 + r : p.N - 1;
  const uint8_t* wp = p.w + (int64_t)wr * p.w_stride + g * 16;
  const uint8_t* xp = p.x + (r < p.M ? r : p.M - 1) * p.x_stride + g * 16;
  float4_t acc = float4_t{0.f, 0.f, 0.f, 0.f};
  struct Batch {
    u32x4_t w[U][2], x[U][2];
  };
  const int full = p.kbytes / 128;
  const auto load16 = [](const uint8_t* q) {
    u32x4_t v;
    __builtin_memcpy(&v, q, 16);
    return v;
  };
  const auto load = [&](Batch& b, int s) {  // the whole steps among s, s + W, ..
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (s + u * W >= full) break;
      const int64_t k = (int64_t)(s + u * W) * 128;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        b.w[u][h] = load16(wp + k + 64 * h);
        b.x[u][h] = load16(xp + k + 64 * h);
      }
    }
  };
  const auto use = [&](const Batch& b, int s) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (s + u * W < full) acc = mma_128b<T>(b.w[u][0], b.w[u][1], b.x[u][0], b.x[u][1], acc);
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
  if (p.kbytes % 128 != 0 && wave == full % W) {  // the reduction's tail
    const int k = full * 128, kb = p.kbytes - g * 16;
    acc = mma_128b<T>(fetch_piece(wp, k, kb), fetch_piece(wp, k + 64, kb), fetch_piece(xp, k, kb),
                      fetch_piece(xp, k + 64, kb), acc);
  }
  part[wave][lane] = acc;
  __syncthreads();
  if (wave > 0) return;
  // the first wave finishes token row lane % 16, columns 4 (lane / 16) ..
  const int col = n0 + 4 * g;
  by_output(p, [&](auto o, auto vec) {
    using O = decltype(o);
    constexpr bool VEC = decltype(vec)::value;
    Raw<O, 4> res[1];
    linear_residual<O, VEC, 1, 1, 4>(p, r, col, res);
    Columns<T, 4> c;
    RowScales<T, 1, 1> rs;
    c.load(p, col);
    rs.load(p, r);
    float4_t sum = part[0][lane];
#pragma unroll
    for (int w = 1; w < W; ++w) sum += part[w][lane];
    float v[1][4] = {{sum[0], sum[1], sum[2], sum[3]}};
    linear_finish<T, O, VEC, 1, 1, 4>(p, r, col, v, c, rs, res);
  });
}

}  // namespace sengine
