// Rotary positions with several axes: each pair (x0, x1) of a head's first 2 P values turns by its token's position on
// the pair's axis,
//   angle = position[token, axis(j)] * frequency[j],   (x0, x1) -> (x0 cos - x1 sin, x0 sin + x1 cos),
// and the values behind them are copied.  Pair j is (x[j], x[P + j]), or (x[2 j], x[2 j + 1]).  The angle is formed and
// reduced to half a turn either way in 64 bits (a position of 10^6 at a radian a step has lost 16 bits of its turn in
// 32), its sine and cosine and the products are fp32, and a result is rounded once.
//
// Bandwidth bound: queries and keys are read and written once, in one launch.  32768 tokens x 40 heads x 128 bf16, neighbouring
// pairs: 118 us (5.7 TB/s; two items a thread in flight 123), pairs P apart 126 (one item 129).  8 x 12544 tokens x 16 heads x
// 48 fp16, pairs P apart: 64 to 69 us (4.5 to 4.8 TB/s; two half lines an access), neighbouring 53; workgroups of twice the
// tokens 69 for 64, of four times 76.  The same in fp32 133 and 115 us (4.6, 5.4 TB/s).  A single token: 3.2 us.
//
// A workgroup takes a few tokens: their sines and cosines, which all heads share, go to LDS; then its threads go through
// the tokens' pieces of VEC values in the order in which they lie in memory.  With a head or two the angles are the time: 62 x
// 8930 tokens of two heads x 32 fp16, 16 pairs, 44 us of the 28 that the bytes take.
#include "token_types.h"

namespace sengine {

struct RotaryParams {
  const void* x[2];  // queries, keys
  void* out[2];
  int64_t x_b[2], x_l[2], x_h[2], o_b[2], o_l[2], o_h[2];  // strides in elements
  const void* pos;
  const float* freq;
  int64_t pos_b, pos_l, tokens;
  int L, Hq, pairs, ends[3];  // ends: the first pair of axes 1, 2, 3
  int turned, pieces;         // items of a head: those that turn pairs, and all
  int per_token, per_wg;      // items of a token, tokens of a workgroup
  uint32_t by_token, by_head;  // 2^32 / per_token and 2^32 / pieces, rounded up
  int pos_float;
};

constexpr int kRotTokens = 64, kRotAngles = 4096, kRotItems = 65536;  // the most of a workgroup

// n / d for n < kRotItems from m = ceil(2^32 / d): exact while n * d < 2^32.
__device__ __forceinline__ int quotient(int n, int d, uint32_t m) { return d == 1 ? n : (int)__umulhi((uint32_t)n, m); }

__device__ __forceinline__ void turn_pair(float& a, float& b, float c, float s) {
  const float x = a, y = b;
  a = __builtin_fmaf(x, c, -(y * s));
  b = __builtin_fmaf(x, s, y * c);
  // fp32 values here on every route: the compiler would form some fp16 results by mixed instructions, which round once
  // where a conversion of the fp32 value rounds twice, so that bits would go by the pieces' size
  asm("" : "+v"(a), "+v"(b));
}

template <class T, int VEC, bool NEAR>  // NEAR: a pair's values are neighbours
__global__ __launch_bounds__(256) void rotary_kernel(RotaryParams p) {
  extern __shared__ float turns[];  // cosines of this workgroup's tokens, then their sines
  __shared__ int64_t base[5][kRotTokens];  // where a token's queries and keys lie, their results, its positions
  const int tid = (int)threadIdx.x;
  const int64_t first = (int64_t)blockIdx.x * p.per_wg;
  const int ntok = p.tokens - first < p.per_wg ? (int)(p.tokens - first) : p.per_wg;
  if (tid < ntok) {
    const int64_t b = (first + tid) / p.L, l = (first + tid) - b * p.L;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      base[w][tid] = b * p.x_b[w] + l * p.x_l[w];
      base[2 + w][tid] = b * p.o_b[w] + l * p.o_l[w];
    }
    base[4][tid] = b * p.pos_b + l * p.pos_l;
  }
  __syncthreads();
  float* const cosines = turns;
  float* const sines = turns + p.per_wg * p.pairs;
  for (int i = tid; i < ntok * p.pairs; i += 256) {
    const int t = i / p.pairs, j = i - t * p.pairs;
    const int64_t at = base[4][t] + (j >= p.ends[0]) + (j >= p.ends[1]) + (j >= p.ends[2]);
    const double pos = p.pos_float ? (double)static_cast<const float*>(p.pos)[at]
                                   : (double)static_cast<const int32_t*>(p.pos)[at];
    double turn = pos * ((double)p.freq[j] * 0.15915494309189535);  // angle / (2 pi)
    turn -= __builtin_rint(turn);
    sincospif((float)(2.0 * turn), &sines[i], &cosines[i]);
  }
  __syncthreads();

  constexpr int U = NEAR ? 1 : 2;  // items of a thread in flight
  const int items = ntok * p.per_token;
  for (int i0 = tid; i0 < items; i0 += 256 * U) {
    float a[U][VEC], b[U][VEC];
    const float *c[U], *s[U];
    T* to[U];
    bool turned[U];
    constexpr bool PAIR = !NEAR || VEC == 1;  // an item that turns has two parts, this far apart
    const int part = NEAR ? 1 : p.pairs;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + 256 * u;
      if (i >= items) break;
      const int t = quotient(i, p.per_token, p.by_token), r = i - t * p.per_token;
      int h = quotient(r, p.pieces, p.by_head);
      const int piece = r - h * p.pieces;
      const int w = h >= p.Hq;
      h -= w ? p.Hq : 0;
      turned[u] = piece < p.turned;
      // where the item begins: a turned piece, or one of those behind the pairs
      const int step = PAIR && NEAR ? 2 : VEC;
      const int at = turned[u] ? piece * step : 2 * p.pairs + (piece - p.turned) * VEC;
      const int j = turned[u] ? (NEAR && VEC > 1 ? piece * (VEC / 2) : piece * VEC) : 0;
      const T* x = static_cast<const T*>(w ? p.x[1] : p.x[0]) + base[w][t] + h * (w ? p.x_h[1] : p.x_h[0]) + at;
      to[u] = static_cast<T*>(w ? p.out[1] : p.out[0]) + base[2 + w][t] + h * (w ? p.o_h[1] : p.o_h[0]) + at;
      c[u] = cosines + t * p.pairs + j;
      s[u] = sines + t * p.pairs + j;
      load_floats<T, VEC>(x, a[u]);
      if (PAIR && turned[u]) load_floats<T, VEC>(x + part, b[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i0 + 256 * u >= items) break;
      if (turned[u]) {
        if constexpr (PAIR) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) turn_pair(a[u][e], b[u][e], c[u][e], s[u][e]);
          store_floats(to[u] + part, b[u]);
        } else {
#pragma unroll
          for (int e = 0; e < VEC; e += 2) turn_pair(a[u][e], a[u][e + 1], c[u][e / 2], s[u][e / 2]);
        }
      }
      store_floats(to[u], a[u]);
    }
  }
}

template <class T, int VEC, bool NEAR>
static hipError_t run(RotaryParams p, int d, bool copies, hipStream_t stream) {
  p.turned = NEAR && VEC > 1 ? 2 * p.pairs / VEC : p.pairs / VEC;
  p.pieces = p.turned + (copies ? (d - 2 * p.pairs) / VEC : 0);
  const int64_t per_token = (int64_t)p.per_token * p.pieces;  // per_token holds the heads so far
  if (per_token > kRotItems) return hipErrorInvalidValue;     // not reached: the entry's limits
  if (per_token == 0) return hipSuccess;
  p.per_token = (int)per_token;
  // Up to four items a thread, as long as that leaves 512 workgroups.
  int64_t n = 1024 / per_token;
  if (n > p.tokens / 512) n = p.tokens / 512;
  if (n > kRotAngles / p.pairs) n = kRotAngles / p.pairs;
  if (n > kRotTokens) n = kRotTokens;
  if (n < 1) n = 1;
  p.per_wg = (int)n;
  p.by_token = (uint32_t)(((1ull << 32) + per_token - 1) / per_token);
  p.by_head = (uint32_t)(((1ull << 32) + p.pieces - 1) / p.pieces);
  const int64_t wgs = (p.tokens + n - 1) / n;
  if (!launchable(wgs, 256)) return hipErrorInvalidConfiguration;
  rotary_kernel<T, VEC, NEAR><<<dim3((unsigned)wgs), dim3(256), (size_t)(n * p.pairs) * 8, stream>>>(p);
  return hipGetLastError();
}

// Pieces of 16 bytes, or the largest part of them that sizes, strides and addresses are multiples of.
template <class T, bool NEAR>
static hipError_t by_piece(const RotaryParams& p, const sengine_rotary_desc* d, bool copies, hipStream_t stream) {
  const auto fits = [&](int vec) {
    if ((NEAR ? 2 * p.pairs : p.pairs) % vec || (d->d - 2 * p.pairs) % vec) return false;
    for (int w = 0; w < (d->Hk ? 2 : 1); ++w) {
      if ((uintptr_t)p.x[w] % (vec * sizeof(T)) || (uintptr_t)p.out[w] % (vec * sizeof(T))) return false;
      const int64_t strides[6] = {p.x_b[w], p.x_l[w], p.x_h[w], p.o_b[w], p.o_l[w], p.o_h[w]};
      const int n[3] = {d->B, d->L, w ? d->Hk : d->Hq};
      for (int i = 0; i < 6; ++i)
        if (n[i % 3] > 1 && strides[i] % vec) return false;
    }
    return true;
  };
  if constexpr (sizeof(T) == 2)
    if (fits(8)) return run<T, 8, NEAR>(p, d->d, copies, stream);
  if (fits(4)) return run<T, 4, NEAR>(p, d->d, copies, stream);
  if (fits(2)) return run<T, 2, NEAR>(p, d->d, copies, stream);
  return run<T, 1, NEAR>(p, d->d, copies, stream);
}

template <class T>
static hipError_t by_order(const RotaryParams& p, const sengine_rotary_desc* d, bool copies, hipStream_t stream) {
  return d->interleaved ? by_piece<T, true>(p, d, copies, stream) : by_piece<T, false>(p, d, copies, stream);
}

}  // namespace sengine

using namespace sengine;

extern "C" int sengine_amd_rotary(const sengine_rotary_desc* d, const void* q, const void* k, const void* positions,
                                  const float* frequencies, void* out_q, void* out_k, hipStream_t stream) {
  if (!d) return set_error(-1, "rotary: null descriptor");
  if (d->B < 0 || d->L < 0 || d->Hq < 1 || d->Hk < 0 || d->d < 1)
    return set_error(-2, "rotary: needs B, L, Hk >= 0 and Hq, d >= 1");
  if (d->axes < 1 || d->axes > 4) return set_error(-2, "rotary: 1 to 4 axes");
  int64_t pairs = 0;
  for (int a = 0; a < d->axes; ++a) {
    if (d->sections[a] < 0) return set_error(-2, "rotary: a section has 0 pairs or more");
    pairs += d->sections[a];
  }
  if (pairs < 1 || 2 * pairs > d->d) return set_error(-2, "rotary: the sections' pairs must fit into a head of d values");
  if (d->type != SENGINE_ENC_F16 && d->type != SENGINE_ENC_BF16 && d->type != SENGINE_ENC_F32)
    return set_error(-2, "rotary: q and k must be fp16, bf16 or fp32");
  if (d->d > 1024 || ((int64_t)d->Hq + d->Hk) * d->d > kRotItems)
    return set_error(-2, "rotary: a head has up to 1024 values, a token's heads together up to 65536");
  if (d->B == 0 || d->L == 0) return 0;
  if (!q || !out_q || !positions || !frequencies || (d->Hk > 0 && (!k || !out_k)))
    return set_error(-1, "rotary: null q, k, positions, frequencies or output");
  // more tokens than a launch has workgroups for, in whatever pieces
  if (!launchable(((int64_t)d->B * d->L + kRotTokens - 1) / kRotTokens, 256)) return (int)hipErrorInvalidConfiguration;
  for (int w = 0; w < (d->Hk ? 2 : 1); ++w) {
    const int32_t n[3] = {d->B, d->L, w ? d->Hk : d->Hq};
    if (!rows_apart(d->d, 3, n, w ? d->out_k_stride : d->out_q_stride))
      return set_error(-2, "rotary: output rows overlap");
  }
  RotaryParams p{};
  p.x[0] = q, p.x[1] = k;
  p.out[0] = out_q, p.out[1] = out_k;
  const int64_t* strides[4] = {d->q_stride, d->k_stride, d->out_q_stride, d->out_k_stride};
  for (int w = 0; w < 2; ++w) {
    p.x_b[w] = strides[w][0], p.x_l[w] = strides[w][1], p.x_h[w] = strides[w][2];
    p.o_b[w] = strides[2 + w][0], p.o_l[w] = strides[2 + w][1], p.o_h[w] = strides[2 + w][2];
  }
  p.pos = positions;
  p.freq = frequencies;
  p.pos_b = d->pos_stride[0], p.pos_l = d->pos_stride[1];
  p.tokens = (int64_t)d->B * d->L;
  p.L = d->L;
  p.Hq = d->Hq;
  p.pairs = (int)pairs;
  for (int a = 0, end = 0; a < 3; ++a) {
    end += a < d->axes ? d->sections[a] : 0;
    p.ends[a] = a + 1 < d->axes ? end : (int)pairs;
  }
  p.per_token = d->Hq + d->Hk;
  p.pos_float = d->pos_float != 0;
  // values behind the pairs that an output has already need no copy
  const auto same = [&](const void* x, const void* out, const int64_t* s, const int64_t* o, int32_t heads) {
    return x == out && (d->B == 1 || s[0] == o[0]) && (d->L == 1 || s[1] == o[1]) && (heads == 1 || s[2] == o[2]);
  };
  const bool copies = !same(q, out_q, d->q_stride, d->out_q_stride, d->Hq) ||
                      (d->Hk > 0 && !same(k, out_k, d->k_stride, d->out_k_stride, d->Hk));
  hipError_t e;
  if (d->type == SENGINE_ENC_F16)
    e = by_order<_Float16>(p, d, copies, stream);
  else if (d->type == SENGINE_ENC_BF16)
    e = by_order<__bf16>(p, d, copies, stream);
  else
    e = by_order<float>(p, d, copies, stream);
  return (int)e;
}
