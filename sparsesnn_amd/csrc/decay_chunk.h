// Decaying linear attention 64 tokens at a time (decay_attention.hip).  With a chunk's rows Q, K, V and the state S that
// it begins with,
//   O  = scale ((Q K^T . D) V + L Q S),   D[i][j] = g^(i - j) for j <= i, else 0,   L[i] = g^(i + 1)
//   S' = g^n S + K^T W V,                 W[j] = g^(n - 1 - j)
// Workgroup = one head of one sequence, or of a segment of it; its waves have 32 columns of V, S and O each, and S stays
// in their registers.  Q, K and V come through LDS, the next chunk's rows on their way in registers beside the products.
//
// All products are 16x16x32 matrix instructions, laid out so that what one leaves is what the next one takes:
//   * K Q^T puts four tokens j of one token i in a lane, two fragments of it are the second operand of the product with
//     V^T (its tokens in the order 4 g .. 4 g + 3, 16 + 4 g ..), V^T and K^T are read transposed from LDS;
//   * K^T (W V) has its rows, dk, permuted so that a lane ends with eight neighbouring ones of a column: as they lie they
//     are the operand of S^T Q^T; the columns, dv, likewise, so that a lane stores eight neighbouring values of O.
//
// Rounding.  S is fp32.  What a 16-bit instruction takes of it and of the fp32 weights Q K^T . D is a sum of two 16-bit
// values (16 bits of them in bf16, 22 in fp16), so that O is as exact as its own rounding; W V, which makes S, is a sum
// of three (bf16) or two (fp16, the second 2^11 times larger so that it does not fall below the type's range).  fp16
// values of S and of the weights are scaled by a power of two a column, and a token, to the type's range: an fp32 state
// passes it easily.
//
// A value of V that is not finite must not reach the tokens before it, and 0 times it would: a chunk that holds one
// takes it out and marks the outputs that it belongs to instead.
#pragma once
#include "lds_copy.h"
#include "linear.h"

namespace sengine {

struct DecayParams {
  const void *q, *k, *v;
  void* out;
  int64_t q_b, q_l, q_h, k_b, k_l, k_h, v_b, v_l, v_h, o_b, o_l, o_h;  // strides in elements
  int64_t s_b, s_h, so_b, so_h;
  const float* decay;
  const float* state;  // or null: zeros
  float* state_out;    // or null
  const int32_t* lengths;
  float* parts;        // (B, H, segs - 1) states
  int B, L, H, dk, dv;
  int segs, seg_len;
  float scale;
  __device__ __forceinline__ int length(int64_t b) const {
    const int n = lengths ? lengths[b] : L;
    return n < 0 ? 0 : n < L ? n : L;
  }
};

constexpr int kDecayChunk = 64;

// Waves of a workgroup: 32 columns each.
__host__ __device__ inline int decay_waves(int dv) { return dv <= 32 ? 1 : dv <= 64 ? 2 : dv <= 128 ? 4 : 8; }

// g^n from log2 g: 1 for n = 0, also of g = 0.
__device__ __forceinline__ float decay_log2(float g) { return log2f(g); }
__device__ __forceinline__ float decay_power(float lg, int n) { return n == 0 ? 1.f : exp2f((float)n * lg); }

// LDS rows of P pieces of 16 bytes, piece j of row r at place j ^ (..): 16 lanes that read a piece of 16 rows, or half of
// it, spread over the banks.
template <int P>
__device__ __forceinline__ int decay_at(int r, int j) {
  constexpr int mask = P >= 16 ? 15 : P - 1;
  return (r * P + (j ^ ((P == 4 ? r >> 1 : r) & mask))) * 16;
}

template <class T>
__device__ __forceinline__ u32x4_t decay_pack(const float (&x)[8]) {
  typedef T vec_t __attribute__((ext_vector_type(8)));
  vec_t v;
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = (T)x[e];
  return __builtin_bit_cast(u32x4_t, v);
}

// x rounded to T, and x becomes what that leaves out.  The fp32 values are made first: fp16's mixed instructions would
// round the product that x is once where a conversion of the fp32 value rounds twice, and the compiler may take one way
// for the value and the other for what it leaves out.
template <class T>
__device__ __forceinline__ u32x4_t decay_term(float (&x)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) asm("" : "+v"(x[e]));
  typedef T vec_t __attribute__((ext_vector_type(8)));
  const u32x4_t r = decay_pack<T>(x);
  const vec_t v = __builtin_bit_cast(vec_t, r);
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] -= (float)v[e];
  return r;
}

// A power of two that brings values up to `most` (its bits, the sign cleared) to fp16's upper range, and its inverse.
__device__ __forceinline__ void decay_range(uint32_t most, float& up, float& down) {
  int e = (int)(most >> 23);
  e = e < 81 ? 81 : e > 250 ? 250 : e;  // not so far up that what is added to them passes fp32
  up = __builtin_bit_cast(float, (uint32_t)(268 - e) << 23);
  down = __builtin_bit_cast(float, (uint32_t)(e - 14) << 23);
}

__device__ __forceinline__ uint32_t decay_most(uint32_t m, float x) {
  const uint32_t b = __builtin_bit_cast(uint32_t, x) & 0x7fffffffu;
  return b > m ? b : m;
}

__device__ __forceinline__ uint32_t decay_across(uint32_t m) {  // over the lanes of a column
  const uint32_t a = __shfl_xor(m, 16, 64);
  m = a > m ? a : m;
  const uint32_t b = __shfl_xor(m, 32, 64);
  return b > m ? b : m;
}

// 1 where a 16-bit value is not finite, else 0, of both halves.
template <class T>
__device__ __forceinline__ bool decay_odd(u32x4_t v) {
  constexpr uint32_t top = __is_same(T, _Float16) ? 0x7c00u : 0x7f80u;
  uint32_t any = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    any |= (uint32_t)((v[i] & top) == top) | (uint32_t)((v[i] & (top << 16)) == (top << 16));
  return any != 0;
}

// DKP: dk rounded up to 32, 64 or 128.  STATE: a segment's state from a state of zeros, without outputs.
template <class T, int DKP, int NW, bool STATE>
__global__ __launch_bounds__(64 * NW) void decay_chunk_kernel(DecayParams p) {
  constexpr bool HALF = __is_same(T, _Float16);
  constexpr int NT = 64 * NW, C = kDecayChunk;
  constexpr int PK = DKP / 8, PV = NW * 4;  // pieces of a row of Q or K, of V
  constexpr int NM = DKP / 32, NK = DKP / 16;
  constexpr int LK = (C * PK + NT - 1) / NT, LV = C * PV / NT;  // pieces of a thread a chunk
  __shared__ __attribute__((aligned(1024))) uint8_t smem[C * 16 * (PK * (STATE ? 1 : 2) + PV)];
  uint8_t* const sK = smem;
  uint8_t* const sV = smem + C * 16 * PK;
  uint8_t* const sQ = smem + C * 16 * (PK + PV);
  const int tid = (int)threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, a = lane & 15;
  // neighbouring heads of a segment on one XCD: where their rows share cache lines they are fetched once
  const int segs = STATE ? p.segs - 1 : p.segs;
  const int id = xcd_order((int)blockIdx.x, p.B * p.H * segs);
  const int h = id % p.H, seg = id / p.H % segs;
  const int64_t b = id / p.H / segs;
  const int n = p.length(b);
  const int begin = seg * p.seg_len;
  const int left = n - begin < 0 ? 0 : n - begin < p.seg_len ? n - begin : p.seg_len;  // tokens of this segment
  // what follows the segment needs no state of it, if it has no tokens
  if (STATE && n - begin <= p.seg_len) return;
  const T* q = static_cast<const T*>(p.q) + b * p.q_b + h * p.q_h + begin * p.q_l;
  const T* k = static_cast<const T*>(p.k) + b * p.k_b + h * p.k_h + begin * p.k_l;
  const T* v = static_cast<const T*>(p.v) + b * p.v_b + h * p.v_h + begin * p.v_l;
  T* out = static_cast<T*>(p.out) + b * p.o_b + h * p.o_h + begin * p.o_l;

  // powers of the decay as the lanes need them
  const float lg = decay_log2(p.decay[h]);
  float inside[4][4], begun[4], weight[4][4];  // scale D by 16-token blocks apart, scale L, W
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    begun[x] = p.scale * decay_power(lg, 16 * x + a + 1);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int apart = 16 * x + a - 4 * g - e;
      inside[x][e] = apart >= 0 ? p.scale * decay_power(lg, apart) : 0.f;
      weight[x][e] = decay_power(lg, C - 1 - (16 * x + 4 * g + e));
    }
  }
  float passed = decay_power(lg, C);

  // S: value i of fragment [f][c] is row 32 (f / 2) + 8 g + 4 (f % 2) + i, column 8 (a / 4) + 4 c + a % 4 of the wave's
  const int dv0 = wave * 32 + 8 * (a >> 2) + (a & 3);
  float4_t S[NK][2];
  const auto state_at = [&](int f, int c, int i) {
    return (int64_t)(32 * (f / 2) + 8 * g + 4 * (f % 2) + i) * p.dv + dv0 + 4 * c;
  };
  const auto has_state = [&](int f, int c, int i) {
    return 32 * (f / 2) + 8 * g + 4 * (f % 2) + i < p.dk && dv0 + 4 * c < p.dv;
  };
  const int64_t bh = b * p.H + h;
  const int64_t matrix = (int64_t)p.dk * p.dv;
  const float* from = STATE ? nullptr
                      : seg > 0 ? (left > 0 ? p.parts + (bh * (p.segs - 1) + seg - 1) * matrix : nullptr)
                      : p.state ? p.state + b * p.s_b + h * p.s_h
                                : nullptr;
#pragma unroll
  for (int f = 0; f < NK; ++f)
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) S[f][c][i] = from && has_state(f, c, i) ? from[state_at(f, c, i)] : 0.f;

  u32x4_t lq[STATE ? 1 : LK], lk[LK], lv[LV];
  const auto fetch = [&](const T* base, int64_t stride, int t, int at, int width) {
    if (t >= left || at >= width) return u32x4_t{0, 0, 0, 0};
    return *reinterpret_cast<const u32x4_t*>(base + (int64_t)t * stride + at);
  };
  const auto load = [&](int t0) {
#pragma unroll
    for (int i = 0; i < LK; ++i) {
      const int at = tid + i * NT, r = at / PK, j = at % PK;
      if (C * PK % NT != 0 && at >= C * PK) break;
      if constexpr (!STATE) lq[i] = fetch(q, p.q_l, t0 + r, j * 8, p.dk);
      lk[i] = fetch(k, p.k_l, t0 + r, j * 8, p.dk);
    }
#pragma unroll
    for (int i = 0; i < LV; ++i) {
      const int at = tid + i * NT, r = at / PV, j = at % PV;
      lv[i] = fetch(v, p.v_l, t0 + r, j * 8, p.dv);
    }
  };
  const auto keep = [&]() {
#pragma unroll
    for (int i = 0; i < LK; ++i) {
      const int at = tid + i * NT, r = at / PK, j = at % PK;
      if (C * PK % NT != 0 && at >= C * PK) break;
      if constexpr (!STATE) *reinterpret_cast<u32x4_t*>(sQ + decay_at<PK>(r, j)) = lq[i];
      *reinterpret_cast<u32x4_t*>(sK + decay_at<PK>(r, j)) = lk[i];
    }
#pragma unroll
    for (int i = 0; i < LV; ++i) {
      const int at = tid + i * NT, r = at / PV, j = at % PV;
      *reinterpret_cast<u32x4_t*>(sV + decay_at<PV>(r, j)) = lv[i];
    }
  };
  const auto rows = [&](const uint8_t* s, int block, int m) {  // 16 rows, values 32 m ..
    return *reinterpret_cast<const u32x4_t*>(s + decay_at<PK>(16 * block + a, 4 * m + g));
  };
  // 32 tokens x 16 columns transposed: the columns 8 p + 4 half .. of four pieces j0 + p
  const auto columns = [&](const uint8_t* s, auto pieces, int step, int j0, int half) {
    constexpr int P = decltype(pieces)::value;
    const int r = 32 * step + 4 * g + (a >> 2), j = j0 + (a & 3);
    return read_transposed(s + decay_at<P>(r, j) + 8 * half, s + decay_at<P>(r + 16, j) + 8 * half);
  };

  load(0);
  for (int t0 = 0; t0 < left; t0 += C) {
    __syncthreads();  // the chunk before has been read
    keep();
    __syncthreads();
    if (t0 + C < left) load(t0 + C);
    const int live = left - t0 < C ? left - t0 : C;
    if (live < C) {  // the last chunk: its weights count from its last token
      passed = decay_power(lg, live);
#pragma unroll
      for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int apart = live - 1 - (16 * x + 4 * g + e);
          weight[x][e] = apart >= 0 ? decay_power(lg, apart) : 0.f;
        }
    }
    u32x4_t V[2][2];  // [tokens 32 x ..][columns 4 c ..]
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int c = 0; c < 2; ++c) V[x][c] = columns(sV, Int<PV>{}, x, 4 * wave, c);

    if constexpr (!STATE) {
      float4_t O[4][2];
#pragma unroll
      for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int c = 0; c < 2; ++c) O[x][c] = float4_t{0.f, 0.f, 0.f, 0.f};
      // S^T Q^T
      float up[2], down[2];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        up[c] = down[c] = 1.f;
        if constexpr (HALF) {
          uint32_t most = 0;
#pragma unroll
          for (int f = 0; f < NK; ++f)
#pragma unroll
            for (int i = 0; i < 4; ++i) most = decay_most(most, S[f][c][i]);
          decay_range(decay_across(most), up[c], down[c]);
        }
      }
#pragma unroll
      for (int m = 0; m < NM; ++m) {
        u32x4_t s[2][2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float x[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = S[2 * m + e / 4][c][e % 4] * up[c];
          s[c][0] = decay_term<T>(x);
          s[c][1] = decay_pack<T>(x);
        }
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const u32x4_t r = rows(sQ, x, m);
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            O[x][c] = mma_64b<T>(s[c][0], r, O[x][c]);
            O[x][c] = mma_64b<T>(s[c][1], r, O[x][c]);
          }
        }
      }
      float back[2][4];  // the columns' factors where O has them
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) back[c][i] = HALF ? __shfl(down[c], 4 * g + i, 64) : 1.f;
      bool odd = false;
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int c = 0; c < 2; ++c) odd |= decay_odd<T>(V[x][c]);
      const bool any_odd = __any(odd);

#pragma unroll
      for (int x = 0; x < 4; ++x) {  // 16 tokens i
        float4_t P[4];
#pragma unroll
        for (int y = 0; y <= x; ++y) {
          P[y] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int m = 0; m < NM; ++m) P[y] = mma_64b<T>(rows(sK, y, m), rows(sQ, x, m), P[y]);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            P[y][i] *= inside[x - y][i];
            if (y == x && 4 * g + i > a) P[y][i] = 0.f;  // whatever the later token holds
          }
        }
#pragma unroll
        for (int y = x + 1; y < 4; ++y) P[y] = float4_t{0.f, 0.f, 0.f, 0.f};
        float pup = 1.f, pdown = 1.f;
        if constexpr (HALF) {
          uint32_t most = 0;
#pragma unroll
          for (int y = 0; y <= x; ++y)
#pragma unroll
            for (int i = 0; i < 4; ++i) most = decay_most(most, P[y][i]);
          decay_range(decay_across(most), pup, pdown);
        }
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int i = 0; i < 4; ++i) O[x][c][i] *= begun[x] * back[c][i] * pup;
#pragma unroll
        for (int y = 0; y <= x / 2; ++y) {
          float w[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) w[e] = P[2 * y + e / 4][e % 4] * pup;
          const u32x4_t hi = decay_term<T>(w), lo = decay_pack<T>(w);
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            u32x4_t V_ = V[y][c];
            if (any_odd) {  // finite values only
              typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));
              constexpr uint16_t top = HALF ? 0x7c00u : 0x7f80u;
              u16x8 t = __builtin_bit_cast(u16x8, V_);
#pragma unroll
              for (int e = 0; e < 8; ++e) t[e] = (t[e] & top) == top ? 0 : t[e];
              V_ = __builtin_bit_cast(u32x4_t, t);
            }
            O[x][c] = mma_64b<T>(V_, hi, O[x][c]);
            O[x][c] = mma_64b<T>(V_, lo, O[x][c]);
          }
        }
        if (any_odd) {  // tokens at or behind a value that is not finite: how many of them there are, by ones
          float4_t count[2] = {float4_t{0.f, 0.f, 0.f, 0.f}, float4_t{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
          for (int y = 0; y <= x / 2; ++y) {
            float w[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = 32 * y + 16 * (e / 4) + 4 * g + e % 4 <= 16 * x + a ? 1.f : 0.f;
            const u32x4_t ones = decay_pack<T>(w);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));
              constexpr uint16_t top = HALF ? 0x7c00u : 0x7f80u, one = HALF ? 0x3c00u : 0x3f80u;
              u16x8 t = __builtin_bit_cast(u16x8, V[y][c]);
#pragma unroll
              for (int e = 0; e < 8; ++e) t[e] = (t[e] & top) == top ? one : 0;
              count[c] = mma_64b<T>(__builtin_bit_cast(u32x4_t, t), ones, count[c]);
            }
          }
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (count[c][i] > 0.f) O[x][c][i] = __builtin_nanf("");
        }
        const int t = 16 * x + a, at = wave * 32 + 8 * g;
        if (t < live && at < p.dv) {
          float o[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) o[e] = O[x][e / 4][e % 4] * pdown;
          *reinterpret_cast<u32x4_t*>(out + (int64_t)(t0 + t) * p.o_l + at) = decay_pack<T>(o);
        }
      }
    }
    // S' = g^n S + K^T W V
#pragma unroll
    for (int f = 0; f < NK; ++f)
#pragma unroll
      for (int c = 0; c < 2; ++c) S[f][c] *= passed;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      u32x4_t w[2][3];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        typedef T vec_t __attribute__((ext_vector_type(8)));
        const vec_t t = __builtin_bit_cast(vec_t, V[x][c]);
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = (float)t[e] * weight[2 * x + e / 4][e % 4];
        w[c][0] = decay_term<T>(y);
        if constexpr (HALF) {
#pragma unroll
          for (int e = 0; e < 8; ++e) y[e] *= 2048.f;
          w[c][1] = decay_pack<T>(y);
        } else {
          w[c][1] = decay_term<T>(y);
          w[c][2] = decay_pack<T>(y);
        }
      }
#pragma unroll
      for (int f = 0; f < NK; ++f) {
        const u32x4_t r = columns(sK, Int<PK>{}, x, 4 * (f / 2), f % 2);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          S[f][c] = mma_64b<T>(r, w[c][0], S[f][c]);
          if constexpr (HALF) {
            const float4_t rest = mma_64b<T>(r, w[c][1], float4_t{0.f, 0.f, 0.f, 0.f});
#pragma unroll
            for (int i = 0; i < 4; ++i) S[f][c][i] = __builtin_fmaf(rest[i], 1.f / 2048.f, S[f][c][i]);
          } else {
            S[f][c] = mma_64b<T>(r, w[c][1], S[f][c]);
            S[f][c] = mma_64b<T>(r, w[c][2], S[f][c]);
          }
        }
      }
    }
  }
  if constexpr (!STATE) {
    // tokens behind the sequence's last one
    const int end = p.L - begin < p.seg_len ? p.L - begin : p.seg_len, pieces = p.dv / 8;
    for (int i = tid; i < (end - left) * pieces; i += NT)
      *reinterpret_cast<u32x4_t*>(out + (int64_t)(left + i / pieces) * p.o_l + i % pieces * 8) = u32x4_t{0, 0, 0, 0};
  }
  float* to = STATE ? p.parts + (bh * (p.segs - 1) + seg) * matrix
              : p.state_out && seg == (n > 0 ? (n - 1) / p.seg_len : 0) ? p.state_out + b * p.so_b + h * p.so_h
                                                                       : nullptr;
  if (!to) return;
#pragma unroll
  for (int f = 0; f < NK; ++f)
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (has_state(f, c, i)) to[state_at(f, c, i)] = S[f][c][i];
}

}  // namespace sengine
