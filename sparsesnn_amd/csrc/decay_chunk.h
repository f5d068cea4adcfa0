// Decaying linear attention 64 tokens at a time (decay_attention.hip).  With a chunk's rows Q, K, V and the state S that
// it begins with,
//   O  = scale ((Q K^T . D) V + L Q S),   D[i][j] = g^(i - j) for j <= i, else 0,   L[i] = g^(i + 1)
//   S' = g^n S + K^T W V,                 W[j] = g^(n - 1 - j)
// Workgroup = one head of one sequence, or of a segment of it, and up to 128 columns of V; a wave has 16 columns of V, S
// and O, and S stays in its registers.  The memory pipeline copies the next chunk's rows into one half of LDS beside the
// products with the other.  The ten 16 x 16 blocks of Q K^T . D that count are shared out over the waves and go through
// LDS; while they are made, the other products need only what the wave has.
//
// All products are 16x16x32 matrix instructions, laid out so that what one leaves is what the next one takes:
//   * K Q^T puts four tokens j of one token i in a lane: two such blocks, side by side in LDS, are the second operand of
//     the product with V^T (its tokens in the order 4 g .. 4 g + 3, 16 + 4 g ..), V^T and K^T are read transposed;
//   * K^T (W V) has its rows, dk, permuted so that a lane ends with eight neighbouring ones of a column: as they lie they
//     are the operand of S^T Q^T.
//
// Rounding.  S is fp32.  What a 16-bit instruction takes of it and of the fp32 weights Q K^T . D is a sum of two 16-bit
// values (of bf16, 16 bits; S of fp16, 22), so that O is as exact as its own rounding; W V, which makes S, is a sum of
// three (bf16) or two (fp16, the second 2^11 times larger so that it does not fall below the type's range).  Weights
// easily pass fp16's range: they are bf16 values always, and fp16 values of V are sums of two of them, exactly.  A
// column of S is scaled by a power of two to fp16's range.
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
constexpr int kDecayColumns = 128;  // most columns of V of a workgroup

// Waves of a workgroup: 16 columns each.
__host__ __device__ inline int decay_waves(int dv) { return dv <= 32 ? 2 : dv <= 48 ? 3 : dv <= 64 ? 4 : 8; }

// g^n from log2 g: 1 for n = 0, also of g = 0.
__device__ __forceinline__ float decay_log2(float g) { return log2f(g); }
__device__ __forceinline__ float decay_power(float lg, int n) { return n == 0 ? 1.f : exp2f((float)n * lg); }

// LDS rows of P pieces of 16 bytes, piece j of row r at place j ^ (..): 16 lanes that read a piece of 16 rows, or half of
// it, spread over the banks.
template <int P>
__device__ __forceinline__ int decay_place(int r, int j) {
  constexpr int mask = P >= 16 ? 15 : P - 1;
  return j ^ ((P == 4 ? r >> 1 : r) & mask);
}
template <int P>
__device__ __forceinline__ int decay_at(int r, int j) {
  return (r * P + decay_place<P>(r, j)) * 16;
}

template <class T, int N>
__device__ __forceinline__ auto decay_pack(const float (&x)[N]) {
  typedef T vec_t __attribute__((ext_vector_type(N)));
  typedef uint32_t words_t __attribute__((ext_vector_type(N / 2)));
  vec_t v;
#pragma unroll
  for (int e = 0; e < N; ++e) v[e] = (T)x[e];
  return __builtin_bit_cast(words_t, v);
}

// x rounded to T, and x becomes what that leaves out.  The fp32 values are made first: fp16's mixed instructions would
// round the product that x is once where a conversion of the fp32 value rounds twice, and the compiler may take one way
// for the value and the other for what it leaves out.
template <class T, int N>
__device__ __forceinline__ auto decay_term(float (&x)[N]) {
#pragma unroll
  for (int e = 0; e < N; ++e) asm("" : "+v"(x[e]));
  typedef T vec_t __attribute__((ext_vector_type(N)));
  const auto r = decay_pack<T>(x);
  const vec_t v = __builtin_bit_cast(vec_t, r);
#pragma unroll
  for (int e = 0; e < N; ++e) x[e] -= (float)v[e];
  return r;
}

// A power of two that brings values up to `most` (its bits, the sign cleared) to fp16's upper range, and its inverse.
__device__ __forceinline__ void decay_range(uint32_t most, float& up, float& down) {
  int e = (int)(most >> 23);
  e = e < 81 ? 81 : e > 250 ? 250 : e;
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

// `instead` in the place of the 16-bit values that are not finite, `others` of the rest where KEEP is false.
template <class T, bool KEEP>
__device__ __forceinline__ u32x4_t decay_replace(u32x4_t v, uint16_t instead) {
  typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));
  constexpr uint16_t top = __is_same(T, _Float16) ? 0x7c00u : 0x7f80u;
  u16x8 t = __builtin_bit_cast(u16x8, v);
#pragma unroll
  for (int e = 0; e < 8; ++e) t[e] = (t[e] & top) == top ? instead : KEEP ? t[e] : (uint16_t)0;
  return __builtin_bit_cast(u32x4_t, t);
}

// DKP: dk rounded up to 32, 64 or 128.  STATE: a segment's state from a state of zeros, without outputs.
template <class T, int DKP, int NW, bool STATE>
__global__ __launch_bounds__(64 * NW, 2) void decay_chunk_kernel(DecayParams p) {
  constexpr bool HALF = __is_same(T, _Float16);
  constexpr int C = kDecayChunk;
  constexpr int PK = DKP / 8, PV = NW == 3 ? 8 : NW * 2;  // pieces of a row of Q or K, of V
  constexpr int NM = DKP / 32, NK = DKP / 16;
  constexpr int NC = PK * (STATE ? 1 : 2) + PV, NCW = (NC + NW - 1) / NW;  // copies of 1 KB a chunk, of a wave
  constexpr int kStage = NC * 1024;
  constexpr int kQ = (PK + PV) * 1024;  // a stage: K, V, Q
  constexpr int kP = 8 * 1024;          // blocks of Q K^T . D: 4 x 2 operands, the first terms and then the second
  __shared__ __attribute__((aligned(1024))) uint8_t smem[2 * kStage + (STATE ? 0 : 2 * kP)];
  __shared__ float powers[C];  // scale g^n
  const int tid = (int)threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, a = lane & 15;
  // neighbouring heads of a segment on one XCD: where their rows share cache lines they are fetched once
  const int segs = STATE ? p.segs - 1 : p.segs;
  const int slices = (p.dv + kDecayColumns - 1) / kDecayColumns;
  int id = xcd_order((int)blockIdx.x, p.B * p.H * segs * slices);
  const int slice = id % slices;
  id /= slices;
  const int h = id % p.H, seg = id / p.H % segs;
  const int64_t b = id / p.H / segs;
  const int width = p.dv - slice * kDecayColumns < kDecayColumns ? p.dv - slice * kDecayColumns : kDecayColumns;
  const int n = p.length(b);
  const int begin = seg * p.seg_len;
  const int left = n - begin < 0 ? 0 : n - begin < p.seg_len ? n - begin : p.seg_len;  // tokens of this segment
  // what follows the segment needs no state of it, if it has no tokens
  if (STATE && n - begin <= p.seg_len) return;
  const uint8_t* q = static_cast<const uint8_t*>(p.q) + (b * p.q_b + h * p.q_h + begin * p.q_l) * 2;
  const uint8_t* k = static_cast<const uint8_t*>(p.k) + (b * p.k_b + h * p.k_h + begin * p.k_l) * 2;
  const uint8_t* v = static_cast<const uint8_t*>(p.v) + (b * p.v_b + h * p.v_h + begin * p.v_l + slice * kDecayColumns) * 2;
  T* out = static_cast<T*>(p.out) + b * p.o_b + h * p.o_h + begin * p.o_l + slice * kDecayColumns;

  // powers of the decay as the lanes need them
  const float lg = decay_log2(p.decay[h]);
  float begun[4], weight[4][4];  // scale L, W
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    begun[x] = p.scale * decay_power(lg, 16 * x + a + 1);
#pragma unroll
    for (int e = 0; e < 4; ++e) weight[x][e] = decay_power(lg, C - 1 - (16 * x + 4 * g + e));
  }
  float passed = decay_power(lg, C);
  if constexpr (!STATE) {
    if (tid < C) powers[tid] = p.scale * decay_power(lg, tid);
    // blocks above the diagonal that share an operand with one that counts stay zeros
    for (int i = tid; i < 2 * kP / 16; i += 64 * NW)
      *reinterpret_cast<u32x4_t*>(smem + 2 * kStage + i * 16) = u32x4_t{0, 0, 0, 0};
  }

  // S: value i of fragment f is row 32 (f / 2) + 8 g + 4 (f % 2) + i, column a of the wave's
  const int column = wave * 16 + a;
  const bool used = wave * 16 < width;  // whether the wave has columns
  float4_t S[NK];
  const auto state_at = [&](int f, int i) {
    return (int64_t)(32 * (f / 2) + 8 * g + 4 * (f % 2) + i) * p.dv + slice * kDecayColumns + column;
  };
  const auto has_state = [&](int f, int i) { return 32 * (f / 2) + 8 * g + 4 * (f % 2) + i < p.dk && column < width; };
  const int64_t bh = b * p.H + h;
  const int64_t matrix = (int64_t)p.dk * p.dv;
  const float* from = STATE ? nullptr
                      : seg > 0 ? (left > 0 ? p.parts + (bh * (p.segs - 1) + seg - 1) * matrix : nullptr)
                      : p.state ? p.state + b * p.s_b + h * p.s_h
                                : nullptr;
#pragma unroll
  for (int f = 0; f < NK; ++f)
#pragma unroll
    for (int i = 0; i < 4; ++i) S[f][i] = from && has_state(f, i) ? from[state_at(f, i)] : 0.f;

  // This wave's copies: c = wave, wave + NW, .. of a stage's PK of K, PV of V, PK of Q.  A lane's 16 bytes are place
  // lane % P of a row; the piece that belongs there is fetched, or nothing where the row has none.
  int voff[NCW];
#pragma unroll
  for (int i = 0; i < NCW; ++i) {
    const int c = wave + i * NW, kind = c < PK ? 0 : c < PK + PV ? 1 : 2;
    const int at = (c - (kind == 0 ? 0 : kind == 1 ? PK : PK + PV)) * 64 + lane;
    const int r = kind == 1 ? at / PV : at / PK;
    const int j = kind == 1 ? decay_place<PV>(r, at % PV) : decay_place<PK>(r, at % PK);
    const int64_t stride = kind == 0 ? p.k_l : kind == 1 ? p.v_l : p.q_l;
    voff[i] = j * 8 < (kind == 1 ? width : p.dk) ? r * (int)stride * 2 + j * 16 : 0x7fffff00;
  }
  const uint32_t lds0 = lds_offset(smem);
  const auto copy = [&](int t0, int stage) {
    const int live = left - t0 < C ? left - t0 : C;  // rows past them are out of the buffers' range
    const u32x4_t kr = row_buffer(k + (int64_t)t0 * p.k_l * 2, ((live - 1) * (int)p.k_l + p.dk) * 2);
    const u32x4_t vr = row_buffer(v + (int64_t)t0 * p.v_l * 2, ((live - 1) * (int)p.v_l + width) * 2);
    const u32x4_t qr = STATE ? kr : row_buffer(q + (int64_t)t0 * p.q_l * 2, ((live - 1) * (int)p.q_l + p.dk) * 2);
#pragma unroll
    for (int i = 0; i < NCW; ++i) {
      const int c = wave + i * NW;
      if (NC % NW != 0 && c >= NC) break;
      lds_copy(c < PK ? kr : c < PK + PV ? vr : qr, lds0 + stage * kStage + c * 1024, voff[i]);
    }
  };
  const auto rows = [&](const uint8_t* s, int block, int m) {  // 16 rows, values 32 m ..
    return *reinterpret_cast<const u32x4_t*>(s + decay_at<PK>(16 * block + a, 4 * m + g));
  };
  // 32 tokens transposed: 16 columns whose pieces of four values are halves `half` of 16-byte pieces j
  const auto columns = [&](const uint8_t* s, auto pieces, int step, int j, int half) {
    constexpr int P = decltype(pieces)::value;
    const int r = 32 * step + 4 * g + (a >> 2);
    return read_transposed(s + decay_at<P>(r, j) + 8 * half, s + decay_at<P>(r + 16, j) + 8 * half);
  };

  if (left > 0) copy(0, 0);
  for (int t0 = 0, stage = 0; t0 < left; t0 += C, stage ^= 1) {
    // this wave's copies have landed and its reads of the other stage and the blocks are done; so are all waves'
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (t0 + C < left) copy(t0 + C, stage ^ 1);
    const uint8_t* const sK = smem + stage * kStage;
    const uint8_t* const sV = sK + PK * 1024;
    const uint8_t* const sQ = sK + kQ;
    uint8_t* const sP = smem + 2 * kStage;
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

    if constexpr (!STATE) {
      // Blocks of K Q^T . D: tokens j of block y, i of block x >= y; the wave's are number wave, wave + NW, ..
      constexpr int NB = (10 + NW - 1) / NW;
      float4_t P[NB];
      int bx[NB], by[NB];
#pragma unroll
      for (int u = 0; u < NB; ++u) {
        const int at = wave + u * NW < 10 ? wave + u * NW : 9;
        bx[u] = at < 1 ? 0 : at < 3 ? 1 : at < 6 ? 2 : 3;
        by[u] = at - bx[u] * (bx[u] + 1) / 2;
        P[u] = float4_t{0.f, 0.f, 0.f, 0.f};
      }
#pragma unroll
      for (int m = 0; m < NM; ++m)
#pragma unroll
        for (int u = 0; u < NB; ++u) P[u] = mma_64b<T>(rows(sK, by[u], m), rows(sQ, bx[u], m), P[u]);
#pragma unroll
      for (int u = 0; u < NB; ++u) {
        float w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int apart = 16 * (bx[u] - by[u]) + a - 4 * g - i;
          w[i] = apart >= 0 ? P[u][i] * powers[apart & (C - 1)] : 0.f;  // whatever a later token holds
        }
        const u32x2_t hi = decay_term<__bf16>(w), lo = decay_pack<__bf16>(w);
        if (wave + u * NW < 10) {
          uint8_t* const at = sP + ((bx[u] * 2 + by[u] / 2) * 64 + lane) * 16 + by[u] % 2 * 8;
          *reinterpret_cast<u32x2_t*>(at) = hi;
          *reinterpret_cast<u32x2_t*>(at + kP) = lo;
        }
      }
    }

    u32x4_t V[2];  // tokens 32 x ..
#pragma unroll
    for (int x = 0; x < 2; ++x) V[x] = columns(sV, Int<PV>{}, x, 2 * wave + ((a & 3) >> 1), a & 1);
    float4_t O[4];
    if constexpr (!STATE) {
#pragma unroll
      for (int x = 0; x < 4; ++x) O[x] = float4_t{0.f, 0.f, 0.f, 0.f};
      if (used) {  // S^T Q^T
        float up = 1.f, down = 1.f;
        if constexpr (HALF) {
          uint32_t most = 0;
#pragma unroll
          for (int f = 0; f < NK; ++f)
#pragma unroll
            for (int i = 0; i < 4; ++i) most = decay_most(most, S[f][i]);
          decay_range(decay_across(most), up, down);
        }
#pragma unroll
        for (int m = 0; m < NM; ++m) {
          float s[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) s[e] = HALF ? S[2 * m + e / 4][e % 4] * up : S[2 * m + e / 4][e % 4];
          const u32x4_t hi = decay_term<T>(s), lo = decay_pack<T>(s);
          u32x4_t r[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) r[x] = rows(sQ, x, m);
#pragma unroll
          for (int x = 0; x < 4; ++x) O[x] = mma_64b<T>(hi, r[x], O[x]);
#pragma unroll
          for (int x = 0; x < 4; ++x) O[x] = mma_64b<T>(lo, r[x], O[x]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float back = HALF ? __shfl(down, 4 * g + i, 64) : 1.f;  // the column's factor where O has it
#pragma unroll
          for (int x = 0; x < 4; ++x) O[x][i] *= HALF ? begun[x] * back : begun[x];
        }
      }
    }
    if (used) {  // S' = g^n S + K^T W V
#pragma unroll
      for (int f = 0; f < NK; ++f) S[f] *= passed;
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        typedef T vec_t __attribute__((ext_vector_type(8)));
        const vec_t t = __builtin_bit_cast(vec_t, V[x]);
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = (float)t[e] * weight[2 * x + e / 4][e % 4];
        u32x4_t w[3];
        w[0] = decay_term<T>(y);
        if constexpr (HALF) {
#pragma unroll
          for (int e = 0; e < 8; ++e) y[e] *= 2048.f;
          w[1] = decay_pack<T>(y);
        } else {
          w[1] = decay_term<T>(y);
          w[2] = decay_pack<T>(y);
        }
        constexpr int G = NK < 4 ? NK : 4;  // fragments at a time, so that none waits for its own sums
#pragma unroll
        for (int f0 = 0; f0 < NK; f0 += G) {
          u32x4_t r[G];
#pragma unroll
          for (int f = 0; f < G; ++f) r[f] = columns(sK, Int<PK>{}, x, 4 * ((f0 + f) / 2) + (a & 3), (f0 + f) % 2);
#pragma unroll
          for (int f = 0; f < G; ++f) S[f0 + f] = mma_64b<T>(r[f], w[0], S[f0 + f]);
          if constexpr (HALF) {
            float4_t rest[G];
#pragma unroll
            for (int f = 0; f < G; ++f) rest[f] = mma_64b<T>(r[f], w[1], float4_t{0.f, 0.f, 0.f, 0.f});
#pragma unroll
            for (int f = 0; f < G; ++f)
#pragma unroll
              for (int i = 0; i < 4; ++i) S[f0 + f][i] = __builtin_fmaf(rest[f][i], 1.f / 2048.f, S[f0 + f][i]);
          } else {
#pragma unroll
            for (int f = 0; f < G; ++f) S[f0 + f] = mma_64b<T>(r[f], w[1], S[f0 + f]);
#pragma unroll
            for (int f = 0; f < G; ++f) S[f0 + f] = mma_64b<T>(r[f], w[2], S[f0 + f]);
          }
        }
      }
    }
    if constexpr (!STATE) {
      if (used) {
        // a value that is not finite, times zero, is not a number in its row
        float4_t odd = mma_64b<T>(V[0], u32x4_t{0, 0, 0, 0}, float4_t{0.f, 0.f, 0.f, 0.f});
        odd = mma_64b<T>(V[1], u32x4_t{0, 0, 0, 0}, odd);
        const float any = (odd[0] + odd[1]) + (odd[2] + odd[3]);
        if (__builtin_expect(__any(any != any), 0)) {
          // its token's outputs and later ones: how many such values there are up to each token, by ones
          constexpr uint16_t one = HALF ? 0x3c00u : 0x3f80u;
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            float4_t count = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int y = 0; y <= x / 2; ++y) {
              float w[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) w[e] = 32 * y + 16 * (e / 4) + 4 * g + e % 4 <= 16 * x + a ? 1.f : 0.f;
              count = mma_64b<T>(decay_replace<T, false>(V[y], one), decay_pack<T>(w), count);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (count[i] > 0.f) O[x][i] = __builtin_nanf("");
          }
#pragma unroll
          for (int y = 0; y < 2; ++y) V[y] = decay_replace<T, true>(V[y], 0);
        }
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the blocks are written
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      if (used) {  // (Q K^T . D) V
        u32x4_t first[2], second[2];
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          first[y] = V[y];
          if constexpr (HALF) {
            typedef T vec_t __attribute__((ext_vector_type(8)));
            const vec_t t = __builtin_bit_cast(vec_t, V[y]);
            float s[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) s[e] = (float)t[e];
            first[y] = decay_term<__bf16>(s);
            second[y] = decay_pack<__bf16>(s);
          }
        }
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          u32x4_t hi[4], lo[4];
#pragma unroll
          for (int x = 2 * y; x < 4; ++x) {
            hi[x] = *reinterpret_cast<const u32x4_t*>(sP + ((x * 2 + y) * 64 + lane) * 16);
            lo[x] = *reinterpret_cast<const u32x4_t*>(sP + kP + ((x * 2 + y) * 64 + lane) * 16);
          }
#pragma unroll
          for (int x = 2 * y; x < 4; ++x) O[x] = mma_64b<__bf16>(first[y], hi[x], O[x]);
#pragma unroll
          for (int x = 2 * y; x < 4; ++x) O[x] = mma_64b<__bf16>(first[y], lo[x], O[x]);
          if constexpr (HALF) {
#pragma unroll
            for (int x = 2 * y; x < 4; ++x) O[x] = mma_64b<__bf16>(second[y], hi[x], O[x]);
          }
        }
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int t = 16 * x + a, at = wave * 16 + 4 * g;
          if (t < live && at < width) {
            const float o[4] = {O[x][0], O[x][1], O[x][2], O[x][3]};
            *reinterpret_cast<u32x2_t*>(out + (int64_t)(t0 + t) * p.o_l + at) = decay_pack<T>(o);
          }
        }
      }
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no copy outlives the workgroup's use of LDS
  if constexpr (!STATE) {
    // tokens behind the sequence's last one
    const int end = p.L - begin < p.seg_len ? p.L - begin : p.seg_len, pieces = width / 8;
    for (int i = tid; i < (end - left) * pieces; i += 64 * NW)
      *reinterpret_cast<u32x4_t*>(out + (int64_t)(left + i / pieces) * p.o_l + i % pieces * 8) = u32x4_t{0, 0, 0, 0};
  }
  float* to = STATE ? p.parts + (bh * (p.segs - 1) + seg) * matrix
              : p.state_out && seg == (n > 0 ? (n - 1) / p.seg_len : 0) ? p.state_out + b * p.so_b + h * p.so_h
                                                                       : nullptr;
  if (!to) return;
#pragma unroll
  for (int f = 0; f < NK; ++f)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (has_state(f, i)) to[state_at(f, i)] = S[f][i];
}

}  // namespace sengine
