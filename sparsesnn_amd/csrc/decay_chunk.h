// Decaying linear attention 64 tokens at a time (decay_attention.hip).  With a chunk's rows Q, K, V and the state S that
// it begins with,
//   O  = scale ((Q K^T . D) V + L Q S),   D[i][j] = g^(i - j) for j <= i, else 0,   L[i] = g^(i + 1)
//   S' = g^n S + K^T W V,                 W[j] = g^(n - 1 - j)
// Workgroup = one head of one sequence, or of a segment of it, and up to 128 columns of V; a wave has 16 or 32 columns of V,
// S and O, and S stays in its registers.  The memory pipeline copies a chunk's rows into LDS once those before have been
// read, and several workgroups a CU fill each other's waits.  The ten 16 x 16 blocks of Q K^T . D that count are shared out
// over the waves and go through LDS; while they are made, the other products need only what the wave has.
//
// Few heads: a first pass makes each segment's state from a state of zeros (K and V only, copies one chunk ahead), and
// decay_scan_kernel joins them, so that K and V are read twice.
//
// Measured: 16 heads of 128 x 128 over 65536 tokens, bf16, in 32 segments: 122 us (4.4 TB/s), 12 and 312 (3.4 TB/s; matrix
// cores 38 %, vector unit 40 %, waves waiting 31 %).  64 heads of 48 x 48 over 12544 tokens, fp16, in 16 segments: 45, 6 and 107
// (2.9 TB/s; 12 %, 30 %, 40 %: a chunk's products, splits and reads follow each other in a wave, and LDS and registers leave
// three waves a SIMD).
//
// All products are 16x16x32 matrix instructions, laid out so that what one leaves is what the next one takes:
//   * K Q^T puts four tokens j of one token i in a lane: two such blocks, side by side in LDS, are the second operand of
//     the product with V^T (its tokens in the order 4 g .. 4 g + 3, 16 + 4 g ..), V^T and K^T are read transposed;
//   * K^T (W V) has its rows, dk, permuted so that a lane ends with eight neighbouring ones of a column: as they lie they
//     are the operand of S^T Q^T.
//
// Rounding.  S is fp32.  What a 16-bit instruction takes of it, and W V, which makes it, are in bf16 sums of three values,
// which have all of its 24 bits whatever the age of a token: later keys may be small or zero, so that an early token is all
// that a state holds, and outputs may be differences of its values.  (Two instead of three: 400 us for 424 at 65536 tokens of
// 16 heads of 128 x 128, 77 for 79 at 8 x 1000; outputs 1.1e-4 for 5.5e-5 of the exact ones' size from those, rounded.)
// In fp16 they are sums of two: 22 bits, S with a column scaled by a power of two to fp16's range; of W V the second one is
// 2^11 times larger, so that a token is off by at most |k| 2^-36 on top, where the decay has taken it below the type's range.
// The fp32 weights Q K^T . D, which only their own chunk sees, are sums of two bf16 values, 16 bits, on both types, as they
// easily pass fp16's range, and fp16 values of V are sums of two of them, exactly; all four products count.
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
  float* begun;        // (B, H) copies of a state that is updated in place, or null
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

// Columns of V of a workgroup, in 16s; how many of them a wave has, and the waves a SIMD that its registers are limited to.
// Measured, us: 64 columns, 64 heads of 64 over 12544 tokens, bf16: a wave 16 columns and two waves a SIMD 157, three 168, 32
// columns 189; 48 columns of fp16: three 155, two 166; 128 columns, 16 heads of 128 over 65536 tokens: a wave 32 columns 438,
// 16 columns 523; the same in fp16, where 32 columns keep 38 registers in memory, 472 and 518.  Keys of more than 64 values do
// not fit three waves a SIMD: 4 x 6000 tokens, 16 heads of 128 x 48, fp16 three 213, two 123 (bf16 156, 120), 128 x 32 108, 104.
__host__ __device__ constexpr int decay_blocks(int dv) { return dv <= 32 ? 2 : dv <= 48 ? 3 : dv <= 64 ? 4 : 8; }
__host__ __device__ constexpr int decay_own(int blocks) { return blocks == 8 ? 2 : 1; }
__host__ __device__ constexpr int decay_waves(int dk, int blocks) { return blocks < 4 && dk <= 64 ? 3 : 2; }

// Workgroups that a CU holds.
inline int decay_resident(int dk, int dv) {
  const int blocks = decay_blocks(dv), pk = dk <= 32 ? 4 : dk <= 64 ? 8 : 16, pv = blocks == 3 ? 8 : blocks * 2;
  const int by_lds = 160 / (2 * pk + pv + 12 + 1), by_waves = 4 * decay_waves(dk, blocks) / (blocks / decay_own(blocks));
  return by_lds < by_waves ? by_lds : by_waves;
}

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
  for (int e = 0; e < N; ++e) {
    if constexpr (__is_same(T, __bf16)) {
      // x - v by the instruction that adds a pair's products to x: a widened v would take one more.  (A neighbour that is
      // not finite makes x a NaN: the sum that both belong to is one anyway.)  The factors (-1, 0) and (0, -1) are kept
      // from the compiler, which takes the first for its inline constant -1, of which the instruction has the other half.
      typedef __bf16 pair_t __attribute__((ext_vector_type(2)));
      uint32_t minus = e % 2 ? 0xbf800000u : 0x0000bf80u;
      asm("" : "+s"(minus));
      const uint32_t word = r[e / 2];
      x[e] = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(pair_t, word), __builtin_bit_cast(pair_t, minus), x[e], false);
    } else {
      x[e] = __builtin_fmaf((float)v[e], -1.f, x[e]);
    }
  }
  return r;
}

// A power of two that brings values up to `most` (its bits, the sign cleared) to fp16's upper range, and its inverse.
__device__ __forceinline__ void decay_range(uint32_t most, float& up, float& down) {
  int e = (int)(most >> 23);
  e = e < 15 ? 15 : e;  // both stay normal values
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

// Place of the operand of tokens j 32 y .. of the tokens i of block x.
__device__ __forceinline__ int decay_operand(int x, int y) { return x < 2 ? x : 2 * x - 2 + y; }

// DKP: dk rounded up to 32, 64 or 128; NW waves of 16 NV columns.  STATE: a segment's state from a state of zeros,
// without outputs.
template <class T, int DKP, int NV, int NW, bool STATE>
__global__ __launch_bounds__(64 * NW, STATE ? 4 : decay_waves(DKP, NV * NW)) void decay_chunk_kernel(DecayParams p) {
  constexpr bool HALF = __is_same(T, _Float16);
  constexpr int C = kDecayChunk, STAGES = STATE ? 2 : 1;
  constexpr int TERMS = HALF ? 2 : 3;  // values of T that the state's products take for one of it
  constexpr int PK = DKP / 8, PV = NV * NW == 3 ? 8 : NV * NW * 2;  // pieces of a row of Q or K, of V
  constexpr int NM = DKP / 32, NK = DKP / 16;
  constexpr int NC = PK * (STATE ? 1 : 2) + PV, NCW = (NC + NW - 1) / NW;  // copies of 1 KB a chunk, of a wave
  constexpr int kStage = NC * 1024;
  constexpr int kQ = (PK + PV) * 1024;  // a stage: K, V, Q
  constexpr int kP = 6 * 1024;          // blocks of Q K^T . D: six operands' first terms, then their second ones
  __shared__ __attribute__((aligned(1024))) uint8_t smem[STAGES * kStage + (STATE ? 0 : 2 * kP)];
  __shared__ float powers[16 + C + 1], behind[2 * C];  // scale g^(n - 16), zeros up to there; g^(C - 1 - j), zeros behind
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
  if (left > 0) copy(0, 0);  // on their way beside the powers and the state

  // powers of the decay as the lanes need them
  const float lg = decay_log2(p.decay[h]);
  for (int i = tid; i < 2 * C; i += 64 * NW) {
    if (i <= 16 + C) powers[i] = i < 16 ? 0.f : p.scale * decay_power(lg, i - 16);
    behind[i] = i < C ? decay_power(lg, C - 1 - i) : 0.f;
  }
  // blocks above the diagonal that share an operand with one that counts stay zeros
  for (int i = tid; i < (STATE ? 0 : 2 * kP / 16); i += 64 * NW)
    *reinterpret_cast<u32x4_t*>(smem + STAGES * kStage + i * 16) = u32x4_t{0, 0, 0, 0};

  // S: value i of fragment [f][c] is row 32 (f / 2) + 8 g + 4 (f % 2) + i, column 16 c + a of the wave's
  const int column = wave * 16 * NV + a;
  const bool used = wave * 16 * NV < width;  // whether the wave has columns
  float4_t S[NK][NV];
  const auto state_at = [&](int f, int c, int i) {
    return (int64_t)(32 * (f / 2) + 8 * g + 4 * (f % 2) + i) * p.dv + slice * kDecayColumns + column + 16 * c;
  };
  const auto has_state = [&](int f, int c, int i, int dk) {
    return 32 * (f / 2) + 8 * g + 4 * (f % 2) + i < dk && column + 16 * c < width;
  };
  const int64_t bh = b * p.H + h;
  const int64_t matrix = (int64_t)p.dk * p.dv;
  const float* from = STATE ? nullptr
                      : seg > 0 ? (left > 0 ? p.parts + (bh * (p.segs - 1) + seg - 1) * matrix : nullptr)
                      : p.begun ? p.begun + bh * matrix
                      : p.state ? p.state + b * p.s_b + h * p.s_h
                                : nullptr;
#pragma unroll
  for (int f = 0; f < NK; ++f)
#pragma unroll
    for (int c = 0; c < NV; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) S[f][c][i] = from && has_state(f, c, i, p.dk) ? from[state_at(f, c, i)] : 0.f;

  // Where in LDS a lane's share begins: of 16 rows, their values 32 m + 8 g ..; of 32 tokens transposed, the columns 32 m + 8 p
  // .. (p = a % 4) of K and 16 c .. of the wave's of V.  What else an address has is the same for all lanes.
  int at_rows[NM], at_k[NM], at_v[NV];
#pragma unroll
  for (int m = 0; m < NM; ++m) {
    at_rows[m] = decay_at<PK>(a, 4 * m + g);
    at_k[m] = decay_at<PK>(4 * g + (a >> 2), 4 * m + (a & 3));
  }
#pragma unroll
  for (int c = 0; c < NV; ++c)
    at_v[c] = PK * 1024 + decay_at<PV>(4 * g + (a >> 2), 2 * (wave * NV + c) + ((a & 3) >> 1)) + 8 * (a & 1);
  const auto transposed = [&](int at, int pitch) { return read_transposed(smem + at, smem + at + 16 * pitch); };
  const auto meet = [&]() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };

  uint8_t* const sP = smem + STAGES * kStage;
  int t0 = 0, stage = 0;
  while (t0 < left) {
    // this wave's copies have landed and its reads of the blocks are done; so are all waves'
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    meet();
    if (STAGES == 2 && t0 + C < left) copy(t0 + C, stage ^ 1);
    const int at0 = STAGES == 2 ? stage * kStage : 0;
    const int live = left - t0 < C ? left - t0 : C;

    if constexpr (!STATE) {
      // Blocks of K Q^T . D: tokens j of block y, i of block x >= y; the wave's are number wave, wave + NW, ..
      constexpr int NB = (10 + NW - 1) / NW;
      float4_t P[NB];
      int bx[NB], by[NB];
      int first = wave;
      asm("" : "+s"(first));  // what follows from it is made here, not kept in registers from chunk to chunk
#pragma unroll
      for (int u = 0; u < NB; ++u) {
        const int at = first + u * NW < 10 ? first + u * NW : 9;
        bx[u] = at < 1 ? 0 : at < 3 ? 1 : at < 6 ? 2 : 3;
        by[u] = at - bx[u] * (bx[u] + 1) / 2;
        P[u] = float4_t{0.f, 0.f, 0.f, 0.f};
      }
#pragma unroll
      for (int m = 0; m < NM; ++m)
#pragma unroll
        for (int u = 0; u < NB; ++u)
          P[u] = mma_64b<T>(*reinterpret_cast<const u32x4_t*>(smem + at_rows[m] + by[u] * 16 * PK * 16),
                            *reinterpret_cast<const u32x4_t*>(smem + kQ + at_rows[m] + bx[u] * 16 * PK * 16), P[u]);
#pragma unroll
      for (int u = 0; u < NB; ++u) {
        const int ahead = 16 * (bx[u] - by[u]) + a - 4 * g;
        float w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = ahead >= i ? P[u][i] * powers[16 + ahead - i] : 0.f;  // whatever a later token holds
        const u32x2_t hi = decay_term<__bf16>(w), lo = decay_pack<__bf16>(w);
        if (first + u * NW < 10) {
          uint8_t* const at = sP + (decay_operand(bx[u], by[u] / 2) * 64 + lane) * 16 + by[u] % 2 * 8;
          *reinterpret_cast<u32x2_t*>(at) = hi;
          *reinterpret_cast<u32x2_t*>(at + kP) = lo;
        }
      }
    }

    u32x4_t V[2][NV];  // tokens 32 x .., columns 16 c ..
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int c = 0; c < NV; ++c)
        V[x][c] = transposed(at0 + at_v[c] + x * 32 * PV * 16, PV * 16);
    float4_t O[4][NV];
    if constexpr (!STATE) {
#pragma unroll
      for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int c = 0; c < NV; ++c) O[x][c] = float4_t{0.f, 0.f, 0.f, 0.f};
      if (used) {  // S^T Q^T
        float up[NV], down[NV];
#pragma unroll
        for (int c = 0; c < NV; ++c) {
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
          u32x4_t part[NV][TERMS], r[4];
#pragma unroll
          for (int c = 0; c < NV; ++c) {
            float s[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) s[e] = HALF ? S[2 * m + e / 4][c][e % 4] * up[c] : S[2 * m + e / 4][c][e % 4];
#pragma unroll
            for (int u = 0; u < TERMS - 1; ++u) part[c][u] = decay_term<T>(s);
            part[c][TERMS - 1] = decay_pack<T>(s);
          }
#pragma unroll
          for (int x = 0; x < 4; ++x)
            r[x] = *reinterpret_cast<const u32x4_t*>(smem + kQ + at_rows[m] + x * 16 * PK * 16);
#pragma unroll
          for (int u = 0; u < TERMS; ++u)
#pragma unroll
            for (int x = 0; x < 4; ++x)
#pragma unroll
              for (int c = 0; c < NV; ++c) O[x][c] = mma_64b<T>(part[c][u], r[x], O[x][c]);
        }
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const float begun = powers[16 + 16 * x + a + 1];  // scale L
#pragma unroll
          for (int c = 0; c < NV; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i)  // a column's factor where O has it
              O[x][c][i] *= HALF ? begun * __shfl(down[c], 4 * g + i, 64) : begun;
        }
      }
    }
    if (used) {  // S' = g^n S + K^T W V
      const float passed = decay_power(lg, live);
#pragma unroll
      for (int f = 0; f < NK; ++f)
#pragma unroll
        for (int c = 0; c < NV; ++c) S[f][c] *= passed;
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        u32x4_t w[NV][TERMS];
#pragma unroll
        for (int c = 0; c < NV; ++c) {
          typedef T vec_t __attribute__((ext_vector_type(8)));
          const vec_t t = __builtin_bit_cast(vec_t, V[x][c]);
          float y[8];
#pragma unroll
          for (int e = 0; e < 8; ++e)  // weights count from the chunk's last token
            y[e] = (float)t[e] * behind[C - live + 32 * x + 16 * (e / 4) + 4 * g + e % 4];
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
        constexpr int G = NK < 4 ? NK : 4;  // fragments at a time, so that none waits for its own sums
#pragma unroll
        for (int f0 = 0; f0 < NK; f0 += G) {
          u32x4_t r[G];
#pragma unroll
          for (int f = 0; f < G; ++f)
            r[f] = transposed(at0 + at_k[(f0 + f) / 2] + 8 * ((f0 + f) % 2) + x * 32 * PK * 16, PK * 16);
#pragma unroll
          for (int c = 0; c < NV; ++c) {
#pragma unroll
            for (int f = 0; f < G; ++f) S[f0 + f][c] = mma_64b<T>(r[f], w[c][0], S[f0 + f][c]);
            if constexpr (HALF) {
              float4_t rest[G];
#pragma unroll
              for (int f = 0; f < G; ++f) rest[f] = mma_64b<T>(r[f], w[c][1], float4_t{0.f, 0.f, 0.f, 0.f});
#pragma unroll
              for (int f = 0; f < G; ++f)
#pragma unroll
                for (int i = 0; i < 4; ++i) S[f0 + f][c][i] = __builtin_fmaf(rest[f][i], 1.f / 2048.f, S[f0 + f][c][i]);
            } else {
#pragma unroll
              for (int u = 1; u < TERMS; ++u)
#pragma unroll
                for (int f = 0; f < G; ++f) S[f0 + f][c] = mma_64b<T>(r[f], w[c][u], S[f0 + f][c]);
            }
          }
        }
      }
    }
    if constexpr (!STATE) {
      if (used) {
        // a value that is not finite, times zero, is not a number in its row
        float4_t odd = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int c = 0; c < NV; ++c) odd = mma_64b<T>(V[x][c], u32x4_t{0, 0, 0, 0}, odd);
        const float any = (odd[0] + odd[1]) + (odd[2] + odd[3]);
        if (__builtin_expect(__any(any != any), 0)) {
          // its token's outputs and later ones: how many such values there are up to each token, by ones
          constexpr uint16_t one = HALF ? 0x3c00u : 0x3f80u;
#pragma unroll
          for (int c = 0; c < NV; ++c) {
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              float4_t count = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
              for (int y = 0; y <= x / 2; ++y) {
                float w[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) w[e] = 32 * y + 16 * (e / 4) + 4 * g + e % 4 <= 16 * x + a ? 1.f : 0.f;
                count = mma_64b<T>(decay_replace<T, false>(V[y][c], one), decay_pack<T>(w), count);
              }
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (count[i] > 0.f) O[x][c][i] = __builtin_nanf("");
            }
#pragma unroll
            for (int y = 0; y < 2; ++y) V[y][c] = decay_replace<T, true>(V[y][c], 0);
          }
        }
      }
    }
    if constexpr (!STATE) meet();  // the blocks are written, and K, V and Q have been read
    if (!STATE && t0 + C < left) copy(t0 + C, 0);
    if constexpr (!STATE) {
      if (used) {  // (Q K^T . D) V
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          u32x4_t first[NV], second[NV], hi[4], lo[4];
#pragma unroll
          for (int c = 0; c < NV; ++c) {
            first[c] = V[y][c];
            if constexpr (HALF) {
              typedef T vec_t __attribute__((ext_vector_type(8)));
              const vec_t t = __builtin_bit_cast(vec_t, V[y][c]);
              float s[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) s[e] = (float)t[e];
              first[c] = decay_term<__bf16>(s);
              second[c] = decay_pack<__bf16>(s);
            }
          }
#pragma unroll
          for (int x = 2 * y; x < 4; ++x) {
            hi[x] = *reinterpret_cast<const u32x4_t*>(sP + (decay_operand(x, y) * 64 + lane) * 16);
            lo[x] = *reinterpret_cast<const u32x4_t*>(sP + kP + (decay_operand(x, y) * 64 + lane) * 16);
          }
#pragma unroll
          for (int x = 2 * y; x < 4; ++x)
#pragma unroll
            for (int c = 0; c < NV; ++c) O[x][c] = mma_64b<__bf16>(first[c], hi[x], O[x][c]);
#pragma unroll
          for (int x = 2 * y; x < 4; ++x)
#pragma unroll
            for (int c = 0; c < NV; ++c) O[x][c] = mma_64b<__bf16>(first[c], lo[x], O[x][c]);
          if constexpr (HALF) {
#pragma unroll
            for (int x = 2 * y; x < 4; ++x)
#pragma unroll
              for (int c = 0; c < NV; ++c) O[x][c] = mma_64b<__bf16>(second[c], hi[x], O[x][c]);
#pragma unroll
            for (int x = 2 * y; x < 4; ++x)
#pragma unroll
              for (int c = 0; c < NV; ++c) O[x][c] = mma_64b<__bf16>(second[c], lo[x], O[x][c]);
          }
        }
      }
      if (used) {
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int t = 16 * x + a;
          if (t >= live) continue;
          T* const row = out + (int64_t)(t0 + t) * p.o_l + wave * 16 * NV + 4 * g;
#pragma unroll
          for (int c = 0; c < NV; ++c) {
            if (wave * 16 * NV + 16 * c + 4 * g >= width) continue;
            const float o[4] = {O[x][c][0], O[x][c][1], O[x][c][2], O[x][c][3]};
            *reinterpret_cast<u32x2_t*>(row + 16 * c) = decay_pack<T>(o);
          }
        }
      }
    }
    t0 += C;
    stage ^= STAGES - 1;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no copy outlives the workgroup's use of LDS
  if constexpr (!STATE) {
    // tokens behind the sequence's last one
    const int end = p.L - begin < p.seg_len ? p.L - begin : p.seg_len, pieces = width / 8;
    for (int64_t i = tid; i < (int64_t)(end - left) * pieces; i += 64 * NW)
      *reinterpret_cast<u32x4_t*>(out + (left + i / pieces) * p.o_l + i % pieces * 8) = u32x4_t{0, 0, 0, 0};
  }
  float* to = STATE ? p.parts + (bh * (p.segs - 1) + seg) * matrix
              : p.state_out && seg == (n > 0 ? (n - 1) / p.seg_len : 0) ? p.state_out + b * p.so_b + h * p.so_h
                                                                       : nullptr;
  if (!to) return;
  int dk = p.dk;
  asm("" : "+s"(dk));  // the comparisons are made again, not kept from the state's loading on
#pragma unroll
  for (int f = 0; f < NK; ++f)
#pragma unroll
    for (int c = 0; c < NV; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (has_state(f, c, i, dk)) to[state_at(f, c, i)] = S[f][c][i];
}

}  // namespace sengine
