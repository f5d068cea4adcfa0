// Tile kernel of cross attention (cross_attention.hip).
//
// The queries that read one key head form rows: row i * group + h is query i of the group's head h.  A
// workgroup takes 16 QF rows a wave of one sequence and key head and a range of its keys, KT keys at a time:
//   S = K Q^T    matrix instructions, keys x rows: a lane has 4 keys a fragment of one row
//   P            exponentials against the row's reference maximum, which is raised (and the sums rescaled)
//                only when a score passes it by 2^8: the result does not depend on the reference.  fp16 weights are
//                those times 2^7: up to 2^15, and down to 2^-31 of the reference before they are lost (kWeightShift)
//   O^T += V^T P^T   the P a lane has is the operand as it lies: the order of the reduction's keys over the
//                lanes is free as long as V's operand, read from LDS transposed, has the same
// K and V are copied into LDS by buffer loads, S tiles in flight.  SHARED: all waves work on the same tile
// and meet once a tile; otherwise (few rows) each wave has tiles and LDS of its own, takes every NW-th tile,
// never meets the others, and their results are joined at the end.  Where a head's row is not whole cache lines and the
// heads lie side by side, HPW key heads share a workgroup and their rows are copied as one: a line that two heads
// share is fetched once (alone they fetched 1.67 times the bytes at d = 48).
//
// A mask is turned into a list of the keys that count, 4096 keys at a time, and only those are fetched: what
// does not count is neither read nor multiplied.  Places of the last tile past the end are filled with zeros
// by the buffer's bounds check and score -infinity.
//
// Bound by, as measured: 4 x 4096 queries x 4001 keys, 16 heads x 128, bf16: 481 us without a mask (1.1 PFLOP/s), 337 to
// 344 with a fifth of the keys and one sequence masked; matrix cores 42 %, vector unit 44 % (the exponentials), LDS
// reads as long as the products.  One query of up to 16384 keys (8 sequences, 8 key heads x 128) 57 us and 64 queries
// of 3136 keys (128 sequences, 8 heads x 48) 113 us: bandwidth, 4.9 and 5.5 TB/s.
//
// The masked kernel of 128 rows keeps 14 of its vector registers in scratch memory at 97 to 128 values (60 bytes a
// lane), that of four merged heads of 32 values 20 bytes; masked kernels keep up to 80 scalar ones in vector registers.
//
// LDS: a key's row has PR 16-byte pieces, piece j at place j ^ f(row): 8 lanes that read a piece of 8 rows, and
// 16 lanes that read 32 bytes of 4 rows, touch every bank once.
#pragma once
#include <type_traits>

#include "lds_copy.h"
#include "token_types.h"

namespace sengine {

using Yes = std::integral_constant<bool, true>;
using No = std::integral_constant<bool, false>;

struct CrossParams {
  const void *q, *k, *v;
  void* out;
  const int32_t* lengths;
  const uint8_t* mask;
  int64_t q_b, q_l, q_h, k_b, k_l, k_h, v_b, v_l, v_h, o_b, o_l, o_h, mask_b;
  int B, Lq, Lk, Hq, Hkv, d;
  float scale;
  int group, rows, blocks;  // rows = Lq * group, in `blocks` row blocks
  int units, inner, unit_heads, spread;  // the order of the workgroups (cross_tile_kernel)
  int parts;                // parts of the keys; more than one: partial results for the join
  float* part_o;            // [part][sequence, key head, row][d], not divided by the sum
  float* part_ml;           // [part][sequence, key head, row][2]: reference (base 2) and sum
};

constexpr int kCrossList = 4096;  // keys of a mask at a time

// The weights are rounded to T for the product with V.  fp16 ends at 2^-24, and many keys that far below the largest
// weigh something together (2^20 keys, 2^-26 each: 1.5 %): the exponent is moved up by what the raised reference leaves
// of the type's range.  It cancels in the division by the sum.  bf16 has fp32's range.
template <class T>
constexpr float kWeightShift = __is_same(T, _Float16) ? 7.f : 0.f;

template <class T>
__device__ __forceinline__ float4_t mma_16(u32x4_t a, u32x4_t b, float4_t c) {
  if constexpr (__is_same(T, _Float16))
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0,
                                                  0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c,
                                                   0, 0, 0);
}

// Largest of the four lanes l, l ^ 16, l ^ 32, l ^ 48.  A swap exchanges one half (32 lanes, or rows of 16)
// of the first register with the other half of the second, so that of two copies one ends with the lane's own
// value and the other with its partner's.  It needs two wait states after its operands are written.
__device__ __forceinline__ float max_of_groups(float x) {
  float y = x;
  asm("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(x), "+v"(y));
  x = fmaxf(x, y);
  y = x;
  asm("s_nop 1\n\tv_permlane16_swap_b32 %0, %1" : "+v"(x), "+v"(y));
  return fmaxf(x, y);
}
template <class T, int DV, int NW, int QF, int KT, int S, int HPW, bool SHARED>
struct CrossTile {
  static constexpr int DK = (DV + 1) / 2;                       // 32-wide steps of q . k
  static constexpr bool MERGED = HPW > 1;                       // a row is that of HPW neighbouring heads, d = 16 DV
  static constexpr int PR = MERGED ? HPW * DV * 2 : DK <= 1 ? 4 : DK <= 2 ? 8 : 16;  // pieces of a row in LDS
  static constexpr int kRow = PR * 16, kOperand = KT * kRow, kStage = 2 * kOperand;
  static constexpr int kAllCopies = 2 * KT * PR / 64;
  static constexpr int WPH = SHARED ? NW / HPW : 1;  // waves, each with rows of its own, of a key head
  static constexpr int kCopies = SHARED ? kAllCopies / NW : kAllCopies;  // of a wave a tile
  static constexpr int kLds = (SHARED ? 1 : NW) * S * kStage;
  static_assert(kAllCopies % (SHARED ? NW : 1) == 0 && KT % 32 == 0 && KT * PR % 64 == 0, "tile");
  static_assert(!MERGED || (PR % 8 == 0 && DV <= 4), "merged rows");
  static_assert(SHARED || (HPW == 1 && NW * 64 * DV * 16 <= kLds), "the waves' results fit");
};

template <class T, int DV, int NW, int QF, int KT, int S, int HPW, bool SHARED, bool LIST, int WPE>
__global__ __launch_bounds__(64 * NW, WPE) void cross_tile_kernel(CrossParams p) {
  using C = CrossTile<T, DV, NW, QF, KT, S, HPW, SHARED>;
  constexpr int DK = C::DK, PR = C::PR, NK = KT / 16;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[C::kLds];
  __shared__ uint16_t list[LIST ? kCrossList : 1];
  __shared__ float joint[SHARED ? 1 : NW][2][16];
  __shared__ int counts[LIST ? NW : 1];
  const int lane = (int)threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int g = lane >> 4, c = lane & 15;

  // workgroup -> unit (sequence, part of the keys, one key head or all) and place in it (row block, key head).
  // Workgroups go to the eight XCDs in turn: a unit stays on one, whose L2 then holds what its workgroups share,
  // and neighbouring units, which are of one sequence and so of one length, go to different ones.
  int unit, in;
  if (p.spread) {
    const int local = (int)blockIdx.x >> 3;
    unit = ((int)blockIdx.x & 7) + 8 * (local / p.inner);
    in = local % p.inner;
    if (unit >= p.units) return;
  } else {
    unit = (int)blockIdx.x / p.inner;
    in = (int)blockIdx.x % p.inner;
  }
  const int block = in % p.blocks;
  int kh = in / p.blocks;
  if (p.unit_heads == 1) {
    kh = unit % (p.Hkv / HPW);
    unit /= p.Hkv / HPW;
  }
  const int kh0 = kh * HPW, hw = SHARED ? wave / C::WPH : 0;  // the workgroup's first key head, the wave's place
  kh = kh0 + hw;
  const int part = unit % p.parts, b = unit / p.parts;

  int n = p.Lk;
  if (p.lengths) {
    const int len = p.lengths[b];
    n = len < 0 ? 0 : len < n ? len : n;
  }
  const int64_t spans = (n + 63) / 64;  // parts take whole 64-key spans
  const int k0 = (int)(spans * part / p.parts) * 64;
  const int64_t kend = spans * (part + 1) / p.parts * 64;
  const int k1 = kend < n ? (int)kend : n;

  // the rows' queries as matrix operands; a negative scale goes into their sign, and one of zero makes them zeros (or
  // NaN, where they are infinite or NaN): with cs = 0 the places past the end, which score -infinity, would be NaN
  const int row0 = (block * C::WPH + (SHARED ? wave % C::WPH : 0)) * 16 * QF;
  u32x4_t q[QF][DK];
  const uint32_t flip = p.scale < 0.f ? 0x80008000u : 0u;
  const bool flat = p.scale == 0.f;
  const float cs = flat ? 1.f : fabsf(p.scale) * 1.4426950408889634f;
#pragma unroll
  for (int f = 0; f < QF; ++f) {
    const int row = row0 + 16 * f + c;
    const T* at = static_cast<const T*>(p.q) + b * p.q_b + (row / p.group) * p.q_l +
                  (kh * p.group + row % p.group) * p.q_h;
#pragma unroll
    for (int t = 0; t < DK; ++t) {
      q[f][t] = u32x4_t{0, 0, 0, 0};
      if (row < p.rows && 32 * t + 8 * g < p.d) {
        q[f][t] = *reinterpret_cast<const u32x4_t*>(at + 32 * t + 8 * g);
#pragma unroll
        for (int i = 0; i < 4; ++i) q[f][t][i] ^= flip;
        if (flat) {
          typedef T vec8_t __attribute__((ext_vector_type(8)));
          vec8_t x = __builtin_bit_cast(vec8_t, q[f][t]);
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] = (T)((float)x[i] * 0.f);
          q[f][t] = __builtin_bit_cast(u32x4_t, x);
        }
      }
    }
  }

  float4_t o[DV][QF];
  float top[QF];
  float4_t total[QF];  // the sum of the weights (all four the same), from a product with ones: of what multiplies V
#pragma unroll
  for (int f = 0; f < QF; ++f) {
    top[f] = -INFINITY;
    total[f] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < DV; ++i) o[i][f] = float4_t{0.f, 0.f, 0.f, 0.f};
  }

  const uint32_t one2 = __is_same(T, _Float16) ? 0x3c003c00u : 0x3f803f80u;
  const u32x4_t ones = u32x4_t{one2, one2, one2, one2};
  uint8_t* ring = smem + (SHARED ? 0 : wave * S * C::kStage);
  const uint32_t ring0 = lds_offset(ring);
  const uint8_t* kbase = reinterpret_cast<const uint8_t*>(static_cast<const T*>(p.k) + b * p.k_b + kh0 * p.k_h);
  const uint8_t* vbase = reinterpret_cast<const uint8_t*>(static_cast<const T*>(p.v) + b * p.v_b + kh0 * p.v_h);
  const int kst = (int)p.k_l * 2, vst = (int)p.v_l * 2;  // bytes between keys
  // where this lane reads K fragments and transposed V fragments
  const int ksw = PR == 4 ? (c >> 1) & 3 : c & 7, hp = C::MERGED ? hw * DV * 2 : 0;  // hp: the head's first piece
  constexpr bool HALF = C::MERGED && DV % 2 == 1;  // the last step of q . k has 16 values: the rest is another head's
  int kat[DK], vat[DV < 4 ? DV : 4];
#pragma unroll
  for (int t = 0; t < DK; ++t)
    kat[t] = c * C::kRow + (((hp + 4 * t + (HALF && t == DK - 1 ? g & 1 : g)) ^ ksw) << 4);
#pragma unroll
  for (int f = 0; f < (DV < 4 ? DV : 4); ++f) {
    const int x = PR == 4 ? (c >> 3) & 1 : c >> 2;
    vat[f] = C::kOperand + (4 * g + (c >> 2)) * C::kRow + (((hp + 2 * f + ((c >> 1) & 1)) ^ (2 * x)) << 4) +
             (c & 1) * 8;
  }

  // All keys.  LATE waves do a tile's exponentials before its neighbour's products, the others after.
  const auto run = [&](auto late) {
    constexpr bool LATE = decltype(late)::value;
    for (int c0 = k0; c0 < k1;) {
      // the keys of this stretch: a list of those that count, or all
      int cnt = k1 - c0, cn = cnt;
      if constexpr (LIST) {
        constexpr int NG = kCrossList / NW / 64;  // 64-key groups of a wave
        cn = cn < kCrossList ? cn : kCrossList;
        const uint8_t* mk = p.mask + b * p.mask_b + c0;
        uint64_t bits[NG];
        int mine = 0;
        __syncthreads();  // the list of the stretch before is no longer read
#pragma unroll
        for (int i = 0; i < NG; ++i) {
          const int key = (wave * NG + i) * 64 + lane;
          bits[i] = __ballot(key < cn && mk[key < cn ? key : 0] != 0);
          mine += __popcll(bits[i]);
        }
        if (lane == 0) counts[wave] = mine;
        __syncthreads();
        int at = 0;
        cnt = 0;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
          at += w < wave ? counts[w] : 0;
          cnt += counts[w];
        }
        cnt = __builtin_amdgcn_readfirstlane(cnt);
#pragma unroll
        for (int i = 0; i < NG; ++i) {
          if (bits[i] >> lane & 1)
            list[at + __popcll(bits[i] & ((1ull << lane) - 1))] = (uint16_t)((wave * NG + i) * 64 + lane);
          at += __popcll(bits[i]);
        }
        __syncthreads();
      }
      const int tiles = (cnt + KT - 1) / KT;
      // This wave's copies: K of tile tk and V of tile tv, into stages sk and sv.  Places past the last key, and tiles
      // past the last or before the first, fetch nothing.
      int off[C::kCopies];
      const auto number = [&](int j) { return SHARED ? wave * C::kCopies + j : j; };
      const auto is_v = [&](int j) { return number(j) >= C::kAllCopies / 2; };
      const auto locate = [&](int tk, int tv) {
#pragma unroll
        for (int j = 0; j < C::kCopies; ++j) {
          const bool v = is_v(j);
          const int place = number(j) % (C::kAllCopies / 2) * 64 + lane, row = place / PR;
          const int sw = v ? (PR == 4 ? (row >> 1 & 1) * 2 : (row & 3) * 2) : (PR == 4 ? row >> 1 & 3 : row & 7);
          const int piece = (place % PR) ^ sw, at = (v ? tv : tk) * KT + row;
          const bool in = (unsigned)at < (unsigned)cnt && (C::MERGED || piece * 8 < p.d);
          int key = row;
          if constexpr (LIST) key = in ? list[at] : 0;
          off[j] = in ? key * (v ? vst : kst) + piece * 16 : 0x7fffff00;
        }
      };
      const auto copy = [&](int tk, int tv, int sk, int sv) {
        const uint8_t* ka = kbase + (LIST ? c0 : c0 + (int64_t)tk * KT) * kst;
        const uint8_t* va = vbase + (LIST ? c0 : c0 + (int64_t)tv * KT) * vst;
#pragma unroll
        for (int j = 0; j < C::kCopies; ++j) {
          const bool v = is_v(j);
          const u32x4_t r = row_buffer(v ? va : ka, 0x7fff0000);
          lds_copy(r, scalar(ring0 + (v ? sv : sk) * C::kStage + number(j) * 1024), off[j]);
        }
      };
      float4_t s[NK][QF];
      u32x4_t pr[KT / 32][QF];
      // O and the sum take on the weights and stage sv's values (V), then the scores of stage sk are formed (K);
      // either may be left out.  Each fragment's operand is read while the products of the one before are made, and
      // no earlier: read further ahead they would not fit the registers.
      const auto products = [&](auto V, int sv, auto K, int sk) {
        constexpr int NVG = decltype(V)::value ? DV : 0, NG = NVG + (decltype(K)::value ? NK : 0);
        const uint8_t *va = ring + sv * C::kStage, *ka = ring + sk * C::kStage;
        u32x4_t vf[2][KT / 32], kf[2][DK];
        const auto read = [&](int n) {
          if (n < NVG) {
#pragma unroll
            for (int u = 0; u < KT / 32; ++u) {
              const uint8_t* at = va + vat[n & 3] + (n >> 2) * 128 + u * 32 * C::kRow;
              vf[n & 1][u] = read_transposed(at, at + 16 * C::kRow);
            }
          } else if (n < NG) {
#pragma unroll
            for (int u = 0; u < DK; ++u)
              kf[n & 1][u] = *reinterpret_cast<const u32x4_t*>(ka + (n - NVG) * 16 * C::kRow + kat[u]);
          }
        };
        read(0);
        if constexpr (NVG > 0) {
#pragma unroll
          for (int u = 0; u < KT / 32; ++u)
#pragma unroll
            for (int f = 0; f < QF; ++f) total[f] = mma_16<T>(ones, pr[u][f], total[f]);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int n = 0; n < NG; ++n) {
          read(n + 1);
          __builtin_amdgcn_sched_barrier(0);
          if (n < NVG) {
#pragma unroll
            for (int u = 0; u < KT / 32; ++u)
#pragma unroll
              for (int f = 0; f < QF; ++f) o[n][f] = mma_16<T>(vf[n & 1][u], pr[u][f], o[n][f]);
          } else {
            const int i = n - NVG;
            if constexpr (HALF) {
#pragma unroll
              for (int e = 0; e < 4; ++e) kf[n & 1][DK - 1][e] = g < 2 ? kf[n & 1][DK - 1][e] : 0;
            }
#pragma unroll
            for (int f = 0; f < QF; ++f) s[i][f] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int u = 0; u < DK; ++u)
#pragma unroll
              for (int f = 0; f < QF; ++f) s[i][f] = mma_16<T>(kf[n & 1][u], q[f][u], s[i][f]);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      };
      const auto weights = [&](int t) {
        const int left = cnt - t * KT;
        if (left < KT) {
#pragma unroll
          for (int i = 0; i < NK; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (16 * i + 4 * g + e >= left) {
#pragma unroll
                for (int f = 0; f < QF; ++f) s[i][f][e] = -INFINITY;
              }
        }
        float high[QF];
        bool raise = false;
#pragma unroll
        for (int f = 0; f < QF; ++f) {
          high[f] = fmaxf(fmaxf(s[0][f][0], s[0][f][1]), s[0][f][2]);  // three at a time
          high[f] = fmaxf(fmaxf(s[0][f][3], s[1][f][0]), high[f]);
          high[f] = fmaxf(fmaxf(s[1][f][1], s[1][f][2]), high[f]);
          if constexpr (NK == 2) {
            high[f] = fmaxf(s[1][f][3], high[f]);
          } else {
            high[f] = fmaxf(fmaxf(s[1][f][3], s[2][f][0]), high[f]);
            high[f] = fmaxf(fmaxf(s[2][f][1], s[2][f][2]), high[f]);
            high[f] = fmaxf(fmaxf(s[2][f][3], s[3][f][0]), high[f]);
            high[f] = fmaxf(fmaxf(s[3][f][1], s[3][f][2]), high[f]);
            high[f] = fmaxf(s[3][f][3], high[f]);
          }
          high[f] = max_of_groups(high[f]) * cs;
          raise |= high[f] > top[f] + 8.f;
        }
        if (__any(raise)) {
#pragma unroll
          for (int f = 0; f < QF; ++f) {
            const float t1 = fmaxf(top[f], high[f]);
            const float back = t1 == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(top[f] - t1);
            top[f] = t1;
            total[f] *= back;
#pragma unroll
            for (int i = 0; i < DV; ++i)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[i][f][e] *= back;
          }
        }
#pragma unroll
        for (int f = 0; f < QF; ++f) {
          // (every score so far is -infinity: they weigh nothing)
          const float ref = top[f] == -INFINITY ? 0.f : kWeightShift<T> - top[f];
#pragma unroll
          for (int u = 0; u < KT / 32; ++u) {
            typedef T vec8_t __attribute__((ext_vector_type(8)));
            vec8_t x;
#pragma unroll
            for (int e = 0; e < 8; ++e)
              x[e] = (T)__builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * u + e / 4][f][e % 4], cs, ref));
            pr[u][f] = __builtin_bit_cast(u32x4_t, x);
          }
        }
      };
      if constexpr (SHARED) {
        // Between meetings t and t + 1 the waves need K of tile t and V of tile t - 1, which meeting t finds landed;
        // K up to t + S - 1 and V up to t + S - 2 are on their way.  The later half of eight waves, which share the
        // SIMDs with the earlier half, does its exponentials first and its products after, so that one half's vector
        // work goes with the other's matrix work.
        int sk = 0, sv = S - 1;  // stages of K of tile t and of V of tile t - 1
        const auto meet = [&](int t) {
          locate(t + S - 1, t + S - 2);
          asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"i"((S - 2) * C::kCopies) : "memory");
          __builtin_amdgcn_s_barrier();
          asm volatile("" ::: "memory");
          copy(t + S - 1, t + S - 2, sv, sv == 0 ? S - 1 : sv - 1);
        };
        const auto next = [&] {
          sv = sk;
          sk = sk + 1 == S ? 0 : sk + 1;
        };
        if (tiles > 0) {
#pragma unroll
          for (int u = 0; u < S - 1; ++u) {
            locate(u, u - 1);
            copy(u, u - 1, u, u == 0 ? S - 1 : u - 1);
          }
          meet(0);
          products(No{}, 0, Yes{}, 0);
          if (!LATE) weights(0);
          for (int t = 1; t < tiles; ++t) {
            next();
            meet(t);
            if (LATE) weights(t - 1);
            products(Yes{}, sv, Yes{}, sk);
            if (!LATE) weights(t);
          }
          next();
          meet(tiles);
          if (LATE) weights(tiles - 1);
          products(Yes{}, sv, No{}, 0);
          asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the copies past the end
        }
        __syncthreads();
      } else {
        // tile i of this wave is tile wave + i * NW of the stretch
        const int own = (tiles - wave + NW - 1) / NW;
        const auto fetch = [&](int i, int stage) {
          locate(wave + i * NW, wave + i * NW);
          copy(wave + i * NW, wave + i * NW, stage, stage);
        };
        int stage = 0;
#pragma unroll
        for (int i = 0; i < S - 1; ++i) fetch(i, i);
        for (int i = 0; i < own; ++i) {
          asm volatile("s_waitcnt vmcnt(%0)" ::"i"((S - 2) * C::kCopies) : "memory");
          fetch(i + S - 1, stage == 0 ? S - 1 : stage - 1);
          products(No{}, 0, Yes{}, stage);
          weights(wave + i * NW);
          products(Yes{}, stage, No{}, 0);
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the stage is read before it is filled again
          stage = stage + 1 == S ? 0 : stage + 1;
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the copies past the end
      }
      c0 += cn;
    }
  };
  // (code of its own for each half: branches inside the loop would move the sums between registers)
  if (SHARED && NW == 8 && wave >= 4)
    run(Yes{});
  else
    run(No{});

  if constexpr (!SHARED) {
    static_assert(QF == 1, "one fragment of rows");
    // join the waves: a common reference, sums and rows of O added up in the waves' order
    if (g == 0) {
      joint[wave][0][c] = top[0];
      joint[wave][1][c] = total[0][0];
    }
    __syncthreads();
    float t1 = joint[0][0][c];
#pragma unroll
    for (int w = 1; w < NW; ++w) t1 = fmaxf(t1, joint[w][0][c]);
    const float back = top[0] == -INFINITY ? (total[0][0] == 0.f ? 0.f : 1.f) : __builtin_amdgcn_exp2f(top[0] - t1);
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float tw = joint[w][0][c];
      sum += joint[w][1][c] * (tw == -INFINITY ? (joint[w][1][c] == 0.f ? 0.f : 1.f) : __builtin_amdgcn_exp2f(tw - t1));
    }
    top[0] = t1;
    total[0][0] = sum;
    float4_t* mine = reinterpret_cast<float4_t*>(smem) + wave * DV * 64 + lane;
#pragma unroll
    for (int i = 0; i < DV; ++i) mine[i * 64] = o[i][0] * back;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < DV; ++i) {
      if (i % NW != wave) continue;
      const float4_t* all = reinterpret_cast<const float4_t*>(smem) + i * 64 + lane;
      o[i][0] = all[0];
#pragma unroll
      for (int w = 1; w < NW; ++w) o[i][0] += all[w * DV * 64];
    }
  }
#pragma unroll
  for (int f = 0; f < QF; ++f) {
    const int row = row0 + 16 * f + c;
    if (row >= p.rows) continue;
    if (p.parts > 1) {
      const int64_t r = (((int64_t)part * p.B + b) * p.Hkv + kh) * p.rows + row;
      if (g == 0 && (SHARED || wave == 0)) {
        p.part_ml[2 * r] = top[f];
        p.part_ml[2 * r + 1] = total[f][0];
      }
#pragma unroll
      for (int i = 0; i < DV; ++i)
        if ((SHARED || i % NW == wave) && 16 * i + 4 * g < p.d)
          *reinterpret_cast<float4_t*>(p.part_o + r * p.d + 16 * i + 4 * g) = o[i][f];
    } else {
      const float inv = total[f][0] == 0.f ? 0.f : 1.f / total[f][0];
      T* out = static_cast<T*>(p.out) + b * p.o_b + (row / p.group) * p.o_l + (kh * p.group + row % p.group) * p.o_h;
#pragma unroll
      for (int i = 0; i < DV; ++i)
        if ((SHARED || i % NW == wave) && 16 * i + 4 * g < p.d) {
          const float x[4] = {o[i][f][0] * inv, o[i][f][1] * inv, o[i][f][2] * inv, o[i][f][3] * inv};
          store_floats<T, 4>(out + 16 * i + 4 * g, x);
        }
    }
  }
}

// Joins the parts of a row, one wave each: lane i has part i's reference and sum, then 32 lanes take 4 columns each
// of every second part.  256 rows of 8 parts of 128 values: 4.9 us.
constexpr int kCrossParts = 64;
template <class T>
__global__ __launch_bounds__(64) void cross_join_kernel(CrossParams p) {
  const int64_t rows = (int64_t)p.B * p.Hkv * p.rows, r = blockIdx.x;
  const int lane = (int)threadIdx.x, at = (lane & 31) * 4;
  float t = -INFINITY, l = 0.f;
  if (lane < p.parts) {
    t = p.part_ml[2 * (lane * rows + r)];
    l = p.part_ml[2 * (lane * rows + r) + 1];
  }
  float top = t;
#pragma unroll
  for (int x = 32; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor(top, x, 64));
  const float w = t == -INFINITY ? (l == 0.f ? 0.f : 1.f) : __builtin_amdgcn_exp2f(t - top);
  float total = l * w;
#pragma unroll
  for (int x = 32; x > 0; x >>= 1) total += __shfl_xor(total, x, 64);
  float4_t o = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
  for (int i0 = 0; i0 < p.parts; i0 += 2) {
    const int i = i0 + (lane >> 5);
    const float wi = __shfl(w, i & 63, 64);
    if (i < p.parts && at < p.d) o += *reinterpret_cast<const float4_t*>(p.part_o + (i * rows + r) * p.d + at) * wi;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e] += __shfl_xor(o[e], 32, 64);
  if (lane >= 32 || at >= p.d) return;
  const float inv = total == 0.f ? 0.f : 1.f / total;
  const int row = (int)(r % p.rows), kh = (int)(r / p.rows % p.Hkv);
  const int64_t b = r / p.rows / p.Hkv;
  const float x[4] = {o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv};
  store_floats<T, 4>(static_cast<T*>(p.out) + b * p.o_b + (row / p.group) * p.o_l +
                         (kh * p.group + row % p.group) * p.o_h + at, x);
}

}  // namespace sengine
