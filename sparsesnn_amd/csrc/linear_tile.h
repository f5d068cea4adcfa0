// Tile kernel of the linear operator (linear.hip): workgroup = BM token rows x BN weight rows, a grid
// of WM x WN waves, each wave TM x TN fragments of 16 x 16.
//
// Per 128 bytes of the reduction both operands' rows are copied into one of S LDS stages by
// buffer_load ... lds, 16 bytes a lane; out-of-range lanes (rows past the end, the reduction's tail)
// receive zeros from the buffer's bounds check.  LDS row r keeps its 16-byte piece j at place
// j ^ (r % 8): eight lanes copy one row's 128 bytes and the 16 lanes that read piece j of
// 16 rows touch every bank evenly.
//
// The stage's rows of a wave are read in four quarters, A = weight rows, B = token rows, each halved:
//   A-lo B-first | A-lo B-second | A-hi B-second | A-hi B-first
// so that each quarter's products need only one new half, which is read during the quarter before it.
// In the middle of the third quarter all reads of the stage are done: there the workgroup meets once, and
// beside the rest of the step's products the freed stage is refilled and the next stage's first operands
// are read.  The second half of B becomes the first of the next step.
//
// Bound by, as measured: 256 x 256 tiles: 8192 x 4096 x 8192 bf16 418 to 424 us (1.31 PFLOP/s), 8192^3 e4m3
// 447 (2.46): matrix cores and the clock that they leave; without the copies 8192^3 bf16 takes 757 of 857 us.
// A wave of 128 x 128 needs two thirds of the LDS reads of eight waves of 128 x 64.  128 x 128 tiles:
// 100352 x 1536 x 384 fp16 with GELU 248 us, 22 a step and 130 for the starts, epilogues and stores of 9408
// tiles.  64 x 64 tiles: 0.2 us a step, three workgroups a CU.  Stages of 64 bytes, twice as many, are
// slower everywhere (8192^3 bf16 974 us): twice the meetings, half lines.
//
// Weight rows are placed so that a lane ends with 8 consecutive output columns: row 16 b + 4 g + e of
// 32 LDS rows holds weight row 8 g + 4 b + e, and value e of fragment (b = i % 2) in lane group g is
// then column 8 g + 4 b + e.
#pragma once
#include "lds_copy.h"
#include "linear.h"

namespace sengine {

constexpr int kLinStep = 128;  // bytes of the reduction a step


// Workgroup -> tile.  Each XCD walks kLinGroup row tiles before the next column tile, so that what runs on it
// at a time is a block of tiles whose operands stay in its L2.
constexpr int kLinGroup = 4;
__device__ __forceinline__ void linear_tile_of(int id, int ntm, int ntn, int& mt, int& nt) {
  const int t = xcd_order(id, ntm * ntn);
  const int group = t / (kLinGroup * ntn), first = group * kLinGroup;
  const int rows = ntm - first < kLinGroup ? ntm - first : kLinGroup;
  const int at = t - first * ntn;
  nt = at / rows;
  mt = first + at - nt * rows;
}

// c += a b on one fragment, in place.  As asm the sums stay in the accumulation registers they have:
// with 64 fragments there are no others to move them through.  The compiler knows neither that this is a
// matrix instruction nor its waits: a and b come from LDS reads (it waits for those by itself), sums of the
// same fragment follow each other at distances the hardware interlocks, and before anything else reads the
// sums the caller lets mma_drain pass, which no instruction is scheduled across.
template <class T, bool ACCUM>  // ACCUM: the sums are in accumulation registers, else in ordinary ones
__device__ __forceinline__ void mma_inplace(u32x4_t a, u32x4_t b, float4_t& c) {
  if constexpr (__is_same(T, _Float16) && ACCUM)
    asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
  else if constexpr (__is_same(T, _Float16))
    asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+v"(c) : "v"(a), "v"(b));
  else if constexpr (ACCUM)
    asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
  else
    asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+v"(c) : "v"(a), "v"(b));
}
template <bool ACCUM>
__device__ __forceinline__ void mma_inplace(u32x8_t a, u32x8_t b, float4_t& c) {
  if constexpr (ACCUM)
    asm volatile("v_mfma_f32_16x16x128_f8f6f4 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
  else
    asm volatile("v_mfma_f32_16x16x128_f8f6f4 %0, %1, %2, %0" : "+v"(c) : "v"(a), "v"(b));
}
__device__ __forceinline__ void mma_drain() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

// A lane's share of a fragment in one step: 16 bytes of each 64-byte half of its row.
struct Fragment {
  u32x8_t v;
  __device__ __forceinline__ void set(int h, u32x4_t x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[4 * h + i] = x[i];
  }
  __device__ __forceinline__ u32x4_t half(int h) const {
    return h ? __builtin_shufflevector(v, v, 4, 5, 6, 7) : __builtin_shufflevector(v, v, 0, 1, 2, 3);
  }
};

template <class T, int BM, int BN, int WM, int WN, int S>
struct LinearTile {
  static constexpr int kWaves = WM * WN;
  static constexpr int TM = BM / WM / 16, TN = BN / WN / 16;
  static constexpr int kStage = (BM + BN) * kLinStep;
  static constexpr int kXCopies = BM / 8 / kWaves, kWCopies = BN / 8 / kWaves;  // LDS copies of a wave a stage
  static constexpr int kCopies = kXCopies + kWCopies;
  static_assert(BM % (8 * kWaves) == 0 && BN % (8 * kWaves) == 0 && TM % 2 == 0 && TN % 2 == 0, "tile");
};

template <class T, int BM, int BN, int WM, int WN, int S, int WGS>
__global__ __launch_bounds__(64 * WM * WN, (WGS * WM * WN + 3) / 4)
void linear_tile_kernel(LinearParams p, int ntm, int ntn) {
  using C = LinearTile<T, BM, BN, WM, WN, S>;
  constexpr int TM = C::TM, TN = C::TN;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[S * C::kStage];
  const int lane = (int)threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave % WN;
  int mt, nt;
  linear_tile_of((int)blockIdx.x, ntm, ntn, mt, nt);
  const int64_t m0 = (int64_t)mt * BM;
  const int n0 = nt * BN;

  // both operands' rows of this tile; the range ends with the last valid row's last byte
  const int mrows = p.M - m0 < BM ? (int)(p.M - m0) : BM;
  const int nrows = p.N - n0 < BN ? p.N - n0 : BN;
  const uint8_t* xb = p.x + m0 * p.x_stride;
  const uint8_t* wb = p.w + (int64_t)n0 * p.w_stride;
  const int xbytes = (mrows - 1) * (int)p.x_stride + p.kbytes;
  const int wbytes = (nrows - 1) * (int)p.w_stride + p.kbytes;
  // this lane's row and piece of each copy of 1024 bytes
  const int lrow = lane >> 3, piece = ((lane & 7) ^ lrow) * 16;
  int voff[C::kCopies];
#pragma unroll
  for (int j = 0; j < C::kXCopies; ++j)
    voff[j] = (8 * (wave * C::kXCopies + j) + lrow) * (int)p.x_stride + piece;
#pragma unroll
  for (int j = 0; j < C::kWCopies; ++j) {
    const int r = 8 * (wave * C::kWCopies + j) + lrow;  // LDS row; its weight row:
    const int n = (r & ~31) + ((r >> 2) & 3) * 8 + ((r >> 4) & 1) * 4 + (r & 3);
    voff[C::kXCopies + j] = n * (int)p.w_stride + piece;
  }
  const uint32_t lds0 = lds_offset(smem);
  // 64 fragments a wave fill the accumulation registers: there the loop is the only way through the steps
  // (two at a time, an odd last one followed by one of zeros), since sums that arrive by several ways would
  // have to be moved, through scratch memory.
  constexpr bool PAIRS = TM * TN >= 64;
  const int total = (p.kbytes + kLinStep - 1) / kLinStep;
  // a part of the reduction (blockIdx.y) or all of it
  const int first = p.partial ? (int)blockIdx.y * p.part_steps : 0;
  const int wanted = p.partial && total - first > p.part_steps ? p.part_steps : total - first;
  const int steps = !PAIRS ? wanted : wanted < 2 ? 2 : (wanted + 1) & ~1;
  // Copy j of a step's rows into a stage.  Steps past the end have empty buffers: their copies fetch
  // nothing and write zeros, so that the number of copies in flight is the same in every step.
  u32x4_t xr, wr;
  uint32_t dst;
  const auto copies_of = [&](int step, int stage) {
    const int k = (first + step) * kLinStep, left = step < wanted ? p.kbytes - k : 0;
    xr = row_buffer(xb + k, left > 0 ? xbytes - k : 0);
    wr = row_buffer(wb + k, left > 0 ? wbytes - k : 0);
    dst = lds0 + stage * C::kStage;
    if (left < kLinStep) {  // the tail: pieces past the row's end are out of range
#pragma unroll
      for (int j = 0; j < C::kCopies; ++j) voff[j] = piece < left ? voff[j] : 0x7fffff00;
    }
  };
  const auto copy = [&](int j) {
    if (j < C::kXCopies)
      lds_copy(xr, dst + (wave * C::kXCopies + j) * 1024, voff[j]);
    else
      lds_copy(wr, dst + BM * kLinStep + (wave * C::kWCopies + j - C::kXCopies) * 1024, voff[j]);
  };

  // what the epilogue needs of the columns and rows that this lane finishes
  constexpr int NV = PAIRS ? 4 : 8, NC = PAIRS ? 1 : TN / 2;
  const int64_t em = m0 + wm * TM * 16 + (PAIRS ? lane >> 5 : lane & 15);
  const int en = n0 + wn * TN * 16 + (PAIRS ? (lane & 31) * 4 : (lane >> 4) * 8);
  Columns<T, NV> cols[NC];
  RowScales<T, TM, 16> rscales;
  if (!p.partial) {
#pragma unroll
    for (int i = 0; i < NC; ++i) cols[i].load(p, en + 32 * i);
    if constexpr (!PAIRS) rscales.load(p, em);
  }

  float4_t acc[TN][TM];
#pragma unroll
  for (int i = 0; i < TN; ++i)
#pragma unroll
    for (int j = 0; j < TM; ++j) acc[i][j] = float4_t{0.f, 0.f, 0.f, 0.f};
  Fragment a[TN], b[TM];
  // this lane's 16 bytes of fragment row lane % 16 in either half of the step: pieces lane / 16 and 4 + lane / 16
  const int fr = (lane & 15) * kLinStep, sw = lane & 7;
  const int at0 = fr + (((lane >> 4) ^ sw) << 4), at1 = fr + (((4 + (lane >> 4)) ^ sw) << 4);
  const int xat = wm * TM * 16 * kLinStep, wat = BM * kLinStep + wn * TN * 16 * kLinStep;
  const auto read_a = [&](int stage_at, int i, int h) {
    a[i].set(h, *reinterpret_cast<const u32x4_t*>(smem + stage_at + wat + i * 16 * kLinStep + (h ? at1 : at0)));
  };
  const auto read_b = [&](int stage_at, int j, int h) {
    b[j].set(h, *reinterpret_cast<const u32x4_t*>(smem + stage_at + xat + j * 16 * kLinStep + (h ? at1 : at0)));
  };
  // Products FROM..TO-1 of the NM of quarter (i0, j0), with hook(n) before product n.
  constexpr int NH = __is_same(T, E4m3) ? 1 : 2;  // 64-byte halves of a step that are products of their own
  constexpr int NM = NH * (TN / 2) * (TM / 2);
  const auto quarter = [&](int i0, int j0, int from, int to, auto hook) {
#pragma unroll
    for (int n = from; n < to; ++n) {
      const int h = n / (TN / 2 * (TM / 2)), i = i0 + n / (TM / 2) % (TN / 2), j = j0 + n % (TM / 2);
      hook(n);
      if constexpr (__is_same(T, E4m3))
        mma_inplace<PAIRS>(a[i].v, b[j].v, acc[i][j]);
      else if constexpr (__is_same(T, E4m3Wide))
        acc[i][j] = mma_64b<T>(a[i].half(h), b[j].half(h), acc[i][j]);
      else
        mma_inplace<T, PAIRS>(a[i].half(h), b[j].half(h), acc[i][j]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // items 0..NI-1 spread evenly over NS slots: calls f for those of slot n
  const auto spread = [&](int n, int ni, int ns, auto f) {
#pragma unroll
    for (int r = 0; r < ni; ++r)
      if (r * ns / ni == n) f(r);
  };

  if (PAIRS || steps > 0) {
#pragma unroll
    for (int s = 0; s < S; ++s) {
      copies_of(s, s);
#pragma unroll
      for (int j = 0; j < C::kCopies; ++j) copy(j);
    }
    asm volatile("s_waitcnt vmcnt(%0)" ::"i"((S - 1) * C::kCopies) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int i = 0; i < TN / 2; ++i) read_a(0, i, h);
#pragma unroll
      for (int j = 0; j < TM / 2; ++j) read_b(0, j, h);
    }
    int stage = 0;  // of the present step
    const auto step = [&](int s, auto flip) {
      constexpr int F = decltype(flip)::value ? TM / 2 : 0, G = TM / 2 - F;  // B's first and second half
      constexpr int SPLIT = NM / 2, REST = NM - SPLIT + NM;
      const int cur = stage * C::kStage;
      const int nstage = stage + 1 == S ? 0 : stage + 1;
      const int nxt = nstage * C::kStage;
      quarter(0, F, 0, NM, [&](int n) {
        spread(n, TM, NM, [&](int r) { read_b(cur, G + r % (TM / 2), r / (TM / 2)); });
      });
      quarter(0, G, 0, NM, [&](int n) {
        spread(n, TN, NM, [&](int r) { read_a(cur, TN / 2 + r % (TN / 2), r / (TN / 2)); });
      });
      quarter(TN / 2, G, 0, SPLIT, [&](int) {});
      // this wave has read the stage (lgkmcnt) and its copies of the next one have landed (vmcnt)
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"i"((S - 2) * C::kCopies) : "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      copies_of(s + S, stage);
      __builtin_amdgcn_sched_barrier(0);
      // the rest of the step: the next one's first operands and the copies
      const auto rest = [&](int n) {
        spread(n, TN + TM, REST, [&](int r) {
          if constexpr (NH == 1) {  // a fragment is one operand: B's only after its last use
            if (r < TN)
              read_a(nxt, r % (TN / 2), r / (TN / 2));
            else
              read_b(nxt, G + (r - TN) % (TM / 2), (r - TN) / (TM / 2));
          } else {
            const int h = r / (TN / 2 + TM / 2), q = r % (TN / 2 + TM / 2);
            if (q < TN / 2)
              read_a(nxt, q, h);
            else
              read_b(nxt, G + q - TN / 2, h);
          }
        });
        spread(n, C::kCopies, REST, [&](int j) { copy(j); });
      };
      quarter(TN / 2, G, SPLIT, NM, [&](int n) { rest(n - SPLIT); });
      quarter(TN / 2, F, 0, NM, [&](int n) { rest(n + NM - SPLIT); });
      stage = nstage;
    };
    if constexpr (PAIRS) {
      int s = 0;
      do {
        step(s, Int<0>{});
        step(s + 1, Int<1>{});
        s += 2;
      } while (s < steps);
    } else {
      int s = 0;
      for (; s + 1 < steps; s += 2) {
        step(s, Int<0>{});
        step(s + 1, Int<1>{});
      }
      if (s < steps) step(s, Int<0>{});
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no copy outlives the workgroup's use of LDS
    mma_drain();  // here, where no other path has joined yet: joining may move the sums
  }
  if constexpr (TM * TN == 4) {
    if (p.partial) {  // this part's sums, as the lanes have them
      const int64_t tile = (int64_t)blockIdx.y * ntm * ntn + (int64_t)mt * ntn + nt;
      float4_t* at = reinterpret_cast<float4_t*>(p.partial) + (tile * C::kWaves + wave) * 256 + lane;
#pragma unroll
      for (int j = 0; j < TM; ++j) {
        if (m0 + (wm * TM + j) * 16 >= p.M) break;  // rows that the join does not read either
#pragma unroll
        for (int i = 0; i < TN; ++i) at[(i * TM + j) * 64] = acc[i][j];
      }
      return;
    }
  }
  if constexpr (!PAIRS) {
    linear_epilogue<T, TM, TN>(p, em, en, acc, cols, rscales);
  } else {
    // 64 fragments: the code that finishes them would be too long laid out one after the other.  The sums
    // go through the wave's part of LDS (once the last copies have landed), TM / RJ fragment rows a round, in
    // which 16-byte piece s of row r lies at place s ^ (r % 16), and a loop takes two rows of 4 columns a
    // lane at a time.
    constexpr int PR = TN * 4;                                               // pieces per row
    constexpr int RJ = TM * 16 * PR * 16 * C::kWaves > S * C::kStage ? 2 : 1;  // rounds
    static_assert(PR == 32 && TM * 16 * PR * 16 * C::kWaves <= RJ * S * C::kStage, "sums of a round fit");
    __syncthreads();
    uint8_t* part = smem + wave * (S * C::kStage / C::kWaves);
    by_output(p, [&](auto o, auto vec) {
      using O = decltype(o);
      constexpr bool VEC = decltype(vec)::value;
      constexpr int U = 8, RR = TM / RJ * 16;  // rows of a lane at a time (two rows apart), rows a round
      Raw<O, 4> next[U];
      RowScales<T, U, 2> nrs;
      linear_residual<O, VEC, U, 2, 4>(p, em, en, next);
      nrs.load(p, em);
#pragma unroll
      for (int q = 0; q < RJ; ++q) {
#pragma unroll
        for (int j = 0; j < TM / RJ; ++j)
#pragma unroll
          for (int i = 0; i < TN; ++i) {
            const int s = (i / 2) * 8 + (lane >> 4) * 2 + i % 2;
            *reinterpret_cast<float4_t*>(part + (16 * j + (lane & 15)) * (PR * 16) + (s ^ (lane & 15)) * 16) =
                acc[i][q * (TM / RJ) + j];
          }
        for (int r0 = 0; r0 < RR; r0 += 2 * U) {
          Raw<O, 4> res[U];
          const RowScales<T, U, 2> rs = nrs;
#pragma unroll
          for (int u = 0; u < U; ++u) res[u] = next[u];
          linear_residual<O, VEC, U, 2, 4>(p, em + q * RR + r0 + 2 * U, en, next);  // clamped past the last row
          nrs.load(p, em + q * RR + r0 + 2 * U);
          float v[U][4];
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const int r = r0 + 2 * u + (lane >> 5);
            const float4_t x = *reinterpret_cast<const float4_t*>(part + r * (PR * 16) + ((lane & 31) ^ (r & 15)) * 16);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[u][e] = x[e];
          }
          linear_finish<T, O, VEC, U, 2, 4>(p, em + q * RR + r0, en, v, cols[0], rs, res);
        }
      }
    });
  }
}

// Joins the parts of a split reduction, one wave per 16 x 32 block of a 64 x 64 tile, and finishes it.
template <class T>
__global__ __launch_bounds__(64) void linear_join_kernel(LinearParams p, int ntn, int tiles, int parts) {
  const int lane = (int)threadIdx.x;
  const int tile = (int)blockIdx.x >> 3, wave = (int)blockIdx.x >> 1 & 3, j = (int)blockIdx.x & 1;
  const int64_t m16 = (int64_t)(tile / ntn) * 64 + (wave >> 1) * 32 + j * 16, m = m16 + (lane & 15);
  if (m16 >= p.M) return;
  const float4_t* at = reinterpret_cast<const float4_t*>(p.partial) + (int64_t)(tile * 4 + wave) * 256 + j * 64 + lane;
  const int n = tile % ntn * 64 + (wave & 1) * 32 + (lane >> 4) * 8;
  Columns<T, 8> cols;
  RowScales<T, 1, 16> rscales;
  cols.load(p, n);
  rscales.load(p, m);
  by_output(p, [&](auto o, auto vec) {
    using O = decltype(o);
    constexpr bool VEC = decltype(vec)::value;
    Raw<O, 8> res[1];  // on its way beside the parts
    linear_residual<O, VEC, 1, 16, 8>(p, m, n, res);
    float4_t lo = at[0], hi = at[128];
#pragma unroll 8
    for (int q = 1; q < parts; ++q) {
      const float4_t* part = at + (int64_t)q * tiles * 4 * 256;
      lo += part[0];
      hi += part[128];
    }
    float v[1][8] = {{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]}};
    linear_finish<T, O, VEC, 1, 16, 8>(p, m, n, v, cols, rscales, res);
  });
}

}  // namespace sengine
