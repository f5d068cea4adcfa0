// Causal linear attention with a decay a head.  Per sequence and head, with a state S (dk x dv, fp32):
//   S_t = g S_{t-1} + k_t^T v_t,   o_t = scale q_t S_t,
// the last state being an output.  g in [0, 1] is fp32, one a head.  Tokens past a sequence's length leave the state
// alone and have outputs of zero.
//
// Two forms.  Few tokens: token by token, the state in registers (decay_step_kernel); its time is the state's reading and
// writing: one token of 128 x 32 heads of 128 x 128, 541 MB, 102 us (5.3 TB/s).  Many: 64 tokens at a time as matrix products
// (decay_chunk.h).
#include "decay_chunk.h"

namespace sengine {

// Workgroup = 64 columns of one state: thread 16 r + c has columns 4 c .. of rows r, 16 + r, ..  Tokens go through LDS
// up to kDecayTokens at a time; a token's output is summed over a wave's rows by lane swaps and over the waves in LDS, in
// a fixed order.
constexpr int kDecayTokens = 16;

template <class T, int R>
__global__ __launch_bounds__(256) void decay_step_kernel(DecayParams p, int slices) {
  __shared__ float sq[kDecayTokens][16 * R], sk[kDecayTokens][16 * R], sv[kDecayTokens][64], so[4][kDecayTokens][64];
  const int tid = (int)threadIdx.x, c = tid & 15, r0 = tid >> 4, wave = tid >> 6;
  const int slice = (int)(blockIdx.x % slices);
  const int64_t bh = blockIdx.x / slices;
  const int64_t b = bh / p.H;
  const int h = (int)(bh - b * p.H);
  const int n = p.length(b), col = slice * 64 + 4 * c;
  const bool mine = col < p.dv;
  const float g = p.decay[h];
  float s[R][4];
#pragma unroll
  for (int i = 0; i < R; ++i) {
#pragma unroll
    for (int e = 0; e < 4; ++e) s[i][e] = 0.f;
    const int row = r0 + 16 * i;
    if (p.state && mine && row < p.dk)
      load_floats<float, 4>(p.state + b * p.s_b + h * p.s_h + (int64_t)row * p.dv + col, s[i]);
  }
  const T* q = static_cast<const T*>(p.q) + b * p.q_b + h * p.q_h;
  const T* k = static_cast<const T*>(p.k) + b * p.k_b + h * p.k_h;
  const T* v = static_cast<const T*>(p.v) + b * p.v_b + h * p.v_h + slice * 64;
  T* out = static_cast<T*>(p.out) + b * p.o_b + h * p.o_h + slice * 64;
  const int width = p.dv - slice * 64 < 64 ? p.dv - slice * 64 : 64;
  for (int t0 = 0; t0 < p.L; t0 += kDecayTokens) {
    const int there = p.L - t0 < kDecayTokens ? p.L - t0 : kDecayTokens;
    const int live = n - t0 < 0 ? 0 : n - t0 < there ? n - t0 : there;
    // rows behind dk are zeros, as are columns behind dv: they add nothing
    for (int i = tid; i < live * 2 * R; i += 256) {  // pieces of eight values
      const int t = i / (2 * R), at = (i - t * 2 * R) * 8;
      float a[8], d[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) a[e] = d[e] = 0.f;
      if (at < p.dk) {
        load_floats<T, 8>(q + (int64_t)(t0 + t) * p.q_l + at, a);
        load_floats<T, 8>(k + (int64_t)(t0 + t) * p.k_l + at, d);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        sq[t][at + e] = a[e] * p.scale;
        sk[t][at + e] = d[e];
      }
    }
    for (int i = tid; i < live * 8; i += 256) {
      const int t = i >> 3, at = (i & 7) * 8;
      float a[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) a[e] = 0.f;
      if (at < width) load_floats<T, 8>(v + (int64_t)(t0 + t) * p.v_l + at, a);
#pragma unroll
      for (int e = 0; e < 8; ++e) sv[t][at + e] = a[e];
    }
    __syncthreads();
    for (int t = 0; t < live; ++t) {
      float o[4] = {0.f, 0.f, 0.f, 0.f}, x[4];
      load_floats<float, 4>(&sv[t][4 * c], x);
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const float kr = sk[t][r0 + 16 * i], qr = sq[t][r0 + 16 * i];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[i][e] = __builtin_fmaf(kr, x[e], g * s[i][e]);
          o[e] = __builtin_fmaf(qr, s[i][e], o[e]);
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        o[e] += __shfl_xor(o[e], 16, 64);
        o[e] += __shfl_xor(o[e], 32, 64);
      }
      if ((r0 & 3) == 0) store_floats(&so[wave][t][4 * c], o);
    }
    __syncthreads();
    for (int i = tid; i < there * 8; i += 256) {
      const int t = i >> 3, at = (i & 7) * 8;
      if (at >= width) continue;
      float o[8];
#pragma unroll
      for (int e = 0; e < 8; ++e)
        o[e] = t < live ? (so[0][t][at + e] + so[1][t][at + e]) + (so[2][t][at + e] + so[3][t][at + e]) : 0.f;
      store_floats(out + (int64_t)(t0 + t) * p.o_l + at, o);
    }
    // the next tokens' q, k and v are written into places that all have read (the barrier above), and their outputs'
    // parts only after the next barrier
  }
  if (!p.state_out || !mine) return;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int row = r0 + 16 * i;
    if (row < p.dk) store_floats(p.state_out + b * p.so_b + h * p.so_h + (int64_t)row * p.dv + col, s[i]);
  }
}

template <class T, int R>
static hipError_t run_step(const DecayParams& p, hipStream_t stream) {
  const int slices = (p.dv + 63) / 64;
  const int64_t wgs = (int64_t)p.B * p.H * slices;
  if (!launchable(wgs, 256)) return hipErrorInvalidConfiguration;
  decay_step_kernel<T, R><<<dim3((unsigned)wgs), dim3(256), 0, stream>>>(p, slices);
  return hipGetLastError();
}

template <class T>
static hipError_t run_steps(const DecayParams& p, hipStream_t stream) {
  if (p.dk <= 32) return run_step<T, 2>(p, stream);
  if (p.dk <= 64) return run_step<T, 4>(p, stream);
  return run_step<T, 8>(p, stream);
}

// Prefix of the segments' states: place s holds what segment s adds to a state of zeros, and afterwards the state that
// segment s + 1 begins with.  Thread = four values of a state.  A state that is updated in place is copied: the segment
// that ends a sequence may write it before the first one has read it.
__global__ __launch_bounds__(256) void decay_scan_kernel(DecayParams p, int per_state) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t bh = i / per_state;
  if (bh >= (int64_t)p.B * p.H) return;
  const int64_t b = bh / p.H;
  const int h = (int)(bh - b * p.H), at = (int)(i - bh * per_state) * 4;
  const int n = p.length(b);
  const int last = n > 0 ? (n - 1) / p.seg_len : 0;  // the last segment with tokens
  float run[4] = {0.f, 0.f, 0.f, 0.f};
  if (p.state) load_floats<float, 4>(p.state + b * p.s_b + h * p.s_h + at, run);
  if (p.begun) store_floats(p.begun + bh * (int64_t)(p.dk * p.dv) + at, run);
  const float g = decay_power(decay_log2(p.decay[h]), p.seg_len);
  float* part = p.parts + bh * (p.segs - 1) * (int64_t)(p.dk * p.dv) + at;
  constexpr int U = 8;  // segments whose loads are under way together
  const int64_t next = (int64_t)p.dk * p.dv;
  for (int s = 0; s < last; s += U, part += U * next) {
    float u[U][4];
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (s + i < last) load_floats<float, 4>(part + i * next, u[i]);
#pragma unroll
    for (int i = 0; i < U; ++i) {
      if (s + i >= last) break;
#pragma unroll
      for (int e = 0; e < 4; ++e) run[e] = __builtin_fmaf(g, run[e], u[i][e]);
      store_floats(part + i * next, run);
    }
  }
}

// Whether wide heads take waves of 16 columns, not of 32: where every workgroup has a CU to itself.  Measured, us, waves of 16
// and of 32: 16 heads of 128 x 128 in bf16, 300 tokens 25 and 29, 1000 tokens 35 and 39; two workgroups a CU, 6 x 12 heads of
// 64 x 80 over 777 tokens, 36 and 31.
static bool decay_narrow(int dv, int64_t workgroups) { return decay_own(decay_blocks(dv)) > 1 && workgroups <= 256; }

struct DecayPlan {
  bool steps;        // token by token
  int segs, seg_len;  // segments of a sequence that are computed beside each other, tokens of one
};

// Most tokens that go one by one.  Measured, us, one by one and as a chunk: 64 x 32 heads of 128 x 128, 16 tokens 80 and 91, 32
// tokens 128 and 101; 16 heads of 128 x 128, 16 tokens 11 and 12, 32 tokens 18 and 12.
constexpr int kDecaySteps = 16;

static DecayPlan plan(const sengine_decay_desc* d) {
  // The chunks' copies have offsets of 31 bits from a chunk's first token on.  A row past the last token must be out of
  // the copies' range, or the last token's own: rows that overlap go one by one.
  const auto copied = [](int64_t stride, int size) { return stride == 0 || (stride >= size && stride < 1 << 23); };
  if (d->L <= kDecaySteps || !copied(d->q_stride[1], d->dk) || !copied(d->k_stride[1], d->dk) ||
      !copied(d->v_stride[1], d->dv))
    return {true, 1, d->L};
  const int chunks = (int)(((int64_t)d->L + kDecayChunk - 1) / kDecayChunk);
  // Rounds of workgroups over the chip, times the chunks of one and a start, half as much again for the pass that makes the
  // segments' states; and two launches more and the states' joining, in the time of chunks, of which narrow waves have
  // two thirds.  Measured, us, without segments and in this many: 16 heads of 128 x 128, 150 tokens 22, 300 tokens 32 and
  // 25 (5); 4000 tokens 49 (16), 53 (32), 80 (63); 8 x 16 heads of them over 500 tokens 50, 54 (4).  Narrow heads, bf16: 8
  // heads of 16 x 16, 150 tokens 12, 193 tokens 15 and 13 (4), 300 tokens 17 and 13 (5); 4 x 8 heads of 48 x 48, 150 tokens 15,
  // 193 tokens 18 and 17 (4), 300 tokens 21 and 17 (5); 4 x 16 heads of 64 x 64, where four segments are two rounds, 193 tokens
  // 17 and 18, 400 tokens 25 and 23 (7).
  const int64_t heads = (int64_t)d->B * d->H * ((d->dv + kDecayColumns - 1) / kDecayColumns);
  const int64_t slots = 256 * decay_resident(d->dk, d->dv);
  const auto pass = [&](int64_t workgroups, int per) {
    return (float)((workgroups + slots - 1) / slots) * (float)(per + 1) * (decay_narrow(d->dv, workgroups) ? 2.f / 3.f : 1.f);
  };
  int best = chunks;  // chunks of a segment
  float least = pass(heads, chunks);
  for (int segs = 2; segs <= chunks && segs <= 256 && (segs - 1) * heads <= 2 * slots; ++segs) {
    const int per = (chunks + segs - 1) / segs;
    const float cost = 1.5f * pass(heads * ((chunks + per - 1) / per), per) + 1.5f + (float)segs / 16.f;
    if (cost < least) least = cost, best = per;
  }
  return {false, (chunks + best - 1) / best, best * kDecayChunk};
}

static size_t workspace_of(const sengine_decay_desc* d, const DecayPlan& q) {
  return (size_t)d->B * d->H * q.segs * d->dk * d->dv * 4;  // the segments' states, and those that the sequences begin with
}

template <class T, int DKP, int BLOCKS>
static hipError_t run_chunks(const DecayParams& p, hipStream_t stream) {
  constexpr int NV = decay_own(BLOCKS), NW = BLOCKS / NV;
  const int64_t heads = (int64_t)p.B * p.H, parts = heads * ((p.dv + kDecayColumns - 1) / kDecayColumns);
  if (!launchable(parts * p.segs, 64 * BLOCKS)) return hipErrorInvalidConfiguration;
  if (p.segs > 1) {
    decay_chunk_kernel<T, DKP, 1, BLOCKS, true>
        <<<dim3((unsigned)(parts * (p.segs - 1))), dim3(64 * BLOCKS), 0, stream>>>(p);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const int per_state = p.dk * p.dv / 4;
    decay_scan_kernel<<<dim3((unsigned)((heads * per_state + 255) / 256)), dim3(256), 0, stream>>>(p, per_state);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  if (NV > 1 && decay_narrow(p.dv, parts * p.segs))
    decay_chunk_kernel<T, DKP, 1, BLOCKS, false><<<dim3((unsigned)(parts * p.segs)), dim3(64 * BLOCKS), 0, stream>>>(p);
  else
    decay_chunk_kernel<T, DKP, NV, NW, false><<<dim3((unsigned)(parts * p.segs)), dim3(64 * NW), 0, stream>>>(p);
  return hipGetLastError();
}

template <class T, int DKP>
static hipError_t by_values(const DecayParams& p, hipStream_t stream) {
  switch (decay_blocks(p.dv)) {
    case 2:
      return run_chunks<T, DKP, 2>(p, stream);
    case 3:
      return run_chunks<T, DKP, 3>(p, stream);
    case 4:
      return run_chunks<T, DKP, 4>(p, stream);
    default:
      return run_chunks<T, DKP, 8>(p, stream);
  }
}

template <class T>
static hipError_t run(DecayParams& p, const DecayPlan& q, hipStream_t stream) {
  if (q.steps) return run_steps<T>(p, stream);
  p.segs = q.segs;
  p.seg_len = q.seg_len;
  if (p.dk <= 32) return by_values<T, 32>(p, stream);
  if (p.dk <= 64) return by_values<T, 64>(p, stream);
  return by_values<T, 128>(p, stream);
}

static const char* refused(const sengine_decay_desc* d) {
  if (d->B < 0 || d->L < 0 || d->H < 1) return "decay_attention: needs B, L >= 0 and H >= 1";
  if (d->dk < 8 || d->dk > 128 || d->dk % 8 || d->dv < 8 || d->dv > 256 || d->dv % 8)
    return "decay_attention: dk is a multiple of 8 up to 128, dv of 8 up to 256";
  if (d->type != SENGINE_ENC_F16 && d->type != SENGINE_ENC_BF16)
    return "decay_attention: q, k and v must be fp16 or bf16";
  if (d->L > 0x7fffff00 || (int64_t)d->B * d->H > 0x7fffffff) return "decay_attention: sizes too large";
  return nullptr;
}

}  // namespace sengine

using namespace sengine;

extern "C" int sengine_amd_decay_attention_ws(const sengine_decay_desc* d, const void* q, const void* k, const void* v,
                                              const float* decay, const float* state, const int32_t* lengths,
                                              void* out, float* state_out, void* workspace, size_t workspace_bytes,
                                              hipStream_t stream) {
  if (!d) return set_error(-1, "decay_attention: null descriptor");
  if (const char* why = refused(d)) return set_error(-2, why);
  if (d->B == 0) return 0;
  if (!decay || (d->L > 0 && (!q || !k || !v || !out)))
    return set_error(-1, "decay_attention: null q, k, v, decay or out");
  const int32_t rows_of[3] = {d->B, d->L, d->H}, states_of[2] = {d->B, d->H};
  if (d->L > 0 && !rows_apart(d->dv, 3, rows_of, d->out_stride))
    return set_error(-2, "decay_attention: output rows overlap");
  const int64_t matrix = (int64_t)d->dk * d->dv;
  if (state_out && !rows_apart(matrix, 2, states_of, d->state_out_stride))
    return set_error(-2, "decay_attention: output states overlap");
  const auto rows = [&](const void* a, const int64_t* s) {
    return (uintptr_t)a % 16 == 0 && (d->B == 1 || s[0] % 8 == 0) && (d->L == 1 || s[1] % 8 == 0) &&
           (d->H == 1 || s[2] % 8 == 0);
  };
  if (d->L > 0 && (!rows(q, d->q_stride) || !rows(k, d->k_stride) || !rows(v, d->v_stride) || !rows(out, d->out_stride)))
    return set_error(-2, "decay_attention: rows of q, k, v and out must begin at multiples of 16 bytes");
  const auto states = [&](const float* a, const int64_t* s) {
    return (uintptr_t)a % 16 == 0 && (d->B == 1 || s[0] % 4 == 0) && (d->H == 1 || s[1] % 4 == 0);
  };
  if ((state && !states(state, d->state_stride)) || (state_out && !states(state_out, d->state_out_stride)))
    return set_error(-2, "decay_attention: states must begin at multiples of 16 bytes");
  if ((uintptr_t)workspace % 16) return set_error(-2, "decay_attention: the workspace must be aligned to 16 bytes");
  DecayParams p{};
  p.q = q, p.k = k, p.v = v, p.out = out;
  p.q_b = d->q_stride[0], p.q_l = d->q_stride[1], p.q_h = d->q_stride[2];
  p.k_b = d->k_stride[0], p.k_l = d->k_stride[1], p.k_h = d->k_stride[2];
  p.v_b = d->v_stride[0], p.v_l = d->v_stride[1], p.v_h = d->v_stride[2];
  p.o_b = d->out_stride[0], p.o_l = d->out_stride[1], p.o_h = d->out_stride[2];
  p.s_b = d->state_stride[0], p.s_h = d->state_stride[1];
  p.so_b = d->state_out_stride[0], p.so_h = d->state_out_stride[1];
  p.decay = decay, p.state = state, p.state_out = state_out, p.lengths = lengths;
  p.B = d->B, p.L = d->L, p.H = d->H, p.dk = d->dk, p.dv = d->dv;
  p.scale = d->scale;
  DecayPlan plan_ = plan(d);
  if (plan_.segs > 1 && (!workspace || workspace_bytes < workspace_of(d, plan_)))
    plan_ = {false, 1, (int)(((int64_t)d->L + kDecayChunk - 1) / kDecayChunk * kDecayChunk)};
  p.parts = static_cast<float*>(workspace);
  if (plan_.segs > 1 && state && state == state_out) p.begun = p.parts + (int64_t)d->B * d->H * (plan_.segs - 1) * matrix;
  return (int)(d->type == SENGINE_ENC_F16 ? run<_Float16>(p, plan_, stream) : run<__bf16>(p, plan_, stream));
}

extern "C" int sengine_amd_decay_attention(const sengine_decay_desc* d, const void* q, const void* k, const void* v,
                                           const float* decay, const float* state, const int32_t* lengths, void* out,
                                           float* state_out, hipStream_t stream) {
  return sengine_amd_decay_attention_ws(d, q, k, v, decay, state, lengths, out, state_out, nullptr, 0, stream);
}

extern "C" int sengine_amd_decay_attention_workspace(const sengine_decay_desc* d, size_t* bytes) {
  if (!d || !bytes) return set_error(-1, "decay_attention_workspace: null argument");
  *bytes = 0;
  if (refused(d) || d->B == 0 || d->L == 0) return 0;  // nothing to do, or refused by the entry
  const DecayPlan q = plan(d);
  if (q.segs > 1) *bytes = workspace_of(d, q);
  return 0;
}
