// Cross attention: Lq queries of every sequence attend to that sequence's Lk encoder states.
//   o[b, i, h] = sum_j p_j v[b, j, g] / sum_j p_j,   p_j = exp(scale * q[b, i, h] . k[b, j, g] - max)
// over the keys j that count: j < lengths[b] (if given) and mask[b, j] != 0 (if given); g = h / (Hq / Hkv).
// A query with no such key gets zeros.  What lies in a key or value that does not count is never
// used, be it infinite or NaN.
//
#include "cross_tile.h"

namespace sengine {

// Any alignment and any strides (rows at odd elements, through the C entry only; keys too far apart for a tile's
// offsets): one query of 1024 masked keys 2^18 elements apart, 128 sequences, 32 heads on 8 x 128: 908 us (the tile
// kernel without the mask 110), bound by its single-element loads.  One wave a query row and head, an online softmax
// over 64 keys at a time, lane j forming the dot product of key j, then the lanes sharing the values' columns.
template <class T>
__global__ __launch_bounds__(64) void cross_row_kernel(CrossParams p) {
  __shared__ float sq[128], sp[64];
  const int lane = (int)threadIdx.x;
  int64_t id = blockIdx.x;
  const int h = (int)(id % p.Hq);
  id /= p.Hq;
  const int i = (int)(id % p.Lq), b = (int)(id / p.Lq);
  const int g = h / (p.Hq / p.Hkv);
  const T* q = static_cast<const T*>(p.q) + b * p.q_b + i * p.q_l + h * p.q_h;
  const T* k = static_cast<const T*>(p.k) + b * p.k_b + g * p.k_h;
  const T* v = static_cast<const T*>(p.v) + b * p.v_b + g * p.v_h;
  int n = p.Lk;
  if (p.lengths) {
    const int len = p.lengths[b];
    n = len < 0 ? 0 : len < n ? len : n;
  }
  for (int c = lane; c < p.d; c += 64) sq[c] = (float)q[c] * p.scale;
  __syncthreads();
  float top = -INFINITY, total = 0.f, o0 = 0.f, o1 = 0.f;
  for (int j0 = 0; j0 < n; j0 += 64) {
    const int j = j0 + lane;
    const bool counts = j < n && (!p.mask || p.mask[b * p.mask_b + j]);
    float s = -INFINITY;
    if (counts) {
      s = 0.f;
      const T* kr = k + j * p.k_l;
      for (int c = 0; c < p.d; ++c) s = __builtin_fmaf(sq[c], (float)kr[c], s);
    }
    const uint64_t any = __ballot(counts);
    if (!any) continue;
    float t = s;
    for (int o = 32; o > 0; o >>= 1) t = fmaxf(t, __shfl_xor(t, o, 64));
    t = fmaxf(t, top);
    const float ref = t == -INFINITY ? 0.f : t;  // every key so far scores -infinity: they weigh nothing
    const float back = __expf(top - ref);
    const float e = counts ? __expf(s - ref) : 0.f;
    float u = e;
    for (int o = 32; o > 0; o >>= 1) u += __shfl_xor(u, o, 64);
    total = total * back + u;
    top = t;
    __syncthreads();
    sp[lane] = e;
    __syncthreads();
    o0 *= back;
    o1 *= back;
    for (int r = 0; r < 64; ++r) {
      if (!(any >> r & 1)) continue;
      const T* vr = v + (int64_t)(j0 + r) * p.v_l;
      if (lane < p.d) o0 = __builtin_fmaf(sp[r], (float)vr[lane], o0);
      if (lane + 64 < p.d) o1 = __builtin_fmaf(sp[r], (float)vr[lane + 64], o1);
    }
  }
  const float inv = 1.f / total;
  T* out = static_cast<T*>(p.out) + b * p.o_b + i * p.o_l + h * p.o_h;
  if (lane < p.d) out[lane] = (T)(total == 0.f ? 0.f : o0 * inv);
  if (lane + 64 < p.d) out[lane + 64] = (T)(total == 0.f ? 0.f : o1 * inv);
}

// Which form, and in how many parts (us, measured as they stand here).
//   rows of a workgroup (rows: the queries of a key head's group): 16, on waves with tiles of their own, where there
//     are no more; else the most of 256, 128, 64 that leave a workgroup for every CU, 256 for heads over 64 values
//     only: 4 x 4096 x 4001, 16 heads x 128: 256 rows 481, 128 rows 530; 4 x 4096 x 4096 x 64: 322, 313 and with 64
//     rows 362; 1000 x 1000, 8 heads x 64: 128 rows 20, 64 rows 15
//   four key heads together where a head's row is not whole cache lines, up to 48 values, and the time is that of
//     reading K and V (they pass 64 MB): 64 x 3136, 128 sequences, 8 heads x 48: 113 (alone 164); one query of 196
//     keys, 4 sequences: 11.6 (alone, with waves of their own: 11.3).  Heads of 16, 32 and 48 values have this form;
//     others whose rows are not whole lines either (24, 40, 56, 80 ..) are read alone, and were not measured merged
//   parts of the keys where there are fewer workgroups than CUs, up to two a CU, of 256 keys or more (512 with 64
//     rows or more): one query of up to 16384 keys, 8 sequences of unequal lengths, 8 key heads x 128: in 8 parts
//     63, in 16 72, in 12 69
constexpr int kCUs = 256;
struct CrossPlan {
  int rows_a_block;
  int heads;  // key heads of a workgroup
  int parts;
};

// Keys and query rows (of all sequences and heads) that the kernels' counts hold.
static bool keys_fit(const sengine_cross_desc* d) { return d->Lk <= 0x3fffffff; }
static bool rows_fit(const sengine_cross_desc* d) {
  const int64_t queries = (int64_t)d->B * d->Lq;
  return queries <= 0x7fffff00 && queries * d->Hq <= 0x7fffff00;  // up to the end of the last block of 256
}

static CrossPlan plan(const sengine_cross_desc* d) {
  const int64_t rows = (int64_t)d->Lq * (d->Hq / d->Hkv);
  const auto wgs_of = [&](int r) { return (int64_t)d->B * d->Hkv * ((rows + r - 1) / r); };
  CrossPlan q{16, 1, 1};
  if (rows > 128 && d->d > 64 && wgs_of(256) >= kCUs)
    q.rows_a_block = 256;
  else if (rows > 64 && wgs_of(128) >= kCUs)
    q.rows_a_block = 128;
  else if (rows > 16)
    q.rows_a_block = 64;
  if (rows <= 64 && d->d <= 48 && d->d % 16 == 0 && d->Hkv % 4 == 0 && d->k_stride[2] == d->d &&
      d->v_stride[2] == d->d && (double)d->B * d->Lk * d->Hkv * d->d >= 1 << 24)
    q.heads = 4;
  const int64_t wgs = (int64_t)d->B * (d->Hkv / q.heads) * ((rows + q.rows_a_block - 1) / q.rows_a_block);
  constexpr int64_t kWant = 2 * kCUs;  // workgroups
  const int64_t least = q.rows_a_block == 16 ? 256 : 512;  // keys of a part
  if (wgs < kCUs) {
    int64_t parts = kWant / wgs;
    if (parts > d->Lk / least) parts = d->Lk / least;
    if (parts > kCrossParts) parts = kCrossParts;
    if (parts > 1) q.parts = (int)parts;
  }
  return q;
}

static size_t cross_workspace(const sengine_cross_desc* d, int parts) {
  return (size_t)parts * d->B * d->Lq * d->Hq * (d->d + 2) * sizeof(float);
}

template <class T, int DV, int NW, int QF, int KT, int S, int HPW, bool SHARED, int WPE>
static hipError_t run_tile(CrossParams& p, hipStream_t stream) {
  constexpr int R = (SHARED ? NW / HPW : 1) * 16 * QF;
  p.blocks = (p.rows + R - 1) / R;
  // units of all key heads where there are enough of them (heads of 48 values share cache lines), else of one;
  // in turn over the XCDs unless that would leave some with less (2.5 units against 3 and the like)
  p.unit_heads = (int64_t)p.B * p.parts >= 32 ? p.Hkv / HPW : 1;
  p.inner = p.blocks * p.unit_heads;
  const int64_t units = (int64_t)p.B * p.parts * (p.Hkv / HPW / p.unit_heads);
  p.spread = units % 8 == 0 || units >= 64;
  p.units = (int)units;
  const int64_t wgs = (p.spread ? (units + 7) / 8 * 8 : units) * p.inner;
  if (!launchable(wgs, 64 * NW)) return hipErrorInvalidConfiguration;
  const dim3 grid((unsigned)wgs), block(64 * NW);
  if (p.mask)
    cross_tile_kernel<T, DV, NW, QF, KT, S, HPW, SHARED, true, WPE><<<grid, block, 0, stream>>>(p);
  else
    cross_tile_kernel<T, DV, NW, QF, KT, S, HPW, SHARED, false, WPE><<<grid, block, 0, stream>>>(p);
  return hipGetLastError();
}

template <class T, int DV>
static hipError_t by_rows(CrossParams& p, const CrossPlan& q, hipStream_t stream) {
  if constexpr (DV < 4) {
    if (q.heads == 4 && q.rows_a_block == 16) return run_tile<T, DV, 4, 1, 32, 3, 4, true, 1>(p, stream);
    if (q.heads == 4) return run_tile<T, DV, 8, 2, 32, 3, 4, true, 2>(p, stream);
  }
  if (q.rows_a_block == 16) return run_tile<T, DV, 4, 1, 32, 2, 1, false, 1>(p, stream);
  if (q.rows_a_block == 64) return run_tile<T, DV, 4, 1, 64, 2, 1, true, 2>(p, stream);
  if (q.rows_a_block == 128) return run_tile<T, DV, 4, 2, 64, 2, 1, true, 2>(p, stream);
  return run_tile<T, DV, 8, 2, 64, 2, 1, true, 2>(p, stream);
}

template <class T>
static hipError_t by_width(CrossParams& p, const CrossPlan& q, hipStream_t stream) {
  const int dv = (p.d + 15) / 16;
  hipError_t e;
  if (dv <= 1)
    e = by_rows<T, 1>(p, q, stream);
  else if (dv <= 2)
    e = by_rows<T, 2>(p, q, stream);
  else if (dv <= 3)
    e = by_rows<T, 3>(p, q, stream);
  else if (dv <= 4)
    e = by_rows<T, 4>(p, q, stream);
  else if (dv <= 6)
    e = by_rows<T, 6>(p, q, stream);
  else
    e = by_rows<T, 8>(p, q, stream);
  if (e != hipSuccess || p.parts == 1) return e;
  const int64_t rows = (int64_t)p.B * p.Hkv * p.rows;
  cross_join_kernel<T><<<dim3((unsigned)rows), dim3(64), 0, stream>>>(p);
  return hipGetLastError();
}

}  // namespace sengine

using namespace sengine;

extern "C" int sengine_amd_cross_attention_ws(const sengine_cross_desc* d, const void* q, const void* k,
                                              const void* v, const int32_t* key_lengths, const void* key_mask,
                                              void* out, void* workspace, size_t workspace_bytes, hipStream_t stream) {
  if (!d) return set_error(-1, "cross_attention: null descriptor");
  if (d->B < 0 || d->Lq < 0 || d->Lk < 0 || d->Hq < 1 || d->Hkv < 1)
    return set_error(-2, "cross_attention: needs B, Lq, Lk >= 0 and heads >= 1");
  if (d->Hq % d->Hkv) return set_error(-2, "cross_attention: the query heads must be a multiple of the key heads");
  if (d->d < 8 || d->d > 128 || d->d % 8)
    return set_error(-2, "cross_attention: the head size must be a multiple of 8 up to 128");
  if (d->type != SENGINE_ENC_F16 && d->type != SENGINE_ENC_BF16)
    return set_error(-2, "cross_attention: q, k and v must be fp16 or bf16");
  if (!keys_fit(d)) return set_error(-2, "cross_attention: more than 2^30 keys");
  if (!rows_fit(d)) return set_error(-2, "cross_attention: too many query rows");
  if (d->B == 0 || d->Lq == 0) return 0;
  if (!q || !out || (d->Lk > 0 && (!k || !v))) return set_error(-1, "cross_attention: null q, k, v or out");
  // rows less than d elements apart: among them the same memory for several sequences, queries or heads
  const auto apart = [&](int32_t n, int64_t s) { return n == 1 || s >= d->d || s <= -d->d; };
  if (!apart(d->B, d->out_stride[0]) || !apart(d->Lq, d->out_stride[1]) || !apart(d->Hq, d->out_stride[2]))
    return set_error(-2, "cross_attention: output rows overlap");
  CrossParams p{};
  p.q = q;
  p.k = k;
  p.v = v;
  p.out = out;
  p.lengths = key_lengths;
  p.mask = static_cast<const uint8_t*>(key_mask);
  p.q_b = d->q_stride[0], p.q_l = d->q_stride[1], p.q_h = d->q_stride[2];
  p.k_b = d->k_stride[0], p.k_l = d->k_stride[1], p.k_h = d->k_stride[2];
  p.v_b = d->v_stride[0], p.v_l = d->v_stride[1], p.v_h = d->v_stride[2];
  p.o_b = d->out_stride[0], p.o_l = d->out_stride[1], p.o_h = d->out_stride[2];
  p.mask_b = d->mask_stride;
  p.B = d->B, p.Lq = d->Lq, p.Lk = d->Lk, p.Hq = d->Hq, p.Hkv = d->Hkv, p.d = d->d;
  p.scale = d->scale;
  p.group = d->Hq / d->Hkv;
  p.rows = d->Lq * p.group;
  if ((uintptr_t)workspace % 16) return set_error(-2, "cross_attention: the workspace must be aligned to 16 bytes");
  // the tile kernel: rows of d values that begin at multiples of 16 bytes, offsets in 31 bits: of a stretch's 4096 keys
  // with a mask, of a tile's 64 without one (whose base moves from tile to tile)
  const auto aligned = [](const void* a, const int64_t* s) {
    return (uintptr_t)a % 16 == 0 && s[0] % 8 == 0 && s[1] % 8 == 0 && s[2] % 8 == 0;
  };
  const int64_t most = key_mask ? 0x3ffff : 0xffffff;
  const auto near = [&](int64_t s) { return s >= 0 && s <= most; };
  if (aligned(q, d->q_stride) && aligned(k, d->k_stride) && aligned(v, d->v_stride) && aligned(out, d->out_stride) &&
      near(p.k_l) && near(p.v_l)) {
    const CrossPlan plan_ = plan(d);
    p.parts = plan_.parts;
    if (p.parts > 1 && (!workspace || workspace_bytes < cross_workspace(d, p.parts))) p.parts = 1;
    p.part_o = static_cast<float*>(workspace);
    p.part_ml = p.part_o + (int64_t)p.parts * p.B * p.Hkv * p.rows * p.d;
    return (int)(d->type == SENGINE_ENC_F16 ? by_width<_Float16>(p, plan_, stream)
                                            : by_width<__bf16>(p, plan_, stream));
  }
  if (!launchable((int64_t)d->B * d->Lq * d->Hq, 64)) return (int)hipErrorInvalidConfiguration;
  const dim3 grid((unsigned)((int64_t)d->B * d->Lq * d->Hq));
  if (d->type == SENGINE_ENC_F16)
    cross_row_kernel<_Float16><<<grid, dim3(64), 0, stream>>>(p);
  else
    cross_row_kernel<__bf16><<<grid, dim3(64), 0, stream>>>(p);
  return (int)hipGetLastError();
}

extern "C" int sengine_amd_cross_attention(const sengine_cross_desc* d, const void* q, const void* k, const void* v,
                                           const int32_t* key_lengths, const void* key_mask, void* out,
                                           hipStream_t stream) {
  return sengine_amd_cross_attention_ws(d, q, k, v, key_lengths, key_mask, out, nullptr, 0, stream);
}

extern "C" int sengine_amd_cross_attention_workspace(const sengine_cross_desc* d, size_t* bytes) {
  if (!d || !bytes) return set_error(-1, "cross_attention_workspace: null argument");
  *bytes = 0;
  if (d->B < 1 || d->Lq < 1 || d->Lk < 1 || d->Hkv < 1 || d->Hq < d->Hkv || d->d < 8 || d->d > 128 ||
      !keys_fit(d) || !rows_fit(d))
    return 0;  // nothing to do, or refused by the entry
  const int parts = plan(d).parts;
  if (parts > 1) *bytes = cross_workspace(d, parts);
  return 0;
}
