// Cross attention: Lq queries of every sequence attend to that sequence's Lk encoder states.
//   o[b, i, h] = sum_j p_j v[b, j, g] / sum_j p_j,   p_j = exp(scale * q[b, i, h] . k[b, j, g] - max)
// over the keys j that count: j < lengths[b] (if given) and mask[b, j] != 0 (if given); g = h / (Hq / Hkv).
// A query with no such key gets zeros.  What lies in a key or value that does not count is never
// used, be it infinite or NaN.
//
// One wave a query row and head, an online softmax over 64 keys at a time: lane j forms the dot product
// of key j, then the lanes share the values' columns.
#include "token_types.h"

namespace sengine {

struct CrossParams {
  const void *q, *k, *v;
  void* out;
  const int32_t* lengths;
  const uint8_t* mask;
  int64_t q_b, q_l, q_h, k_b, k_l, k_h, v_b, v_l, v_h, o_b, o_l, o_h, mask_b;
  int B, Lq, Lk, Hq, Hkv, d;
  float scale;
};

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

}  // namespace sengine

using namespace sengine;

extern "C" int sengine_amd_cross_attention(const sengine_cross_desc* d, const void* q, const void* k, const void* v,
                                           const int32_t* key_lengths, const void* key_mask, void* out,
                                           hipStream_t stream) {
  if (!d) return set_error(-1, "cross_attention: null descriptor");
  if (d->B < 0 || d->Lq < 0 || d->Lk < 0 || d->Hq < 1 || d->Hkv < 1)
    return set_error(-2, "cross_attention: needs B, Lq, Lk >= 0 and heads >= 1");
  if (d->Hq % d->Hkv) return set_error(-2, "cross_attention: the query heads must be a multiple of the key heads");
  if (d->d < 8 || d->d > 128 || d->d % 8)
    return set_error(-2, "cross_attention: the head size must be a multiple of 8 up to 128");
  if (d->type != SENGINE_ENC_F16 && d->type != SENGINE_ENC_BF16)
    return set_error(-2, "cross_attention: q, k and v must be fp16 or bf16");
  if ((int64_t)d->B * d->Lq * d->Hq > 0x7fffffffll) return set_error(-2, "cross_attention: too many query rows");
  if (d->B == 0 || d->Lq == 0) return 0;
  if (!q || !out || (d->Lk > 0 && (!k || !v))) return set_error(-1, "cross_attention: null q, k, v or out");
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
  const dim3 grid((unsigned)((int64_t)d->B * d->Lq * d->Hq));
  if (d->type == SENGINE_ENC_F16)
    cross_row_kernel<_Float16><<<grid, dim3(64), 0, stream>>>(p);
  else
    cross_row_kernel<__bf16><<<grid, dim3(64), 0, stream>>>(p);
  return (int)hipGetLastError();
}
