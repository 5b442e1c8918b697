// Attention over the pages of a paged KV cache.
//
//   out = sum_j p_j v_j / sum_j p_j,  p_j = exp(s_j - max s),  s_j = cap(q . k_j scale) - slope (pos - j)
//
// over the positions j that a row sees, in one pass with the running maximum and
// sum of the softmax, all in f32.
#include "paged.h"

#include <algorithm>
#include <cmath>

namespace rai {

namespace {

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
  for (int d = 32; d; d >>= 1) x = fmaxf(x, __shfl_xor(x, d));
  return x;
}
__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
  for (int d = 32; d; d >>= 1) x += __shfl_xor(x, d);
  return x;
}

// One row of one head by one wave: positions lo .. hi - 1 of the sequence whose
// table row is `table`, lane t holding key base + t and dimensions t, t + 64, ...
// of the output.  Keys that are not there or masked are not read into the sums at
// all, whatever they hold.
template <class T>
__device__ void wave_row(const AttnArgs &a, const LayerView<T> &kv, const int *table, int head, const float *q, int pos,
                         int lo, int hi, float &m, float &l, float (&o)[4]) {
  const int lane = threadIdx.x & 63, hd = kv.hd, kvh = head / (a.heads / kv.nkv), mask = (1 << kv.shift) - 1;
  const float slope = a.slopes ? a.slopes[head] : 0.0f;
  m = -INFINITY;
  l = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = 0.0f;
  for (int base = lo; base < hi; base += 64) {
    const int j = base + lane;
    const int page = j < hi ? page_of(table, j, kv.shift, kv.pages) : -1;
    float s = -INFINITY;
    if (page >= 0) {
      const T *k = kv.k + key_at(page, kvh, j & mask, kv.nkv, hd, kv.shift);
      float d = 0.0f;
      for (int e = 0; e < hd; ++e) d = fmaf(q[e], to_f32(k[e]), d);
      s = d * a.scale;
      if (a.softcap > 0.0f) s = a.softcap * tanhf(s / a.softcap);
      s -= slope * (float)(pos - j);
    }
    float mn = fmaxf(m, wave_max(s));
    if (__any(s != s)) mn = NAN;
    if (mn == -INFINITY) continue;
    const float scale = exp2f((m - mn) * kLog2e), p = exp2f((s - mn) * kLog2e);
    l = l * scale + wave_sum(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] *= scale;
    for (int t = 0; t < 64 && base + t < hi; ++t) {
      const int pg = __shfl(page, t);
      const float pt = __shfl(p, t);
      if (pg < 0) continue;
      const T *v = kv.v + value_at(pg, kvh, (base + t) & mask, kv.nkv, hd, kv.shift);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (lane + 64 * i < hd) o[i] = fmaf(pt, to_f32(v[(size_t)(lane + 64 * i) << kv.shift]), o[i]);
    }
    m = mn;
  }
}

// A wave per (row, head).
template <class T>
__global__ __launch_bounds__(256) void k_rows(AttnArgs a, LayerView<T> kv, BatchView b) {
  const SeqSpan sp = seq_span(b, blockIdx.y);
  const int unit = blockIdx.x * 4 + (threadIdx.x >> 6), j = unit / a.heads, head = unit % a.heads, lane = threadIdx.x & 63;
  if (j >= sp.nq) return;
  const int pos = sp.n - sp.nq + j;
  float m, l, o[4];
  wave_row(a, kv, b.tables + (size_t)blockIdx.y * b.stride, head,
           a.q + (size_t)(sp.q0 + j) * a.q_stride + (size_t)head * kv.hd, pos, first_seen(pos, a.window), pos + 1, m, l,
           o);
  float *out = a.out + (size_t)(sp.q0 + j) * a.out_stride + (size_t)head * kv.hd;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (lane + 64 * i < kv.hd) out[lane + 64 * i] = l == 0.0f ? 0.0f : o[i] / l;
}

}  // namespace

size_t paged_attention_work(int, int, int, const BatchView &, int) { return 0; }

template <class T>
void launch_paged_attention(const AttnArgs &a, const LayerView<T> &kv, const BatchView &b, void *, size_t,
                            hipStream_t s) {
  const size_t units = (size_t)b.max_q * a.heads;
  k_rows<T><<<dim3((unsigned)((units + 3) / 4), b.seqs), 256, 0, s>>>(a, kv, b);
}

template void launch_paged_attention<float>(const AttnArgs &, const LayerView<float> &, const BatchView &, void *, size_t,
                                            hipStream_t);
template void launch_paged_attention<_Float16>(const AttnArgs &, const LayerView<_Float16> &, const BatchView &, void *,
                                               size_t, hipStream_t);
template void launch_paged_attention<Bf16>(const AttnArgs &, const LayerView<Bf16> &, const BatchView &, void *, size_t,
                                           hipStream_t);

}  // namespace rai
