// Beam search's selection: of beams * vocab candidates per group, those with the
// largest scores[beam] + logit - log sum exp(logits of the beam), equal ones by
// beam, then logit, then token.
#include <hip/hip_runtime.h>

#include <cmath>

#include "paged.h"

namespace rai {

namespace {

struct BeamArgs {
  const float *logits;
  size_t stride;
  int vocab;
  const float *scores;
  const uint8_t *done;
  int end_token, beams, take;
  int *parent, *token;
  float *score;
};

// A row's chunk: kChunkLogits logits of one block, 16 a thread.
constexpr int kThreads = 256, kPer = 16, kChunkLogits = kThreads * kPer;

size_t chunks_of(size_t vocab) { return (vocab + kChunkLogits - 1) / kChunkLogits; }

// What a chunk leaves behind: its largest logit, the sum of exp(logit - largest),
// and its `take` best logits as keys, best first.
struct Parts {
  double *sum;    // [row][chunk]
  float *top;     // [row][chunk]
  uint64_t *key;  // [group][place][beam][chunk]
};

// Logit and token in one number that orders candidates of a row: larger logits
// first, then lower tokens; both zeros are one.  0: no candidate (NaN, -inf).
__device__ __forceinline__ uint64_t key_of(float x, int tok) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  const uint32_t up = u & 0x80000000u ? ~u : u | 0x80000000u;
  return x > -INFINITY ? (uint64_t)up << 32 | (uint32_t)~tok : 0;
}
__device__ __forceinline__ int token_of(uint64_t k) { return (int)~(uint32_t)k; }
__device__ __forceinline__ float logit_of(uint64_t k) {
  const uint32_t up = (uint32_t)(k >> 32);
  return __uint_as_float(up & 0x80000000u ? up & 0x7fffffffu : ~up);
}

// exp(x - top), x <= top: the product with log2 e carries its rounding along, so
// that only the half steps of the difference and of the exponential are left.  A
// row's log-sum: half steps of a difference of up to log(vocab), 21, in the mean, two of
// the exponential, one of the correction, 15 of a thread's sum: 3e-6 together at most.
__device__ __forceinline__ float exp_near(float x, float top) {
  constexpr float kLog2e = 1.4426950408889634f, kLow = 1.9259629911266175e-8f, kLn2 = 0.6931471805599453f;
  const float d = fmaxf(x - top, -200.0f), t = d * kLog2e;
  const float low = fmaf(d, kLow, fmaf(d, kLog2e, -t)), e = __builtin_amdgcn_exp2f(t);
  return fmaf(e * kLn2, low, e);
}

__device__ __forceinline__ uint64_t shfl_of(uint64_t v, int d) { return __shfl_xor((unsigned long long)v, d); }
__device__ __forceinline__ float shfl_of(float v, int d) { return __shfl_xor(v, d); }
__device__ __forceinline__ double shfl_of(double v, int d) { return __shfl_xor(v, d); }

// The smallest of the maxima of `groups` interleaved groups of the block's threads
// (a power of two up to 64): at least `groups` of the block's values reach it, and
// few more where they are spread evenly.
template <class V, class Before>
__device__ __forceinline__ V threshold(V v, int groups, V *red, Before better) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  auto pick = [&](V o) { v = better(o, v) ? o : v; };
  for (int d = 32; d >= groups; d >>= 1) pick(shfl_of(v, d));
  __syncthreads();
  if (lane < groups) red[wave * 64 + lane] = v;
  __syncthreads();
  v = red[lane & (groups - 1)];
#pragma unroll
  for (int w = 1; w < kThreads / 64; ++w) pick(red[w * 64 + (lane & (groups - 1))]);
  for (int d = groups >> 1; d; d >>= 1) {
    const V o = shfl_of(v, d);
    v = better(v, o) ? o : v;
  }
  return v;
}

constexpr int kList = 512;  // candidates of a chunk that are placed by counting

// Block (chunk, row): one pass over the logits, all of them in registers.  Bound by
// the vector instructions, some 555 a wave of 1024 logits (35 for each of a lane's 16),
// and the loads before them: the candidates are cut by their f32 value first, and by
// value and token only where too many are equal.  215 rows of 50304: 20 us, 2.2 TB/s
// (with 32 logits a thread 22).
__global__ __launch_bounds__(kThreads) void k_beam_chunk(BeamArgs a, Parts out, int groups, bool vec) {
  __shared__ uint64_t list[kList], red[kThreads];
  __shared__ double sums[kThreads / 64];
  __shared__ float tops[kThreads / 64];
  __shared__ int count;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const size_t row = blockIdx.y, at = row * gridDim.x + blockIdx.x;
  if (a.done && a.done[row]) return;  // its only candidate is known
  const float *x = a.logits + row * a.stride;
  const int base = blockIdx.x * kChunkLogits;
  float v[kPer];
  if (vec && base + kChunkLogits <= a.vocab) {
#pragma unroll
    for (int i = 0; i < kPer / 4; ++i) {
      const float4 y = *reinterpret_cast<const float4 *>(x + base + 4 * (tid + kThreads * i));
      v[4 * i] = y.x, v[4 * i + 1] = y.y, v[4 * i + 2] = y.z, v[4 * i + 3] = y.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int e = base + 4 * (tid + kThreads * (i / 4)) + i % 4;
      v[i] = e < a.vocab ? x[e] : -INFINITY;
    }
  }
  auto token = [&](int i) { return base + 4 * (tid + kThreads * (i / 4)) + i % 4; };
  if (tid == 0) count = 0;
  float mine = -INFINITY, top;
#pragma unroll
  for (int i = 0; i < kPer; ++i) mine = fmaxf(mine, v[i]);
  top = mine;
#pragma unroll
  for (int d = 32; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
  if (lane == 0) tops[wave] = top;
  const float least = threshold(mine, groups, reinterpret_cast<float *>(red), [](float p, float q) { return p > q; });
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) top = fmaxf(top, tops[w]);
  // The candidates that can be among the best, in any order.
  uint32_t hits = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) hits |= (v[i] >= least && v[i] > -INFINITY ? 1u : 0u) << i;
  if (hits) {
    int n = atomicAdd(&count, __popc(hits));
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (hits >> i & 1) {
        if (n < kList) list[n] = key_of(v[i], token(i));
        ++n;
      }
  }
  float sum = 0.0f;  // -inf and NaN add nothing
  if (fabsf(top) < INFINITY)
#pragma unroll
    for (int i = 0; i < kPer; ++i) sum += exp_near(v[i], top);
  double total = sum;
#pragma unroll
  for (int d = 32; d; d >>= 1) total += __shfl_xor(total, d);
  if (lane == 0) sums[wave] = total;
  __syncthreads();
  if (tid == 0) {
    out.sum[at] = (sums[0] + sums[1]) + (sums[2] + sums[3]);
    out.top[at] = top;
  }
  // [group][place][beam][chunk]: the merge reads first places first.
  const size_t lists = (size_t)a.beams * gridDim.x;
  uint64_t *keys = out.key + (row / a.beams) * a.take * lists + row % a.beams * gridDim.x + blockIdx.x;
  int n = count;
  if (n > kList) {
    uint64_t best = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) best = max(best, key_of(v[i], token(i)));
    auto larger = [](uint64_t p, uint64_t q) { return p > q; };
    const uint64_t cut = threshold(best, groups, red, larger);
    if (tid == 0) count = 0;
    __syncthreads();
    if (best >= cut)
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const uint64_t k = key_of(v[i], token(i));
        if (k && k >= cut) {
          const int m = atomicAdd(&count, 1);
          if (m < kList) list[m] = k;
        }
      }
    __syncthreads();
    n = count;
    if (n > kList) {  // the best sit in a few threads: one after the other
      uint64_t last = ~(uint64_t)0;
      for (int p = 0; p < a.take; ++p) {
        uint64_t next = 0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          const uint64_t k = key_of(v[i], token(i));
          if (k < last) next = max(next, k);
        }
        last = threshold(next, 1, red, larger);
        if (tid == 0) keys[p * lists] = last;
      }
      return;
    }
  }
  // A candidate's place is the number of better ones.
  for (int i = tid; i < n; i += kThreads) {
    const uint64_t k = list[i];
    int place = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) place += list[j] > k;
    if (place < a.take) keys[place * lists] = k;
  }
  for (int i = n + tid; i < a.take; i += kThreads) keys[i * lists] = 0;
}

constexpr int kBatch = 2048;  // candidates looked at in one go

// One block per group: the chunks' lists merged, their first places first.  A
// batch's candidates that reach the threshold (and the last of the best so far)
// are placed by counting.  Bound by the latency of its few dependent steps; `per`
// threads (a power of two) share the chunks of a beam.  8 beams of 13 chunks, 16 taken:
// 9 us, 4 of them an empty kernel's.
__global__ __launch_bounds__(kThreads) void k_beam_merge(BeamArgs a, Parts in, int chunks, int groups, int per, Div by_lists,
                                                         Div by_chunks) {
  __shared__ double base[64], less[64], tops[64], sc[kBatch + 64];
  __shared__ uint64_t key[kBatch + 64];
  __shared__ int bm[kBatch + 64];
  __shared__ double red[kThreads], kept_sc[64];
  __shared__ uint64_t kept_key[64];
  __shared__ int kept_beam[64];
  __shared__ int count, have;
  const int g = blockIdx.x, tid = threadIdx.x;
  const uint32_t lists = by_lists.d, all = lists * a.take;
  const uint64_t *keys = in.key + (size_t)g * all;
  constexpr int kN = kBatch / kThreads;
  uint64_t k[kN];
  auto load = [&](uint32_t from) {
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const uint32_t e = from + tid + kThreads * i;
      k[i] = e < all ? keys[e] : 0;
    }
  };
  load(0);
  // Each beam's score (-inf where there is nothing to choose), its largest logit
  // and the logarithm of its sum: apart, since a large logit would swallow the others.
  for (int b = tid / per; b < a.beams; b += kThreads / per) {
    const size_t row = (size_t)g * a.beams + b;
    const bool done = a.done && a.done[row];
    float s = a.scores[row], top = -INFINITY;
    double sum = 0.0;
    if (!done) {
      for (int c = tid & (per - 1); c < chunks; c += per) {
        const float t = in.top[row * chunks + c];
        const double w = in.sum[row * chunks + c];
        if (!(t > -INFINITY)) continue;
        const float m = fmaxf(top, t);
        sum = sum * exp((double)top - (double)m) + w * exp((double)t - (double)m);
        top = m;
      }
      for (int d = per >> 1; d; d >>= 1) {
        const float t = __shfl_xor(top, d), m = fmaxf(top, t);
        const double w = __shfl_xor(sum, d);
        sum = (sum > 0.0 ? sum * exp((double)top - (double)m) : 0.0) + (w > 0.0 ? w * exp((double)t - (double)m) : 0.0);
        top = m;
      }
    }
    if ((tid & (per - 1)) == 0) {
      base[b] = fabsf(s) < INFINITY && (done || fabsf(top) < INFINITY) ? (double)s : -(double)INFINITY;
      less[b] = log(sum);
      tops[b] = done ? INFINITY : top;  // infinite: a finished beam
    }
  }
  if (tid == 0) have = 0;
  __syncthreads();
  for (uint32_t from = 0; from < all; from += kBatch) {
    double score[kN], mine = -INFINITY;
    uint64_t ck[kN];
    int beam[kN];
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const uint32_t e = from + tid + kThreads * i, list = e - by_lists(e) * lists;
      beam[i] = (int)by_chunks(list);
      ck[i] = k[i];
      double s = base[beam[i]];
      if (tops[beam[i]] == INFINITY) {
        ck[i] = key_of(0.0f, a.end_token);
        if (e >= lists || beam[i] * by_chunks.d != list) s = -INFINITY;
      } else {
        s += (double)logit_of(ck[i]) - tops[beam[i]] - less[beam[i]];
        if (ck[i] == 0 || !(base[beam[i]] > -INFINITY)) s = -INFINITY;
      }
      score[i] = e < all ? s : -INFINITY;
      mine = fmax(mine, score[i]);
    }
    load(from + kBatch < all ? from + kBatch : all);
    if (tid == 0) count = 0;
    double least = threshold(mine, groups, red, [](double p, double q) { return p > q; });
    const int kept = have;
    if (kept == a.take) least = fmax(least, kept_sc[kept - 1]);
    int found = 0;
#pragma unroll
    for (int i = 0; i < kN; ++i)
      if (score[i] > -INFINITY && score[i] >= least) {
        const int at = atomicAdd(&count, 1);
        sc[at] = score[i];
        key[at] = ck[i];
        bm[at] = beam[i];
        found = 1;
      }
    found = __syncthreads_or(found);
    if (found) {
      const int n = count + kept;
      if (tid < kept) {
        sc[count + tid] = kept_sc[tid];
        key[count + tid] = kept_key[tid];
        bm[count + tid] = kept_beam[tid];
      }
      __syncthreads();
      for (int i = tid; i < n; i += kThreads) {
        const double s = sc[i];
        const uint64_t x = key[i];
        const int b = bm[i];
        int place = 0, equal = 0;
#pragma unroll 8
        for (int j = 0; j < n; ++j) {
          const double o = sc[j];
          place += o > s;
          equal += o == s;
        }
        if (equal > 1)
          for (int j = 0; j < n; ++j) place += sc[j] == s && (bm[j] < b || (bm[j] == b && key[j] > x));
        if (place < a.take) {
          kept_sc[place] = s;
          kept_key[place] = x;
          kept_beam[place] = b;
        }
      }
      if (tid == 0) have = min(n, a.take);
      __syncthreads();
    } else if (kept == a.take && lists <= kBatch) {
      break;  // a place of every list was among these: the later ones are behind it
    }
  }
  __syncthreads();
  if (tid < a.take) {
    const size_t o = (size_t)g * a.take + tid;
    const bool ok = tid < have;
    a.parent[o] = ok ? g * a.beams + kept_beam[tid] : -1;
    a.token[o] = ok ? token_of(kept_key[tid]) : -1;
    a.score[o] = ok ? (float)kept_sc[tid] : -INFINITY;
  }
}

size_t beam_work(size_t vocab, size_t groups, size_t beams, size_t take) {
  return groups * beams * chunks_of(vocab) * (sizeof(double) + sizeof(uint64_t) * take + sizeof(float));
}

void check_beam(size_t vocab, size_t groups, size_t beams, size_t take) {
  if (vocab == 0) fail(RAI_E_SHAPE, "selection over an empty row");
  if (beams == 0 || beams > 64) fail(RAI_E_SHAPE, "beams must be 1 to 64");
  if (take == 0 || take > 64) fail(RAI_E_SHAPE, "take must be 1 to 64");
  if (vocab > (size_t(1) << 30) || groups > 65535 || groups * beams > 65535) fail(RAI_E_SHAPE, "dimensions overflow");
}

}  // namespace

}  // namespace rai

extern "C" {

int rai_beam_select_workspace(size_t vocab, size_t groups, size_t beams, size_t take, size_t *bytes) {
  RAI_API_BODY({
    if (!bytes) rai::fail(RAI_E_ARG, "null argument");
    rai::check_beam(vocab, groups, beams, take);
    *bytes = rai::beam_work(vocab, groups, beams, take);
  });
}

int rai_beam_select_dev(const float *logits, size_t stride, size_t vocab, const float *scores, const uint8_t *done,
                        int32_t end_token, size_t groups, size_t beams, size_t take, int32_t *parent,
                        int32_t *token, float *score, void *work, size_t work_bytes, void *stream) {
  RAI_API_BODY({
    rai::check_beam(vocab, groups, beams, take);
    if (groups == 0) return RAI_OK;
    if (!logits || !scores || !parent || !token || !score || !work) rai::fail(RAI_E_ARG, "null argument");
    if (stride < vocab) rai::fail(RAI_E_SHAPE, "logits rows overlap: the stride is shorter than a row");
    if (done && (end_token < 0 || (size_t)end_token >= vocab)) rai::fail(RAI_E_RANGE, "end_token is out of range");
    if ((uintptr_t)work % 16) rai::fail(RAI_E_ARG, "work must be 16-byte aligned");
    if (work_bytes < rai::beam_work(vocab, groups, beams, take))
      rai::fail(RAI_E_SHAPE, "work is smaller than rai_beam_select_workspace");
    const rai::BeamArgs a{logits, stride, (int)vocab, scores, done, end_token, (int)beams, (int)take, parent, token, score};
    const size_t rows = groups * beams, chunks = rai::chunks_of(vocab);
    rai::Parts p;
    p.sum = static_cast<double *>(work);
    p.key = reinterpret_cast<uint64_t *>(p.sum + rows * chunks);
    p.top = reinterpret_cast<float *>(p.key + rows * chunks * take);
    int few = 1;
    while ((size_t)few < take) few *= 2;
    const bool vec = (uintptr_t)logits % 16 == 0 && stride % 4 == 0;
    hipStream_t s = (hipStream_t)stream;
    rai::k_beam_chunk<<<dim3((unsigned)chunks, (unsigned)rows), rai::kThreads, 0, s>>>(a, p, few, vec);
    int per = 1;
    while (per < 64 && (size_t)per < chunks && per * beams < rai::kThreads) per *= 2;
    rai::k_beam_merge<<<(unsigned)groups, rai::kThreads, 0, s>>>(a, p, (int)chunks, few, per,
                                                                 rai::Div((uint32_t)(beams * chunks)),
                                                                 rai::Div((uint32_t)chunks));
    RAI_HIP_CHECK(hipGetLastError());
  });
}

}  // extern "C"
