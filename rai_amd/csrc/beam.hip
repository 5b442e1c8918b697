// Beam search's selection: of beams * vocab candidates per group, those with the
// largest scores[beam] + logit - log sum exp(logits of the beam), equal ones by
// beam, then token.
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
  uint64_t *key;  // [row][chunk][take]
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

// exp(x - top) with the rounding of the difference and of its product with log2 e
// carried along: only the half step of the exponential itself is left.
__device__ __forceinline__ float exp_near(float x, float top) {
  constexpr float kLog2e = 1.4426950408889634f, kLow = 1.9259629911266175e-8f;
  const float d = x - top, v = d - x, err = (x - (d - v)) - (top + v);
  const float t = d * kLog2e;
  if (t < -150.0f) return 0.0f;
  const float low = fmaf(d, kLog2e, -t) + fmaf(d, kLow, err * kLog2e);
  const float e = __builtin_amdgcn_exp2f(t);
  return fmaf(e, low * 0.6931471805599453f, e);
}

__device__ __forceinline__ uint64_t shfl_of(uint64_t v, int d) { return __shfl_xor((unsigned long long)v, d); }

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

// Block (chunk, row): one pass over the logits, all of them in registers.
__global__ __launch_bounds__(kThreads) void k_beam_chunk(BeamArgs a, Parts out, int groups, bool vec) {
  __shared__ uint64_t list[kChunkLogits], red[kThreads];
  __shared__ double sums[kThreads / 64];
  __shared__ float tops[kThreads / 64];
  __shared__ int count;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const size_t row = blockIdx.y, at = row * gridDim.x + blockIdx.x;
  if (a.done && a.done[row]) return;  // its only candidate is known
  const float *x = a.logits + row * a.stride;
  const int base = blockIdx.x * kChunkLogits;
  float v[kPer];
#pragma unroll
  for (int i = 0; i < kPer / 4; ++i) {
    const int e = base + 4 * (tid + kThreads * i);
    if (vec && e + 4 <= a.vocab) {
      const float4 y = *reinterpret_cast<const float4 *>(x + e);
      v[4 * i] = y.x, v[4 * i + 1] = y.y, v[4 * i + 2] = y.z, v[4 * i + 3] = y.w;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[4 * i + j] = e + j < a.vocab ? x[e + j] : -INFINITY;
    }
  }
  if (tid == 0) count = 0;
  float top = -INFINITY;
  uint64_t best = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    top = fmaxf(top, v[i]);
    best = max(best, key_of(v[i], base + 4 * (tid + kThreads * (i / 4)) + i % 4));
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
  if (lane == 0) tops[wave] = top;
  const uint64_t least = threshold(best, groups, red, [](uint64_t p, uint64_t q) { return p > q; });
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) top = fmaxf(top, tops[w]);
  // The candidates that can be among the best, in any order.
  if (best >= least)
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const uint64_t k = key_of(v[i], base + 4 * (tid + kThreads * (i / 4)) + i % 4);
      if (k && k >= least) list[atomicAdd(&count, 1)] = k;
    }
  float sum = 0.0f;
  if (fabsf(top) < INFINITY)
#pragma unroll
    for (int i = 0; i < kPer; ++i) sum += v[i] > -INFINITY ? exp_near(v[i], top) : 0.0f;
  double total = sum;
#pragma unroll
  for (int d = 32; d; d >>= 1) total += __shfl_xor(total, d);
  if (lane == 0) sums[wave] = total;
  __syncthreads();
  if (tid == 0) {
    out.sum[at] = (sums[0] + sums[1]) + (sums[2] + sums[3]);
    out.top[at] = top;
  }
  // A candidate's place is the number of better ones.
  const int n = count;
  uint64_t *keys = out.key + at * a.take;
  for (int i = tid; i < n; i += kThreads) {
    const uint64_t k = list[i];
    int place = 0;
    for (int j = 0; j < n; ++j) place += list[j] > k;
    if (place < a.take) keys[place] = k;
  }
  for (int i = n + tid; i < a.take; i += kThreads) keys[i] = 0;
}

// A candidate of a group and the order of the selection.
struct Cand {
  double score;  // -inf: none
  uint64_t key;
  int beam;
};
__device__ __forceinline__ bool before(const Cand &x, const Cand &y) {
  if (x.score != y.score) return x.score > y.score;
  return x.beam != y.beam ? x.beam < y.beam : x.key > y.key;
}
__device__ __forceinline__ Cand shfl_of(const Cand &c, int d) {
  return {__shfl_xor(c.score, d), shfl_of(c.key, d), __shfl_xor(c.beam, d)};
}

constexpr int kBatch = 2048;  // candidates looked at in one go

// One block per group: the chunks' lists merged, their first places first.  A
// batch's candidates that reach the threshold (and the last of the best so far)
// are placed by counting; a whole row of places without one ends the search.
__global__ __launch_bounds__(kThreads) void k_beam_merge(BeamArgs a, Parts in, int chunks, int groups) {
  __shared__ double base[64], less[64], tops[64], sc[kBatch + 64];
  __shared__ uint64_t key[kBatch + 64];
  __shared__ int bm[kBatch + 64];
  __shared__ Cand red[kThreads], best[64];
  __shared__ int count, have;
  const int g = blockIdx.x, tid = threadIdx.x;
  // Each beam's score (-inf where there is nothing to choose), its largest logit
  // and the logarithm of its sum: apart, since a large logit would swallow the others.
  for (int b = tid; b < a.beams; b += kThreads) {
    const size_t row = (size_t)g * a.beams + b;
    double s = a.scores[row], sum = 0.0;
    float top = -INFINITY;
    if (!(a.done && a.done[row])) {
      for (int c = 0; c < chunks; ++c) top = fmaxf(top, in.top[row * chunks + c]);
      for (int c = 0; c < chunks; ++c) {
        const float t = in.top[row * chunks + c];
        if (t > -INFINITY) sum += in.sum[row * chunks + c] * exp((double)t - (double)top);
      }
      if (!(fabsf(top) < INFINITY)) s = -INFINITY;
    }
    tops[b] = top;
    less[b] = log(sum);
    base[b] = fabs(s) < INFINITY ? s : -(double)INFINITY;
  }
  if (tid == 0) have = 0;
  __syncthreads();
  const long long lists = (long long)a.beams * chunks, all = lists * a.take;
  const Cand none{-(double)INFINITY, 0, 0};
  for (long long from = 0; from < all; from += kBatch) {
    Cand c[kBatch / kThreads], mine = none;
#pragma unroll
    for (int i = 0; i < kBatch / kThreads; ++i) {
      const long long e = from + tid + kThreads * i;
      c[i] = none;
      if (e < all) {
        const long long list = e % lists;
        const int place = (int)(e / lists), beam = (int)(list / chunks), chunk = (int)(list % chunks);
        const size_t row = (size_t)g * a.beams + beam;
        c[i].beam = beam;
        if (a.done && a.done[row]) {
          if (place == 0 && chunk == 0) c[i] = {base[beam], key_of(0.0f, a.end_token), beam};
        } else {
          const uint64_t k = in.key[(row * chunks + chunk) * a.take + place];
          if (k) c[i] = {base[beam] + ((double)logit_of(k) - tops[beam] - less[beam]), k, beam};
        }
        if (before(c[i], mine)) mine = c[i];
      }
    }
    if (tid == 0) count = 0;
    Cand least = threshold(mine, groups, red, before);
    const int kept = have;
    if (kept == a.take && before(best[kept - 1], least)) least = best[kept - 1];
    int found = 0;
#pragma unroll
    for (int i = 0; i < kBatch / kThreads; ++i)
      if (c[i].score > -INFINITY && !before(least, c[i])) {
        const int at = atomicAdd(&count, 1);
        sc[at] = c[i].score;
        key[at] = c[i].key;
        bm[at] = c[i].beam;
        found = 1;
      }
    found = __syncthreads_or(found);
    if (found) {
      const int n = count + kept;
      if (tid < kept) {
        sc[count + tid] = best[tid].score;
        key[count + tid] = best[tid].key;
        bm[count + tid] = best[tid].beam;
      }
      __syncthreads();
      for (int i = tid; i < n; i += kThreads) {
        const Cand x{sc[i], key[i], bm[i]};
        int place = 0;
        for (int j = 0; j < n; ++j) place += before(Cand{sc[j], key[j], bm[j]}, x);
        if (place < a.take) best[place] = x;
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
    a.parent[o] = ok ? g * a.beams + best[tid].beam : -1;
    a.token[o] = ok ? token_of(best[tid].key) : -1;
    a.score[o] = ok ? (float)best[tid].score : -INFINITY;
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
    rai::k_beam_merge<<<(unsigned)groups, rai::kThreads, 0, s>>>(a, p, (int)chunks, few);
    RAI_HIP_CHECK(hipGetLastError());
  });
}

}  // extern "C"
