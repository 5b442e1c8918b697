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

__device__ __forceinline__ double block_sum(double x, double *red) {
  const int tid = threadIdx.x;
  red[tid] = x;
  for (int d = 128; d; d >>= 1) {
    __syncthreads();
    if (tid < d) red[tid] += red[tid + d];
  }
  __syncthreads();
  const double r = red[0];
  __syncthreads();
  return r;
}

// log sum exp of a row; NaN counts as -inf.
__global__ __launch_bounds__(256) void k_beam_lse(BeamArgs a, double *lse) {
  __shared__ double red[256];
  const float *x = a.logits + (size_t)blockIdx.x * a.stride;
  float m = -INFINITY;
  for (int i = threadIdx.x; i < a.vocab; i += 256) m = fmaxf(m, x[i]);
  red[threadIdx.x] = m;
  for (int d = 128; d; d >>= 1) {
    __syncthreads();
    if (threadIdx.x < d) red[threadIdx.x] = fmax(red[threadIdx.x], red[threadIdx.x + d]);
  }
  __syncthreads();
  const float top = (float)red[0];
  __syncthreads();
  double sum = 0.0;
  if (std::isfinite(top))
    for (int i = threadIdx.x; i < a.vocab; i += 256) {
      const float v = x[i];
      sum += v == v ? exp((double)v - (double)top) : 0.0;
    }
  sum = block_sum(sum, red);
  if (threadIdx.x == 0) lse[blockIdx.x] = std::isfinite(top) ? (double)top + log(sum) : (double)INFINITY;
}

// A candidate and the order of the selection.
struct Cand {
  double score;
  float logit;
  int beam, tok;  // beam < 0: none
};
__device__ __forceinline__ bool before(const Cand &x, const Cand &y) {
  if (x.beam < 0 || y.beam < 0) return x.beam >= 0 && y.beam < 0;
  if (x.score != y.score) return x.score > y.score;
  if (x.beam != y.beam) return x.beam < y.beam;
  if (x.logit != y.logit) return x.logit > y.logit;
  return x.tok < y.tok;
}

// One block per group: the best candidate behind the last one chosen, `take`
// times over all candidates.
__global__ __launch_bounds__(256) void k_beam_pick(BeamArgs a, const double *lse) {
  __shared__ Cand best[256];
  const int g = blockIdx.x, tid = threadIdx.x;
  const long long n = (long long)a.beams * a.vocab;
  Cand last{0.0, 0.0f, -1, 0};
  for (int k = 0; k < a.take; ++k) {
    Cand b{0.0, 0.0f, -1, 0};
    for (long long i = tid; i < n && (k == 0 || last.beam >= 0); i += 256) {
      const int beam = (int)(i / a.vocab), tok = (int)(i % a.vocab), row = g * a.beams + beam;
      Cand c{(double)a.scores[row], 0.0f, beam, tok};
      if (a.done && a.done[row]) {
        if (tok != a.end_token) continue;
      } else {
        c.logit = a.logits[(size_t)row * a.stride + tok];
        c.score += (double)c.logit - lse[row];
      }
      if (c.score > -INFINITY && (k == 0 || before(last, c)) && before(c, b)) b = c;
    }
    best[tid] = b;
    for (int d = 128; d; d >>= 1) {
      __syncthreads();
      if (tid < d && before(best[tid + d], best[tid])) best[tid] = best[tid + d];
    }
    __syncthreads();
    last = best[0];
    __syncthreads();
    if (tid == 0) {
      const size_t o = (size_t)g * a.take + k;
      const bool ok = last.beam >= 0;
      a.parent[o] = ok ? g * a.beams + last.beam : -1;
      a.token[o] = ok ? last.tok : -1;
      a.score[o] = ok ? (float)last.score : -INFINITY;
    }
  }
}

size_t beam_work(size_t, size_t groups, size_t beams, size_t) { return groups * beams * sizeof(double); }

void check_beam(size_t vocab, size_t groups, size_t beams, size_t take) {
  if (vocab == 0) fail(RAI_E_SHAPE, "selection over an empty row");
  if (beams == 0 || beams > 64) fail(RAI_E_SHAPE, "beams must be 1 to 64");
  if (take == 0 || take > 64) fail(RAI_E_SHAPE, "take must be 1 to 64");
  if (vocab > INT32_MAX || groups > 65535) fail(RAI_E_SHAPE, "dimensions overflow");
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
    double *lse = static_cast<double *>(work);
    hipStream_t s = (hipStream_t)stream;
    rai::k_beam_lse<<<(unsigned)(groups * beams), 256, 0, s>>>(a, lse);
    rai::k_beam_pick<<<(unsigned)groups, 256, 0, s>>>(a, lse);
    RAI_HIP_CHECK(hipGetLastError());
  });
}

}  // extern "C"
