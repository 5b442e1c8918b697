// Shared by the paged cache's kernels: one layer of a pool, its element types,
// and the launchers (asynchronous, validate nothing).
#ifndef RAI_PAGED_H
#define RAI_PAGED_H

#include <hip/hip_runtime.h>

#include "common.h"
#include "paged_index.h"

#define RAI_HIP_CHECK(expr)                                                                \
  do {                                                                                     \
    hipError_t e_ = (expr);                                                                \
    if (e_ != hipSuccess)                                                                  \
      rai::fail(e_ == hipErrorOutOfMemory ? RAI_E_OOM : RAI_E_HIP,                         \
                std::string(#expr) + ": " + hipGetErrorString(e_));                        \
  } while (0)

namespace rai {

struct Bf16 {
  uint16_t b;
};

// One layer of the pool.
template <class T>
struct LayerView {
  T *k, *v;
  int pages, shift, nkv, hd;
};

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(_Float16 x) { return (float)x; }
__device__ __forceinline__ float to_f32(Bf16 x) { return __uint_as_float((uint32_t)x.b << 16); }

// Round to nearest, ties to even; a NaN stays one.
template <class T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) {
  return x;
}
template <>
__device__ __forceinline__ _Float16 from_f32<_Float16>(float x) {
  return (_Float16)x;
}
template <>
__device__ __forceinline__ Bf16 from_f32<Bf16>(float x) {
  const uint32_t u = __float_as_uint(x);
  if ((u & 0x7fffffffu) > 0x7f800000u) return Bf16{(uint16_t)((u >> 16) | 0x40)};
  return Bf16{(uint16_t)((u + 0x7fffu + ((u >> 16) & 1)) >> 16)};
}

// n / d for n < 2^31: the high half of n times ceil(2^(32 + s) / d) - 2^32, plus n.
struct Div {
  uint32_t d, m, s;
  explicit Div(uint32_t by) : d(by), s(0) {
    while ((uint64_t(1) << s) < by) ++s;
    m = (uint32_t)(((uint64_t(1) << 32) * ((uint64_t(1) << s) - by)) / by + 1);
  }
  __device__ __forceinline__ uint32_t operator()(uint32_t n) const { return (__umulhi(m, n) + n) >> s; }
};

struct AttnArgs {
  const float *q;
  float *out;
  size_t q_stride, out_stride;
  int heads;
  float scale, softcap;
  int window;  // 0: everything
  const float *slopes;
};

// Bytes of work that launch_paged_attention can use for these bounds and elements of
// `size` bytes.
size_t paged_attention_work(int nkv, int heads, int hd, int size, const BatchView &b, int window);
template <class T>
void launch_paged_attention(const AttnArgs &a, const LayerView<T> &kv, const BatchView &b, void *work,
                            size_t work_bytes, hipStream_t s);

}  // namespace rai

#endif
