// Attention over the pages of a paged KV cache.
//
//   out = sum_j p_j v_j / sum_j p_j,  p_j = exp(s_j - max s),  s_j = cap(q . k_j scale) - slope (pos - j)
//
// over the positions j that a row sees, in one pass with the running maximum and
// sum of the softmax.  The rows of one kv head (new tokens x the query heads on
// it) share its keys and values: S^T = K Q^T and O^T = V^T P^T are tiles of the
// 16-bit matrix instructions, with f32 sums.
//
// f32 accuracy from 16-bit operands.  An f32 value is the exact sum of three bf16
// ones (8 + 8 + 8 bits, each cut off), so a product with a bf16 value is three
// exact products, and one of two f32 values the six largest of nine: the others are
// below 2^-21 of it together, 1.8 half steps of f32 in a normal row's result.  Against f16
// values two f16 parts do (11 + 11 bits and the sign of the second), the queries of a
// row scaled by a power of two that brings the largest to 2^14 .. 2^15, the
// probabilities by 2^14: what is below 2^-17 of the largest has fewer bits, to 2^-39 of it.  The f32 matrix instructions run at
// a sixteenth of the 16-bit rate: three or six products are the faster way.
//
// Layout.  The instruction leaves row 4 g + i (16 x 16) or 8 b + 4 h + c (32 x 32)
// of S^T in lane group g or h; the keys are dealt to the rows so that a lane ends
// up with eight keys in a row for one query, which is what the second product
// takes as its operand: the probabilities never leave their lane.
//
// Results that are not finite (a NaN or an infinity in what the row sees, or in
// what a neighbour sees: 0 x inf in the shared products) are computed again row by
// row, from the keys that the row sees alone.
#include "kernels.h"
#include "paged.h"

#include <algorithm>
#include <cmath>

namespace rai {

namespace {

constexpr float kLog2e = 1.4426950408889634f;

typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));

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

// tanh.  Near zero, where 1 - 2 / (e^2x + 1) cancels, x + x^3 P(x^2) with P fitted to
// the smallest relative error over 0..0.625 (6e-9).
constexpr float kTanhNear = 0.625f;
__device__ __forceinline__ float tanh_near(float x) {
  const float y = x * x;
  const float p = fmaf(fmaf(fmaf(fmaf(-0.005717044f, y, 0.020650586f), y, -0.053743497f), y, 0.13331491f), y, -0.33333284f);
  return fmaf(x * y, p, x);
}
__device__ __forceinline__ float cap_tanh(float x) {
  const float e = __builtin_amdgcn_exp2f(2.0f * kLog2e * fabsf(x));
  const float far = 1.0f - 2.0f * __builtin_amdgcn_rcpf(e + 1.0f);
  return fabsf(x) < kTanhNear ? tanh_near(x) : copysignf(far, x);
}

// A score in the log2 domain: x = q . k * scale.
struct Score {
  float softcap, inv_cap, slope;
  bool plain;
  __device__ __forceinline__ float operator()(float x, int away) const {
    if (plain) return x * kLog2e;
    if (softcap > 0.0f) x = softcap * cap_tanh(x * inv_cap);
    return (x - slope * (float)away) * kLog2e;
  }
};
__device__ __forceinline__ Score score_of(const AttnArgs &a, int head) {
  return {a.softcap, a.softcap > 0.0f ? 1.0f / a.softcap : 0.0f, a.slopes ? a.slopes[head] : 0.0f,
          a.softcap == 0.0f && !a.slopes};
}

// ------------------------------------------------------------ rows and splits --

// Rows of a sequence on one kv head: r = token * per + query head of the group.
// Tile t holds rows t * R .. of them and reads positions lo .. hi - 1.
struct Tile {
  int lo, hi;  // lo: a multiple of 64
};
__device__ __forceinline__ Tile tile_of(const SeqSpan &sp, int t, int R, int per, int window) {
  const int base = sp.n - sp.nq, first = t * R / per, last = min(sp.nq - 1, (t * R + R - 1) / per);
  return {first_seen(base + first, window) & ~63, max(base + last + 1, 0)};
}
// A tile's positions in equal splits of whole 128, as many as `len` asks for.
struct Share {
  int count, len;
};
__device__ __forceinline__ Share share_of(const Tile &t, int len) {
  const int span = t.hi - t.lo;
  if (span <= len) return {1, len};
  const int n = (span + len - 1) / len, each = ((span + n - 1) / n + 127) & ~127;
  return {(span + each - 1) / each, each};
}

constexpr int kFewRows = 16;    // a tile of k_few
constexpr int kManyRows = 128;  // a tile of k_many

// Sequences of at most few_max rows a kv head go to k_few, others to k_many.  How
// the key axis is split, and where the parts of a row's softmax lie: [row][split] x hd
// values, and maximum and sum.  k_few's rows are 16 few_tiles to a (sequence, kv head),
// k_many's the heads of the batch's rows.
struct Parts {
  int len, most;
  float *o;
  float2 *ml;
  __device__ __forceinline__ size_t at(size_t row, int split) const { return row * most + split; }
};
struct Splits {
  int few_max, few_tiles;
  Parts few, many;
  __device__ __forceinline__ bool is_few(int nq, int per) const { return nq * per <= few_max; }
  __device__ __forceinline__ size_t few_row(int seq, int kvh, int nkv, int r) const {
    return ((size_t)seq * nkv + kvh) * few_tiles * kFewRows + r;
  }
};

// -------------------------------------------------------------------- one row --

// One row of one head by one wave: positions lo .. hi - 1 of the sequence whose
// table row is `table`, lane t holding key base + t and dimensions t, t + 64, ...
// of the output.  Keys that are not there or masked are not read into the sums at
// all, whatever they hold.  m is in the log2 domain; o is the weighted mean so far
// (a sum of large values could leave f32's range), l the sum of the weights.
template <class T>
__device__ __forceinline__ void wave_row(const AttnArgs &a, const LayerView<T> &kv, const int *table, int head,
                                         const float *q, int pos, int lo, int hi, float &m, float &l, float (&o)[4]) {
  const int lane = threadIdx.x & 63, hd = kv.hd, kvh = head / (a.heads / kv.nkv), mask = (1 << kv.shift) - 1;
  const Score score = score_of(a, head);
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
      s = score(d * a.scale, pos - j);
    }
    float mn = fmaxf(m, wave_max(s));
    if (__any(s != s)) mn = NAN;
    if (mn == -INFINITY) continue;
    const float p = exp2f(s - mn), old = l * exp2f(m - mn), sum = old + wave_sum(p), inv = 1.0f / sum;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] *= old * inv;
    for (int t = 0; t < 64 && base + t < hi; ++t) {
      const int pg = __shfl(page, t);
      const float pt = __shfl(p, t) * inv;
      if (pg < 0) continue;
      const T *v = kv.v + value_at(pg, kvh, (base + t) & mask, kv.nkv, hd, kv.shift);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (lane + 64 * i < hd) o[i] = fmaf(pt, to_f32(v[(size_t)(lane + 64 * i) << kv.shift]), o[i]);
    }
    m = mn;
    l = sum;
  }
}

// A row's result again, from its own keys of positions lo .. hi - 1; as part `at` of
// `parts` where the row is split.
template <class T>
__device__ __forceinline__ void redo_row(const AttnArgs &a, const LayerView<T> &kv, const int *table, int row, int head,
                                         int pos, int lo, int hi, const Parts &parts, size_t at, bool split) {
  const int lane = threadIdx.x & 63;
  float m, l, o[4];
  wave_row(a, kv, table, head, a.q + (size_t)row * a.q_stride + (size_t)head * kv.hd, pos,
           max(lo, first_seen(pos, a.window)), min(hi, pos + 1), m, l, o);
  float *out = a.out + (size_t)row * a.out_stride + (size_t)head * kv.hd;
  if (split) {
    out = parts.o + at * kv.hd;
    // The sum as parts hold it; where that leaves f32's range, the mean with all weight in the maximum.
    bool over = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) over = over || (fabsf(o[i]) < INFINITY && !(fabsf(o[i] * l) < INFINITY));
    over = __any(over);
    if (lane == 0) parts.ml[at] = over ? make_float2(m + log2f(l), 1.0f) : make_float2(m, l);
    if (!over)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] *= l;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (lane + 64 * i < kv.hd) out[lane + 64 * i] = o[i];
}

// ------------------------------------------------------------- 16-bit operands --

// Eight values of the cache as a matrix operand, in KP parts; P parts of an f32
// operand against them; the products that count, largest last.
template <class T>
struct Form;

__device__ __forceinline__ u4 cut3(const float (&x)[8], u4 &mid, u4 &low) {
  u4 h;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t a = __float_as_uint(x[2 * i]), b = __float_as_uint(x[2 * i + 1]);
    h[i] = __builtin_amdgcn_perm(b, a, 0x07060302);
    const float ra = x[2 * i] - __uint_as_float(a & 0xffff0000u), rb = x[2 * i + 1] - __uint_as_float(b & 0xffff0000u);
    const uint32_t c = __float_as_uint(ra), d = __float_as_uint(rb);
    mid[i] = __builtin_amdgcn_perm(d, c, 0x07060302);
    const float la = ra - __uint_as_float(c & 0xffff0000u), lb = rb - __uint_as_float(d & 0xffff0000u);
    low[i] = __builtin_amdgcn_perm(__float_as_uint(lb), __float_as_uint(la), 0x07060302);
  }
  return h;
}

struct Bf16Form {
  static constexpr int P = 3;
  static constexpr float kLift = 0.0f;
  static __device__ __forceinline__ f4 mma16(u4 x, u4 y, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, x), __builtin_bit_cast(b8, y), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f16v mma32(u4 x, u4 y, f16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8, x), __builtin_bit_cast(b8, y), c, 0, 0, 0);
  }
  static __device__ __forceinline__ void parts(const float (&x)[8], u4 (&p)[3]) { p[0] = cut3(x, p[1], p[2]); }
  static __device__ __forceinline__ int row_exponent(float) { return 0; }
};
template <>
struct Form<float> : Bf16Form {
  static constexpr int KP = 3;
};
template <>
struct Form<Bf16> : Bf16Form {
  static constexpr int KP = 1;
};
template <>
struct Form<_Float16> {
  static constexpr int P = 2, KP = 1;
  static constexpr float kLift = 14.0f;  // probabilities times 2^14: f16's subnormals start 2^-28 below the largest
  static __device__ __forceinline__ f4 mma16(u4 x, u4 y, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, x), __builtin_bit_cast(h8, y), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f16v mma32(u4 x, u4 y, f16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, x), __builtin_bit_cast(h8, y), c, 0, 0, 0);
  }
  static __device__ __forceinline__ void parts(const float (&x)[8], u4 (&p)[2]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const h2 h = {(_Float16)x[2 * i], (_Float16)x[2 * i + 1]};
      const h2 l = {(_Float16)(x[2 * i] - (float)h[0]), (_Float16)(x[2 * i + 1] - (float)h[1])};
      p[0][i] = __builtin_bit_cast(uint32_t, h);
      p[1][i] = __builtin_bit_cast(uint32_t, l);
    }
  }
  // The power of two that brings a row's largest value to 2^14..2^15.
  static __device__ __forceinline__ int row_exponent(float most) {
    return most > 0.0f && most < INFINITY ? 14 - ilogbf(most) : 0;
  }
};

// c += the product of a cache operand x (KP parts) and an f32 operand y (P parts).
template <class F, class C, int KP, int P, class M>
__device__ __forceinline__ C products(const u4 (&x)[KP], const u4 (&y)[P], C c, M mma) {
#pragma unroll
  for (int w = KP + P - 2 < P - 1 ? KP + P - 2 : P - 1; w >= 0; --w)  // parts i + j = w, smallest first
#pragma unroll
    for (int i = 0; i < KP; ++i)
      if (w - i >= 0 && w - i < P) c = mma(x[i], y[w - i], c);
  return c;
}

// Eight cache values in flight, and as the parts of an operand.
template <class T>
struct Raw {
  u4 v[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T *p) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) v[i] = reinterpret_cast<const u4 *>(p)[i];
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) v[i] = u4{0, 0, 0, 0};
  }
  // A lane's values of an operand in LDS (f32: in two halves of 64 lanes).
  __device__ __forceinline__ void fetch(const u4 *at) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) v[i] = at[64 * i];
  }
  // Keeps elements from .. to - 1 of the eight.
  __device__ __forceinline__ void keep(int from, int to) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const bool in = e >= from && e < to;
      if constexpr (sizeof(T) == 4)
        v[e / 4][e % 4] = in ? v[e / 4][e % 4] : 0u;
      else
        v[0][e / 2] = in ? v[0][e / 2] : v[0][e / 2] & (e % 2 ? 0x0000ffffu : 0xffff0000u);
    }
  }
  __device__ __forceinline__ void parts(u4 (&x)[Form<T>::KP]) const {
    if constexpr (sizeof(T) == 4) {
      float f[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = __uint_as_float(v[e / 4][e % 4]);
      x[0] = cut3(f, x[1], x[2]);
    } else {
      x[0] = v[0];
    }
  }
};

// Values of a lane's keys in k_few: 16 bytes either way, eight of f16 or bf16, four
// of f32.
template <class T>
struct Keys : Raw<T> {};
template <>
struct Keys<float> {
  u4 v[1];
  __device__ __forceinline__ void load(const float *p) { v[0] = *reinterpret_cast<const u4 *>(p); }
  __device__ __forceinline__ void zero() { v[0] = u4{0, 0, 0, 0}; }
  __device__ __forceinline__ void keep(int from, int to) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[0][e] = e >= from && e < to ? v[0][e] : 0u;
  }
};

// Query values e .. e + 7 of a row (zero from hd on); `vec`: 16-byte loads fit.
__device__ __forceinline__ void query8(const float *q, int e, int hd, bool vec, float (&x)[8]) {
  if (e >= hd) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = 0.0f;
  } else if (vec) {
    const f4 a = *reinterpret_cast<const f4 *>(q + e), b = *reinterpret_cast<const f4 *>(q + e + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = a[i], x[4 + i] = b[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = q[e + i];
  }
}

__device__ __forceinline__ bool finite4(f4 x) {
  return fabsf(x[0]) < INFINITY && fabsf(x[1]) < INFINITY && fabsf(x[2]) < INFINITY && fabsf(x[3]) < INFINITY;
}

// -------------------------------------------------------------------- few rows --

// At most 64 rows a kv head: one token of a sequence, or a verify batch.  Block
// (split, tile of 16 rows, kv head; sequence); the keys go to the waves 32 at a time (16
// of f32), straight from the pages into the operands (a tile reads each once, so there
// is nothing to stage), and the waves' softmaxes are joined in LDS.  Bound by memory:
// the next step's page ids, keys and values are on their way while a step is worked on,
// and f32 values go into the f32 instructions as they come (64 a step of 16 keys, four
// times as fast as memory delivers; cutting the values took some 700 vector instructions
// a step).  The tiles of one split run side by side on one XCD (blocks 8 apart), whose L2
// gives the later ones the same keys.  32 sequences of up to 4096 positions, 32 heads on
// 8 of 128 dimensions, bf16: 79 us, 4.4 TB/s; 9 tokens of 8 sequences, 16 heads, f32:
// 77 us, 4.1 TB/s.  Short contexts of few heads are all latency, some 6 us and 1.5 to 2
// a round of the waves: eight waves and no split there (plan_of).
// HC: head size in steps of 32, rounded up; W: waves.
template <class T, int HC, int W>
__global__ __launch_bounds__(64 * W, W > 4 ? 2 : HC <= 4 ? 3 : 1) void k_few(AttnArgs a, LayerView<T> kv, BatchView b, Splits sl, bool vec) {
  using F = Form<T>;
  constexpr int KP = F::KP, P = F::P, D = 2 * HC;
  constexpr bool kF32 = sizeof(T) == 4;
  constexpr int TK = kF32 ? 1 : 2, STEP = 16 * TK, N = 4 * TK;  // score tiles, keys of a step and of a lane
  constexpr float kLift = kF32 ? 0.0f : F::kLift;
  __shared__ float ml[2][W][16];
  __shared__ f4 part[W / 2][D][64];
  __shared__ uint32_t bad_rows;
  const int seq = blockIdx.y, per = a.heads / kv.nkv, hd = kv.hd;
  const int t0 = (blockIdx.x >> 3) % sl.few_tiles * kFewRows;  // the tile's first row
  const int unit = (blockIdx.x >> 3) / sl.few_tiles * 8 + (blockIdx.x & 7), kvh = unit % kv.nkv, split = unit / kv.nkv;
  const SeqSpan sp = seq_span(b, seq);
  const int rows = min(sp.nq * per - t0, kFewRows);
  if (rows <= 0 || !sl.is_few(sp.nq, per)) return;
  const Tile tile = tile_of(sp, t0 / kFewRows, kFewRows, per, a.window);
  const Share each = share_of(tile, sl.few.len);
  const int splits = each.count;
  if (split >= splits) return;
  const int lo = tile.lo + split * each.len, hi = min(tile.hi, lo + each.len);
  const int seen = first_seen(sp.n - sp.nq + t0 / per, a.window);  // no row sees less
  const size_t row0 = sl.few_row(seq, kvh, kv.nkv, t0);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, g = lane >> 4;
  const int *table = b.tables + (size_t)seq * b.stride;
  const int mask = (1 << kv.shift) - 1;
  // The row of this lane's column.
  const int r = t0 + min(col, rows - 1), tok = r / per, head = kvh * per + r % per, pos = sp.n - sp.nq + tok;
  const int first = first_seen(pos, a.window);
  const Score score = score_of(a, head);
  // The rows' queries as operands, the same for every wave, lane after lane.
  constexpr int QP = kF32 ? 2 : P;
  __shared__ u4 ql[HC][QP][64];
  float back = a.scale;
  {
    const float *x = a.q + (size_t)(sp.q0 + tok) * a.q_stride + (size_t)head * hd;
    if constexpr (kF32) {
      for (int c = wave; c < HC; c += W) {
        float v[8];
        query8(x, 32 * c + 8 * g, hd, vec, v);
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) ql[c][j][lane][i] = __float_as_uint(v[4 * j + i]);
      }
    } else {
      float v[HC][8], most = 0.0f;
#pragma unroll
      for (int c = 0; c < HC; ++c) {
        query8(x, 32 * c + 8 * g, hd, vec, v[c]);
#pragma unroll
        for (int i = 0; i < 8; ++i) most = fmaxf(most, fabsf(v[c][i]));
      }
      most = fmaxf(most, __shfl_xor(most, 16));
      most = fmaxf(most, __shfl_xor(most, 32));
      const int up = F::row_exponent(most);
#pragma unroll
      for (int c = 0; c < HC; ++c) {
        if (up)
#pragma unroll
          for (int i = 0; i < 8; ++i) v[c][i] = ldexpf(v[c][i], up);
        u4 q[P];
        F::parts(v[c], q);
        if (c % W == wave)
#pragma unroll
          for (int j = 0; j < P; ++j) ql[c][j][lane] = q[j];
      }
      back = ldexpf(a.scale, -up);
    }
  }
  __syncthreads();
  f4 o[D];
#pragma unroll
  for (int d = 0; d < D; ++d) o[d] = f4{0, 0, 0, 0};
  float m = -INFINITY, l = 0.0f;
  // Lane's key rows of the score tiles: base + N (col / 4) + 4 t + col % 4; its keys
  // in S^T and in V^T: base + N g ...
  auto page_at = [&](int key) { return key < hi ? page_of(table, key, kv.shift, kv.pages) : -1; };
  Raw<T> kr[TK][HC];
  Keys<T> vr[D];
  auto load_keys = [&](int kk, int page) {
#pragma unroll
    for (int t = 0; t < TK; ++t) {
      const int key = kk + 4 * t + (col & 3);
      const bool in = page >= 0 && key < hi && key >= seen;
      const T *p = kv.k + key_at(max(page, 0), kvh, key & mask, kv.nkv, hd, kv.shift) + 8 * g;
#pragma unroll
      for (int c = 0; c < HC; ++c) {
        if (in && 32 * c + 8 * g < hd)
          kr[t][c].load(p + 32 * c);
        else
          kr[t][c].zero();
      }
    }
  };
  auto load_values = [&](int vk, int page) {
    const T *p = kv.v + value_at(max(page, 0), kvh, vk & mask, kv.nkv, hd, kv.shift) + ((size_t)col << kv.shift);
#pragma unroll
    for (int d = 0; d < D; ++d) {
      if (page >= 0 && 16 * d + col < hd)
        vr[d].load(p + ((size_t)(16 * d) << kv.shift));
      else
        vr[d].zero();
    }
  };
  constexpr int ALL = W * STEP;  // a step of every wave
  const int ko = N * (col >> 2), vo = N * g;
  int base = lo + STEP * wave, vpage = page_at(base + vo), knext = page_at(base + ALL + ko), vnext = page_at(base + ALL + vo);
  load_keys(base + ko, page_at(base + ko));
  load_values(base + vo, vpage);
  for (; base < hi; base += ALL) {
    asm volatile("" ::: "memory");  // the queries are read from LDS each time: registers are for what is in flight
    const int vk = base + vo;
    f4 s[TK];
#pragma unroll
    for (int t = 0; t < TK; ++t) s[t] = f4{0, 0, 0, 0};
#pragma unroll
    for (int c = 0; c < HC; ++c) {
      u4 q[QP];
#pragma unroll
      for (int j = 0; j < QP; ++j) q[j] = ql[c][j][lane];
      if constexpr (kF32) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
#pragma unroll
          for (int t = 0; t < TK; ++t)
            s[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kr[t][c].v[e / 4][e % 4]),
                                                        __uint_as_float(q[e / 4][e % 4]), s[t], 0, 0, 0);
      } else {
#pragma unroll
        for (int t = 0; t < TK; ++t) {
          u4 x[KP];
          kr[t][c].parts(x);
          s[t] = products<F>(x, q, s[t], [](u4 x, u4 y, f4 c) { return F::mma16(x, y, c); });
        }
      }
    }
    if (base + ALL < hi) load_keys(base + ALL + ko, knext);  // while this step's softmax and values go on
    float x[N], top = -INFINITY;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const int key = vk + e;
      const bool in = vpage >= 0 && key <= pos && key >= first && key < hi;
      x[e] = in ? score(s[e / 4][e % 4] * back, pos - key) : -INFINITY;
      top = fmaxf(top, x[e]);
    }
    top = fmaxf(top, __shfl_xor(top, 16));
    top = fmaxf(top, __shfl_xor(top, 32));
    const float mn = fmaxf(m, top), ref = (mn == -INFINITY ? 0.0f : mn) - kLift;
    const float alpha = m == mn ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
    m = mn;
    float sum = 0.0f;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      x[e] = __builtin_amdgcn_exp2f(x[e] - ref);
      sum += x[e];
    }
    l = l * alpha + sum;
    if (__any(alpha != 1.0f))
#pragma unroll
      for (int d = 0; d < D; ++d) o[d] *= alpha;
    // Slots that hold no key of these rows: whatever lies there stays out.
    if (base < seen || base + STEP > hi)
#pragma unroll
      for (int d = 0; d < D; ++d) vr[d].keep(seen - vk, hi - vk);
    if constexpr (kF32) {
#pragma unroll
      for (int e = 0; e < N; ++e)
#pragma unroll
        for (int d = 0; d < D; ++d)
          o[d] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(vr[d].v[e / 4][e % 4]), x[e], o[d], 0, 0, 0);
    } else {
      u4 p[P];
      F::parts(x, p);
#pragma unroll
      for (int d = 0; d < D; ++d) {
        u4 y[KP];
        vr[d].parts(y);
        o[d] = products<F>(y, p, o[d], [](u4 x, u4 y, f4 c) { return F::mma16(x, y, c); });
      }
    }
    vpage = vnext;
    if (base + ALL < hi) load_values(base + ALL + vo, vpage);
    knext = page_at(base + 2 * ALL + ko);
    vnext = page_at(base + 2 * ALL + vo);
  }
  // The waves' softmaxes, after the four lane groups' shares of the sum.
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
  if (g == 0) ml[0][wave][col] = m, ml[1][wave][col] = l;
  __syncthreads();
  float top = ml[0][0][col];
#pragma unroll
  for (int w = 1; w < W; ++w) top = fmaxf(top, ml[0][w][col]);
  float sum = 0.0f;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    const float mw = ml[0][w][col];
    sum += ml[1][w][col] * (mw == top ? 1.0f : __builtin_amdgcn_exp2f(mw - top));
  }
  const float mine = m == top ? 1.0f : __builtin_amdgcn_exp2f(m - top);
#pragma unroll
  for (int d = 0; d < D; ++d) o[d] *= mine;
#pragma unroll
  for (int from = W / 2; from; from >>= 1) {
    if (wave >= from && wave < 2 * from)
#pragma unroll
      for (int d = 0; d < D; ++d) part[wave - from][d][lane] = o[d];
    __syncthreads();
    if (wave < from)
#pragma unroll
      for (int d = 0; d < D; ++d) o[d] += part[wave][d][lane];
    __syncthreads();
  }
  if (wave == 0) {
    bool bad = !(fabsf(sum) < INFINITY);
#pragma unroll
    for (int d = 0; d < D; ++d) bad = bad || !finite4(o[d]);
    const uint64_t all = __ballot(bad);
    if (lane == 0) bad_rows = (uint32_t)(all | all >> 16 | all >> 32 | all >> 48) & 0xffffu;
    if (col < rows) {
      const size_t at = sl.few.at(row0 + col, split);
      float *out = a.out + (size_t)(sp.q0 + tok) * a.out_stride + (size_t)head * hd;
      float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
      bool wide = vec;
      if (splits > 1) {
        out = sl.few.o + at * hd;
        if (g == 0) sl.few.ml[at] = make_float2(top - kLift, sum);
        inv = 1.0f;
        wide = true;
      }
#pragma unroll
      for (int d = 0; d < D; ++d) {
        const int e = 16 * d + 4 * g;
        if (e >= hd) continue;
        const f4 y = o[d] * inv;
        if (wide)
          *reinterpret_cast<f4 *>(out + e) = y;
        else
          for (int i = 0; i < 4; ++i) out[e + i] = y[i];
      }
    }
  }
  __syncthreads();
  if (bad_rows == 0) return;
  for (int i = wave; i < rows; i += W)
    if (bad_rows >> i & 1)
      redo_row(a, kv, table, sp.q0 + (t0 + i) / per, kvh * per + (t0 + i) % per, sp.n - sp.nq + (t0 + i) / per, lo, hi,
               sl.few, sl.few.at(row0 + i, split), splits > 1);
}

// ------------------------------------------------------------------- many rows --

// Chunks of a prompt.  Block (row tile x kv head, split, sequence): each of four
// waves has 32 rows, and stages of 32 keys and values pass through LDS for all of
// them, as they are in the pages but dealt operand by operand, lane after lane (so
// that reads are linear).  They get there by DMA, a stage ahead and without a
// register.  Two blocks share a CU, one's softmax beside the other's products.
constexpr int kStage = 32;

template <class T, int HC>
constexpr size_t many_lds() {
  return (size_t)kStage * HC * 32 * 2 * (sizeof(T) == 4 ? 4 + 3 * 2 : 2 * 2);
}

typedef __attribute__((address_space(3))) void lds_void;
typedef const __attribute__((address_space(1))) void global_void;

// Eight cache values of each lane (p: the lane's) to a 64-lane operand in LDS: f32
// in two halves.
template <class T>
__device__ __forceinline__ void dma(const T *p, u4 *to) {
  __builtin_amdgcn_global_load_lds((global_void *)p, (lds_void *)to, 16, 0, 0);
  if constexpr (sizeof(T) == 4) __builtin_amdgcn_global_load_lds((global_void *)(p + 4), (lds_void *)(to + 64), 16, 0, 0);
}

// Key of its 32 that row r of a 32 x 32 operand holds.
__device__ __forceinline__ int row_key(int r) { return (r & 16) + 2 * (r & 4) + ((r & 8) >> 1) + (r & 3); }

template <class T, int HC>
__global__ __launch_bounds__(256, HC <= 4 ? 2 : 1) void k_many(AttnArgs a, LayerView<T> kv, BatchView b, Splits sl, bool vec) {
  using F = Form<T>;
  constexpr int KP = F::KP, P = F::P, S = kStage, KS = 2 * HC;
  constexpr int OP = 64 * sizeof(T) / 2, BUF = KS * OP;  // an operand, and a stage of keys or of values, in 16 bytes
  constexpr bool CUT = KP > 1;
  constexpr int kPair = CUT ? 2 : 4;
  constexpr int BUFS = CUT ? 1 : 2, PART = 64 * KP;  // an operand in parts
  extern __shared__ __align__(16) uint8_t lds[];
  u4 *kl = reinterpret_cast<u4 *>(lds), *vl = kl + BUFS * BUF;
  u4 *kparts = CUT ? vl + BUF : kl, *vparts = CUT ? kparts + KS * PART : vl;
  const int seq = blockIdx.z, split = blockIdx.y, per = a.heads / kv.nkv, hd = kv.hd;
  const SeqSpan sp = seq_span(b, seq);
  const int rows = sp.nq * per, tiles = (rows + kManyRows - 1) / kManyRows;
  // Kv heads side by side (an XCD keeps those of its own in L2), the longest rows first.
  const int kvh = blockIdx.x % kv.nkv, t = tiles - 1 - (int)(blockIdx.x / kv.nkv);
  if (t < 0 || sl.is_few(sp.nq, per)) return;
  const Tile tile = tile_of(sp, t, kManyRows, per, a.window);
  const Share each = share_of(tile, sl.many.len);
  const int splits = each.count;
  if (split >= splits) return;
  const int lo = tile.lo + split * each.len, hi = min(tile.hi, lo + each.len);
  const int base0 = sp.n - sp.nq;
  const int seen = first_seen(base0 + t * kManyRows / per, a.window);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, col = lane & 31, h = lane >> 5;
  const int *table = b.tables + (size_t)seq * b.stride;
  const int mask = (1 << kv.shift) - 1;
  const int r0 = t * kManyRows + 32 * wave, r = min(r0 + col, rows - 1), tok = r / per, head = kvh * per + r % per;
  const int pos = base0 + tok, first = first_seen(pos, a.window);
  // The wave's rows see nothing before wlo, nothing from whi on; all of them see
  // everything between alo and ahi.
  const int tok0 = min(r0, rows - 1) / per, tok1 = min(r0 + 31, rows - 1) / per;
  const bool idle = r0 >= rows;
  const int wlo = first_seen(base0 + tok0, a.window), whi = base0 + tok1 + 1;
  const int alo = first_seen(base0 + tok1, a.window), ahi = base0 + tok0 + 1;
  const Score score = score_of(a, head);
  u4 q[KS][P];
  float back;
  {
    const float *x = a.q + (size_t)(sp.q0 + tok) * a.q_stride + (size_t)head * hd;
    const float sign = a.scale < 0.0f ? -1.0f : 1.0f;  // the scale is positive from here on
    float most = 0.0f;
    int up = 0;
    if (F::kLift != 0.0f) {  // f16
      for (int c = 0; c < KS; ++c) {
        float v[8];
        query8(x, 16 * c + 8 * h, hd, vec, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) most = fmaxf(most, fabsf(v[i]));
      }
      most = fmaxf(most, __shfl_xor(most, 32));
      up = F::row_exponent(most);
    }
#pragma unroll
    for (int c = 0; c < KS; ++c) {
      float v[8];
      query8(x, 16 * c + 8 * h, hd, vec, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = F::kLift != 0.0f ? ldexpf(v[i] * sign, up) : v[i] * sign;
      F::parts(v, q[c]);
    }
    back = ldexpf(fabsf(a.scale), -up);
  }
  // Scores that are only scaled go into the exponential with one multiply-add.
  const bool direct = score.plain && __all(back * kLog2e > 0.0f && back * kLog2e < INFINITY);
  const float mul = direct ? back * kLog2e : 1.0f;
  f16v o[HC];
#pragma unroll
  for (int d = 0; d < HC; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[d][i] = 0.0f;
  float m = -INFINITY, l = 0.0f;

  // What is never loaded (dimensions past the head, keys that are not there) is
  // zero, or a value of an earlier stage.
  for (int i = tid; i < 2 * BUFS * BUF; i += 256) kl[i] = u4{0, 0, 0, 0};
  const int kkey = row_key(col);
  // Pages of the two halves of a stage: even and odd lanes look them up (the entry
  // of the last position past the end), and each is a scalar only where it is used,
  // a stage later: a scalar at once would wait for the DMA in flight.
  auto entries = [&](int kb) { return table[min(kb + 16 * (lane & 1), hi - 1) >> kv.shift]; };
  auto page_of_half = [&](int entry, int kb, int u) {
    const int p = __builtin_amdgcn_readlane(entry, u);
    return kb + 16 * u < hi && (unsigned)p < (unsigned)kv.pages ? p : -1;
  };
  // This wave's operands of a stage: every fourth of the keys' (16 dimensions each)
  // and of the values' (16 keys x 32 dimensions).
  auto load = [&](int kb, const int (&page)[2], int buf) {
    const int key = kb + kkey, kpage = kkey & 16 ? page[1] : page[0];
    if (kpage >= 0 && key < hi && key >= seen) {
      const T *p = kv.k + key_at(kpage, kvh, key & mask, kv.nkv, hd, kv.shift) + 8 * h;
#pragma unroll
      for (int f = 0; f < KS; f += 4)
        if (f + wave < KS && 16 * (f + wave) + 8 * h < hd) dma(p + 16 * (f + wave), kl + buf * BUF + (f + wave) * OP);
    }
#pragma unroll
    for (int f = 0; f < KS; f += 4) {
      const int u = (f + wave) / HC, d = 32 * ((f + wave) % HC) + col, vpage = u ? page[1] : page[0];
      if (f + wave < KS && vpage >= 0 && d < hd)
        dma(kv.v + value_at(vpage, kvh, (kb + 16 * u + 8 * h) & mask, kv.nkv, hd, kv.shift) + ((size_t)d << kv.shift),
            vl + buf * BUF + (f + wave) * OP);
    }
  };
  int next = 0, page[2] = {-1, -1};
  __syncthreads();
  if (lo < hi) {
    next = entries(lo);
    page[0] = page_of_half(next, lo, 0);
    page[1] = page_of_half(next, lo, 1);
    next = entries(lo + S);
    load(lo, page, 0);
  }
  int cur = 0;
  for (int kb = lo; kb < hi; kb += S, cur ^= BUFS - 1) {
    const u4 *kbuf = kparts + cur * BUF;
    u4 *vbuf = vparts + cur * BUF;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    const bool now[2] = {page[0] >= 0, page[1] >= 0}, inside = kb >= seen && kb + S <= hi && now[0] && now[1];
    auto ahead = [&] {
      if (kb + S >= hi) return;
      page[0] = page_of_half(next, kb + S, 0);
      page[1] = page_of_half(next, kb + S, 1);
      next = entries(kb + 2 * S);
      load(kb + S, page, CUT ? 0 : cur ^ 1);
    };
    if (!CUT) ahead();
    if (CUT || !inside) {
      // Slots that hold no key of these rows: whatever lies there becomes zero.
#pragma unroll
      for (int f = wave; f < KS; f += 4) {
        const int u = f / HC, vk = kb + 16 * u + 8 * h;
        Raw<T> r;
        u4 x[KP];
        if constexpr (CUT) {
          r.fetch(kl + f * OP + lane);
          r.parts(x);
#pragma unroll
          for (int j = 0; j < KP; ++j) kparts[f * PART + 64 * j + lane] = x[j];
        }
        r.fetch((CUT ? vl : vbuf) + f * OP + lane);
        if (!inside) r.keep(now[u] ? seen - vk : 8, hi - vk);
        r.parts(x);
#pragma unroll
        for (int j = 0; j < KP; ++j) vbuf[f * PART + 64 * j + lane] = x[j];
      }
      __syncthreads();
    }
    if (CUT) ahead();
    if (idle || kb >= whi || kb + S <= wlo) continue;
    f16v s;
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = 0.0f;
#pragma unroll
    for (int c = 0; c < KS; ++c) {
      u4 x[KP];
#pragma unroll
      for (int j = 0; j < KP; ++j) x[j] = kbuf[c * PART + 64 * j + lane];
      s = products<F>(x, q[c], s, [](u4 x, u4 y, f16v c) { return F::mma32(x, y, c); });
    }
    // Register 8 u + j of a lane is key kb + 16 u + 8 h + j.
    if (!direct) {
      if (score.softcap > 0.0f) {
        const float in = back * score.inv_cap, out = score.softcap * kLog2e;
        float most = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          s[i] *= in;
          most = fmaxf(most, fabsf(s[i]));
        }
        if (__all(most < kTanhNear))
#pragma unroll
          for (int i = 0; i < 16; ++i) s[i] = out * tanh_near(s[i]);
        else
#pragma unroll
          for (int i = 0; i < 16; ++i) s[i] = out * cap_tanh(s[i]);
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] *= back * kLog2e;
      }
      if (a.slopes)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          s[i] = fmaf(-score.slope * kLog2e, (float)(pos - (kb + 16 * (i / 8) + 8 * h + i % 8)), s[i]);
    }
    if (!(inside && kb >= alo && kb + S <= ahi))
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int key = kb + 16 * (i / 8) + 8 * h + i % 8;
        s[i] = (now[i / 8] & (key <= pos) & (key >= first) & (key < hi)) ? s[i] : -INFINITY;
      }
    float top = s[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) top = fmaxf(top, s[i]);
    top = fmaxf(top, __shfl_xor(top, 32));
    const float mn = fmaxf(m, top * mul), ref = (mn == -INFINITY ? 0.0f : mn) - F::kLift;
    const float alpha = m == mn ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
    m = mn;
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], mul, -ref));
      sum += s[i];
    }
    l = l * alpha + sum;
    if (__any(alpha != 1.0f))
#pragma unroll
      for (int d = 0; d < HC; ++d) o[d] *= alpha;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      float y[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = s[8 * u + j];
      u4 p[P];
      F::parts(y, p);
      // Two dimension tiles at a time: their sums do not wait for each other.
#pragma unroll
      for (int d0 = 0; d0 < HC; d0 += kPair) {
        u4 v[kPair][KP];
#pragma unroll
        for (int d = 0; d < kPair; ++d)
          if (d0 + d < HC)
#pragma unroll
            for (int j = 0; j < KP; ++j) v[d][j] = vbuf[(u * HC + d0 + d) * PART + 64 * j + lane];
#pragma unroll
        for (int w = (KP + P - 2 < P - 1 ? KP + P - 2 : P - 1); w >= 0; --w)
#pragma unroll
          for (int i = 0; i < KP; ++i)
#pragma unroll
            for (int d = 0; d < kPair; ++d)
              if (d0 + d < HC && w - i >= 0 && w - i < P) o[d0 + d] = F::mma32(v[d][i], p[w - i], o[d0 + d]);
      }
    }
  }
  l += __shfl_xor(l, 32);
  bool bad = !(fabsf(l) < INFINITY);
#pragma unroll
  for (int d = 0; d < HC; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) bad = bad || !(fabsf(o[d][i]) < INFINITY);
  if (r0 + col < rows) {
    const size_t at = sl.many.at((size_t)(sp.q0 + tok) * a.heads + head, split);
    float *out = a.out + (size_t)(sp.q0 + tok) * a.out_stride + (size_t)head * hd;
    float inv = l == 0.0f ? 0.0f : 1.0f / l;
    bool wide = vec;
    if (splits > 1) {
      out = sl.many.o + at * hd;
      if (h == 0) sl.many.ml[at] = make_float2(m - F::kLift, l);
      inv = 1.0f;
      wide = true;
    }
#pragma unroll
    for (int d = 0; d < HC; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int e = 32 * d + 8 * i + 4 * h;
        if (e >= hd) continue;
        const f4 y = f4{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]} * inv;
        if (wide)
          *reinterpret_cast<f4 *>(out + e) = y;
        else
          for (int j = 0; j < 4; ++j) out[e + j] = y[j];
      }
  }
  const uint64_t all = __ballot(bad);
  for (uint32_t rest = (uint32_t)(all | all >> 32); rest; rest &= rest - 1) {
    const int i = r0 + __builtin_ctz(rest);
    const int row = sp.q0 + i / per, hq = kvh * per + i % per;
    if (i < rows)
      redo_row(a, kv, table, row, hq, base0 + i / per, lo, hi, sl.many, sl.many.at((size_t)row * a.heads + hq, split),
               splits > 1);
  }
}

// ------------------------------------------------------------------------ join --

// Splits of a row joined: 32 lanes x 4 dimensions (twice over for heads past 128)
// by `shares` (1 to 16, a power of two) that take the splits in turn; a block has 16
// / shares rows.  Block (rows, sequence).  Bound by the latency of its loads: a row's
// maxima are read first, a share's parts eight at a time.  32 rows of 65 parts: 8 us;
// 32768 of two: 16.
constexpr int kShares = 16;
__global__ __launch_bounds__(32 * kShares) void k_join(AttnArgs a, BatchView b, Splits sl, int nkv, int hd, int shares,
                                                       bool vec) {
  __shared__ f4 part[kShares][64];
  const SeqSpan sp = seq_span(b, blockIdx.y);
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, share = w & (shares - 1);
  const int unit = blockIdx.x * (kShares / shares) + w / shares, j = unit / a.heads, head = unit % a.heads;
  const int per = a.heads / nkv, kvh = head / per, r = j * per + head % per;
  const bool few = sl.is_few(sp.nq, per), mine = j < sp.nq;
  const int R = few ? kFewRows : kManyRows;
  const Parts &parts = few ? sl.few : sl.many;
  const int splits = mine ? share_of(tile_of(sp, r / R, R, per, a.window), parts.len).count : 0;
  const size_t row = few ? sl.few_row(blockIdx.y, kvh, nkv, r) : (size_t)(sp.q0 + j) * a.heads + head;
  f4 o[2] = {f4{0, 0, 0, 0}, f4{0, 0, 0, 0}};
  if (splits > 1) {
    const float2 *ml = parts.ml + parts.at(row, 0);
    const float *p = parts.o + parts.at(row, 0) * hd + 4 * lane;
    float top = -INFINITY, l = 0.0f;
#pragma unroll 4
    for (int s = lane; s < splits; s += 32) top = fmaxf(top, ml[s].x);
#pragma unroll
    for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
    auto weight = [&](float2 x) { return x.x == top ? 1.0f : __builtin_amdgcn_exp2f(x.x - top); };
#pragma unroll 4
    for (int s = lane; s < splits; s += 32) l += weight(ml[s]) * ml[s].y;
#pragma unroll
    for (int d = 16; d; d >>= 1) l += __shfl_xor(l, d);
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll 8
    for (int s = share; s < splits; s += shares) {
      const float w = weight(ml[s]) * inv;
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (4 * lane + 128 * i < hd) o[i] += *reinterpret_cast<const f4 *>(p + (size_t)s * hd + 128 * i) * w;
    }
  }
  if (shares > 1) {
    part[w][lane] = o[0];
    part[w][lane + 32] = o[1];
    __syncthreads();
    if (share) return;
#pragma unroll 4
    for (int s = 1; s < shares; ++s) {
      o[0] += part[w + s][lane];
      o[1] += part[w + s][lane + 32];
    }
  }
  if (splits < 2) return;
  float *out = a.out + (size_t)(sp.q0 + j) * a.out_stride + (size_t)head * hd;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int e = 4 * lane + 128 * i;
    if (e >= hd) continue;
    if (vec)
      *reinterpret_cast<f4 *>(out + e) = o[i];
    else
      for (int k = 0; k < 4; ++k) out[e + k] = o[i][k];
  }
}

// --------------------------------------------------------------------- launch --

constexpr int kFewMax = 64;   // rows a kv head: four tiles read the keys as often from L2, a block of k_many
                              // has half of its 128 rows idle (9 tokens x 4 heads at 2200 positions, eight
                              // sequences: f32 90 us there)
// Blocks of k_few: pieces that even out sequences of different lengths, or, of one
// sequence, about as many as the chip holds at once (one token at 32768 positions: 40
// us with 65 parts a row, 44 with 129, 46 with 43).
constexpr size_t kFewBlocks = 2048, kFewBlocksOne = 640;
constexpr size_t kManySlots = 512;  // two blocks a CU

// What a tile can read at most: its rows' windows, from a multiple of 64 on.
int most_keys(const BatchView &b, int window) {
  const long long span = window > 0 ? (long long)window + b.max_q + 63 : b.max_kv;
  return (int)std::max(1LL, std::min<long long>(b.max_kv, span));
}

int whole128(size_t n) { return (int)((n + 127) / 128 * 128); }

// k_many's splits, for sequences at their bounds: the number that lets the chip end
// soonest.  Tiles near the start of a prompt read few keys, so that blocks of equal
// rows are not blocks of equal length: while all fit the chip at once the longest
// counts, beyond that their sum and half of the longest.  In positions of a block
// (0.07 to 0.09 us each): the join costs about 100, its launch, and 90 a split for
// 32768 rows x heads of 128, the parts written and read (1024 rows x 32 heads: 8 us
// a split).  Up to 8 tiles stand for all; `fit`: parts that the scratch holds.
int many_split(size_t units, size_t tiles, int keys, int max_q, size_t row_bytes, size_t fit) {
  const int samples = (int)std::min<size_t>(tiles, 8);
  int best_len = std::max(128, whole128(keys));
  double best = 0.0;
  for (int n = 1; n <= (int)std::min<size_t>(fit, 16); ++n) {
    const int len = whole128(((size_t)keys + n - 1) / n);
    double blocks = 0.0, sum = 0.0, longest = 0.0;
    for (int i = 0; i < samples; ++i) {
      const double span = std::max(1.0, keys - (double)max_q * (samples - 1 - i) / samples);
      const double parts = std::ceil(span / len);
      blocks += parts;
      sum += span;
      longest = std::max(longest, span / parts);
    }
    const double scale = (double)units * tiles / samples;
    const double join = len < keys ? 100.0 + 90.0 * n * (double)row_bytes / (32768.0 * 128 * 4) : 0.0;
    const double cost =
        join + (blocks * scale <= kManySlots ? longest : std::max(longest, sum * scale / kManySlots + 0.5 * longest));
    if (n == 1 || cost < best) best = cost, best_len = len;
  }
  return best_len;
}

struct Plan {
  int few_len, many_len, few, many;  // split lengths and counts
  int few_max, few_tiles, few_waves;
  size_t few_rows, many_rows, many_tiles;
  size_t few_parts() const { return few > 1 ? few * few_rows : 0; }
  size_t many_parts() const { return many > 1 ? many * many_rows : 0; }
};

Plan plan_of(int nkv, int heads, int hd, int size, const BatchView &b, int window, size_t work_bytes) {
  Plan p;
  const int per = heads / nkv, keys = most_keys(b, window);
  const size_t rows = (size_t)b.max_q * per, units = (size_t)b.seqs * nkv;
  size_t left = work_bytes / (4 * (size_t)hd + 8);  // parts that fit
  auto count = [&](int &len, size_t part_rows) {
    int n = (keys + len - 1) / len;
    const size_t fit = std::max<size_t>(1, left / part_rows);
    if ((size_t)n > fit) {
      len = whole128(((size_t)keys + fit - 1) / fit);
      n = (keys + len - 1) / len;
    }
    if (n > 1) left -= n * part_rows;
    return n;
  };
  // One sequence with a chunk: no launch for what is not there (should it have few
  // rows all the same, k_many takes them).
  p.few_max = b.seqs == 1 && rows > kFewMax ? 0 : kFewMax;
  p.few_tiles = p.few_max ? (int)((std::min<size_t>(rows, kFewMax) + kFewRows - 1) / kFewRows) : 0;
  p.few_rows = units * p.few_tiles * kFewRows;
  p.many_rows = (size_t)b.tokens * heads;
  p.many_tiles = rows > (size_t)p.few_max ? (rows + kManyRows - 1) / kManyRows : 0;
  p.few = p.many = 1;
  p.few_len = p.many_len = std::max(256, whole128(keys));
  // Few heads, short contexts: eight waves a block and no split while the join costs
  // more than the one CU's time for the keys and values of a head, up to some 330 KB
  // (one token, 32 heads, 8 waves against splits: 8 heads of 128 in f32, 300 positions
  // 15 and 20 us, 500 21 and 20; 4 of 64 in bf16, 500 positions 9 and 13, 1000 13 and 14).
  p.few_waves = hd <= 128 && units * p.few_tiles <= 256 && (size_t)keys * hd * size * 2 <= 330000 ? 8 : 4;
  if (p.few_tiles && p.few_waves == 4) {
    const size_t want = std::max<size_t>(1, (b.seqs == 1 ? kFewBlocksOne : kFewBlocks) / (units * p.few_tiles));
    p.few_len = std::max(256, whole128(((size_t)keys + want - 1) / want));
    p.few = count(p.few_len, p.few_rows);
  }
  if (p.many_tiles) {
    p.many_len = many_split(units, p.many_tiles, keys, b.max_q, p.many_rows * hd * 4, left / p.many_rows);
    p.many = count(p.many_len, p.many_rows);
  }
  return p;
}

template <class T, int HC>
void launch_of(const AttnArgs &a, const LayerView<T> &kv, const BatchView &b, const Plan &p, const Splits &sl, bool vec,
               hipStream_t s) {
  if (p.many_tiles) {
    constexpr size_t lds = many_lds<T, HC>();
    dynamic_lds<k_many<T, HC>>(lds);
    k_many<T, HC><<<dim3((unsigned)(p.many_tiles * kv.nkv), p.many, b.seqs), 256, lds, s>>>(a, kv, b, sl, vec);
  }
  if (p.few_tiles) {
    const unsigned units = ((unsigned)p.few * kv.nkv + 7) / 8 * 8;
    const dim3 grid(units * p.few_tiles, b.seqs);
    if (HC <= 4 && p.few_waves == 8)
      k_few<T, HC <= 4 ? HC : 4, 8><<<grid, 512, 0, s>>>(a, kv, b, sl, vec);
    else
      k_few<T, HC, 4><<<grid, 256, 0, s>>>(a, kv, b, sl, vec);
  }
}

}  // namespace

size_t paged_attention_work(int nkv, int heads, int hd, int size, const BatchView &b, int window) {
  const Plan p = plan_of(nkv, heads, hd, size, b, window, SIZE_MAX);
  return (p.few_parts() + p.many_parts()) * (4 * (size_t)hd + 8);
}

template <class T>
void launch_paged_attention(const AttnArgs &a, const LayerView<T> &kv, const BatchView &b, void *work,
                            size_t work_bytes, hipStream_t s) {
  const Plan p = plan_of(kv.nkv, a.heads, kv.hd, (int)sizeof(T), b, a.window, work_bytes);
  Splits sl;
  sl.few_max = p.few_max;
  sl.few_tiles = p.few_tiles;
  sl.few = Parts{p.few_len, p.few, static_cast<float *>(work), nullptr};
  sl.many = Parts{p.many_len, p.many, sl.few.o + p.few_parts() * kv.hd, nullptr};
  sl.few.ml = reinterpret_cast<float2 *>(sl.many.o + p.many_parts() * kv.hd);
  sl.many.ml = sl.few.ml + p.few_parts();
  const bool vec = ((uintptr_t)a.q | (uintptr_t)a.out) % 16 == 0 && a.q_stride % 4 == 0 && a.out_stride % 4 == 0;
  switch ((kv.hd + 31) / 32) {
    case 1: launch_of<T, 1>(a, kv, b, p, sl, vec, s); break;
    case 2: launch_of<T, 2>(a, kv, b, p, sl, vec, s); break;
    case 3: launch_of<T, 3>(a, kv, b, p, sl, vec, s); break;
    case 4: launch_of<T, 4>(a, kv, b, p, sl, vec, s); break;
    default: launch_of<T, 8>(a, kv, b, p, sl, vec, s); break;
  }
  if (p.few > 1 || p.many > 1) {
    // Rows that can be split, and shares by what most of them have.
    const int most = p.many > 1 ? p.many : p.few, per = a.heads / kv.nkv;
    const int rows = p.many > 1 ? b.max_q : std::min(b.max_q, std::max(kFewMax / per, 1));
    int shares = 1;
    while (shares < kShares && 4 * shares < most) shares *= 2;
    const int block = kShares / shares;
    k_join<<<dim3((unsigned)((rows * a.heads + block - 1) / block), b.seqs), 32 * kShares, 0, s>>>(a, b, sl, kv.nkv, kv.hd,
                                                                                                   shares, vec);
  }
}

template void launch_paged_attention<float>(const AttnArgs &, const LayerView<float> &, const BatchView &, void *, size_t,
                                            hipStream_t);
template void launch_paged_attention<_Float16>(const AttnArgs &, const LayerView<_Float16> &, const BatchView &, void *,
                                               size_t, hipStream_t);
template void launch_paged_attention<Bf16>(const AttnArgs &, const LayerView<Bf16> &, const BatchView &, void *, size_t,
                                           hipStream_t);

}  // namespace rai
