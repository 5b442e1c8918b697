// The paged KV cache: what fills it (rotary positions and the store), what forks
// and moves its pages, and the checks of its entry points.  The attention over it
// is in paged_attn.hip.
#include "paged.h"

#include <algorithm>
#include <cmath>
#include <cstring>

namespace rai {

namespace {

constexpr int kMaxHd = 256;  // the angles of 32 positions: 32 KB of LDS at most

// ------------------------------------------------------------------- store --

struct RopeView {
  const double *inv;
  int rot;
  bool inter;
  float gain;
};

struct StoreArgs {
  float *q_out;
  const float *q, *k, *v;
  size_t qo_ld, q_ld, k_ld, v_ld;
  int heads;
  RopeView rope;
};

// cos and sin of pos * inv, both times gain.  The angle and its reduction to a
// quarter turn and f, -1/2..1/2 of one, in f64 (an f32 angle of a far position is
// off by more than the rotation may be); sin and cos of f quarter turns as
// polynomials in f^2 with the smallest relative error (with coefficients rounded to f32
// 3.4e-8 and 8e-9, a half step of f32 being 6e-8; evaluated in f32 1.3e-7 and 8e-8).
__device__ __forceinline__ void rope_angle(int pos, double inv, float gain, float &c, float &s) {
  const double a = (double)pos * (inv * 0.63661977236758138);
  const double n = rint(a);
  const float f = (float)(a - n), z = f * f;
  const int k = (int)(n - 4.0 * floor(n * 0.25));
  const float sf = f * fmaf(fmaf(fmaf(-0.00460165786f, z, 0.079680033f), z, -0.64596349f), z, 1.57079637f);
  const float cf = fmaf(fmaf(fmaf(fmaf(0.00090336299f, z, -0.0208599363f), z, 0.253669173f), z, -1.23370051f), z, 1.0f);
  c = gain * (k & 1 ? sf : cf) * ((k + 1) & 2 ? -1.0f : 1.0f);
  s = gain * (k & 1 ? cf : sf) * (k & 2 ? -1.0f : 1.0f);
}

// The pair (e0, e1) of rotated pair i.
__device__ __forceinline__ void pair_of(const RopeView &r, int i, int &e0, int &e1) {
  e0 = r.inter ? 2 * i : i;
  e1 = r.inter ? 2 * i + 1 : i + r.rot / 2;
}

constexpr int kTokens = 32;   // positions of a block, from a multiple of it on
constexpr int kValueDims = 64;  // value elements of a block

// Four elements as they go to the cache.
template <class T>
__device__ __forceinline__ void put4(T *o, const float (&x)[4]) {
  T y[4] = {from_f32<T>(x[0]), from_f32<T>(x[1]), from_f32<T>(x[2]), from_f32<T>(x[3])};
  if constexpr (sizeof(T) == 4)
    *reinterpret_cast<uint4 *>(o) = __builtin_bit_cast(uint4, y);
  else
    *reinterpret_cast<uint2 *>(o) = __builtin_bit_cast(uint2, y);
}

__device__ __forceinline__ void get4(const float *p, float (&x)[4]) {
  const float4 v = *reinterpret_cast<const float4 *>(p);
  x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
}

// Block (32 positions, part, sequence).  Parts below qk rotate a few heads of the
// queries and keys, the angles of their positions computed once; the others take 64
// elements of the values' rows: a thread has one element of eight positions, which
// lie side by side in the page.  Bound by memory: 4 or 8 elements at a time (VEC: rows
// 16-byte aligned, pairs in whole fours), each line of the pages written by one block.
// 2241 rows of 32 + 8 + 8 heads of 128, bf16: 31 us, 3.3 TB/s.
template <class T, bool VEC>
__global__ __launch_bounds__(256) void k_store(StoreArgs a, LayerView<T> kv, BatchView b, int qk, int heads, Div by_units, Div by_half) {
  extern __shared__ __align__(16) float angles[];  // cosines [position][pair], sines behind them
  __shared__ int pages[kTokens];
  const SeqSpan sp = seq_span(b, blockIdx.z);
  const int base = sp.n - sp.nq, p0 = ((base >> 5) + (int)blockIdx.x) * kTokens, tid = threadIdx.x, hd = kv.hd;
  const int j0 = max(p0 - base, 0), j1 = min(sp.nq, p0 + kTokens - base);
  if (j0 >= j1) return;
  const int *table = b.tables + (size_t)blockIdx.z * b.stride;
  const int mask = (1 << kv.shift) - 1, part = blockIdx.y;
  if (part >= qk) {
    const int e = (part - qk) * kValueDims + (tid & 63), p = p0 + 8 * (tid >> 6);
    if (e >= kv.nkv * hd || p + 8 <= base + j0 || p >= base + j1 || p + 7 < 0) return;
    // Eight positions from a multiple of eight on share a page.
    const int page = page_of(table, max(p, 0), kv.shift, kv.pages);
    if (page < 0) return;
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int j = p + i - base;
      x[i] = j >= j0 && j < j1 ? a.v[(size_t)(sp.q0 + j) * a.v_ld + e] : 0.0f;
    }
    T *o = kv.v + value_at(page, e / hd, p & mask, kv.nkv, hd, kv.shift) + ((size_t)(e % hd) << kv.shift);
    if (p >= base + j0 && p + 8 <= base + j1 && p >= 0) {
      put4(o, {x[0], x[1], x[2], x[3]});
      put4(o + 4, {x[4], x[5], x[6], x[7]});
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (p + i >= max(base + j0, 0) && p + i < base + j1) o[i] = from_f32<T>(x[i]);
    }
    return;
  }
  const int half = a.rope.rot / 2, rows = j1 - j0;
  float *const cs = angles, *const sn = angles + kTokens * half;
  for (int i = tid; i < rows * half; i += 256) {
    const int t = by_half(i), f = i - t * half;
    rope_angle(base + j0 + t, a.rope.inv[f], a.rope.gain, cs[t * half + f], sn[t * half + f]);
  }
  for (int t = tid; t < rows; t += 256)
    pages[t] = base + j0 + t >= 0 ? page_of(table, base + j0 + t, kv.shift, kv.pages) : -1;
  __syncthreads();
  // Units of a row of a head: fours of pairs, then fours of other elements; or, one
  // by one, pairs, then elements.  Four units a thread are read before they are
  // written (the output may be the input: a unit writes what it alone reads).
  const int h0 = part * heads, h1 = min(h0 + heads, a.heads + kv.nkv), units = by_units.d;
  const int pairs = VEC ? (a.rope.inter ? a.rope.rot / 4 : a.rope.rot / 8) : half;
  const int bits = 32 - __clz(rows - 1), total = ((h1 - h0) << bits) * units;  // clz(0) is 32
  constexpr int N = VEC ? 4 : 1, B = 4;
  for (int i0 = tid; i0 < total; i0 += 256 * B) {
    float y[B][N], z[B][N];
    int unit[B], tok[B], head[B];
#pragma unroll
    for (int k = 0; k < B; ++k) {
      const int i = i0 + 256 * k, r = by_units(i), u = i - r * units, t = r & ((1 << bits) - 1), h = h0 + (r >> bits);
      const bool key = h >= a.heads, in = i < total && t < rows && (!key || pages[t] >= 0);
      unit[k] = in ? u : -1;
      tok[k] = t;
      head[k] = h;
      if (!in) continue;
      const size_t row = sp.q0 + j0 + t;
      const float *x = key ? a.k + row * a.k_ld + (size_t)(h - a.heads) * hd : a.q + row * a.q_ld + (size_t)h * hd;
      int e0 = u, e1 = half + u;
      if (VEC && u >= pairs)
        e0 = a.rope.rot + 4 * (u - pairs);
      else if (VEC)
        e0 = 4 * u, e1 = half + 4 * u;
      else if (u >= pairs)
        e0 = a.rope.rot + u - pairs;
      else if (a.rope.inter)
        e0 = 2 * u, e1 = 2 * u + 1;
      if constexpr (VEC) {
        get4(x + e0, y[k]);
        if (u < pairs && !a.rope.inter) get4(x + e1, z[k]);
      } else {
        y[k][0] = x[e0];
        if (u < pairs) z[k][0] = x[e1];
      }
    }
#pragma unroll
    for (int k = 0; k < B; ++k) {
      const int u = unit[k], t = tok[k], h = head[k];
      if (u < 0) continue;
      const bool key = h >= a.heads;
      const size_t row = sp.q0 + j0 + t;
      float *qo = a.q_out + row * a.qo_ld + (size_t)h * hd;
      T *ko = kv.k + key_at(max(pages[t], 0), key ? h - a.heads : 0, (base + j0 + t) & mask, kv.nkv, hd, kv.shift);
      if constexpr (VEC) {
        auto out = [&](int e, const float (&v)[4]) {
          if (key)
            put4(ko + e, v);
          else
            *reinterpret_cast<float4 *>(qo + e) = make_float4(v[0], v[1], v[2], v[3]);
        };
        const float(&p)[4] = y[k], (&q)[4] = z[k];
        if (u >= pairs) {
          out(a.rope.rot + 4 * (u - pairs), p);
        } else if (a.rope.inter) {
          const float c0 = cs[t * half + 2 * u], s0 = sn[t * half + 2 * u], c1 = cs[t * half + 2 * u + 1], s1 = sn[t * half + 2 * u + 1];
          out(4 * u, {p[0] * c0 - p[1] * s0, p[1] * c0 + p[0] * s0, p[2] * c1 - p[3] * s1, p[3] * c1 + p[2] * s1});
        } else {
          float c[4], s[4];
          get4(&cs[t * half + 4 * u], c);
          get4(&sn[t * half + 4 * u], s);
          out(4 * u, {p[0] * c[0] - q[0] * s[0], p[1] * c[1] - q[1] * s[1], p[2] * c[2] - q[2] * s[2], p[3] * c[3] - q[3] * s[3]});
          out(half + 4 * u,
              {q[0] * c[0] + p[0] * s[0], q[1] * c[1] + p[1] * s[1], q[2] * c[2] + p[2] * s[2], q[3] * c[3] + p[3] * s[3]});
        }
      } else {
        auto out = [&](int e, float v) {
          if (key)
            ko[e] = from_f32<T>(v);
          else
            qo[e] = v;
        };
        if (u < pairs) {
          int e0, e1;
          pair_of(a.rope, u, e0, e1);
          out(e0, y[k][0] * cs[t * half + u] - z[k][0] * sn[t * half + u]);
          out(e1, z[k][0] * cs[t * half + u] + y[k][0] * sn[t * half + u]);
        } else {
          out(a.rope.rot + u - pairs, y[k][0]);
        }
      }
    }
  }
}

template <class T>
void launch_store(const StoreArgs &a, const LayerView<T> &kv, const BatchView &b, hipStream_t s) {
  const int rot = a.rope.rot, hd = kv.hd;
  const uintptr_t all = (uintptr_t)a.q | (uintptr_t)a.q_out | (uintptr_t)a.k;
  const bool vec = all % 16 == 0 && (a.q_ld | a.qo_ld | a.k_ld) % 4 == 0 && rot % (a.rope.inter ? 4 : 8) == 0;
  const int pairs = vec ? rot / (a.rope.inter ? 4 : 8) : rot / 2, units = pairs + (vec ? (hd - rot) / 4 : hd - rot);
  // Two heads a block: all blocks of a large batch are then on the chip at once, and
  // each has few loads to wait for (2241 rows of 32 + 8 heads: 31 us, with five 38).
  const int tiles = (b.max_q + kTokens - 2) / kTokens + 1, all_heads = a.heads + kv.nkv;
  const int heads = (size_t)tiles * b.seqs * all_heads < 1024 ? 1 : 2;
  const int qk = (all_heads + heads - 1) / heads, parts = qk + (kv.nkv * hd + kValueDims - 1) / kValueDims;
  const dim3 grid(tiles, parts, b.seqs);
  const size_t lds = (size_t)kTokens * rot * sizeof(float);
  if (vec)
    k_store<T, true><<<grid, 256, lds, s>>>(a, kv, b, qk, heads, Div(units), Div(std::max(rot / 2, 1)));
  else
    k_store<T, false><<<grid, 256, lds, s>>>(a, kv, b, qk, heads, Div(units), Div(std::max(rot / 2, 1)));
}

// ----------------------------------------------------------- forks and moves --

// The pool as bytes: a page of one layer's keys (or values) is `bytes` long, a
// multiple of 16.
struct PoolBytes {
  uint4 *k, *v;
  size_t layer_vecs, page_vecs;
  int layers, pages;
};

// Keys and values of a page are copied by `parts` blocks, 32 KB of each at most: some
// hundred blocks even for a few forked pages.  Bound by memory: 300 pages of 22 layers
// 91 us, 4.8 TB/s of reads and writes.
constexpr size_t kCopyVecs = 2048;

__device__ __forceinline__ void copy_page(const PoolBytes &p, int layer, int src, int dst, int part) {
  const size_t base = (size_t)layer * p.layer_vecs, from = part * kCopyVecs;
  const size_t to = min(p.page_vecs, from + kCopyVecs);
  const uint4 *ks = p.k + base + (size_t)src * p.page_vecs, *vs = p.v + base + (size_t)src * p.page_vecs;
  uint4 *kd = p.k + base + (size_t)dst * p.page_vecs, *vd = p.v + base + (size_t)dst * p.page_vecs;
#pragma unroll 4
  for (size_t i = from + threadIdx.x; i < to; i += 256) {
    const uint4 x = ks[i], y = vs[i];
    kd[i] = x;
    vd[i] = y;
  }
}

// Block (layer x part, child): the first one's blocks write the table row too.
__global__ __launch_bounds__(256) void k_fork(PoolBytes p, const int *tables, size_t stride, const int *lengths,
                                              int seqs, const int *parent, const int *fresh, int parts, int *tables_out,
                                              int *lengths_out, int *used, int shift) {
  const int i = blockIdx.y, par = parent[i], tid = threadIdx.x;
  const bool ok = (unsigned)par < (unsigned)seqs;
  const size_t most = stride << shift;
  int len = ok ? max(lengths[par], 0) : 0, f = fresh[i];
  if ((size_t)len > most) len = (int)most;
  int again = 0;
  for (int j = tid; j < i; j += 256) again |= parent[j] == par;
  again = __syncthreads_or(again);
  const bool part = (len & ((1 << shift) - 1)) != 0;
  const int last = len >> shift;  // the part-filled page's place
  // A last page that is not there has nothing to copy: the fresh page, which holds what
  // another sequence left in it, stays free, and the children name what the parent names.
  const int src = ok && part && again ? tables[(size_t)par * stride + last] : -1;
  const bool take = (unsigned)src < (unsigned)p.pages;
  if (!take || (unsigned)f >= (unsigned)p.pages) f = -1;
  if (blockIdx.x == 0) {
    for (size_t c = tid; c < stride; c += 256) {
      int id = ok ? tables[(size_t)par * stride + c] : -1;
      if (take && c == (size_t)last) id = f;
      tables_out[(size_t)i * stride + c] = id;
    }
    if (tid == 0) {
      lengths_out[i] = len;
      used[i] = take && f >= 0;
    }
  }
  if (f < 0) return;
  copy_page(p, blockIdx.x / parts, src, f, blockIdx.x % parts);
}

constexpr int kRename = 2048;  // pairs looked through in one go

// Blocks 0 .. renames - 1: table entries, one a thread; the others: (pair, layer x part).
__global__ __launch_bounds__(256) void k_move(PoolBytes p, const int *src, const int *dst, int n, int parts, int *tables,
                                              size_t entries, int renames) {
  __shared__ __align__(16) int from[kRename];
  const int tid = threadIdx.x;
  if ((int)blockIdx.x >= renames) {
    const int copies = p.layers * parts, i = (blockIdx.x - renames) / copies, c = (blockIdx.x - renames) % copies;
    const int a = src[i], b = dst[i];
    if ((unsigned)a < (unsigned)p.pages && (unsigned)b < (unsigned)p.pages) copy_page(p, c / parts, a, b, c % parts);
    return;
  }
  for (size_t e0 = (size_t)blockIdx.x * 256; e0 < entries; e0 += (size_t)renames * 256) {
    const size_t e = e0 + tid;
    const int id = e < entries ? tables[e] : -1;
    int at = -1;
    for (int i0 = 0; i0 < n; i0 += kRename) {
      const int m = min(kRename, n - i0), m4 = (m + 3) & ~3;
      __syncthreads();
      for (int i = tid; i < m4; i += 256) from[i] = i < m ? src[i0 + i] : -1;
      __syncthreads();
#pragma unroll 4
      for (int i = 0; i < m4; i += 4) {
        const int4 f = *reinterpret_cast<const int4 *>(from + i);
        at = f.x == id ? i0 + i : f.y == id ? i0 + i + 1 : f.z == id ? i0 + i + 2 : f.w == id ? i0 + i + 3 : at;
      }
    }
    if ((unsigned)id >= (unsigned)p.pages || at < 0) continue;
    const int to = dst[at];
    if ((unsigned)to < (unsigned)p.pages) tables[e] = to;
  }
}

// ------------------------------------------------------------------ checks --

size_t type_bytes(int type) { return type == RAI_CACHE_F32 ? 4 : 2; }

int page_shift(size_t page_size) {
  int s = 0;
  while ((size_t(1) << s) < page_size) ++s;
  return s;
}

void check_pages(const rai_pages *p) {
  if (!p || !p->k || !p->v) fail(RAI_E_ARG, "null argument");
  if (p->type != RAI_CACHE_F32 && p->type != RAI_CACHE_F16 && p->type != RAI_CACHE_BF16)
    fail(RAI_E_ARG, "unknown cache type");
  if (p->page_size < 16 || p->page_size > 1024 || (p->page_size & (p->page_size - 1)))
    fail(RAI_E_SHAPE, "page_size must be a power of two from 16 to 1024");
  if (p->head_dim == 0 || p->head_dim % 8 || p->head_dim > kMaxHd)
    fail(RAI_E_SHAPE, "head_dim must be a multiple of 8 up to 256");
  if (p->layers == 0 || p->pages == 0 || p->kv_heads == 0) fail(RAI_E_SHAPE, "the pool must not be empty");
  if (p->layers > 65535 || p->pages > INT32_MAX || p->kv_heads > 4096) fail(RAI_E_SHAPE, "dimensions overflow");
  if ((uintptr_t)p->k % 16 || (uintptr_t)p->v % 16) fail(RAI_E_ARG, "the pages must be 16-byte aligned");
}

// Null only where there is nothing to do (no sequences or no rows).
bool check_batch(const rai_page_batch *b, const rai_pages *p, BatchView *v) {
  if (!b) fail(RAI_E_ARG, "null argument");
  if (b->seqs == 0 || b->tokens == 0 || b->max_q == 0) return false;
  if (!b->tables || !b->q_start || !b->kv_len) fail(RAI_E_ARG, "null argument");
  if (b->table_stride == 0) fail(RAI_E_SHAPE, "table_stride must be non-zero");
  if (b->seqs > 65535) fail(RAI_E_SHAPE, "at most 65535 sequences");
  if (b->tokens > INT32_MAX / 2 || b->table_stride > INT32_MAX || b->max_kv > INT32_MAX / 2)
    fail(RAI_E_SHAPE, "dimensions overflow");
  if (b->tokens >= size_t(1) << 24) fail(RAI_E_SHAPE, "at most 2^24 - 1 rows in one call");
  const size_t most = std::min<size_t>(b->max_kv, b->table_stride * p->page_size);
  *v = BatchView{b->tables, b->table_stride, b->q_start, b->kv_len, (int)b->seqs, (int)b->tokens,
                 (int)std::min(b->max_q, b->tokens), (int)most};
  return true;
}

void check_rows(const void *p, size_t stride, size_t heads, size_t hd, const char *what) {
  if (!p) fail(RAI_E_ARG, "null argument");
  if (stride < heads * hd) fail(RAI_E_SHAPE, std::string(what) + " rows overlap: the stride is shorter than a row");
}

template <class T>
LayerView<T> layer_view(const rai_pages *p, size_t layer) {
  const size_t n = layer * p->pages * p->kv_heads * p->page_size * p->head_dim;
  return {static_cast<T *>(p->k) + n, static_cast<T *>(p->v) + n, (int)p->pages, page_shift(p->page_size),
          (int)p->kv_heads, (int)p->head_dim};
}

PoolBytes pool_bytes(const rai_pages *p) {
  const size_t page = p->kv_heads * p->page_size * p->head_dim * type_bytes(p->type) / 16;
  return {static_cast<uint4 *>(p->k), static_cast<uint4 *>(p->v), p->pages * page, page, (int)p->layers, (int)p->pages};
}

// f(LayerView of the pool's type).
template <class F>
void with_layer(const rai_pages *p, size_t layer, F f) {
  if (p->type == RAI_CACHE_F32)
    f(layer_view<float>(p, layer));
  else if (p->type == RAI_CACHE_F16)
    f(layer_view<_Float16>(p, layer));
  else
    f(layer_view<Bf16>(p, layer));
}

void check_heads(size_t heads, const rai_pages *p) {
  if (heads == 0 || heads % p->kv_heads || heads > 16384)
    fail(RAI_E_SHAPE, "heads must be a positive multiple of kv_heads");
}

// Rows of a batch, head by head: the launches' bound.
void check_rows_heads(const BatchView &b, size_t heads) {
  if ((size_t)b.tokens * heads >= size_t(1) << 24) fail(RAI_E_SHAPE, "at most 2^24 - 1 rows x heads in one call");
}

void check_options(const rai_attention_options *o) {
  if (!o) fail(RAI_E_ARG, "null argument");
  if (!std::isfinite(o->scale)) fail(RAI_E_ARG, "scale must be finite");
  if (!(o->softcap == 0.0f || (o->softcap >= 1e-30f && o->softcap <= 1e30f)))
    fail(RAI_E_ARG, "softcap must be 0 or from 1e-30 to 1e30");
}

int window_of(const rai_attention_options *o) { return (int)std::min<size_t>(o->window, INT32_MAX / 2); }

}  // namespace

}  // namespace rai

extern "C" {

int rai_rope_frequencies(int scaling, double theta, size_t rot, double factor, double trained, double low, double high,
                         double *inv, float *gain) {
  RAI_API_BODY({
    if (!inv || !gain) rai::fail(RAI_E_ARG, "null argument");
    if (rot == 0 || rot % 2) rai::fail(RAI_E_SHAPE, "rot_dim must be positive and even");
    if (!std::isfinite(theta) || theta <= 0.0) rai::fail(RAI_E_ARG, "theta must be finite and positive");
    if (scaling < RAI_ROPE_NONE || scaling > RAI_ROPE_YARN) rai::fail(RAI_E_ARG, "unknown rope scaling");
    if (scaling != RAI_ROPE_NONE && !(std::isfinite(factor) && factor >= 1.0))
      rai::fail(RAI_E_ARG, "factor must be finite and at least 1");
    if (scaling >= RAI_ROPE_LLAMA3 && !(std::isfinite(trained) && trained > 0.0))
      rai::fail(RAI_E_ARG, "trained_context must be finite and positive");
    if (scaling == RAI_ROPE_LLAMA3 && !(std::isfinite(high) && low > 0.0 && low < high))
      rai::fail(RAI_E_ARG, "0 < low_freq < high_freq must hold");
    if (scaling == RAI_ROPE_YARN && theta == 1.0) rai::fail(RAI_E_ARG, "theta 1 has no wavelengths to blend by");
    const double two_pi = 6.283185307179586;
    double lo = 0.0, hi = 1.0;  // YaRN: the pairs (as indexes) that turn 32 times and once in the trained context
    if (scaling == RAI_ROPE_YARN) {
      const auto pair_turning = [&](double n) { return rot * std::log(trained / (n * two_pi)) / (2.0 * std::log(theta)); };
      lo = std::max(std::floor(pair_turning(32.0)), 0.0);
      hi = std::min(std::ceil(pair_turning(1.0)), (double)rot - 1.0);
    }
    for (size_t i = 0; i < rot / 2; ++i) {
      const double f = std::pow(theta, -2.0 * (double)i / (double)rot);
      double keep = 1.0;  // share of the unscaled frequency
      if (scaling == RAI_ROPE_LINEAR) keep = 0.0;
      if (scaling == RAI_ROPE_LLAMA3) keep = (trained * f / two_pi - low) / (high - low);
      if (scaling == RAI_ROPE_YARN) keep = 1.0 - ((double)i - lo) / std::max(hi - lo, 0.001);
      keep = std::min(std::max(keep, 0.0), 1.0);
      inv[i] = scaling == RAI_ROPE_NONE ? f : f * (keep + (1.0 - keep) / factor);
    }
    *gain = scaling == RAI_ROPE_YARN ? (float)(0.1 * std::log(factor) + 1.0) : 1.0f;
  });
}

int rai_paged_store_dev(const rai_pages *pages, size_t layer, const rai_page_batch *batch, const rai_rope *rope,
                        float *q_out, size_t q_out_stride, const float *q, size_t q_stride, size_t heads,
                        const float *k, size_t k_stride, const float *v, size_t v_stride, void *stream) {
  RAI_API_BODY({
    rai::check_pages(pages);
    if (layer >= pages->layers) rai::fail(RAI_E_RANGE, "layer is out of range");
    rai::BatchView b;
    const bool work = rai::check_batch(batch, pages, &b);
    rai::RopeView r{nullptr, 0, false, 1.0f};
    if (rope) {
      if (!rope->inv_freq) rai::fail(RAI_E_ARG, "null argument");
      if (rope->rot_dim == 0 || rope->rot_dim % 2 || rope->rot_dim > pages->head_dim)
        rai::fail(RAI_E_SHAPE, "rot_dim must be positive, even and at most head_dim");
      if (!std::isfinite(rope->gain)) rai::fail(RAI_E_ARG, "gain must be finite");
      r = rai::RopeView{rope->inv_freq, (int)rope->rot_dim, rope->interleaved != 0, rope->gain};
    }
    if (heads > 16384) rai::fail(RAI_E_SHAPE, "dimensions overflow");
    if (!work) return RAI_OK;
    if (heads) {
      rai::check_rows(q, q_stride, heads, pages->head_dim, "q");
      rai::check_rows(q_out, q_out_stride, heads, pages->head_dim, "q_out");
      if (q == q_out && q_stride != q_out_stride) rai::fail(RAI_E_SHAPE, "q rotated in place needs one stride");
    }
    rai::check_rows(k, k_stride, pages->kv_heads, pages->head_dim, "k");
    rai::check_rows(v, v_stride, pages->kv_heads, pages->head_dim, "v");
    const rai::StoreArgs a{q_out, q, k, v, q_out_stride, q_stride, k_stride, v_stride, (int)heads, r};
    rai::with_layer(pages, layer, [&](auto kv) { rai::launch_store(a, kv, b, (hipStream_t)stream); });
    RAI_HIP_CHECK(hipGetLastError());
  });
}

int rai_paged_attention_workspace(size_t heads, const rai_pages *pages, const rai_page_batch *batch,
                                  const rai_attention_options *options, size_t *bytes) {
  RAI_API_BODY({
    if (!bytes) rai::fail(RAI_E_ARG, "null argument");
    rai::check_pages(pages);
    rai::check_heads(heads, pages);
    rai::check_options(options);
    rai::BatchView b;
    *bytes = 0;
    if (!rai::check_batch(batch, pages, &b)) return RAI_OK;
    rai::check_rows_heads(b, heads);
    *bytes = rai::paged_attention_work((int)pages->kv_heads, (int)heads, (int)pages->head_dim,
                                       (int)rai::type_bytes(pages->type), b, rai::window_of(options));
  });
}

int rai_paged_attention_dev(float *out, size_t out_stride, const float *q, size_t q_stride, size_t heads,
                            const rai_pages *pages, size_t layer, const rai_page_batch *batch,
                            const rai_attention_options *options, void *work, size_t work_bytes, void *stream) {
  RAI_API_BODY({
    rai::check_pages(pages);
    if (layer >= pages->layers) rai::fail(RAI_E_RANGE, "layer is out of range");
    rai::check_heads(heads, pages);
    rai::check_options(options);
    rai::BatchView b;
    if (!rai::check_batch(batch, pages, &b)) return RAI_OK;
    rai::check_rows_heads(b, heads);
    rai::check_rows(q, q_stride, heads, pages->head_dim, "q");
    rai::check_rows(out, out_stride, heads, pages->head_dim, "out");
    if (out == q) rai::fail(RAI_E_ARG, "out must not be q");
    if (!work && work_bytes) rai::fail(RAI_E_ARG, "null argument");
    if ((uintptr_t)work % 16) rai::fail(RAI_E_ARG, "work must be 16-byte aligned");
    const rai::AttnArgs a{q, out, q_stride, out_stride, (int)heads, options->scale, options->softcap,
                          rai::window_of(options), options->slopes};
    rai::with_layer(pages, layer,
                    [&](auto kv) { rai::launch_paged_attention(a, kv, b, work, work_bytes, (hipStream_t)stream); });
    RAI_HIP_CHECK(hipGetLastError());
  });
}

int rai_paged_fork_dev(const rai_pages *pages, const int32_t *tables, size_t table_stride, const int32_t *lengths,
                       size_t seqs, const int32_t *parent, const int32_t *fresh, size_t n, int32_t *tables_out,
                       int32_t *lengths_out, int32_t *used, void *stream) {
  RAI_API_BODY({
    rai::check_pages(pages);
    if (n == 0) return RAI_OK;
    if (!tables || !lengths || !parent || !fresh || !tables_out || !lengths_out || !used)
      rai::fail(RAI_E_ARG, "null argument");
    if (seqs == 0 || table_stride == 0) rai::fail(RAI_E_SHAPE, "the tables must not be empty");
    if (n > 65535 || seqs > 65535) rai::fail(RAI_E_SHAPE, "at most 65535 sequences");
    if (table_stride > INT32_MAX) rai::fail(RAI_E_SHAPE, "dimensions overflow");
    if (tables_out < tables + seqs * table_stride && tables < tables_out + n * table_stride)
      rai::fail(RAI_E_ARG, "tables_out overlaps tables");
    if (lengths_out < lengths + seqs && lengths < lengths_out + n) rai::fail(RAI_E_ARG, "lengths_out overlaps lengths");
    const rai::PoolBytes p = rai::pool_bytes(pages);
    const int parts = (int)((p.page_vecs + rai::kCopyVecs - 1) / rai::kCopyVecs);
    if ((size_t)p.layers * parts > (size_t(1) << 23)) rai::fail(RAI_E_SHAPE, "dimensions overflow");
    rai::k_fork<<<dim3(p.layers * parts, n), 256, 0, (hipStream_t)stream>>>(
        p, tables, table_stride, lengths, (int)seqs, parent, fresh, parts, tables_out, lengths_out, used,
        rai::page_shift(pages->page_size));
    RAI_HIP_CHECK(hipGetLastError());
  });
}

int rai_paged_move_dev(const rai_pages *pages, const int32_t *src, const int32_t *dst, size_t n, int32_t *tables,
                       size_t entries, void *stream) {
  RAI_API_BODY({
    rai::check_pages(pages);
    if (n == 0) return RAI_OK;
    if (!src || !dst || (!tables && entries)) rai::fail(RAI_E_ARG, "null argument");
    if (n > 65535) rai::fail(RAI_E_SHAPE, "at most 65535 pages in one call");
    const rai::PoolBytes p = rai::pool_bytes(pages);
    const size_t parts = (p.page_vecs + rai::kCopyVecs - 1) / rai::kCopyVecs, renames = std::min<size_t>(256, (entries + 255) / 256);
    if (n * p.layers * parts >= size_t(1) << 23) rai::fail(RAI_E_SHAPE, "too many pages x layers in one call");
    rai::k_move<<<(unsigned)(renames + n * p.layers * parts), 256, 0, (hipStream_t)stream>>>(p, src, dst, (int)n, (int)parts,
                                                                                        tables, entries, (int)renames);
    RAI_HIP_CHECK(hipGetLastError());
  });
}

}  // extern "C"
