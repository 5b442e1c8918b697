// Where a batch's rows and positions lie in the pages of a paged KV cache: the
// bounds that device-side lengths and page ids are cut to (no HIP here, so that
// the host can test them alone).
#ifndef RAI_PAGED_INDEX_H
#define RAI_PAGED_INDEX_H

#include <cstddef>
#include <cstdint>

#ifdef __HIPCC__
#define RAI_HD __host__ __device__ __forceinline__
#else
#define RAI_HD inline
#endif

namespace rai {

// A batch as the kernels take it (rai_page_batch); max_kv is at most the
// positions of a table row.
struct BatchView {
  const int *tables;
  size_t stride;
  const int *q_start, *kv_len;
  int seqs, tokens, max_q, max_kv;
};

// Rows q0 .. q0 + nq - 1 of a sequence of n positions; row q0 + j is position
// n - nq + j (negative where the length is shorter than the rows).
struct SeqSpan {
  int q0, nq, n;
};

RAI_HD int clamp_int(int v, int lo, int hi) { return v < lo ? lo : v > hi ? hi : v; }

// Any contents of q_start and kv_len give rows inside 0 .. tokens - 1, at most
// max_q of them, and a length of 0 .. max_kv.
RAI_HD SeqSpan seq_span(const BatchView &b, int s) {
  SeqSpan r;
  r.q0 = clamp_int(b.q_start[s], 0, b.tokens);
  const int end = clamp_int(b.q_start[s + 1], r.q0, b.tokens);
  r.nq = end - r.q0 < b.max_q ? end - r.q0 : b.max_q;
  r.n = clamp_int(b.kv_len[s], 0, b.max_kv);
  return r;
}

// The page of position pos (0 <= pos < stride << shift) in a table row, -1 where
// there is none.
RAI_HD int page_of(const int *row, int pos, int shift, int pages) {
  const int p = row[pos >> shift];
  return (unsigned)p < (unsigned)pages ? p : -1;
}

// Element offsets of (page, kv head, slot) in a layer's keys, and of (page, kv
// head, dimension 0, slot) in its values.
RAI_HD size_t key_at(int page, int head, int slot, int heads, int hd, int shift) {
  return (((((size_t)page * heads + head) << shift) + slot)) * hd;
}
RAI_HD size_t value_at(int page, int head, int slot, int heads, int hd, int shift) {
  return ((((size_t)page * heads + head) * hd) << shift) + slot;
}

// The first position that a row at `pos` sees (window 0: all of them).
RAI_HD int first_seen(int pos, int window) {
  return window > 0 && pos - window + 1 > 0 ? pos - window + 1 : 0;
}

}  // namespace rai

#endif
