// Host check of paged_index.h: whatever the lengths, row starts and page ids
// hold, rows, positions and addresses stay inside the arrays they index.
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#include "paged_index.h"

using namespace rai;

#define CHECK(c)                                       \
  do {                                                 \
    if (!(c)) {                                        \
      std::printf("line %d: %s\n", __LINE__, #c);      \
      std::exit(1);                                    \
    }                                                  \
  } while (0)

int main() {
  std::mt19937 rng(1);
  const int odd[] = {0, 1, -1, 5, 16, 17, 1 << 20, INT32_MAX, INT32_MIN, INT32_MAX - 1};
  auto pick = [&](int n) { return (int)(rng() % n); };
  for (int it = 0; it < 200000; ++it) {
    const int shift = 4 + pick(7), stride = 1 + pick(5), pages = 1 + pick(9), heads = 1 + pick(3), hd = 8 * (1 + pick(32));
    const int seqs = 1 + pick(4);
    std::vector<int> starts(seqs + 1), lens(seqs), tab(seqs * stride);
    for (int &v : starts) v = pick(2) ? odd[pick(10)] : pick(40);
    for (int &v : lens) v = pick(2) ? odd[pick(10)] : pick(200);
    for (int &v : tab) v = pick(2) ? odd[pick(10)] : pick(pages);
    BatchView b{tab.data(), (size_t)stride, starts.data(), lens.data(), seqs, 1 + pick(40), 0, 0};
    b.max_q = 1 + pick(b.tokens);
    b.max_kv = pick((stride << shift) + 1);
    for (int s = 0; s < seqs; ++s) {
      const SeqSpan r = seq_span(b, s);
      CHECK(r.q0 >= 0 && r.nq >= 0 && r.q0 + r.nq <= b.tokens && r.nq <= b.max_q);
      CHECK(r.n >= 0 && r.n <= b.max_kv);
      for (int j = 0; j < r.nq; ++j) {
        const int pos = r.n - r.nq + j;
        CHECK(pos < b.max_kv);
        const int window = pick(3) ? pick(50) : odd[pick(10)] < 0 ? 0 : odd[pick(10)] & INT32_MAX;
        const int first = first_seen(pos, window > INT32_MAX / 2 ? INT32_MAX / 2 : window);
        CHECK(first >= 0);
        for (int p = first; p <= pos; p += 1 + pick(20)) {
          const int pg = page_of(tab.data() + (size_t)s * stride, p, shift, pages);
          CHECK(pg >= -1 && pg < pages);
          if (pg < 0) continue;
          const int h = pick(heads), slot = p & ((1 << shift) - 1);
          const size_t all = ((size_t)pages * heads << shift) * hd;
          CHECK(key_at(pg, h, slot, heads, hd, shift) + hd <= all);
          CHECK(value_at(pg, h, slot, heads, hd, shift) + ((size_t)(hd - 1) << shift) < all);
        }
      }
    }
  }
  // Offsets past 32 bits.
  CHECK(key_at(1 << 20, 7, 15, 8, 128, 4) == ((((size_t)(1 << 20) * 8 + 7) << 4) + 15) * 128);
  CHECK(value_at(1 << 20, 7, 15, 8, 128, 4) == ((((size_t)(1 << 20) * 8 + 7) * 128) << 4) + 15);
  std::puts("ok");
  return 0;
}
