// Replays the addresses of a paged key/value cache (kernelcodegen_amd/csrc/kv_cache_index.h) over
// slots, page tables and lengths that a kernel must not trust: every row is inside the cache or -1,
// a slot's row is its own, and offsets do not wrap where they pass 32 bits.
#include <stdio.h>
#include <initializer_list>

#include "kv_cache_index.h"

using namespace kcg;

static int failures = 0;
#define CHECK(x)                                             \
  do {                                                       \
    if (!(x) && failures++ < 10) printf("line %d: %s\n", __LINE__, #x); \
  } while (0)

int main() {
  const int bad[] = {-2147483647 - 1, -2147483647, -65536, -17, -1, 0, 1, 3, 4, 15, 16, 63, 64, 65, 1023, 1 << 20, 2147483647};
  const KvShape shapes[] = {{1, 4, 1}, {4, 4, 8}, {65, 5, 3}, {524287, 8, 8}, {8388607, 8, 65536}};
  for (const KvShape &c : shapes) {
    const int64_t rows = (int64_t{c.pages} * c.heads) << c.log2_page;
    const int page = 1 << c.log2_page;
    for (int head : {0, c.heads / 2, c.heads - 1}) {
      for (int p : bad)
        for (int place : {0, 1, page - 1}) {
          const int64_t r = kv_row(c, p, head, place);
          const bool in = p >= 0 && p < c.pages;
          CHECK(in ? r >= 0 && r < rows : r == -1);
          if (in) CHECK(r == (int64_t{p} * c.heads + head) * page + place);
        }
      for (int s : bad) {
        const int64_t r = kv_slot_row(c, s, head);
        const bool in = s >= 0 && s / page < c.pages;
        CHECK(in ? r >= 0 && r < rows : r == -1);
        if (in) CHECK(r == (int64_t{s / page} * c.heads + head) * page + s % page);
      }
    }
    // the last slot of the last head is the last row
    if (int64_t{c.pages} * page <= 0x7fffffff)
      CHECK(kv_slot_row(c, c.pages * page - 1, c.heads - 1) == rows - 1);
  }
  for (int context : bad)
    for (int drafts : bad)
      for (int n : {1, 2, 13, 63, 64})
        for (int64_t capacity : {int64_t{16}, int64_t{17 * 16}, int64_t{1} << 20, int64_t{0x7fffffff}}) {
          const KvLens l = kv_lens(context, drafts, n, capacity);
          CHECK(l.context >= 0 && l.drafts >= 0 && l.drafts <= n && l.queries >= l.drafts && l.queries <= n);
          CHECK(int64_t{l.context} + l.drafts <= capacity);
          if (context >= 0 && drafts >= 0 && drafts <= n && int64_t{context} + drafts <= capacity)
            CHECK(l.context == context && l.drafts == drafts && l.queries == drafts);
        }
  const uint64_t words[] = {0, 1, ~uint64_t{0}, uint64_t{1} << 63, 0xaaaaaaaaaaaaaaaaull};
  for (int drafts = 0; drafts <= 64; ++drafts)
    for (int n = 0; n < 64; ++n) {
      for (int i = 0; i < 5; ++i) {
        const uint64_t w = kv_seen(words, i, n, drafts);
        for (int j = 0; j < 64; ++j) CHECK(((w >> j) & 1) == (j < drafts ? (words[i] >> j) & 1 : 0));
      }
      const uint64_t w = kv_seen(nullptr, 0, n, drafts);
      for (int j = 0; j < 64; ++j) CHECK(((w >> j) & 1) == (j < drafts && j <= n ? 1u : 0u));
    }
  if (failures) return 1;
  printf("all inside\n");
  return 0;
}
