// Where a token of a paged key/value cache lies.  Host and device code share these functions:
// the CPU tests replay them over tables and lengths that a kernel must not trust.
#pragma once

#include <stdint.h>

#if defined(__HIP__)
#define KCG_HD __host__ __device__ inline __attribute__((always_inline))
#else
#define KCG_HD inline
#endif

namespace kcg {

// [pages][heads][page][dim], page = 2^log2_page tokens
struct KvShape {
  int pages, log2_page, heads;
};

// Row (of `dim` elements) of a token in page `page` at place `place`; -1: no such page.
KCG_HD int64_t kv_row(const KvShape &c, int page, int head, int place) {
  if (page < 0 || page >= c.pages) return -1;
  return ((static_cast<int64_t>(page) * c.heads + head) << c.log2_page) + place;
}

// Row of a slot (page * page_size + place); -1: outside the cache.
KCG_HD int64_t kv_slot_row(const KvShape &c, int slot, int head) {
  if (slot < 0) return -1;
  return kv_row(c, slot >> c.log2_page, head, slot & ((1 << c.log2_page) - 1));
}

// The keys of one sequence: `context` that every query sees, then `drafts`; both clamped to
// what the table has room for and to the call's N.
struct KvLens {
  int context, drafts;  // context + drafts <= capacity
  int queries;          // rows of the output that are written
};

KCG_HD KvLens kv_lens(int context, int drafts, int n, int64_t capacity) {
  KvLens r;
  r.queries = drafts < 0 ? 0 : (drafts > n ? n : drafts);
  const int64_t c = context < 0 ? 0 : context;
  r.context = static_cast<int>(c < capacity ? c : capacity);
  const int64_t room = capacity - r.context;
  r.drafts = static_cast<int>(r.queries < room ? r.queries : room);
  return r;
}

// The drafted keys that query n sees, as bits.
KCG_HD uint64_t kv_seen(const uint64_t *tree_mask, int64_t index, int n, int drafts) {
  const uint64_t all = drafts >= 64 ? ~uint64_t{0} : (uint64_t{1} << drafts) - 1;
  const uint64_t chain = n >= 63 ? ~uint64_t{0} : (uint64_t{2} << n) - 1;
  return (tree_mask ? tree_mask[index] : chain) & all;
}

}  // namespace kcg
