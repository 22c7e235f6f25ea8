// seq.cuh -- packed sequences and pages: which rows a sequence has, which page a key is in.
#pragma once
#include "attn.cuh"
#include "srdit_internal.h"

namespace srdit {

// Rows of packed sequences: sequence b has rows [at[b], at[b + 1]) of `rows` (clamped to them
// and to ascending order), or without offsets `each` rows each.
struct Offsets {
  const int32_t* at;
  int rows, each;
  SRDIT_DEV int begin(int b) const { return at ? min(max(__ldg(at + b), 0), rows) : b * each; }
  SRDIT_DEV int end(int b) const {
    return at ? max(begin(b), min(__ldg(at + b + 1), rows)) : b * each + each;
  }
};

// The sequence among B that packed row t belongs to, by one warp (B: behind the last one).
// Rows before the first offset are no sequence's either.
SRDIT_DEV int find_sequence(const Offsets& o, int B, int t, Divisor by_each) {
  if (!o.at) return by_each.div(t);
  const int lane = threadIdx.x & 31;
  int b = 0;
  for (int base = 0; base < B; base += 32) {  // offsets that are not above t
    const int n = base + lane;
    const unsigned below = __ballot_sync(0xffffffffu, n < B && __ldg(o.at + n + 1) <= t);
    b = base + __popc(below);
    if (below != 0xffffffffu) break;
  }
  return b < B && t >= __ldg(o.at) ? b : B;
}

// A sequence's pages.
struct Table {
  const int32_t* at;
  long long stride;
  int width, pages, page_size;
  Divisor by_page;
  // the page of a sequence's n-th page, or -1 where the table has none or one out of range
  SRDIT_DEV int page(int b, int n) const {
    if (n < 0 || n >= width) return -1;
    const int p = __ldg(at + b * stride + n);
    return p >= 0 && p < pages ? p : -1;
  }
  // a sequence's length, no more than its pages hold
  SRDIT_DEV int clamp_len(int len) const {
    const long long most = static_cast<long long>(width) * page_size;
    return static_cast<int>(min(max(static_cast<long long>(len), 0ll), most));
  }
};

inline Table table_of(const srdit_kv_pages& p) {
  return {p.table, p.table_stride, p.table_width, p.pages, p.page_size,
          Divisor::of(p.page_size > 0 ? p.page_size : 1)};
}

// Argument checks of a cache's pages that every entry point makes.
int check_pages(const srdit_kv_pages& p);

}  // namespace srdit
