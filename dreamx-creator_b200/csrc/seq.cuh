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
// Rows before the first offset are no sequence's either. With `lens`, len is its entry of it, and
// begin and end are the sequence's rows: all of them come with one trip to memory, of up to 32
// sequences, and another for each 32 times as many.
SRDIT_DEV int find_sequence(const Offsets& o, int B, int t, Divisor by_each, const int32_t* lens,
                            int& len, int& begin, int& end) {
  if (!o.at) {
    const int b = by_each.div(t);
    begin = b * o.each;
    end = begin + o.each;
    len = lens ? __ldg(lens + b) : 0;
    return b;
  }
  const int lane = threadIdx.x & 31;
  int base = 0, count = B;  // it is among these, or none
  while (count > 32) {      // offsets that are not above t, one of each 32nd of them
    const int each = (count + 31) >> 5, n = (lane + 1) * each;
    const int k = __popc(__ballot_sync(0xffffffffu, n < count && __ldg(o.at + base + n) <= t));
    base += k * each;
    count = min(each, count - k * each);
  }
  const int n = base + lane;
  const bool on = lane < count;
  const int to = on ? __ldg(o.at + n + 1) : 0x7fffffff, from = on ? __ldg(o.at + n) : 0;
  const int l = on && lens ? __ldg(lens + n) : 0;
  const int x = __popc(__ballot_sync(0xffffffffu, to <= t));  // (of ascending offsets)
  if (x >= count) return B;
  begin = max(__shfl_sync(0xffffffffu, from, x), 0);
  end = min(__shfl_sync(0xffffffffu, to, x), o.rows);
  len = __shfl_sync(0xffffffffu, l, x);
  return t >= begin ? base + x : B;
}
SRDIT_DEV int find_sequence(const Offsets& o, int B, int t, Divisor by_each) {
  int len, begin, end;
  return find_sequence(o, B, t, by_each, nullptr, len, begin, end);
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
