// The positions and places that the attention block's kernels work out from what the batch says in device memory: plain integers,
// for the kernels and for a host program that tries them on every kind of nonsense (tests/attn_index.cpp).
#pragma once
#ifdef __HIPCC__
#define ATTN_FN __host__ __device__ inline
#else
#define ATTN_FN inline
#endif
namespace attn {
ATTN_FN int lower(int a, int b) { return a < b ? a : b; }
ATTN_FN int upper(int a, int b) { return a > b ? a : b; }

struct Seq {
  int r0;    // its first row
  int n;     // its rows that this launch takes (at most max_rows)
  int p0;    // the position of its first row (below 0 where len says less than the rows)
  int len;
};
// rows held to [0, T], the length to what the table holds
ATTN_FN Seq seq_at(int row0, int row1, int length, int T, int max_rows, int most_len) {
  Seq q;
  q.r0 = lower(upper(row0, 0), T);
  const int all = lower(upper(row1, q.r0), T) - q.r0;
  q.n = lower(all, max_rows);
  q.len = lower(upper(length, 0), most_len);
  q.p0 = q.len - all;
  return q;
}
// The positions [lo, hi) that a row at position p sees (none: lo >= hi; a row below position 0 sees none, whatever the prefix).
ATTN_FN void sees(int p, int len, int window, int prefix, int first, int& lo, int& hi) {
  hi = p < 0 ? 0 : lower(len, upper(p + 1, prefix));
  lo = upper(first, 0);
  if (window) lo = upper(lo, p - window + 1);
}
// The keys [lo, hi) of all rows together in steps of `unit` (a power of two) from a whole one on; no step where no row sees any,
// whatever lo is then.
struct Span {
  int base, steps;
};
ATTN_FN Span span_of(int lo, int hi, int unit) {
  Span s = {0, 0};
  if (lo < hi) {
    s.base = lo & -unit;
    s.steps = (hi - s.base + unit - 1) / unit;
  }
  return s;
}
// The steps [z0, z1) of piece z of `pieces`, at least `least` to a piece that has any (behind the last step: none, from there on).
struct Part {
  int z0, z1;
};
ATTN_FN Part part_of(int steps, int pieces, int least, int z) {
  const int share = upper((steps + pieces - 1) / pieces, least);
  Part p;
  p.z0 = lower(z * share, steps);
  p.z1 = lower(p.z0 + share, steps);
  return p;
}
// Where the i-th tile of `tile` positions (a power of two) from a whole one on begins, for rows at [from, to); -1: there is none.  (Work-groups
// are launched for the most rows of any sequence: i * tile alone may lead past 2^31.)
ATTN_FN int tile_at(int from, int to, int tile, int i) {
  const int t0 = from & -tile;
  return from < to && i <= (to - 1 - t0) / tile ? t0 + i * tile : -1;
}
// Where the table has the page of a position: within its row of ldt entries also for a position behind the last key (up to 4096
// behind it; most_len is at most 2^31 - 4096).
ATTN_FN int entry_of(int p, int ps, int ldt) { return lower(p >> ps, ldt - 1); }
}  // namespace attn
