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
// Sequences behind a shared prefix.  Group g has sequences [groups[g], groups[g + 1]), whose rows are one behind the other; without groups g is a
// sequence.  Its rows, held to the buffers; len: its first sequence (held to those there are, whether it has rows or not).
ATTN_FN Seq part_at(const int* groups, const int* rows, int g, int seqs, int T, int max_rows) {
  int s0 = g, s1 = g + 1;
  if (groups) {
    s0 = lower(upper(groups[g], 0), seqs);
    s1 = lower(upper(groups[g + 1], s0), seqs);
  }
  Seq q;
  q.r0 = lower(upper(rows[s0], 0), T);
  q.n = lower(lower(upper(rows[s1], q.r0), T) - q.r0, max_rows);
  q.p0 = 0;
  q.len = lower(s0, seqs - 1);
  return q;
}
// The part of a row's interval [from, to) in front of `split`, or behind it, inside a table of `most` positions.
ATTN_FN void part_of_span(int from, int to, int split, bool front, int most, int& lo, int& hi) {
  lo = upper(from, front ? 0 : upper(split, 0));
  hi = lower(lower(to, front ? split : to), most);
}
// The sequence of [s0, s1) that row t belongs to: tried first where rows of equal numbers would have it (a decode step's tokens: one look), then
// searched for; some one of them where the rows are in no order.
ATTN_FN int seq_of_row(const int* rows, int s0, int s1, int r0, int n, int t) {
  const int at = s0 + (int)((long long)(t - r0) * (s1 - s0) / upper(n, 1)), guess = lower(upper(at, s0), s1 - 1);
  if (rows[guess] <= t && t < rows[guess + 1]) return guess;
  int a = s0, b = s1;
  while (b - a > 1) {
    const int m = a + (b - a) / 2;
    if (rows[m] <= t) a = m;
    else b = m;
  }
  return a;
}
// Where a row's pieces are among those of a batch: row t, the i-th of sequence s -- `per` places for each sequence, or (0) one for each row of the buffers.
ATTN_FN int place_of(int per, int s, int i, int t) { return per ? s * per + i : t; }
// The group that a sequence is in (n of them, in order), -1: in none.
ATTN_FN int group_of(const int* groups, int n, int s) {
  int a = 0, b = n;   // (the last group that does not begin behind s lies in [a, b))
  while (b - a > 1) {
    const int m = a + (b - a) / 2;
    if (groups[m] <= s) a = m;
    else b = m;
  }
  return n > 0 && groups[a] <= s && s < groups[a + 1] ? a : -1;
}
// What a plan does to a sequence: `add` tokens behind the `before` that it has, or -add taken off, in pages of 2^ps tokens, `ldt` of them at most.  Its pages
// are then the entries [0, has) of the table, [0, had) before; `take` of them new, or those from `has` on, `give` of them, given back -- never
// those that lie whole in the first `shared` positions.  fits: no more than max_rows tokens, no more pages than the table has.
struct Change {
  int before, len, rows, had, has, take, give;
  bool fits;
};
ATTN_FN Change change_of(int before, int add, int shared, int ps, int ldt, int max_rows) {
  const int most = ldt << ps, mask = (1 << ps) - 1;   // (most: at most 2^31 - 4096)
  Change c;
  c.before = lower(upper(before, 0), most);
  c.had = (c.before + mask) >> ps;
  c.fits = add <= max_rows && add <= most - c.before;
  c.rows = c.fits ? upper(add, 0) : 0;
  c.len = add < 0 ? (c.before > -(add + 1) ? c.before + add : 0) : c.before + c.rows;
  c.has = (c.len + mask) >> ps;
  if (add < 0) c.has = lower(c.had, upper(c.has, lower(upper(shared, 0), most) >> ps));
  c.take = upper(c.has - c.had, 0);
  c.give = upper(c.had - c.has, 0);
  return c;
}
// ... and the change that a plan takes: no row in one of the whole pages of the first `shared` positions, which are others' too -- what is written there
// would be theirs as well, and a page that is taken for it would be given back by nobody, since those entries stay.
ATTN_FN Change planned(int before, int add, int shared, int ps, int ldt, int max_rows) {
  Change c = change_of(before, add, shared, ps, ldt, max_rows);
  if (add > 0 && c.before < lower(upper(shared, 0), ldt << ps) >> ps << ps) {
    c.fits = false;
    c.rows = c.take = 0;
    c.len = c.before;
    c.has = c.had;
  }
  return c;
}
// The i-th place behind `from` in a ring of n (from below n, i at most n).
ATTN_FN unsigned ring_at(unsigned from, unsigned i, unsigned n) {
  const unsigned k = from + i;   // (below 2^32: n is below 2^31)
  return k >= n ? k - n : k;
}
}  // namespace attn
