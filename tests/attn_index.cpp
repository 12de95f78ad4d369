// What the attention block's kernels make of a batch in device memory (kernels/attn_index.h), tried on the host with every kind of
// rows, lengths, prefixes, first positions and windows: each row, table entry and cache position that a kernel would take has to
// lie in its buffer.  The walks are those of attn_few (32 keys a step, four waves) and attn_many (tiles of 32 or 64 keys).
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#include "../arcinferzero_amd/csrc/kernels/attn_index.h"

static long checks = 0;
#define NEED(x)                                                                                                  \
  do {                                                                                                           \
    ++checks;                                                                                                    \
    if (!(x)) { printf("%s:%d: %s does not hold\n", __FILE__, __LINE__, #x); exit(1); }                          \
  } while (0)

int main() {
  std::mt19937 rng(5);
  const int edge[] = {-2147483647 - 1, -2147483647, -70000, -33, -1, 0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 255, 256, 1000, 4095, 70000, 2147479551, 2147483646, 2147483647};
  auto any = [&](int small) {
    const unsigned k = rng() % 4;
    return k == 0 ? edge[rng() % (sizeof edge / sizeof *edge)] : k == 1 ? (int)rng() : (int)(rng() % (unsigned)(small + 1));
  };
  for (int trial = 0; trial < 400000; ++trial) {
    const int ps = 4 + (int)(rng() % 5), T = 1 + (int)(rng() % 300), max_rows = 1 + (int)(rng() % 300), G = 1 + (int)(rng() % 16);
    // (the table's size: small, or the largest that a call takes)
    const int ldt = rng() % 8 ? 1 + (int)(rng() % 40) : 0x7FFFF000 >> ps, most_len = ldt << ps;
    const attn::Seq q = attn::seq_at(any(300), any(300), any(most_len), T, max_rows, most_len);
    NEED(q.r0 >= 0 && q.n >= 0 && q.n <= max_rows && q.r0 + q.n <= T && q.len >= 0 && q.len <= most_len && q.p0 + q.n <= q.len && q.p0 >= -T);
    if (!q.n) continue;
    const int window = rng() % 2 ? 0 : (int)(rng() % 3 ? rng() % 100 + 1 : 1 << 30), prefix = rng() % 2 ? 0 : any(most_len);
    const bool docs = rng() % 2;
    int all_lo = 0x7FFFFFFF, all_hi = 0, lo, hi, u;
    for (int i = 0; i < q.n; ++i) {
      attn::sees(q.p0 + i, q.len, window, prefix, docs ? any(most_len) : 0, lo, hi);
      NEED(lo >= 0 && hi <= q.len);
      if (lo < hi && lo < all_lo) all_lo = lo;
      if (lo < hi && hi > all_hi) all_hi = hi;
    }
    if (!docs) {   // (attn_few's way: the first row's beginning, the last row's end)
      int l, h;
      attn::sees(q.p0, q.len, window, prefix, 0, l, u);
      attn::sees(q.p0 + q.n - 1, q.len, window, prefix, 0, u, h);
      NEED(all_lo >= all_hi || (l <= all_lo && h == all_hi));
      all_lo = l;
      all_hi = h;
    }
    for (int unit = 32; unit <= 64; unit *= 2) {
      const attn::Span s = attn::span_of(all_lo, all_hi, unit);
      NEED(s.base >= 0 && s.base % unit == 0 && s.steps >= 0 && (s.steps == 0 || (s.base <= all_lo && s.base + (s.steps - 1) * unit < all_hi)));
      // the last work-group's steps and what it looks up ahead of them: up to 12 steps of 32 (three waves on, two rounds ahead), or
      // two tiles of 64
      const int last = s.steps, ahead = unit == 32 ? 12 : 2;
      // (pieces: one behind the other, the last to the end; what a piece without steps looks up is no further than that)
      const int pieces = 1 + (int)(rng() % 1024), least = rng() % 2 ? 1 : 1 + (int)(rng() % 64);
      int behind = 0;
      for (int z = 0; z < pieces; ++z) {
        const attn::Part p = attn::part_of(s.steps, pieces, least, z);
        NEED(p.z0 == behind && p.z0 <= p.z1 && p.z1 <= s.steps);
        behind = p.z1;
      }
      NEED(behind == s.steps);
      for (int st : {0, 1, last / 2, last - 1, last, last + ahead}) {
        if (st < 0) continue;
        for (int t = 0; t < unit; t += 4) {
          const int p = s.base + st * unit + t, e = attn::entry_of(p, ps, ldt);
          NEED(p >= 0 && e >= 0 && e < ldt);
          if (st < s.steps && p < q.len) NEED(e == p >> ps);
        }
      }
    }
    // kv_write and kv_read: positions of rows, and tiles of them up to the last that is launched for 2^30 rows
    const int from = attn::upper(q.p0, 0), to = q.p0 + q.n, tile = 1 << (rng() % 9);
    int next = from & -tile;
    for (int i = 0; i < 302; ++i) {
      const int t0 = attn::tile_at(from, to, tile, i);
      NEED(from < to && next < to ? t0 == next : t0 == -1);
      if (t0 >= 0) {
        NEED((t0 >> ps) >= 0 && (attn::lower(t0 + tile, to) - 1) >> ps < ldt);
        next += tile;
      }
    }
    for (int i : {1000, 1 << 20, (1 << 30) / tile + 1}) NEED(attn::tile_at(from, to, tile, i) == -1);
    for (int i = 0; i < q.n; ++i)
      if (q.p0 + i >= 0) NEED((q.p0 + i) >> ps < ldt);
  }
  printf("%ld places in their buffers\n", checks);
  return 0;
}
