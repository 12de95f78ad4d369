// What a plan does to a sequence (kernels/attn_index.h: change_of, ring_at), against 64-bit arithmetic, for every kind of nonsense that the
// device buffers may hold.
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <random>

#include "../arcinferzero_amd/csrc/kernels/attn_index.h"

static long checks = 0;
#define NEED(x) \
  do { \
    ++checks; \
    if (!(x)) { \
      printf("line %d: %s (before %d, add %d, shared %d, ps %d, ldt %d, max_rows %d)\n", __LINE__, #x, before, add, shared, ps, ldt, max_rows); \
      exit(1); \
    } \
  } while (0)

int main() {
  std::mt19937_64 rng(5);
  const int far[] = {0, 1, -1, 15, 16, 17, 255, 256, 4096, 0x7FFFFFFF, (int)0x80000000, (int)0x80000001, 0x7FFFF000, 1 << 30};
  auto any = [&](int most) {
    switch (rng() % 4) {
      case 0: return far[rng() % (sizeof far / sizeof *far)];
      case 1: return (int)rng();
      default: return (int)(rng() % (2 * (uint64_t)most + 3)) - (int)(rng() % 3 ? 0 : most);
    }
  };
  for (int round = 0; round < 400000; ++round) {
    const int ps = 4 + (int)(rng() % 5), ldt = rng() % 8 ? 1 + (int)(rng() % 300) : 0x7FFFF000 >> ps, max_rows = rng() % 4 ? (int)(rng() % 5000) : 0x7FFFFFFF;
    const int near = ldt <= 300 ? ldt << ps : 1 << 20, before = any(near), add = any(near), shared = any(near);
    const attn::Change c = attn::change_of(before, add, shared, ps, ldt, max_rows);
    const int64_t page = 1 << ps, most = (int64_t)ldt << ps, b = before < 0 ? 0 : before > most ? most : before, to = b + add < 0 ? 0 : b + add;
    const bool fits = add <= max_rows && to <= most;
    const int64_t had = (b + page - 1) / page;
    NEED(c.before == b && c.had == had && c.fits == fits);
    NEED(c.rows >= 0 && c.rows == (fits && add > 0 ? add : 0));
    NEED(c.len == (fits ? to : b) && c.len >= 0 && c.len <= most);
    NEED(c.take >= 0 && c.give >= 0 && (c.take == 0 || c.give == 0));
    if (fits && add >= 0) NEED(c.has == (to + page - 1) / page && c.take == c.has - c.had && c.give == 0);
    if (add < 0) {
      const int64_t kept = (shared < 0 ? 0 : shared > most ? most : shared) / page, need = (to + page - 1) / page, first = need > kept ? need : kept;
      NEED(c.take == 0 && c.give == (had > first ? had - first : 0) && c.has + c.give == had);
    }
    // every entry that is looked at lies in the table's row
    NEED(c.had >= 0 && c.had <= ldt && c.has >= 0 && c.has <= ldt);
    if (c.rows) NEED((c.before + c.rows - 1) >> ps < c.has && (c.before >> ps) <= c.had);
    const unsigned n = 1 + (unsigned)(rng() % 0x7FFFFFFFu), from = (unsigned)(rng() % n), i = (unsigned)(rng() % ((uint64_t)n + 1));
    NEED(attn::ring_at(from, i, n) == (unsigned)(((uint64_t)from + i) % n));
  }
  printf("%ld places of plans\n", checks);
  return 0;
}
