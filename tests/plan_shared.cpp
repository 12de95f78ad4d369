// Plans of sequences whose first pages are also others' (kernels/attn_index.h: planned), played through page by page on the host: no row ever
// lies in a page that another sequence has too, and every page is in one place -- the ring, the prefix, one sequence's table.
#include <algorithm>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#include "../arcinferzero_amd/csrc/kernels/attn_index.h"

static long checks = 0;
#define NEED(x) \
  do { \
    ++checks; \
    if (!(x)) { \
      printf("line %d: %s\n", __LINE__, #x); \
      exit(1); \
    } \
  } while (0)

struct Pool {
  int ps, ldt, shared, prefix;   // (pages 0 ... prefix - 1 are the shared ones)
  std::vector<int> ring, len;
  std::vector<std::vector<int>> table;
  Pool(int seqs, int ps_, int ldt_, int shared_, int free) : ps(ps_), ldt(ldt_), shared(shared_), prefix(shared_ >> ps_), len(seqs, shared_ >> ps_ << ps_) {
    for (int i = 0; i < free; ++i) ring.push_back(prefix + i);
    table.assign(seqs, std::vector<int>(ldt, -1));
    for (auto& t : table)
      for (int e = 0; e < prefix; ++e) t[e] = e;
  }
  // A plan of one sequence, as the kernel carries it out; false: refused.
  bool plan(int s, int add, int max_rows = 1 << 20) {
    const attn::Change c = attn::planned(len[s], add, shared, ps, ldt, max_rows);
    if (!c.fits || c.take > (int)ring.size()) {
      NEED(c.fits || (c.rows == 0 && c.take == 0 && c.give == 0 && c.len == c.before && c.has == c.had));
      return false;
    }
    for (int i = 0; i < c.give; ++i) {
      ring.push_back(table[s][c.has + i]);
      table[s][c.has + i] = -1;
    }
    for (int i = 0; i < c.take; ++i) {
      table[s][c.had + i] = ring.front();
      ring.erase(ring.begin());
    }
    for (int i = 0; i < c.rows; ++i) NEED(table[s][(c.before + i) >> ps] >= prefix);   // (its own page)
    len[s] = c.len;
    return true;
  }
  void conserved(int free) const {
    std::vector<int> all(ring);
    for (auto& t : table) {
      for (int e = 0; e < prefix; ++e) NEED(t[e] == e);
      for (int e = prefix; e < ldt; ++e)
        if (t[e] >= 0) all.push_back(t[e]);
    }
    std::sort(all.begin(), all.end());
    NEED((int)all.size() == free);
    for (int i = 0; i < free; ++i) NEED(all[i] == prefix + i);
  }
};

int main() {
  {   // taken back into the prefix, given tokens, ended, begun again
    Pool p(2, 4, 12, 64, 20);
    NEED(p.plan(0, 36) && p.len[0] == 100);
    NEED(p.plan(0, -60) && p.len[0] == 40 && p.ring.size() == 20);
    NEED(!p.plan(0, 10) && p.len[0] == 40);
    NEED(p.plan(0, (int)0x80000000) && p.len[0] == 0 && p.ring.size() == 20);
    NEED(!p.plan(0, 64) && !p.plan(0, 1));
    p.conserved(20);
    p.len[0] = 64;   // (behind the prefix once more)
    NEED(p.plan(0, 1) && p.len[0] == 65);
    p.conserved(20);
  }
  std::mt19937_64 rng(3);
  for (int round = 0; round < 4000; ++round) {
    const int ps = 4 + (int)(rng() % 3), ldt = 2 + (int)(rng() % 12), shared = (int)(rng() % ((ldt - 1) << ps)), seqs = 1 + (int)(rng() % 4), free = (int)(rng() % 30);
    Pool p(seqs, ps, ldt, shared, free);
    for (int step = 0; step < 40; ++step) {
      const int s = (int)(rng() % seqs);
      const int add = rng() % 8 == 0 ? (int)0x80000000 : (int)(rng() % 90) - 40;
      if (rng() % 6 == 0) p.len[s] = std::max(p.len[s], p.prefix << ps);
      p.plan(s, add);
      p.conserved(free);
    }
  }
  printf("%ld places of plans behind prefixes\n", checks);
  return 0;
}
