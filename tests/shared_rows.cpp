// Which rows the joining of a shared prefix's parts takes, a row of the batch at a time (kernels/attn_index.h: seq_of_row, part_at): each
// sequence's first max_rows and no others, whatever a sequence's length; inside the buffers whatever these hold.
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
      printf("line %d: %s (round %d)\n", __LINE__, #x, round); \
      exit(1); \
    } \
  } while (0)

int main() {
  std::mt19937_64 rng(17);
  const int far[] = {0, 1, -1, 64, 0x7FFFFFFF, (int)0x80000000};
  for (int round = 0; round < 60000; ++round) {
    const int seqs = 1 + (int)(rng() % 60), T = 1 + (int)(rng() % 700), max_rows = rng() % 3 ? (int)(rng() % 40) : 0x7FFFFFFF;
    const bool sound = rng() % 4 != 0;
    std::vector<int> rows(seqs + 1), of(T, -1);
    if (sound) {
      int r = rng() % 3 ? 0 : (int)(rng() % 9);
      const int most = 1 + (int)(rng() % 30);
      for (int& x : rows) {
        x = r < T ? r : T;
        r += rng() % 20 == 0 ? (int)(rng() % 200) : (int)(rng() % most);   // (one of many rows beside others of few, or none)
      }
      for (int s = 0; s < seqs; ++s)
        for (int t = rows[s]; t < rows[s + 1]; ++t)
          if (t - rows[s] < max_rows) of[t] = s;
    } else {
      for (int& r : rows) r = rng() % 4 ? (int)(rng() % (2 * T)) - (int)(rng() % 30) : far[rng() % (sizeof far / sizeof *far)];
    }
    for (int t = 0; t < T; ++t) {
      const int s = attn::seq_of_row(rows.data(), 0, seqs, 0, T, t);
      NEED(s >= 0 && s < seqs);
      const attn::Seq q = attn::part_at(nullptr, rows.data(), s, seqs, T, max_rows);
      const bool takes = t >= q.r0 && t - q.r0 < q.n;
      if (sound) NEED(takes ? of[t] == s : of[t] == -1);
    }
    // the places of their pieces: one for each row, inside what there is of them, and found again from the sequence and its row
    const int most = max_rows < T ? max_rows : T, per = (long long)seqs * most <= T ? most : 0, places = per ? seqs * per : T;
    std::vector<char> used(places, 0);
    for (int s = 0; s < seqs; ++s) {
      const attn::Seq q = attn::part_at(nullptr, rows.data(), s, seqs, T, most);
      for (int i = 0; i < q.n; ++i) {
        const int u = attn::place_of(per, s, i, q.r0 + i);
        NEED(u >= 0 && u < places);
        if (sound) NEED(!used[u]);
        used[u] = 1;
        if (per) NEED(u / per == s && u % per == i);
        else NEED(u == q.r0 + i);
      }
    }
  }
  printf("%ld rows of batches\n", checks);
  return 0;
}
