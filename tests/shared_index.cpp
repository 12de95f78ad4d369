// Where the rows and keys of sequences behind a shared prefix are (kernels/attn_index.h: part_at, part_of_span, group_of): inside the buffers
// whatever these hold, and the two parts of a row's interval the whole of it.
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
  std::mt19937_64 rng(11);
  const int far[] = {0, 1, -1, 64, 0x7FFFFFFF, (int)0x80000000, 0x7FFFF000};
  auto any = [&](int most) { return rng() % 4 == 0 ? far[rng() % (sizeof far / sizeof *far)] : (int)(rng() % (2 * (uint64_t)most + 3)) - (int)(rng() % 2 ? 0 : most); };
  for (int round = 0; round < 100000; ++round) {
    const int seqs = 1 + (int)(rng() % 40), n = (int)(rng() % 9), T = 1 + (int)(rng() % 500), max_rows = (int)(rng() % 3 ? rng() % 600 : 0x7FFFFFFF);
    const bool sound = rng() % 2;
    std::vector<int> groups(n + 1), rows(seqs + 1);
    if (sound) {
      int s = (int)(rng() % 3), r = 0;
      for (int& g : groups) { g = s < seqs ? s : seqs; s += (int)(rng() % 8); }
      for (int& x : rows) { x = r < T ? r : T; r += (int)(rng() % 20); }
    } else {
      for (int& g : groups) g = any(seqs);
      for (int& r : rows) r = any(T);
    }
    for (int g = 0; g < n; ++g) {
      const attn::Seq q = attn::part_at(groups.data(), rows.data(), g, seqs, T, max_rows);
      NEED(q.r0 >= 0 && q.n >= 0 && q.r0 + q.n <= T && q.n <= max_rows && q.len >= 0 && q.len < seqs);
      const int s1 = attn::lower(attn::upper(groups[g + 1], q.len + 1), seqs);
      for (int i = 0; i < q.n; ++i) {
        const int s = attn::seq_of_row(rows.data(), q.len, s1, q.r0, q.n, q.r0 + i);
        NEED(s >= q.len && s < s1);
        if (sound) NEED(rows[s] <= q.r0 + i && q.r0 + i < rows[s + 1]);
      }
      if (sound && q.n) NEED(q.len == groups[g] && q.r0 == rows[groups[g]] && q.n == attn::lower(rows[groups[g + 1]] - q.r0, max_rows));
    }
    for (int s = 0; s < seqs; ++s) {
      const attn::Seq q = attn::part_at(nullptr, rows.data(), s, seqs, T, max_rows);
      NEED(q.r0 >= 0 && q.n >= 0 && q.r0 + q.n <= T && q.n <= max_rows && q.len == s);
      const int g = attn::group_of(groups.data(), n, s);
      NEED(g >= -1 && g < n);
      if (sound) {
        int in = -1;
        for (int k = 0; k < n; ++k)
          if (groups[k] <= s && s < groups[k + 1]) in = k;
        NEED(g == in);
      }
    }
    const int most = 16 * (1 + (int)(rng() % 100)), from = any(most), to = any(most), split = any(most);
    int a, b, c, d;
    attn::part_of_span(from, to, split, true, most, a, b);
    attn::part_of_span(from, to, split, false, most, c, d);
    NEED(a >= 0 && b <= most && c >= 0 && d <= most);
    for (int j = 0; j < most; ++j) {
      const bool front = j >= a && j < b, behind = j >= c && j < d;
      NEED(!(front && behind) && (front || behind) == (j >= from && j < to));
    }
  }
  printf("%ld places of shared prefixes\n", checks);
  return 0;
}
