// "ops" module: a token from each row of logits.
//
// With m the row's largest logit and t its temperature a token's weight is w = e^((x - m) / t).  Kept are the k highest logits, of these the fewest
// highest whose weights make p of theirs, of these the ones with w >= q; of equal logits the lower index comes first.  Each cut leaves the
// first ones of the same order, so what is kept is one pair: the last logit and, among its equals, the last index.  The token is then the first kept one in
// the vocabulary's order whose running sum of weights passes u times the sum.
//
// Numbers: which token a draw gives hangs on the last digits of sums of a hundred thousand weights, whatever order they are added in.  So a weight is a
// whole number of 2^-43 (exponent and fraction from 64-bit steps, 2^-42 of the weight; weights below 2^-44 are none), every sum is one of whole
// numbers and the same in any order, and two rows of the same logits give the same token.
//
// A work-group has a row.  The row is read once for its largest logit, and then again, out of the caches, for what the cuts ask for:
//   k up to 512: the k-th of the threads' largest logits is one that at least k tokens reach; those that do -- few more than k -- go to LDS, and the rest
//     happens there.
//   else: a histogram of the row over the weight's logarithm, 64 bins an octave, counts and sums of weights; the bin in which a cut lies
//     is found from it, its tokens go to LDS and give the cut itself.  Another pass adds up what is kept, and the token is found in a sixteenth of a
//     sixteenth of the row.
// Where more tokens meet in a bin than LDS takes (thousands of equal logits, a very high temperature) their logits' digits are counted
// over the whole row instead, eight bits at a time.
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace {
typedef unsigned long long u64;
constexpr int THREADS = 1024, WAVES = 16, CAP = 512, SMALL_K = 512, BINS = 3072;   // (48 octaves)
constexpr int PER = WAVES * CAP / THREADS;                                        // tokens of the list a thread
constexpr uint32_t NONE = 0x007FFFFFu;                                             // the key of -inf: no token

struct Lds {
  double pow2[256];   // 2^(j / 256)
  u64 sum[BINS];
  uint32_t count[BINS];
  uint32_t key[WAVES * CAP], at[WAVES * CAP];
  u64 digit_sum[256];
  uint32_t digit[256];
  u64 part[WAVES];
  int number[WAVES];
  float top[WAVES];
  int where[WAVES];
  u64 found[2];
  int place[4];
};

// Logits in their order as whole numbers; -0 is 0, and what is no number is -inf.
__device__ inline uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x == 0.0f ? 0.0f : x);
  return x == x ? (b & 0x80000000u ? ~b : b | 0x80000000u) : NONE;
}
__device__ inline float logit_of(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k); }

struct Row {
  const float* x;   // (of V logits; the units of four begin `skew` values in front of it, where addresses are multiples of 16)
  int V, skew, units;
  double most, scale;   // the largest logit; 256 log2(e) / t
  bool endless;         // the largest is +inf: tokens of it alone, each of weight 1
};
__device__ inline float4 load(const Row& r, int unit) {
  const int i = 4 * unit - r.skew;
  if (i >= 0 && i + 3 < r.V) return *(const float4*)(r.x + i);
  float4 v;
  float* e = (float*)&v;
#pragma unroll
  for (int j = 0; j < 4; ++j) e[j] = i + j >= 0 && i + j < r.V ? r.x[i + j] : -INFINITY;
  return v;
}
// The weight's logarithm in 1 / 256 of an octave, at least -15360, and what is left of it (in the same, within a half).
__device__ inline int octaves(const Row& r, float x, double& rest) {
  constexpr double MAGIC = 6755399441055744.0;   // 1.5 * 2^52: its last place is 1
  const double y = fmax(((double)x - r.most) * r.scale, -15360.0), k = y + MAGIC;
  rest = y - (k - MAGIC);
  return (int)(uint32_t)__double_as_longlong(k);
}
__device__ inline u64 weight(const Row& r, const double* pow2, float x) {
  if (!(x > -INFINITY)) return 0;
  if (r.endless) return x == INFINITY ? 1ull << 43 : 0;
  double f;
  const int n = octaves(r, x, f);
  // 2^(f / 256) to f^3: what is cut off is 2^-42 at most
  constexpr double A = 0.0027076061740622863, B = 3.665565596910106e-06, C = 3.308302680541371e-09;   // (ln 2 / 256)^i / i!
  const double w = pow2[n & 255] * fma(f, fma(f, fma(f, C, B), A), 1.0);
  return (u64)__double_as_longlong(__builtin_ldexp(w, 43 + (n >> 8)) + 4503599627370496.0) & 0xFFFFFFFFFFFFFull;   // (+ 2^52: rounded to a whole number)
}
__device__ inline int bin(const Row& r, float x) {   // (of a token: 0 for the largest)
  if (r.endless) return x == INFINITY ? 0 : BINS - 1;
  double f;
  return min(-octaves(r, x, f) >> 2, BINS - 1);
}

__device__ inline int wave() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }
__device__ inline int lane() { return threadIdx.x & 63; }
template <class T>
__device__ inline T up_sum(T v) {   // (over the lanes up to this one)
#pragma unroll
  for (int o = 1; o < 64; o *= 2) {
    const T w = __shfl_up(v, o);
    if (lane() >= o) v += w;
  }
  return v;
}
__device__ inline u64 wave_sum(u64 v) {
#pragma unroll
  for (int o = 32; o; o /= 2) v += __shfl_xor(v, o);
  return v;
}
// The sum over the threads in front of this one, and of all.
__device__ inline u64 scan(Lds& s, u64 v, u64& total) {
  const u64 up = up_sum(v);
  __syncthreads();
  if (lane() == 63) s.part[wave()] = up;
  __syncthreads();
  u64 front = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    front += w < wave() ? s.part[w] : 0;
    total += s.part[w];
  }
  return front + up - v;
}
// A wave's units [a, b) in their order, 64 at a time: f(logits of this lane's unit, its first index); lanes behind the end have -inf at V.
template <class F>
__device__ inline void walk(const Row& r, int a, int b, F f) {
  constexpr int N = 4;   // (loads on their way at once)
  for (int u0 = a; u0 < b; u0 += 64 * N) {
    float4 v[N];
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int u = u0 + 64 * k + lane();
      v[k] = u < b ? load(r, u) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
    }
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int u = u0 + 64 * k + lane();
      if (u0 + 64 * k < b) f(v[k], u < b ? 4 * u - r.skew : r.V);
    }
  }
}
// ... each wave its sixteenth of [a, b)
struct Range {
  int a, b;
};
__device__ inline Range share(Range all, int w) {
  const int per = (all.b - all.a + WAVES - 1) / WAVES;
  const int a = min(all.a + w * per, all.b);
  return {a, min(a + per, all.b)};
}

// Of 256 sums, from the last one down, the one in which the running sum reaches `need`: its number in place[0], found[0] the sum in front of it.
// (The sums reach it.)
template <class T>
__device__ inline void pick(Lds& s, const T* sums, T need) {
  __syncthreads();
  if (wave() == 0) {
    T v[4], own = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) own += v[j] = sums[255 - 4 * lane() - j];
    T front = up_sum(own) - own;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (front < need && front + v[j] >= need) {
        s.place[0] = 255 - 4 * lane() - j;
        s.found[0] = front;
      }
      front += v[j];
    }
  }
  __syncthreads();
}

// Tokens in LDS in the vocabulary's order: each wave's run of them one behind the other, PER or fewer to a thread.
struct List {
  uint32_t key[PER];
  int at[PER];
  bool in[PER];
  int n;
};
// The tokens of the row for which f says so; false: there are more than LDS takes.
template <class F>
__device__ inline bool gather(Lds& s, const Row& r, List& l, F f) {
  const Range mine = share({0, r.units}, wave());
  int have = 0;
  __syncthreads();   // (the last list is not looked at any more)
  walk(r, mine.a, mine.b, [&](const float4& v, int i) {
    const float* e = (const float*)&v;
    u64 vote[4];
    int front = have, all = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool yes = e[j] > -INFINITY && f(e[j], i + j);
      vote[j] = __ballot(yes);
      front += __builtin_amdgcn_mbcnt_hi((uint32_t)(vote[j] >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)vote[j], 0));
      all += __popcll(vote[j]);
    }
    if (all == 0) return;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (vote[j] >> lane() & 1) {
        if (front < CAP) {
          s.key[wave() * CAP + front] = key_of(e[j]);
          s.at[wave() * CAP + front] = i + j;
        }
        ++front;
      }
    have += all;
  });
  if (lane() == 0) s.number[wave()] = have;
  __syncthreads();
  bool fits = true;
  int starts[WAVES];
  l.n = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    starts[w] = l.n;
    l.n += s.number[w];
    fits = fits && s.number[w] <= CAP;
  }
  if (!fits) return false;
  const int per = (l.n + THREADS - 1) / THREADS;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int g = threadIdx.x * per + j;
    l.in[j] = j < per && g < l.n;
    l.key[j] = 0;
    l.at[j] = 0;
    if (l.in[j]) {
      int w = 0;
#pragma unroll
      for (int k = 1; k < WAVES; ++k) w = starts[k] <= g ? k : w;
      int from = 0;
#pragma unroll
      for (int k = 1; k < WAVES; ++k) from = k == w ? starts[k] : from;
      l.key[j] = s.key[w * CAP + g - from];
      l.at[j] = s.at[w * CAP + g - from];
    }
  }
  return true;
}

// A cut: tokens above `key` are kept, and those of it up to index `last`.
struct Cut {
  uint32_t key;
  int last;
  __device__ bool keeps(uint32_t k, int i) const { return k > key || (k == key && i <= last); }
};

// The cut behind which the count (or, by weight, the sum of weights) of the tokens that f goes over first reaches `need` -- which all of them together do.
// each(g): g(key, index) for the tokens, in any order; nth(key, n): the index of the n-th token (from 0) of that key.  sum: of the weights that it keeps of these.
template <bool BY_WEIGHT, class E, class N>
__device__ inline Cut select(Lds& s, const Row& r, u64 need, E each, N nth) {
  uint32_t prefix = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    __syncthreads();
    if (threadIdx.x < 256) {
      s.digit[threadIdx.x] = 0;
      s.digit_sum[threadIdx.x] = 0;
    }
    __syncthreads();
    each([&](uint32_t k, int) {
      if (shift < 24 && k >> (shift + 8) != prefix) return;
      if (BY_WEIGHT) atomicAdd(&s.digit_sum[k >> shift & 255], weight(r, s.pow2, logit_of(k)));
      else atomicAdd(&s.digit[k >> shift & 255], 1u);
    });
    if (BY_WEIGHT) pick<u64>(s, s.digit_sum, need);
    else pick<uint32_t>(s, s.digit, (uint32_t)need);
    need -= s.found[0];
    prefix = prefix << 8 | (uint32_t)s.place[0];
    __syncthreads();
  }
  // (all tokens of one key have the same weight, which is not 0 where a sum had to be reached)
  const u64 w = BY_WEIGHT ? weight(r, s.pow2, logit_of(prefix)) : 1;
  return {prefix, nth(prefix, (int)((need + w - 1) / w) - 1)};
}
__device__ inline int list_nth(Lds& s, const List& l, uint32_t key, int n) {
  int own = 0;
#pragma unroll
  for (int j = 0; j < PER; ++j) own += l.in[j] && l.key[j] == key;
  u64 total;
  int front = (int)scan(s, (u64)own, total);
#pragma unroll
  for (int j = 0; j < PER; ++j)
    if (l.in[j] && l.key[j] == key) {
      if (front == n) s.place[1] = l.at[j];
      ++front;
    }
  __syncthreads();
  return s.place[1];
}
template <bool BY_WEIGHT>
__device__ inline Cut list_select(Lds& s, const Row& r, const List& l, u64 need) {
  return select<BY_WEIGHT>(
      s, r, need,
      [&](auto g) {
#pragma unroll
        for (int j = 0; j < PER; ++j)
          if (l.in[j]) g(l.key[j], l.at[j]);
      },
      [&](uint32_t key, int n) { return list_nth(s, l, key, n); });
}
// ... over the row's tokens for which f says so
template <bool BY_WEIGHT, class F>
__device__ inline Cut row_select(Lds& s, const Row& r, u64 need, F f) {
  const Range mine = share({0, r.units}, wave());
  return select<BY_WEIGHT>(
      s, r, need,
      [&](auto g) {
        walk(r, mine.a, mine.b, [&](const float4& v, int i) {
          const float* e = (const float*)&v;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (e[j] > -INFINITY && f(e[j], i + j)) g(key_of(e[j]), i + j);
        });
      },
      [&](uint32_t key, int n) {
        auto count = [&](Range a, auto see) {
          int have = 0;
          walk(r, a.a, a.b, [&](const float4& v, int i) {
            const float* e = (const float*)&v;
            int own = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) own += key_of(e[j]) == key && f(e[j], i + j);
            const int up = up_sum(own);
            see(v, i, have + up - own);
            have += __shfl(up, 63);
          });
          return have;
        };
        const int have = count(mine, [](const float4&, int, int) {});
        __syncthreads();
        if (lane() == 0) s.number[wave()] = have;
        __syncthreads();
        int front = 0;
        for (int w = 0; w < wave(); ++w) front += s.number[w];
        if (front <= n && n < front + have)
          count(mine, [&](const float4& v, int i, int before) {
            const float* e = (const float*)&v;
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (key_of(e[j]) == key && f(e[j], i + j)) {
                if (front + before == n) s.place[1] = i + j;
                ++before;
              }
          });
        __syncthreads();
        return s.place[1];
      });
}

// The point that a draw looks for: below the sum, whatever u is.
__device__ inline double target(float u, u64 sum) {
  const double all = (double)sum, below = __longlong_as_double(__double_as_longlong(all) - 1);
  return fmin(u > 0.0f ? (double)u * all : 0.0, below);
}
}  // namespace

// temp, top_k, top_p, min_p: of each row, or none.  grid T, 1024.
extern "C" __global__ __launch_bounds__(1024) void sample(const float* __restrict__ logits, int ld, int off, int V, const float* __restrict__ temp,
                                                          const int* __restrict__ top_k, const float* __restrict__ top_p, const float* __restrict__ min_p,
                                                          const float* __restrict__ u, int* __restrict__ token, float* __restrict__ prob) {
  __shared__ Lds s;
  const int row = blockIdx.x;
  Row r;
  r.x = logits + (size_t)row * ld + off;
  r.V = V;
  r.skew = (int)((uintptr_t)r.x >> 2 & 3);
  r.units = (V + r.skew + 3) / 4;
  const float t = temp ? temp[row] : 1.0f, draw = u[row], q = min_p ? min_p[row] : 0.0f, p = top_p ? top_p[row] : 1.0f;
  const int k = top_k ? top_k[row] : 0;
  auto answer = [&](int i, float pr) {
    token[row] = i;
    if (prob) prob[row] = pr;
  };

  // ---- the largest logit, and where
  const Range mine = share({0, r.units}, wave());
  float top = -INFINITY;
  int where = 0x7FFFFFFF;
  walk(r, mine.a, mine.b, [&](const float4& v, int i) {
    const float* e = (const float*)&v;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (e[j] > top) { top = e[j]; where = i + j; }
  });
  const float own = top;   // (this thread's)
#pragma unroll
  for (int o = 32; o; o /= 2) {
    const float a = __shfl_xor(top, o);
    const int b = __shfl_xor(where, o);
    if (a > top || (a == top && b < where)) { top = a; where = b; }
  }
  if (lane() == 0) { s.top[wave()] = top; s.where[wave()] = where; }
  if (threadIdx.x < 256) s.pow2[threadIdx.x] = exp2((double)threadIdx.x / 256.0);
  __syncthreads();
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    const float a = s.top[w];
    const int b = s.where[w];
    if (a > top || (a == top && b < where)) { top = a; where = b; }
  }
  if (!(top > -INFINITY)) {   // (nothing can be drawn)
    if (threadIdx.x == 0) answer(-1, 0.0f);
    return;
  }
  if (!(t > 0.0f)) {
    if (threadIdx.x == 0) answer(where, 1.0f);
    return;
  }
  r.most = (double)top;
  r.endless = top == INFINITY;
  r.scale = 369.3299304675746 / (double)t;   // 256 log2(e) / t
  const uint32_t most_key = key_of(top);
  const double least = (double)fminf(fmaxf(q, 0.0f), 1.0f) * 8796093022208.0;   // (2^43; a NaN is 0)
  auto heavy = [&](uint32_t key, u64 w) { return (double)w >= least || key == most_key; };
  const bool by_p = p < 1.0f;
  auto goal = [&](u64 sum) { return (u64)fmax(1.0, ceil((double)fmaxf(p, 0.0f) * (double)sum)); };
  List l;

  // ---- few highest: all in LDS
  bool by_k = k > 0 && k < V;
  if (by_k && k <= SMALL_K) {
    // two digits of the k-th of the threads' largest: at least k tokens reach it
    const uint32_t key = key_of(own);
    uint32_t prefix = 0, need = (uint32_t)k;
#pragma unroll
    for (int shift = 24; shift >= 16; shift -= 8) {
      __syncthreads();
      if (threadIdx.x < 256) s.digit[threadIdx.x] = 0;
      __syncthreads();
      if (shift == 24 || key >> 24 == prefix) atomicAdd(&s.digit[key >> shift & 255], 1u);
      pick<uint32_t>(s, s.digit, need);
      need -= (uint32_t)s.found[0];
      prefix = prefix << 8 | (uint32_t)s.place[0];
    }
    const uint32_t least_key = prefix << 16;
    if (gather(s, r, l, [&](float x, int) { return key_of(x) >= least_key; })) {
      auto keep = [&](const Cut& c) {
#pragma unroll
        for (int j = 0; j < PER; ++j) l.in[j] = l.in[j] && c.keeps(l.key[j], l.at[j]);
      };
      if (l.n > k) keep(list_select<false>(s, r, l, (u64)k));
      u64 w[PER], mine_sum, sum;
      auto weigh = [&] {
        mine_sum = 0;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
          w[j] = l.in[j] ? weight(r, s.pow2, logit_of(l.key[j])) : 0;
          mine_sum += w[j];
        }
      };
      weigh();
      scan(s, mine_sum, sum);
      if (by_p) keep(list_select<true>(s, r, l, goal(sum)));
#pragma unroll
      for (int j = 0; j < PER; ++j) l.in[j] = l.in[j] && heavy(l.key[j], w[j]);
      weigh();
      u64 at = scan(s, mine_sum, sum);
      const double to = target(draw, sum);
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        if (w[j] && (double)at <= to && (double)(at + w[j]) > to) answer(l.at[j], (float)((double)w[j] / (double)sum));
        at += w[j];
      }
      return;
    }
  }

  // ---- the cuts out of a histogram
  Cut cut = {NONE, 0x7FFFFFFF};
  if (by_k || by_p) {
    __syncthreads();
    for (int b = threadIdx.x; b < BINS; b += THREADS) {
      s.sum[b] = 0;
      s.count[b] = 0;
    }
    __syncthreads();
    walk(r, mine.a, mine.b, [&](const float4& v, int) {
      const float* e = (const float*)&v;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (e[j] > -INFINITY) {
          const int b = bin(r, e[j]);
          if (by_k) atomicAdd(&s.count[b], 1u);
          if (by_p && b < BINS - 1) atomicAdd(&s.sum[b], weight(r, s.pow2, e[j]));
        }
    });
    __syncthreads();
    // the bin in which a running sum over the bins reaches `need` (found[1]: the sum in front of it, found[0] of all); BINS: none does
    auto reach = [&](auto value, u64 need) {
      u64 v[BINS / THREADS], mine_sum = 0, total;
#pragma unroll
      for (int j = 0; j < BINS / THREADS; ++j) mine_sum += v[j] = value(threadIdx.x * (BINS / THREADS) + j);
      if (threadIdx.x == 0) s.place[2] = BINS;
      u64 front = scan(s, mine_sum, total);
#pragma unroll
      for (int j = 0; j < BINS / THREADS; ++j) {
        if (front < need && front + v[j] >= need) {
          s.place[2] = threadIdx.x * (BINS / THREADS) + j;
          s.found[1] = front;
        }
        front += v[j];
      }
      __syncthreads();
      const int b = s.place[2];
      __syncthreads();
      return b;
    };
    auto sums = [&](int to) {   // of the bins in front of `to`
      u64 v = 0, total;
      for (int b = threadIdx.x; b < to; b += THREADS) v += s.sum[b];
      scan(s, v, total);
      return total;
    };
    int bk = BINS;
    bool listed = false;   // the list has bin bk
    u64 rest = 0;          // the sum of weights that the cut by k leaves of bk
    if (by_k) {
      bk = reach([&](int b) { return (u64)s.count[b]; }, (u64)k);
      if (bk >= BINS - 1) {
        by_k = false;   // (all tokens, or all that have a weight)
        bk = BINS;
      } else {
        const u64 need = (u64)k - s.found[1];
        auto there = [&](float x, int) { return bin(r, x) == bk; };
        listed = gather(s, r, l, there);
        cut = listed ? list_select<false>(s, r, l, need) : row_select<false>(s, r, need, there);
        if (by_p) {
          u64 v = 0;
          if (listed) {
#pragma unroll
            for (int j = 0; j < PER; ++j)
              if (l.in[j]) {
                l.in[j] = cut.keeps(l.key[j], l.at[j]);
                if (l.in[j]) v += weight(r, s.pow2, logit_of(l.key[j]));
              }
          } else {
            walk(r, mine.a, mine.b, [&](const float4& x, int i) {
              const float* e = (const float*)&x;
#pragma unroll
              for (int j = 0; j < 4; ++j)
                if (e[j] > -INFINITY && there(e[j], 0) && cut.keeps(key_of(e[j]), i + j)) v += weight(r, s.pow2, e[j]);
            });
          }
          scan(s, v, rest);
        }
      }
    }
    if (by_p) {
      const u64 front = sums(bk), need = goal(front + rest);
      const int bp = need <= front ? reach([&](int b) { return b < bk ? s.sum[b] : 0ull; }, need) : bk;
      if (bp < bk) {
        const u64 before = s.found[1];
        auto there = [&](float x, int) { return bin(r, x) == bp; };
        cut = gather(s, r, l, there) ? list_select<true>(s, r, l, need - before) : row_select<true>(s, r, need - before, there);
      } else if (by_k) {   // (the cut by p lies among what the one by k leaves of its bin)
        const Cut last = cut;
        cut = listed ? list_select<true>(s, r, l, need - front)
                     : row_select<true>(s, r, need - front, [&](float x, int i) { return bin(r, x) == bk && last.keeps(key_of(x), i); });
      }
    }
  }

  // ---- what is kept, added up in the vocabulary's order; the sixteenth of the row in which the sum passes the draw's, a sixteenth of that, and the
  // token
  auto kept = [&](float x, int i) -> u64 {
    const uint32_t key = key_of(x);
    if (key <= NONE || !cut.keeps(key, i)) return 0;
    const u64 w = weight(r, s.pow2, x);
    return heavy(key, w) ? w : 0;
  };
  Range all = {0, r.units};
  u64 before = 0, sum = 0;
  double to = 0.0;
  for (int level = 0; level < 2; ++level) {
    const Range part = share(all, wave());
    u64 v = 0;
    walk(r, part.a, part.b, [&](const float4& x, int i) {
      const float* e = (const float*)&x;
#pragma unroll
      for (int j = 0; j < 4; ++j) v += kept(e[j], i + j);
    });
    v = wave_sum(v);
    __syncthreads();
    if (lane() == 0) s.part[wave()] = v;
    __syncthreads();
    if (level == 0) {
      for (int w = 0; w < WAVES; ++w) sum += s.part[w];
      to = target(draw, sum);
    }
    int w = 0;
    for (; w < WAVES - 1 && !((double)(before + s.part[w]) > to); ++w) before += s.part[w];
    all = share(all, w);
  }
  if (wave() == 0) {
    bool done = false;
    walk(r, all.a, all.b, [&](const float4& x, int i) {
      if (done) return;
      const float* e = (const float*)&x;
      u64 w[4], own_sum = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) own_sum += w[j] = kept(e[j], i + j);
      const u64 up = up_sum(own_sum);
      u64 at = before + up - own_sum;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (w[j] && (double)at <= to && (double)(at + w[j]) > to) answer(i + j, (float)((double)w[j] / (double)sum));
        at += w[j];
      }
      before += __shfl(up, 63);
      done = (double)before > to;
    });
  }
}
