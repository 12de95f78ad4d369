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
//   k up to 960: the k-th of the threads' largest logits is one that at least k tokens reach; those that do -- few more than k -- go to LDS, and the rest
//     happens there.
//   else: a histogram of the row over the weight's logarithm, 64 bins an octave, counts and sums of weights; the bin in which a cut lies
//     is found from it, its tokens go to LDS and give the cut itself.  Another pass adds up what is kept, and the token is found in a sixteenth of a
//     sixteenth of the row.
// Of up to 256 listed tokens the cut is found by the place of each among them; of more their digits are counted, as below.  Where all that is kept is listed
// the token comes out of the list.
// Where more tokens meet in a bin than LDS takes (thousands of equal logits, a very high temperature) their logits' digits are counted
// over the whole row instead, eight bits at a time.
// Bound: the 64-bit steps of the weights, some twenty instructions a token each time that they are wanted -- once for the histogram, once for the sums --, and for
// few rows the steps themselves, of which none begins before the last one's sums have met.  A row is read from HBM once and from the caches after that.
// Measured, 256 rows of 151936: the largest logit 27 us (5.7 TB/s), by k and p 60, drawn among all 74, by min_p 60, by p 139; 37 rows of 32001 of all kinds 36; one row of
// 151936 by sixteen work-groups, by k and p 26 us, by p 34; 16 bytes of scratch a lane in sample and sample_draw.  A cut in rows that are almost flat (a temperature of 1000) takes 560.
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace {
typedef unsigned long long u64;
constexpr int THREADS = 1024, WAVES = 16, LIST = 512, BINS = 3 * THREADS;   // (48 octaves)
// The highest k that is looked for among the threads' largest logits (of 1024: the nearer to them all, the more tokens reach the k-th).  Measured, us, this
// way / by the histogram: 256 rows of 151936, k = 512 65 / 175, 960 80 / 173; with a cut by p behind it 73 / 190, 91 / 189; one row, k = 960 37 / 35, with p 46 / 116.
constexpr int SMALL_K = 960;
// Listed tokens of which each is compared with all others.  37 rows of 32001, by k and p: k = 50 21 us (by digits 36), k = 200, 220 tokens, 32, k = 256, which go by
// digits, 33.  (Going down the bits of up to 512 in one wave's registers: 42 for 100, 58 for 400.)
constexpr int FEW = 256;
// Kept logits of 256 that are put together before their weights are worked out.  Measured, us, all where they lie / put together: 256 rows of 151936 cut by
// min_p 75 / 60, one row of 32001 by p 36 / 33, one of 151936 by k = 2000 and p 135 / 116; rows of which half is kept 138 / 139 (of which all is: where they lie,
// 74; with the votes 80).
constexpr int SPARSE = 128;
constexpr uint32_t NONE = 0x007FFFFFu;                                             // the key of -inf: no token

// CAP: tokens of a wave that the list takes.
template <int CAP_>
struct LdsOf {
  static constexpr int CAP = CAP_;
  double pow2[16];   // 2^(43 + j / 16)
  u64 sum[BINS];
  uint32_t count[BINS];
  uint32_t key[WAVES * CAP], at[WAVES * CAP];   // the list: a run of each wave's, in the row's order
  uint32_t few_key[FEW], few_at[FEW];           // ... of few members, the runs behind one another
  u64 few_weight[FEW];
  float held[WAVES * (64 + SPARSE)];            // logits that are kept, a wave's on their way to their weights
  u64 digit_sum[256];
  uint32_t digit[256];
  u64 part[WAVES], kept[WAVES];
  int number[WAVES], equal[WAVES];
  float top[WAVES];
  int where[WAVES];
  u64 found[3];
  uint32_t place[3];
};
typedef LdsOf<LIST> Lds;

// Logits in their order as whole numbers; -0 is 0, and what is no number is -inf.
__device__ inline uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x == 0.0f ? 0.0f : x);
  return x == x ? (b & 0x80000000u ? ~b : b | 0x80000000u) : NONE;
}
__device__ inline float logit_of(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k); }

struct Row {
  const float* x;   // (of V logits; the units of four begin `skew` values in front of it, where addresses are multiples of 16)
  int V, skew, units;
  double most, scale;   // the largest logit, 16 log2(e) / t; where it is +inf, above all finite ones, whose weights are then 0
};
__device__ inline float4 load(const Row& r, int unit) {
  const int i = 4 * unit - r.skew;
  if (i >= 0 && i + 3 < r.V) return *(const float4*)(r.x + i);
  float4 v;
  float* e = (float*)&v;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    e[j] = r.x[min(max(i + j, 0), r.V - 1)];
    e[j] = (i + j >= 0) & (i + j < r.V) ? e[j] : -INFINITY;
  }
  return v;
}
// A weight's logarithm in 1 / 16 of an octave, down to 60 octaves -- of -inf and of what is no number --, its whole part and the rest of it, within a half.
struct Octaves {
  double y, rest;
  int n;
};
__device__ inline Octaves octaves(const Row& r, float x) {
  constexpr double MAGIC = 6755399441055744.0;   // 1.5 * 2^52: its last place is 1
  Octaves o;
  o.y = fmin(fmax(((double)x - r.most) * r.scale, -960.0), 0.0);
  const double k = o.y + MAGIC;
  o.n = __double2loint(k);
  o.rest = o.y - (k - MAGIC);
  return o;
}
__device__ inline u64 weight_at(const double* pow2, const Octaves& o) {
  // 2^(f / 16) to f^5: what is cut off is 2^-42 at most.  (Sixteen powers: no two of them lie in one bank of the LDS.)
  constexpr double A = 0.04332169878499658, B = 0.0009383847928089871, C = 1.3550807779497455e-05, D = 1.467610032291943e-07, E = 1.271587195055813e-09;   // (ln 2 / 16)^i / i!
  const double f = o.rest, p = fma(f, fma(f, fma(f, fma(f, fma(f, E, D), C), B), A), 1.0), t = pow2[o.n & 15];
  const double w = fma(__hiloint2double(__double2hiint(t) + ((o.n >> 4) << 20), __double2loint(t)), p, 4503599627370496.0);   // (+ 2^52: rounded to a whole number)
  return (u64)(uint32_t)(__double2hiint(w) & 0xFFFFF) << 32 | (uint32_t)__double2loint(w);
}
__device__ inline u64 weight(const Row& r, const double* pow2, float x) {
  return weight_at(pow2, octaves(r, x));
}
// 64 bins an octave: of a token, 0 for the largest, the last one of all that have no weight.
__device__ inline int bin_at(const Octaves& o) { return min((int)(o.y * -4.0), BINS - 1); }
__device__ inline int bin(const Row& r, float x) {
  return bin_at(octaves(r, x));
}

__device__ inline int wave() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }
__device__ inline int lane() { return threadIdx.x & 63; }
template <int DPP, int ROWS>
__device__ inline uint32_t moved(uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, DPP, ROWS, 0xF, false); }
template <int DPP, int ROWS>
__device__ inline u64 moved(u64 v) { return (u64)moved<DPP, ROWS>((uint32_t)(v >> 32)) << 32 | moved<DPP, ROWS>((uint32_t)v); }
// The sum over the lanes up to this one: in each row of sixteen, then the rows' ends.
template <class T>
__device__ inline T up_sum(T v) {
  v += moved<0x111, 0xF>(v);
  v += moved<0x112, 0xF>(v);
  v += moved<0x114, 0xF>(v);
  v += moved<0x118, 0xF>(v);
  v += moved<0x142, 0xA>(v);   // (lane 15 to the next row, 47 likewise)
  v += moved<0x143, 0xC>(v);   // (lane 31 to the second half)
  return v;
}
__device__ inline u64 wave_sum(u64 v) {
  v = up_sum(v);
  return (u64)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), 63) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
// The sum over the threads in front of this one, and of all.
template <class S>
__device__ inline u64 scan(S& s, u64 v, u64& total) {
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
// N: loads on their way at once.
template <int N, class F>
__device__ inline void walk(const Row& r, int a, int b, F f) {
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

// A cut: tokens above `key` are kept, and those of it up to index `last`.
struct Cut {
  uint32_t key;
  int last;
  __device__ bool keeps(uint32_t k, int i) const { return (k > key) | ((k == key) & (i <= last)); }
};
__device__ inline Cut higher(const Cut& a, const Cut& b) { return a.key > b.key || (a.key == b.key && a.last <= b.last) ? a : b; }
// What lanes of a wave have written to LDS is there for its other lanes behind this, and what they have read may be written over.
__device__ inline void met() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}
// Tokens of a row whose keys lie in [lo, hi] and that `within` keeps; listed: in LDS.
struct Members {
  uint32_t lo, hi;
  Cut within;
  bool listed;
  __device__ bool has(uint32_t k, int i) const { return (k >= lo) & (k <= hi) & within.keeps(k, i); }
};
// Over units of the row: its members (of a range; `within` everything) to LDS -- false: there are more than it takes --, and where `add` the weights of those that
// `floor` keeps added up, each wave's to part[] (where it keeps everything there are no members).
template <class S>
__device__ inline bool pass(S& s, const Row& r, const Range& all, const Members& m, bool add, const Cut& floor) {
  constexpr int CAP = S::CAP;
  const Range mine = share(all, wave());
  const bool any = m.lo <= m.hi;
  const float lo = any ? logit_of(m.lo) : INFINITY, hi = any ? logit_of(m.hi) : -INFINITY, edge = logit_of(floor.key);
  int have = 0;
  u64 sum = 0;
  __syncthreads();   // (the last list is not looked at any more)
  auto members = [&](const float4& v, int i) {
    const float* e = (const float*)&v;
    bool some = false;
#pragma unroll
    for (int j = 0; j < 4; ++j) some |= (e[j] >= lo) & (e[j] <= hi);
    if (!__any(some)) return;
    u64 vote[4];
    int front = have;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      vote[j] = __ballot((e[j] >= lo) & (e[j] <= hi));
      front += __builtin_amdgcn_mbcnt_hi((uint32_t)(vote[j] >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)vote[j], 0));
      have += __popcll(vote[j]);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (vote[j] >> lane() & 1) {
        if (front < CAP) {
          s.key[wave() * CAP + front] = key_of(e[j]);
          s.at[wave() * CAP + front] = i + j;
        }
        ++front;
      }
  };
  if (!add) {
    walk<8>(r, mine.a, mine.b, members);
  } else {
    // Where few are kept of 256 they are put together first, so that a wave works out the weights of 64 of them at a time.
    float* const held = s.held + wave() * (64 + SPARSE);
    const bool every = floor.key <= NONE;
    int pending = 0;
    walk<4>(r, mine.a, mine.b, [&](const float4& v, int i) {
      const float* e = (const float*)&v;
      bool keep[4];
      u64 vote[4];
      int n = 0;
      if (every) {
#pragma unroll
        for (int j = 0; j < 4; ++j) sum += weight(r, s.pow2, e[j]);
        return;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        keep[j] = (e[j] > edge) | ((e[j] == edge) & (i + j <= floor.last));
        vote[j] = __ballot(keep[j]);
        n += __popcll(vote[j]);
      }
      if (n > SPARSE) {
#pragma unroll
        for (int j = 0; j < 4; ++j) sum += weight(r, s.pow2, keep[j] ? e[j] : -INFINITY);   // (of weight 0)
      } else if (n) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int at = pending + __builtin_amdgcn_mbcnt_hi((uint32_t)(vote[j] >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)vote[j], 0));
          if (keep[j]) held[at] = e[j];
          pending += __popcll(vote[j]);
        }
        met();
        while (pending >= 64) {
          pending -= 64;
          sum += weight(r, s.pow2, held[pending + lane()]);
        }
        met();
      }
      if (any) members(v, i);
    });
    if (pending) sum += weight(r, s.pow2, lane() < pending ? held[lane()] : -INFINITY);
    sum = wave_sum(sum);
  }
  if (lane() == 0) {
    s.number[wave()] = have;
    s.part[wave()] = sum;
  }
  __syncthreads();
  bool fits = true;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) fits = fits && s.number[w] <= CAP;
  return fits;
}
// g(key, index) for the members, this wave's share of them in the row's order, 64 at a time; lanes without one: key 0.
template <class G>
__device__ inline void each(Lds& s, const Row& r, const Members& m, G g) {
  if (m.listed) {
    const int n = s.number[wave()];
    for (int p0 = 0; p0 < n; p0 += 64) {
      const int p = min(p0 + lane(), n - 1);
      const uint32_t k = s.key[wave() * LIST + p];
      const int i = s.at[wave() * LIST + p];
      g(p0 + lane() < n && m.has(k, i) ? k : 0u, i);
    }
    return;
  }
  const Range mine = share({0, r.units}, wave());
  auto value = [&](int u0) {   // (a value a lane, of sixteen units)
    const int u = u0 + (lane() >> 2), i = 4 * u + (lane() & 3) - r.skew;
    return u < mine.b && i >= 0 && i < r.V ? r.x[i] : -INFINITY;
  };
  float x[4] = {value(mine.a), value(mine.a + 16), value(mine.a + 32), value(mine.a + 48)};   // (four of them on their way)
  for (int u0 = mine.a; u0 < mine.b; u0 += 16) {
    const uint32_t k = key_of(x[0]);
    const int i = 4 * (u0 + (lane() >> 2)) + (lane() & 3) - r.skew;
    x[0] = x[1];
    x[1] = x[2];
    x[2] = x[3];
    x[3] = value(u0 + 64);
    g(k > NONE && m.has(k, i) ? k : 0u, i);
  }
}
// The cut behind which the count (by_weight: the sum of weights) of the members first reaches `need` -- which all of them together do -- going down from the
// highest; kept: the sum of weights that it leaves of them.
__device__ inline Cut select(Lds& s, const Row& r, const Members& m, bool by_weight, u64 need, u64& kept) {
  const uint32_t differ = m.lo ^ m.hi;
  int all = 0, run = 0;
  for (int w = 0; w < WAVES; ++w) {
    run = w == wave() ? all : run;
    all += s.number[w];
  }
  if (m.listed && all <= FEW) {
    if (threadIdx.x < FEW) {
      s.digit[threadIdx.x] = 0;
      s.digit_sum[threadIdx.x] = 0;
    }
    for (int p = lane(); p < s.number[wave()]; p += 64) {
      const uint32_t k = s.key[wave() * LIST + p];
      const int i = s.at[wave() * LIST + p];
      const bool has = m.has(k, i);
      s.few_key[run + p] = has ? k : 0;
      s.few_weight[run + p] = has ? weight(r, s.pow2, logit_of(k)) : 0;
      s.few_at[run + p] = i;
    }
    __syncthreads();
    // how many members lie in front of each, and what they weigh: four waves for 64 of them, each against a fourth of all
    constexpr int EACH = WAVES * 64 / FEW;
    const int mine = wave() / EACH * 64 + lane();
    if (wave() / EACH * 64 < all) {
      const uint32_t key = mine < all ? s.few_key[mine] : 0;
      uint32_t rank = 0;
      u64 front = 0;
      for (int p = wave() % EACH; p < all; p += EACH) {
        const uint32_t k = s.few_key[p];
        const bool before = (k > key) | ((k == key) & (p < mine));
        rank += before ? 1 : 0;
        front += before ? s.few_weight[p] : 0;
      }
      if (key && rank) {
        atomicAdd(&s.digit[mine], rank);
        atomicAdd(&s.digit_sum[mine], front);
      }
    }
    __syncthreads();
    if ((int)threadIdx.x < all) {   // (FEW at most)
      const uint32_t key = s.few_key[threadIdx.x], rank = s.digit[threadIdx.x];
      const u64 w = s.few_weight[threadIdx.x], front = s.digit_sum[threadIdx.x];
      if (key && (by_weight ? front < need && front + w >= need : rank == need - 1)) {
        s.place[0] = key;
        s.place[1] = s.few_at[threadIdx.x];
        s.found[0] = front + w;
      }
    }
    __syncthreads();
    kept = s.found[0];
    return {s.place[0], (int)s.place[1]};
  }
  int shift = differ ? (31 - __clz((int)differ)) / 8 * 8 : 0;
  uint32_t prefix = shift == 24 ? 0 : m.lo >> (shift + 8);
  kept = 0;
  for (; shift >= 0; shift -= 8) {
    __syncthreads();
    if (threadIdx.x < 256) {
      s.digit[threadIdx.x] = 0;
      s.digit_sum[threadIdx.x] = 0;
    }
    __syncthreads();
    each(s, r, m, [&](uint32_t k, int) {
      if (k == 0 || (shift < 24 && k >> (shift + 8) != prefix)) return;
      atomicAdd(&s.digit_sum[k >> shift & 255], weight(r, s.pow2, logit_of(k)));
      atomicAdd(&s.digit[k >> shift & 255], 1u);
    });
    __syncthreads();
    // the digit in which the running sum, from 255 down, reaches what is needed
    if (wave() == 0) {
      u64 v[4], w[4], own = 0, own_w = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int d = 255 - 4 * lane() - j;
        w[j] = s.digit_sum[d];
        v[j] = by_weight ? w[j] : s.digit[d];
        own += v[j];
        own_w += w[j];
      }
      u64 front = up_sum(own) - own, front_w = up_sum(own_w) - own_w;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (front < need && front + v[j] >= need) {
          s.place[0] = (uint32_t)(255 - 4 * lane() - j);
          s.found[0] = front;
          s.found[1] = front_w;
        }
        front += v[j];
        front_w += w[j];
      }
    }
    __syncthreads();
    need -= s.found[0];
    kept += s.found[1];
    prefix = prefix << 8 | s.place[0];
  }
  // Tokens of one logit have one weight (not 0, where a sum had to be reached): so many of the first ones.
  const u64 w = weight(r, s.pow2, logit_of(prefix));
  const int n = by_weight ? (int)((need + w - 1) / w) : (int)need;
  kept += (u64)n * w;
  int have = 0;
  each(s, r, m, [&](uint32_t k, int) { have += __popcll(__ballot(k == prefix)); });
  if (lane() == 0) s.equal[wave()] = have;
  __syncthreads();
  int front = 0;
  for (int v = 0; v < wave(); ++v) front += s.equal[v];
  if (front < n && n <= front + have)
    each(s, r, m, [&](uint32_t k, int i) {
      const u64 vote = __ballot(k == prefix);
      const int mine = front + __builtin_amdgcn_mbcnt_hi((uint32_t)(vote >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)vote, 0));
      if (k == prefix && mine == n - 1) s.place[1] = i;
      front += __popcll(vote);
    });
  __syncthreads();
  return {prefix, (int)s.place[1]};
}
// The lowest key up to the largest for whose logit f holds, which it does for all above it.
template <class F>
__device__ inline uint32_t lowest(const Row& r, F f) {
  uint32_t lo = NONE + 1, hi = key_of((float)r.most);
#pragma unroll 1
  while (lo < hi) {   // (64 keys of the range at a time)
    const uint32_t k = lo + (uint32_t)((u64)(hi - lo) * lane() >> 6);
    const u64 vote = __ballot(f(logit_of(k)));
    const int first = vote ? __ffsll((long long)vote) - 1 : 64;
    const uint32_t below = __shfl(k, max(first - 1, 0)) + 1;
    hi = first < 64 ? __shfl(k, min(first, 63)) : hi;
    lo = first > 0 ? below : hi;
  }
  return __builtin_amdgcn_readfirstlane(lo);
}

// The point that a draw looks for: below the sum, whatever u is.
__device__ inline double target(float u, u64 sum) {
  const double all = (double)sum, below = __longlong_as_double(__double_as_longlong(all) - 1);
  return fmin(u > 0.0f ? (double)u * all : 0.0, below);
}

// What a row is drawn by.
struct Form {
  float t, draw, q, p;
  int k;
  __device__ bool by_k(int V) const { return k > 0 && k < V; }
  __device__ bool by_p() const { return p < 1.0f; }
  __device__ u64 goal(u64 sum) const { return (u64)fmax(1.0, ceil((double)fmaxf(p, 0.0f) * (double)sum)); }
};
#define SAMPLE_ARGS                                                                                                                                     \
  const float *__restrict__ logits, int ld, int off, int V, const float *__restrict__ temp, const int *__restrict__ top_k,                              \
      const float *__restrict__ top_p, const float *__restrict__ min_p, const float *__restrict__ u, int *__restrict__ token, float *__restrict__ prob
__device__ inline Row row_of(const float* logits, int ld, int off, int V, int row) {
  Row r;
  r.x = logits + (size_t)row * ld + off;
  r.V = V;
  r.skew = (int)((uintptr_t)r.x >> 2 & 3);
  r.units = (V + r.skew + 3) / 4;
  r.most = r.scale = 0.0;
  return r;
}
__device__ inline Form form_of(const float* temp, const int* top_k, const float* top_p, const float* min_p, const float* u, int row) {
  return {temp ? temp[row] : 1.0f, u[row], min_p ? min_p[row] : 0.0f, top_p ? top_p[row] : 1.0f, top_k ? top_k[row] : 0};
}
__device__ inline void measure(Row& r, float top, float t) {
  r.most = top == INFINITY ? 1e300 : (double)top;
  r.scale = fmax(23.083120654223414 / (double)t, top == INFINITY ? 1e-200 : 0.0);   // 16 log2(e) / t
}
__device__ inline void first_of(float& top, int& where, float a, int b) {
  if (a > top || (a == top && b < where)) { top = a; where = b; }
}
// The largest logit of some units and its first place, for all threads; own: this thread's.
template <class S>
__device__ inline void find_top(S& s, const Row& r, const Range& all, float& top, int& where, float& own) {
  const Range mine = share(all, wave());
  top = -INFINITY;
  where = 0x7FFFFFFF;
  walk<8>(r, mine.a, mine.b, [&](const float4& v, int i) {
    const float* e = (const float*)&v;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (e[j] > top) { top = e[j]; where = i + j; }
  });
  own = top;
#pragma unroll
  for (int o = 32; o; o /= 2) first_of(top, where, __shfl_xor(top, o), __shfl_xor(where, o));
  if (lane() == 0) { s.top[wave()] = top; s.where[wave()] = where; }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < WAVES; ++w) first_of(top, where, s.top[w], s.where[w]);
}
template <class S>
__device__ inline void powers(S& s) {
  if (threadIdx.x < 16) s.pow2[threadIdx.x] = exp2(43.0 + threadIdx.x / 16.0);
}
// A key that at least k tokens reach, out of the threads' largest logits: two digits of the k-th of them.
template <class S>
__device__ inline uint32_t reached(S& s, float own, int k) {
  const uint32_t key = key_of(own);
  uint32_t prefix = 0, left = (uint32_t)k;
#pragma unroll 1
  for (int shift = 24; shift >= 16; shift -= 8) {
    __syncthreads();
    if (threadIdx.x < 256) s.digit[threadIdx.x] = 0;
    __syncthreads();
    if (shift == 24 || key >> 24 == prefix) atomicAdd(&s.digit[key >> shift & 255], 1u);
    __syncthreads();
    if (wave() == 0) {
      uint32_t v[4], sum = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) sum += v[j] = s.digit[255 - 4 * lane() - j];
      uint32_t above = up_sum(sum) - sum;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (above < left && above + v[j] >= left) {
          s.place[0] = (uint32_t)(255 - 4 * lane() - j);
          s.found[0] = above;
        }
        above += v[j];
      }
    }
    __syncthreads();
    left -= (uint32_t)s.found[0];
    prefix = prefix << 8 | s.place[0];
  }
  __syncthreads();
  return max(prefix << 16, NONE + 1);
}
// Counts and sums of weights of some units by bins.
template <class S>
__device__ inline void histogram(S& s, const Row& r, const Range& all, bool by_k, bool by_p) {
  __syncthreads();
  for (int b = threadIdx.x; b < BINS; b += THREADS) {
    s.sum[b] = 0;
    s.count[b] = 0;
  }
  __syncthreads();
  const Range mine = share(all, wave());
  walk<4>(r, mine.a, mine.b, [&](const float4& v, int) {
    const float* e = (const float*)&v;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const Octaves o = octaves(r, e[j]);
      const int b = bin_at(o);
      const u64 w = weight_at(s.pow2, o);
      if (by_k && e[j] > -INFINITY) atomicAdd(&s.count[b], 1u);
      if (by_p && w) atomicAdd(&s.sum[b], w);
    }
  });
  __syncthreads();
}
// The bin in which the running sum of counts, or of the weights of the bins in front of bk (where they and `rest` make p of their sum), reaches what is
// needed -- BINS: none --; need: what is left of that behind `front`, the sum in front of it.
template <class S>
__device__ inline int reach(S& s, const Form& f, bool by_weight, int bk, u64 rest, u64& need, u64& front) {
  constexpr int B = BINS / THREADS;
  u64 v[B], mine_sum = 0, total;
#pragma unroll
  for (int j = 0; j < B; ++j) {
    const int b = threadIdx.x * B + j;
    mine_sum += v[j] = !by_weight ? s.count[b] : b < bk ? s.sum[b] : 0;
  }
  u64 up = scan(s, mine_sum, total);
  need = by_weight ? f.goal(total + rest) : (u64)f.k;
  if (threadIdx.x == 0) s.place[2] = (uint32_t)BINS;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < B; ++j) {
    if (up < need && up + v[j] >= need) {
      s.place[2] = threadIdx.x * B + j;
      s.found[2] = up;
    }
    up += v[j];
  }
  __syncthreads();
  const int b = (int)s.place[2];
  front = b < BINS ? s.found[2] : total;
  need -= min(need, front);
  return b;
}
// The members of bin b.
__device__ inline Members members_of(const Row& r, int b, uint32_t most_key) {
  uint32_t edge[2];   // (where the bin begins, and the one in front of it)
#pragma unroll 1
  for (int j = 0; j < 2; ++j) edge[j] = lowest(r, [&](float x) { return bin(r, x) <= b - j; });
  return {edge[0], b ? edge[1] - 1 : most_key, {NONE, 0x7FFFFFFF}, true};
}
// min_p as a cut: the lowest logit whose weight is no less than q of the largest's, 2^43.
template <class S>
__device__ inline Cut least_of(S& s, const Row& r, float q) {
  const u64 fewest = (u64)ceil((double)fminf(fmaxf(q, 0.0f), 1.0f) * 8796093022208.0);   // (a NaN is 0)
  return {fewest ? lowest(r, [&](float x) { return weight(r, s.pow2, x) >= fewest; }) : NONE, 0x7FFFFFFF};
}
// One wave finds the token in some units: `before` is the sum in front of them.
template <class S>
__device__ inline void find(S& s, const Row& r, const Range& all, const Cut& cut, u64 before, u64 sum, double to, int* token, float* prob) {
  bool done = false;
  walk<4>(r, all.a, all.b, [&](const float4& x, int i) {
    if (done) return;
    const float* e = (const float*)&x;
    u64 w[4], own_sum = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) own_sum += w[j] = weight(r, s.pow2, cut.keeps(key_of(e[j]), i + j) ? e[j] : -INFINITY);
    const u64 up = up_sum(own_sum);
    u64 at = before + up - own_sum;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (w[j] && (double)at <= to && (double)(at + w[j]) > to) {
        *token = i + j;
        if (prob) *prob = (float)((double)w[j] / (double)sum);
      }
      at += w[j];
    }
    before += __shfl(up, 63);
    done = (double)before > to;
  });
}
// The token where all that is kept is listed.
__device__ inline void from_list(Lds& s, const Row& r, const Cut& cut, float draw, int* token, float* prob) {
  const int n = s.number[wave()];
  auto entry = [&](int p, int& i) {   // (its weight)
    if (p >= n) return (u64)0;
    const uint32_t k = s.key[wave() * LIST + p];
    i = s.at[wave() * LIST + p];
    return cut.keeps(k, i) ? weight(r, s.pow2, logit_of(k)) : 0;
  };
  u64 own = 0;
  int i = 0;
  for (int p = lane(); p < n; p += 64) own += entry(p, i);
  own = wave_sum(own);
  __syncthreads();
  if (lane() == 0) s.kept[wave()] = own;
  __syncthreads();
  u64 sum = 0, at = 0;
  for (int w = 0; w < WAVES; ++w) {
    at += w < wave() ? s.kept[w] : 0;
    sum += s.kept[w];
  }
  const double to = target(draw, sum);
  if ((double)at > to || !((double)(at + own) > to)) return;
  for (int p0 = 0; p0 < n; p0 += 64) {
    const u64 w = entry(p0 + lane(), i), up = up_sum(w), front = at + up - w;
    if (w && (double)front <= to && (double)(front + w) > to) {
      *token = i;
      if (prob) *prob = (float)((double)w / (double)sum);
    }
    at += __shfl(up, 63);
  }
}
// A row by one work-group.
__device__ __forceinline__ void one_row(Lds& s, Row r, const Form& f, int* token, float* prob) {
  const Range whole = {0, r.units};
  float top, own;
  int where;
  powers(s);
  find_top(s, r, whole, top, where, own);
  if (!(top > -INFINITY) || !(f.t > 0.0f)) {   // (nothing can be drawn; greedy)
    if (threadIdx.x == 0) {
      *token = top > -INFINITY ? where : -1;
      if (prob) *prob = top > -INFINITY ? 1.0f : 0.0f;
    }
    return;
  }
  measure(r, top, f.t);
  const uint32_t most_key = key_of(top);
  const Cut least = least_of(s, r, f.q);

  // ---- the cuts, one within the other: by k out of a list of few (step 0) or out of the histogram (1), by p (2)
  const bool by_p = f.by_p();
  bool by_k = f.by_k(r.V), small = false, counted = false, added = false;
  Cut cut = {NONE, 0x7FFFFFFF};
  Members m = {1, 0, cut, true};
  u64 front = 0, rest = 0;   // the weights in front of the members, and of those of them that the cut by k keeps
  int bk = BINS;             // the bin of the cut by k
#pragma unroll 1
  for (int step = 0; step < 3; ++step) {
    if (step == 2 ? !by_p : !by_k || small) continue;
    if (step == 0 && f.k > SMALL_K) continue;
    u64 need = (u64)f.k;
    bool look = true;   // (other members than the list has)
    if (step == 0) {
      m.lo = reached(s, own, f.k);
      m.hi = most_key;
    } else if (step == 2 && small) {
      need = f.goal(rest);
      look = false;
      m.within = cut;
    } else {
      if (!counted) histogram(s, r, whole, by_k, by_p);
      counted = true;
      const int b = reach(s, f, step == 2, bk, rest, need, front);
      if (step == 1 && b >= BINS - 1) {   // (all tokens, or all that have a weight)
        by_k = false;
        continue;
      }
      if (step == 1) bk = b;
      look = b < BINS;
      if (look) m = members_of(r, b, most_key);
      else m.within = cut;   // (the cut by p lies among what the one by k leaves of its bin)
    }
    if (look) {
      added = step == 2 || !by_p;   // (the last cut: what lies above its members is added up on the way)
      m.listed = pass(s, r, whole, m, added && step > 0, higher({m.hi, -1}, least));
      added = added && m.listed;
      if (step == 0 && !m.listed) continue;
    }
    if (step == 0) {
      small = added = true;   // (nothing lies above these members)
      int n = 0;
      for (int w = 0; w < WAVES; ++w) n += s.number[w];
      need = min(need, (u64)n);
    }
    cut = select(s, r, m, step == 2, need, rest);
  }

  cut = higher(cut, least);
  if (small) {
    from_list(s, r, cut, f.draw, token, prob);
    return;
  }
  // ---- the sum of what is kept, of each wave's sixteenth of the row: what lies above the members and what is kept of them, or everything
  if (!added) {
    m = {1, 0, cut, true};
    pass(s, r, whole, m, true, cut);
  }
  u64 v = s.part[wave()];
  if (added) {
    u64 w = 0;
    each(s, r, m, [&](uint32_t k, int i) {
      if (k == 0 || !cut.keeps(k, i)) return;
      w += weight(r, s.pow2, logit_of(k));
    });
    v += wave_sum(w);
  }
  // ---- the sixteenth in which the running sum passes the draw's point, a sixteenth of that, and the token
  Range all = whole;
  u64 before = 0, sum = 0;
  double to = 0.0;
#pragma unroll 1
  for (int level = 0; level < 2; ++level) {
    if (level == 1) {
      const Range part = share(all, wave());
      v = 0;
      walk<2>(r, part.a, part.b, [&](const float4& x, int i) {
        const float* e = (const float*)&x;
#pragma unroll
        for (int j = 0; j < 4; ++j) v += weight(r, s.pow2, cut.keeps(key_of(e[j]), i + j) ? e[j] : -INFINITY);
      });
      v = wave_sum(v);
    }
    __syncthreads();
    if (lane() == 0) s.kept[wave()] = v;
    __syncthreads();
    if (level == 0) {
      for (int w = 0; w < WAVES; ++w) sum += s.kept[w];
      to = target(f.draw, sum);
    }
    int w = 0;
    for (; w < WAVES - 1 && !((double)(before + s.kept[w]) > to); ++w) before += s.kept[w];
    all = share(all, w);
  }
  if (wave() == 0) find(s, r, all, cut, before, sum, to, token, prob);
}
}  // namespace

// temp, top_k, top_p, min_p: of each row, or none.  grid T, 1024.
extern "C" __global__ __launch_bounds__(1024) void sample(SAMPLE_ARGS) {
  __shared__ Lds s;
  const int row = blockIdx.x;
  one_row(s, row_of(logits, ld, off, V, row), form_of(temp, top_k, top_p, min_p, u, row), token + row, prob ? prob + row : nullptr);
}

// ---- few rows: sixteen work-groups a row, in four launches -- the largest logits; what the cuts ask for of each work-group's sixteenth (the few
// highest, a histogram, or the sums where nothing is cut); the tokens of the bin with the cut, and the sums above it; the token.
namespace {
constexpr int PARTS = 16, RUN = LIST;   // (tokens of a work-group that the row's list takes)
enum Mode { ANSWERED, SMALL, BINNED, LISTED, SUMS, WHOLE };
struct Place {   // a row's in the room (arcinferzero_amd/csrc/engine_sample.h has its size)
  u64 sum[BINS];
  uint32_t count[BINS];
  u64 part[PARTS * WAVES];   // sums of weights, by sixteenths of sixteenths
  float top[PARTS];
  int where[PARTS];
  float most[THREADS];       // the largest of each sixteen threads
  int number[PARTS];         // tokens in each run of the list (-1: more than it takes)
  uint32_t lo, hi;
  int mode, then;
  u64 need;
  uint32_t key[PARTS * RUN], at[PARTS * RUN];
};
static_assert(sizeof(Place) == 108760, "engine_sample.h");
typedef LdsOf<128> LdsPart;

// The row's largest logit, out of its parts'; false: nothing is to be drawn by weight.
__device__ inline bool known(Row& r, const Place& g, const Form& f, float& top, int& where) {
  top = -INFINITY;
  where = 0x7FFFFFFF;
  const float t = g.top[lane() % PARTS];
  const int w = g.where[lane() % PARTS];
  for (int i = 0; i < PARTS; ++i)
    first_of(top, where, __uint_as_float(__builtin_amdgcn_readlane((int)__float_as_uint(t), i)), __builtin_amdgcn_readlane(w, i));
  if (!(top > -INFINITY) || !(f.t > 0.0f)) return false;
  measure(r, top, f.t);
  return true;
}
// A work-group's list as its run of the row's.
__device__ inline void publish(const LdsPart& s, Place& g, int part, bool fits) {
  int front = 0, all = 0;
  for (int w = 0; w < WAVES; ++w) {
    front = w == wave() ? all : front;
    all += s.number[w];
  }
  fits = fits && all <= RUN;
  if (threadIdx.x == 0) g.number[part] = fits ? all : -1;
  if (!fits) return;
  for (int p = lane(); p < s.number[wave()]; p += 64) {
    g.key[part * RUN + front + p] = s.key[wave() * LdsPart::CAP + p];
    g.at[part * RUN + front + p] = s.at[wave() * LdsPart::CAP + p];
  }
}
}  // namespace

extern "C" __global__ __launch_bounds__(1024) void sample_top(SAMPLE_ARGS, char* __restrict__ room) {
  __shared__ LdsPart s;
  const int part = blockIdx.x, row = blockIdx.y;
  Place& g = ((Place*)room)[row];
  const Row r = row_of(logits, ld, off, V, row);
  float top, own;
  int where;
  find_top(s, r, share({0, r.units}, part), top, where, own);
#pragma unroll
  for (int o = 1; o < PARTS; o *= 2) own = fmaxf(own, __shfl_xor(own, o));
  if (threadIdx.x % PARTS == 0) g.most[part * (THREADS / PARTS) + threadIdx.x / PARTS] = own;
  if (threadIdx.x == 0) { g.top[part] = top; g.where[part] = where; }
  for (int b = part * (BINS / PARTS) + threadIdx.x; b < (part + 1) * (BINS / PARTS); b += THREADS) {
    g.sum[b] = 0;
    g.count[b] = 0;
  }
}

extern "C" __global__ __launch_bounds__(1024) void sample_scan(SAMPLE_ARGS, char* __restrict__ room) {
  __shared__ LdsPart s;
  const int part = blockIdx.x, row = blockIdx.y;
  Place& g = ((Place*)room)[row];
  Row r = row_of(logits, ld, off, V, row);
  const Form f = form_of(temp, top_k, top_p, min_p, u, row);
  const Range mine = share({0, r.units}, part);
  const bool first = part == 0 && threadIdx.x == 0, by_k = f.by_k(V), by_p = f.by_p();
  const float most = g.most[threadIdx.x];
  float top;
  int where;
  if (!known(r, g, f, top, where)) {
    if (first) {
      token[row] = top > -INFINITY ? where : -1;
      if (prob) prob[row] = top > -INFINITY ? 1.0f : 0.0f;
      g.mode = ANSWERED;
    }
    return;
  }
  powers(s);
  __syncthreads();
  if (by_k && f.k <= SMALL_K) {
    const Members m = {reached(s, most, f.k), key_of(top), {NONE, 0x7FFFFFFF}, true};
    if (first) {
      g.lo = m.lo;
      g.hi = m.hi;
      g.mode = SMALL;
    }
    publish(s, g, part, pass(s, r, mine, m, false, m.within));
  } else if (by_k && by_p) {
    if (first) g.mode = WHOLE;   // (the cut by p needs the one by k first: by one work-group)
  } else if (by_k || by_p) {
    if (first) g.mode = BINNED;
    histogram(s, r, mine, by_k, by_p);
    for (int b = threadIdx.x; b < BINS; b += THREADS) {   // (whole numbers: in any order)
      if (s.sum[b]) atomicAdd(&g.sum[b], s.sum[b]);
      if (s.count[b]) atomicAdd(&g.count[b], s.count[b]);
    }
  } else {
    if (first) g.mode = SUMS;
    const Cut least = least_of(s, r, f.q);
    pass(s, r, mine, {1, 0, least, true}, true, least);
    if (threadIdx.x < WAVES) g.part[part * WAVES + threadIdx.x] = s.part[threadIdx.x];
  }
}

extern "C" __global__ __launch_bounds__(1024) void sample_cut(SAMPLE_ARGS, char* __restrict__ room) {
  __shared__ LdsPart s;
  const int part = blockIdx.x, row = blockIdx.y;
  Place& g = ((Place*)room)[row];
  if (g.mode != BINNED) return;
  Row r = row_of(logits, ld, off, V, row);
  const Form f = form_of(temp, top_k, top_p, min_p, u, row);
  const bool first = part == 0 && threadIdx.x == 0, by_p = f.by_p();
  float top;
  int where;
  if (!known(r, g, f, top, where)) return;
  powers(s);
  for (int b = threadIdx.x; b < BINS; b += THREADS) {
    s.sum[b] = g.sum[b];
    s.count[b] = g.count[b];
  }
  __syncthreads();
  u64 need, front;
  const int b = reach(s, f, by_p, BINS, 0, need, front);
  const Cut least = least_of(s, r, f.q);
  const bool all = !by_p && b >= BINS - 1;   // (all tokens are kept, or all that have a weight)
  const Members m = all ? Members{1, 0, least, true} : members_of(r, b, key_of(top));
  const bool fits = pass(s, r, share({0, r.units}, part), m, true, all ? least : higher({m.hi, -1}, least));
  if (threadIdx.x < WAVES) g.part[part * WAVES + threadIdx.x] = s.part[threadIdx.x];
  if (first) {
    g.then = all ? SUMS : LISTED;
    g.lo = m.lo;
    g.hi = m.hi;
    g.need = need;
  }
  if (!all) publish(s, g, part, fits);
}

extern "C" __global__ __launch_bounds__(1024) void sample_draw(SAMPLE_ARGS, char* __restrict__ room) {
  __shared__ Lds s;
  const int row = blockIdx.x;
  const Place& g = ((const Place*)room)[row];
  Row r = row_of(logits, ld, off, V, row);
  const Form f = form_of(temp, top_k, top_p, min_p, u, row);
  // (all on its way at once)
  const int told = g.mode, then = g.then, number = g.number[lane() % PARTS];
  const uint32_t lo = g.lo, hi = g.hi, key = g.key[wave() * RUN + lane()], at = g.at[wave() * RUN + lane()];
  const u64 need = g.need, sums = threadIdx.x < PARTS * WAVES ? g.part[threadIdx.x] : 0;
  float top;
  int where;
  const bool drawn = known(r, g, f, top, where);
  if (told == ANSWERED) return;
  int mode = told == BINNED ? then : told, members = 0;
  if (mode == SMALL || mode == LISTED) {
    for (int i = 0; i < PARTS; ++i) members += __builtin_amdgcn_readlane(number, i);
    if (__any((uint32_t)number > (uint32_t)RUN)) mode = WHOLE;
  }
  if (mode == WHOLE) {
    one_row(s, r, f, token + row, prob ? prob + row : nullptr);
    return;
  }
  if (!drawn) return;
  powers(s);
  if (threadIdx.x < PARTS * WAVES) s.sum[threadIdx.x] = sums;
  if (mode != SUMS) {
    const int n = __builtin_amdgcn_readlane(number, wave());
    s.key[wave() * LIST + lane()] = key;
    s.at[wave() * LIST + lane()] = at;
    for (int p = 64 + lane(); p < n; p += 64) {
      s.key[wave() * LIST + p] = g.key[wave() * RUN + p];
      s.at[wave() * LIST + p] = g.at[wave() * RUN + p];
    }
    if (lane() == 0) s.number[wave()] = n;
  }
  __syncthreads();
  const Cut least = least_of(s, r, f.q);
  Cut cut = least;
  if (mode != SUMS) {
    Members m = {lo, hi, {NONE, 0x7FFFFFFF}, true};
    u64 rest;
    cut = select(s, r, m, mode == LISTED && f.by_p(), mode == SMALL ? (u64)min(f.k, members) : need, rest);
    if (mode == SMALL && f.by_p()) {
      m.within = cut;
      cut = select(s, r, m, true, f.goal(rest), rest);
    }
    cut = higher(cut, least);
    if (mode == SMALL) {
      from_list(s, r, cut, f.draw, token + row, prob ? prob + row : nullptr);
      return;
    }
    // the members that are kept, to the sums of their units
    const Range c = share({0, r.units}, wave());
    const int per = max((c.b - c.a + WAVES - 1) / WAVES, 1);
    each(s, r, m, [&](uint32_t k, int i) {
      if (k == 0 || !cut.keeps(k, i)) return;
      atomicAdd(&s.sum[wave() * WAVES + min((((i + r.skew) >> 2) - c.a) / per, WAVES - 1)], weight(r, s.pow2, logit_of(k)));
    });
  }
  __syncthreads();
  if (wave()) return;
  // ---- the units in which the running sum passes the draw's point
  constexpr int N = PARTS * WAVES / 64;
  u64 v[N], own = 0;
#pragma unroll
  for (int j = 0; j < N; ++j) own += v[j] = s.sum[N * lane() + j];
  const u64 up = up_sum(own), sum = __shfl(up, 63);
  const double to = target(f.draw, sum);
  u64 front = up - own, before = 0;
  int part = -1;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    if ((double)front <= to && (double)(front + v[j]) > to) {
      part = N * lane() + j;
      before = front;
    }
    front += v[j];
  }
  const u64 vote = __ballot(part >= 0);
  const int l = __ffsll((long long)vote) - 1;
  if (l < 0) return;
  part = __builtin_amdgcn_readlane(part, l);
  before = __shfl(before, l);
  find(s, r, share(share({0, r.units}, part / WAVES), part % WAVES), cut, before, sum, to, token + row, prob ? prob + row : nullptr);
}
