// "attn" module: where a pass's new tokens go -- the batch that the cache's calls take, made on the GPU.
//
// Sequence s gets add[s] tokens (or loses -add[s] of its last ones).  With the pages that hold n tokens, ceil(n / page):
//   rows = the running sum of max(add, 0);  len = max(0, before + add);  the table's entries [pages(before), pages(len)) come from a ring
//   of free pages, in the order of the sequences; those that a shorter sequence leaves go to the ring's end;  row i of a sequence has the
//   position before + i and the place page * (tokens a page) + position % (tokens a page).
// What is taken lies in front of what is given back, so a page that one sequence loses is not another's in the same plan, and no
// work depends on the order in which it is done.  All or nothing: where the pages, the table or the rows do not suffice, or a row would lie in
// a page that other sequences share, nothing is changed and no sequence has rows.
//
// Bound: latency -- one work-group for all sequences, since the sums run over them: the counts, their sums in three steps over the
// waves, then the ring's entries and the table's, a thread each.  Places of many rows are a launch of their own (kv_places), a work-group for
// 1024 of one sequence's, behind it.
// Measured: 256 sequences of a token 3.8 us, 1024 5.6, 256 of eight 5.6, 64 prompts of 256 tokens 6.7 in two launches, 1024 of up to 500 12.0 (13.6 with one page of a thread's looked up
// at a time); a launch that does
// nothing takes 2.5.
#include "attn.h"

using attn::Change;

constexpr int PLAN = 1024;

// The sums of three values over the threads in front of this one, and of all.
struct Three {
  int rows, take, give;
};
__device__ inline Three scan(Three v, Three& total, Three (&part)[PLAN / 64]) {
  const int lane = threadIdx.x & 63, wave = wave_id(), waves = blockDim.x >> 6;
  Three sum = v;
#pragma unroll
  for (int o = 1; o < 64; o *= 2) {
    const int a = __shfl_up(sum.rows, o), b = __shfl_up(sum.take, o), c = __shfl_up(sum.give, o);
    if (lane >= o) { sum.rows += a; sum.take += b; sum.give += c; }
  }
  if (lane == 63) part[wave] = sum;
  __syncthreads();
  Three front = {0, 0, 0};
  total = {0, 0, 0};
  for (int w = 0; w < waves; ++w) {
    const Three p = part[w];
    if (w < wave) { front.rows += p.rows; front.take += p.take; front.give += p.give; }
    total.rows += p.rows; total.take += p.take; total.give += p.give;
  }
  return {front.rows + sum.rows - v.rows, front.take + sum.take - v.take, front.give + sum.give - v.give};
}
// The last of the work-group's places (those behind the last sequence hold the total, which no search reaches) whose sum is not above i.
__device__ inline int find(const int (&sums)[PLAN], int i) {
  int at = 0;
  for (int step = blockDim.x / 2; step; step /= 2)
    if (sums[at + step] <= i) at += step;
  return at;
}

// Of `total` things, so many of each sequence, one a thread, four of a thread's on their way at once: put(sequence, thing, get(sequence, thing)).
template <class G, class P>
__device__ inline void deal(const int (&sums)[PLAN], int total, G get, P put) {
  const unsigned local = blockDim.x, all = total;   // (no sum here passes 32 bits: total is below 2^31)
  unsigned i0 = 0;
  for (; all > i0 + local; i0 += 4 * local) {
    int at[4] = {0, 0, 0, 0}, i[4], v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) i[k] = (int)min(i0 + k * local + threadIdx.x, all - 1);
    for (int step = local / 2; step; step /= 2)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (sums[at[k] + step] <= i[k]) at[k] += step;
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = get(at[k], i[k]);
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (i0 + k * local + threadIdx.x < all) put(at[k], i[k], v[k]);
  }
  if (i0 + threadIdx.x < all) {
    const int i = (int)(i0 + threadIdx.x), at = find(sums, i);
    put(at, i, get(at, i));
  }
}

// state, after: the ring's first place, how many pages it holds, what was missing (0: nothing; pages; -1: rows or table), the rows of the plan.
// before may be len, state may be after.  grid 1, local 256 (no more sequences than that) or 1024.  with_rows: pos and slot too.
extern "C" __global__ __launch_bounds__(PLAN) void kv_plan(const int* __restrict__ add, const int* before, int* len, int* __restrict__ rows, int* __restrict__ table,
                                                           int ldt, int* __restrict__ ring, const int* state, int* after, const int* __restrict__ shared,
                                                           int* __restrict__ pos, int* __restrict__ slot, int seqs, int T, int max_rows, int pages, int ps,
                                                           int with_rows) {
  __shared__ Three part[2][PLAN / 64];
  __shared__ int s_rows[PLAN], s_take[PLAN], s_give[PLAN], s_had[PLAN], s_has[PLAN], s_before[PLAN];
  __shared__ unsigned long long sums[3];
  const int local = blockDim.x, mask = (1 << ps) - 1;
  auto change = [&](int s) { return attn::planned(before[s], add[s], shared ? shared[s] : 0, ps, ldt, max_rows); };
  auto place = [&](int pg, int p) { return (unsigned)pg < (unsigned)pages ? (pg << ps) + (p & mask) : -1; };
  Change c = {0, 0, 0, 0, 0, 0, 0, true};   // (of this thread's first sequence)
  if ((int)threadIdx.x < seqs) c = change(threadIdx.x);
  const int head = state[0], count = state[1];
  // (the page that its first new row falls into, if the sequence has it already)
  const int last = slot && with_rows && c.rows > 0 && (c.before & mask) ? table[(size_t)threadIdx.x * ldt + (c.before >> ps)] : -1;
  // ---- the whole batch first: whether it fits.  Where there is a thread for each sequence the sums in front of it are those of the
  // batch too, unless they may not fit 32 bits.
  if (threadIdx.x < 3) sums[threadIdx.x] = 0;
  Three total, front = scan({c.rows, c.take, c.give}, total, part[0]);
  const bool many = seqs > local || __syncthreads_or(c.rows > 1 << 20 || c.take > 1 << 20 || c.give > 1 << 20);
  long long n = total.rows, take = total.take, give = total.give;
  bool fits = c.fits;
  if (many) {
    n = take = give = 0;
    for (int s = threadIdx.x; s < seqs; s += local) {
      const Change k = change(s);
      n += k.rows;
      take += k.take;
      give += k.give;
      fits = fits && k.fits;
    }
    __syncthreads();
    atomicAdd(&sums[0], (unsigned long long)n);
    atomicAdd(&sums[1], (unsigned long long)take);
    atomicAdd(&sums[2], (unsigned long long)give);
    __syncthreads();
    n = (long long)sums[0];
    take = (long long)sums[1];
    give = (long long)sums[2];
  }
  const bool misfit = __syncthreads_or(!fits);   // (everything that may be brought on in place has been read)
  const bool sound = (unsigned)head < (unsigned)pages && (unsigned)count <= (unsigned)pages && count + give <= pages;
  const long long lacks = take - count;
  const int missing = !sound || misfit || n > T ? -1 : lacks <= 0 ? 0 : (int)(lacks < 0x7FFFFFFF ? lacks : 0x7FFFFFFF);
  if (threadIdx.x == 0) {
    after[0] = missing ? head : (int)attn::ring_at(head, (unsigned)take, pages);
    after[1] = missing ? count : (int)(count - take + give);
    after[2] = missing;
    after[3] = missing ? 0 : (int)n;
    rows[seqs] = missing ? 0 : (int)n;
  }
  if (missing) {
    for (int s = threadIdx.x; s < seqs; s += local) {
      rows[s] = 0;
      len[s] = before[s];
    }
    return;
  }
  // ---- a thread's sequence at a time
  const unsigned tail = attn::ring_at(head, count, pages);
  Three at = {0, 0, 0};   // (of the sequences in front)
  for (int s0 = 0; s0 < seqs; s0 += local) {
    const int s = s0 + threadIdx.x;
    if (s0) {
      c = s < seqs ? change(s) : Change{0, 0, 0, 0, 0, 0, 0, true};
      __syncthreads();   // (the places of the last ones are not looked at any more)
      front = scan({c.rows, c.take, c.give}, total, part[s0 / local & 1]);
    }
    if (s < seqs) {
      rows[s] = at.rows + front.rows;
      len[s] = c.len;
    }
    // Up to eight rows a sequence (tokens, drafts): its own thread writes their pages and places (256 sequences of four 4.4 us, of eight 5.6; shared
    // out 6.1, 8.6; of twelve 11.0 shared out).  Else, and for pages given back, of which
    // a sequence that ends has many, the work-group shares them out.
    const bool apart = max_rows > 8;
    if (!apart && s < seqs) {
      int* const to = table + (size_t)s * ldt;
      for (int i = 0; i < c.take; ++i) to[c.had + i] = ring[attn::ring_at(head, at.take + front.take + i, pages)];
      if (with_rows)
        for (int i = 0; i < c.rows; ++i) {
          const int p = c.before + i, e = p >> ps, r = at.rows + front.rows + i;
          if (pos) pos[r] = p;
          if (slot) slot[r] = place(e >= c.had ? ring[attn::ring_at(head, at.take + front.take + (e - c.had), pages)] : s0 ? to[e] : last, p);
        }
    }
    if (apart || total.give) {
      s_rows[threadIdx.x] = front.rows;
      s_take[threadIdx.x] = front.take;
      s_give[threadIdx.x] = front.give;
      s_had[threadIdx.x] = c.had;
      s_has[threadIdx.x] = c.has;
      s_before[threadIdx.x] = c.before;
      __syncthreads();
      deal(s_give, total.give, [&](int j, int i) { return table[(size_t)(s0 + j) * ldt + s_has[j] + (i - s_give[j])]; },
           [&](int, int i, int page) { ring[attn::ring_at(tail, at.give + i, pages)] = page; });
    }
    if (apart) {
      deal(s_take, total.take, [&](int, int i) { return ring[attn::ring_at(head, at.take + i, pages)]; },
           [&](int j, int i, int page) { table[(size_t)(s0 + j) * ldt + s_had[j] + (i - s_take[j])] = page; });
      if (with_rows)
        for (int i = threadIdx.x; i < total.rows; i += local) {
          const int j = find(s_rows, i), p = s_before[j] + (i - s_rows[j]), e = p >> ps;
          if (pos) pos[at.rows + i] = p;
          if (slot)   // (a new page is looked up where the table has it from)
            slot[at.rows + i] = place(e < s_had[j] ? table[(size_t)(s0 + j) * ldt + e] : ring[attn::ring_at(head, at.take + s_take[j] + (e - s_had[j]), pages)], p);
        }
    }
    at.rows += total.rows;
    at.take += total.take;
    at.give += total.give;
  }
}

// Positions and places of a plan's rows.  grid (ceil(max_rows / 1024), seqs), four rows a thread.
extern "C" __global__ __launch_bounds__(256) void kv_places(const int* __restrict__ rows, const int* __restrict__ len, const int* __restrict__ table, int ldt,
                                                            int* __restrict__ pos, int* __restrict__ slot, int T, int max_rows, int pages, int ps) {
  const int s = blockIdx.y;
  const Seq sq = seq_of(rows, len, s, T, max_rows, ldt << ps);
  table += (size_t)s * ldt;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int i = blockIdx.x * 1024 + k * 256 + threadIdx.x, p = sq.p0 + i;
    if (i >= sq.n || p < 0) continue;
    if (pos) pos[sq.r0 + i] = p;
    if (slot) {
      const int pg = table[p >> ps];
      slot[sq.r0 + i] = (unsigned)pg < (unsigned)pages ? (pg << ps) + (p & ((1 << ps) - 1)) : -1;
    }
  }
}
