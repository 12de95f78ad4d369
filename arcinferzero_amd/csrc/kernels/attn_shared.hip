// "attn" module: attention for sequences that share a prefix.
//
// The softmax over a row's keys is made of two parts: over the keys that its group has in common, [0, P), and over its own behind them.
// Each part leaves sums o, the reference m of its weights and their sum l; with m the larger reference
//   out = (o1 2^(m1 - m) + o2 2^(m2 - m)) / (l1 2^(m1 - m) + l2 2^(m2 - m)).
// The first part takes the rows of all sequences of a group as rows of one (attn_many.inc), so the prefix is read once for all of them and
// its products are those of matrices; the second is attention as it is, from P on.  Both leave pieces, as where keys are shared out, and one
// launch joins them.  Both cut the same interval of a row's keys, so that together they see what attention without groups sees, whatever
// the form.
//
// Bound: the prefix's products on the matrix pipe (rows and weights in two halves, so twice the operations), the sequences' own keys by latency, the pieces by
// the caches.  Measured, 128 tokens of 32 heads over 8 of 128 values behind 16384 shared keys and up to 600 of their own: 80 + 24 + 10 us (attention that reads the
// prefix once a sequence 426); the first of them makes 69 G operations, 860 TFLOP/s, in one round of 256 work-groups of 1024 keys each, the matrix pipe busy 47 % of
// the cycles (62 % where a work-group has ten times the keys).  24 questions of up to 90 tokens behind three documents of 4000, 16 heads over 8 of 256 values, a cap: 312 + 58 + 30 us (425): one work-group a compute
// unit, 2.5 rounds of the pieces' tiles, tiles of which the last is half empty, and 128 values of each lane's registers for the sums alone.
// The pieces: a row's are read once, eight at a time.
// Those 128 tokens with a window of 2048 keys 64 us, with a bias by distance 127, capped 131 (116 on the same card with neither).
// Registers that do not fit: 36 bytes of scratch a lane in eight waves with a bias, 12 in heads of 256 with a scale for each few keys and a cap.
#include "attn_many.inc"

// A call's workspace, the room: what these launches leave for the last one, each from its own byte on.
__device__ inline float* in_room(char* room, size_t at) { return (float*)(room + at); }

// The sequence that a row belongs to, the row being the same in all lanes, each of which looks at one of 64 boundaries at a time; some one of them where
// the rows are in no order.
__device__ inline int seq_of_one_row(const int* __restrict__ rows, int seqs, int t) {
  int a = 0, n = seqs;   // (one of [a, a + n))
  while (n > 1) {
    const int step = (n + 63) / 64, b = a + step * ((int)(threadIdx.x & 63) + 1), end = a + n;
    a += step * __popcll(__ballot(b < end && rows[min(b, seqs)] <= t));
    n = min(step, end - a);
  }
  return a;
}

// The parts joined: a row and head has n1 pieces of its group's keys and n2 of its own: sums [piece][places][heads][hd], then reference and sum of weights
// [piece][places][heads][2], a place for each row of the buffers or, where that is less, for each of the most rows of every sequence.  (So the room, and this
// launch, are no larger than the batch may be, however unlike its sequences are: one of 2048 tokens beside 255 of a token, 64 heads of 128 values, 0.15 GB; blocks of the
// longest one's rows for each would be 8.8.)  Rows past the group's `most1`, past max_rows of a sequence, or of none, are left as they are.
// grid (places x heads / (1024 / hd)), 256.
extern "C" __global__ __launch_bounds__(256) void attn_meet(char* __restrict__ room, size_t at1, int n1, size_t at2, int n2, int hd, const int* __restrict__ rows, int T,
                                                            int max_rows, int heads, const int* __restrict__ groups, const int* __restrict__ shared, int n, int seqs,
                                                            int most1, int places, int per, float* __restrict__ out, int ldo, int o_off) {
  const unsigned at = blockIdx.x * (1024u / hd) + threadIdx.x / (hd / 4), u = at / heads, hq = at - u * heads;   // (the host holds places * heads below 2^31)
  const int d = threadIdx.x % (hd / 4) * 4;
  int s = 0, t = (int)u;
  if (per) {
    s = min(u / per, (unsigned)(seqs - 1));
  } else {
    const int t0 = min(__builtin_amdgcn_readfirstlane(t), T - 1), s0 = seq_of_one_row(rows, seqs, t0);
    s = t <= t0 ? s0 : attn::seq_of_row(rows, s0, seqs, t0, T - t0, t);   // (few heads: a wave has values of several rows)
  }
  if (u >= (unsigned)places) return;
  const Seq sq = attn::part_at(nullptr, rows, s, seqs, T, max_rows);
  if (per) t = sq.r0 + ((int)u - s * per);
  if (t < sq.r0 || t - sq.r0 >= sq.n) return;
  const int g = attn::group_of(groups, n, s);
  if (g >= 0) {
    const int ig = t - attn::part_at(groups, rows, g, seqs, T, T).r0;   // (its place among the group's rows)
    if (ig < 0 || ig >= most1) return;
  }
  const bool both = g >= 0 && shared[g] > 0;
  const size_t all = (size_t)places * heads;
  float top = NOTHING, l = 0.0f;
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  auto add = [&](const float* ws, int n) {
    const float* const ml_of = ws + n * all * hd;
    constexpr int N = 8;   // (pieces on the way at once; past the last: the last again, of no weight)
    for (int z = 0; z < n; z += N) {
      float4 v[N];
      float2 ml[N];
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const size_t q = min(z + k, n - 1) * all + at;
        v[k] = *(const float4*)(ws + q * hd + d);
        ml[k] = *(const float2*)(ml_of + 2 * q);
      }
      float t = top;
#pragma unroll
      for (int k = 0; k < N; ++k) t = fmaxf(t, ml[k].x);
      const float f0 = exp2_f(top - t);
      o.x *= f0; o.y *= f0; o.z *= f0; o.w *= f0;
      l *= f0;
      top = t;
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const float f = z + k < n ? exp2_f(ml[k].x - t) : 0.0f;
        l = fmaf(ml[k].y, f, l);
        o.x = fmaf(v[k].x, f, o.x); o.y = fmaf(v[k].y, f, o.y); o.z = fmaf(v[k].z, f, o.z); o.w = fmaf(v[k].w, f, o.w);
      }
    }
  };
  if (both) add(in_room(room, at1), n1);
  add(in_room(room, at2), n2);
  float* to = out + (size_t)t * ldo + o_off + (size_t)hq * hd + d;
  const float f = l == 0.0f ? 0.0f : 1.0f / l;
  if (l == 0.0f) o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  to[0] = o.x * f; to[1] = o.y * f; to[2] = o.z * f; to[3] = o.w * f;
}

// front: the groups' part, of the rows of `max_rows` tokens of a group at most; else each sequence's own
#define PART(NAME, HD, KT, NW, W, FINE, F)                                                                                                                      \
  extern "C" __global__ __launch_bounds__(64 * NW, W) void NAME(                                                                                                \
      const float* q, int ldq, int q_off, const int8_t* kq, const int8_t* vq, const float* ks, const float* vs, int pages, int ps, int bs, const int* rows,     \
      const int* lens, const int* table, int ldt, int T, int max_rows, int heads, int kvh, float scale, float cap2, int window, const float* slopes,            \
      const int* prefix, const int* first, const int* groups, const int* shared, int n, int seqs, int most_rows, int front, int places, int per, char* room,   \
      size_t at, int nsplit, int tiles, int vec) {                                                                                                              \
    many_body<HD, KT, NW, FINE, (F & 1) != 0, (F & 2) != 0, true>(q, ldq, q_off, kq, vq, ks, vs, pages, ps, bs, rows, lens, table, ldt, T, max_rows, heads,     \
                                                                  kvh, nullptr, 0, 0, scale, cap2, window, slopes, prefix, first, in_room(room, at), nsplit,    \
                                                                  tiles, vec, {groups, shared, lens, n, seqs, most_rows, front, places, per});                  \
  }
#define PART4(HD, KT, NW, W, FINE, S)                                     \
  PART(attn_part__HD##HD##_FINE##FINE##_FORM0##S, HD, KT, NW, W, FINE, 0) \
  PART(attn_part__HD##HD##_FINE##FINE##_FORM1##S, HD, KT, NW, W, FINE, 1) \
  PART(attn_part__HD##HD##_FINE##FINE##_FORM2##S, HD, KT, NW, W, FINE, 2) \
  PART(attn_part__HD##HD##_FINE##FINE##_FORM3##S, HD, KT, NW, W, FINE, 3)
PART4(64, 64, 4, 2, 0, )
PART4(64, 64, 4, 2, 1, )
PART4(128, 32, 4, 2, 0, )
PART4(128, 32, 4, 2, 1, )
PART4(128, 64, 8, 2, 0, _W81)
PART4(256, 32, 4, 1, 0, )
PART4(256, 32, 4, 1, 1, )
