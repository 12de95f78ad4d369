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
// the caches.  Measured, 128 tokens of 32 heads over 8 of 128 values behind 16384 shared keys and up to 600 of their own: 80 + 23 + 9.6 us (attention that reads the
// prefix once a sequence 426); the first of them makes 69 G operations, 860 TFLOP/s, in one round of 256 work-groups of 1024 keys each, the matrix pipe busy 47 % of
// the cycles (62 % where a work-group has ten times the keys).  24 questions of up to 90 tokens behind three documents of 4000, 16 heads over 8 of 256 values, a cap: 313 + 59 + 31 us (425): one work-group a compute
// unit, 2.5 rounds of the pieces' tiles, tiles of which the last is half empty, and 128 values of each lane's registers for the sums alone.
// The pieces: a row's are read once, eight at a time.
#include "attn_many.inc"

// A call's workspace, the room: what these launches leave for the last one, each from its own byte on.
__device__ inline float* in_room(char* room, size_t at) { return (float*)(room + at); }

// The parts joined: the group's rows have n1 pieces in blocks of b1, the sequence's n2 in blocks of b2, t1 and t2 blocks each; a piece is sums
// [b][hd], then reference and sum of weights [b][2].  Rows past the group's `most1` are left as they are.  grid (sequences x kv heads, row groups
// of 1024 / hd), 256.
extern "C" __global__ __launch_bounds__(256) void attn_meet(char* __restrict__ room, size_t at1, int n1, int b1, int t1, int most1, size_t at2, int n2, int b2, int t2, int hd,
                                                            const int* __restrict__ rows, const int* __restrict__ lens, int most_len, int T, int max_rows, int heads,
                                                            int kvh, const int* __restrict__ groups, const int* __restrict__ shared, int n, int seqs,
                                                            float* __restrict__ out, int ldo, int o_off) {
  const float *const ws1 = in_room(room, at1), *const ws2 = in_room(room, at2);
  const int s = blockIdx.x / kvh, h = blockIdx.x - s * kvh, G = heads / kvh, per = 1024 / hd;
  const Seq sq = seq_of(rows, lens, s, T, max_rows, most_len);
  const int r = blockIdx.y * per + threadIdx.x / (hd / 4), d = threadIdx.x % (hd / 4) * 4;
  if (blockIdx.y * per >= sq.n * G) return;
  const int g = attn::group_of(groups, n, s), first_row = g < 0 ? 0 : attn::part_at(groups, rows, g, seqs, T, T).r0;
  if (r >= sq.n * G || r >= t2 * b2) return;
  const int i = r / G, ig = sq.r0 + i - first_row;   // (its place among the group's rows)
  if (g >= 0 && (ig < 0 || ig >= most1)) return;
  const bool both = g >= 0 && shared[g] > 0;
  const int rg = both ? ig * G + r - i * G : 0;
  float top = NOTHING, l = 0.0f;
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  auto add = [&](const float* ws, size_t block, int n, int b, int row) {
    const size_t piece = (size_t)b * (hd + 2);
    const float* p = ws + block * n * piece;
    constexpr int N = 8;   // (pieces on the way at once; past the last: the last again, of no weight)
    for (int z = 0; z < n; z += N) {
      float4 v[N];
      float2 ml[N];
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const float* q = p + min(z + k, n - 1) * piece;
        v[k] = *(const float4*)(q + (size_t)row * hd + d);
        ml[k] = *(const float2*)(q + (size_t)b * hd + 2 * row);
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
  if (both) add(ws1, (size_t)(g * kvh + h) * t1 + rg / b1, n1, b1, rg % b1);
  add(ws2, (size_t)blockIdx.x * t2 + r / b2, n2, b2, r % b2);
  float* to = out + (size_t)(sq.r0 + i) * ldo + o_off + (h * G + r - i * G) * hd + d;
  const float f = l == 0.0f ? 0.0f : 1.0f / l;
  if (l == 0.0f) o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  to[0] = o.x * f; to[1] = o.y * f; to[2] = o.z * f; to[3] = o.w * f;
}

// front: the groups' part, of the rows of `max_rows` tokens of a group at most; else each sequence's own
#define PART(NAME, HD, KT, NW, W, FINE, F)                                                                                                                      \
  extern "C" __global__ __launch_bounds__(64 * NW, W) void NAME(                                                                                                \
      const float* q, int ldq, int q_off, const int8_t* kq, const int8_t* vq, const float* ks, const float* vs, int pages, int ps, int bs, const int* rows,     \
      const int* lens, const int* table, int ldt, int T, int max_rows, int heads, int kvh, float scale, float cap2, int window, const float* slopes,            \
      const int* prefix, const int* first, const int* groups, const int* shared, int n, int seqs, int most_rows, int front, char* room, size_t at,             \
      int nsplit, int tiles, int vec) {                                                                                                                         \
    many_body<HD, KT, NW, FINE, (F & 1) != 0, (F & 2) != 0, true>(q, ldq, q_off, kq, vq, ks, vs, pages, ps, bs, rows, lens, table, ldt, T, max_rows, heads,     \
                                                                  kvh, nullptr, 0, 0, scale, cap2, window, slopes, prefix, first, in_room(room, at), nsplit,    \
                                                                  tiles, vec, {groups, shared, lens, n, seqs, most_rows, front});                               \
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
