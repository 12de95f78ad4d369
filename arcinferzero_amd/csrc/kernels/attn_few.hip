// "attn" module: attention of few rows over the 8-bit cache -- single tokens, drafts -- and the joining of pieces.
//
// Per kv head the rows are the sequence's tokens times the query heads that share it, at most 16 or 32.  Reading the cache
// bounds it: 2 hd bytes a key.  A work-group takes a piece of the keys, its four waves 32 of them at a time in turn, straight
// from memory into registers: no byte passes through LDS, nothing waits for another wave, and each wave keeps its own softmax
// until the end.
//
//   S^T = K Q^T   16 x 16 x 32 products, A = 16 keys, B = 16 rows: a lane has four keys' scores of one row
//   O^T += V^T P^T  A = 16 of the head's values, B = the weights just as the scores' product left them: a lane's eight keys of
//                  two tiles are the eight of its k slot, so the weights go from one product into the other in registers
//
// Pieces of one length for all sequences, about two work-groups a compute unit where all are long; they are joined in this launch by the
// last work-group of their rows to come (joined by a launch of its own: 41 us more behind 131072 keys).
// Measured, heads of 128 values: one token behind 131072, 40 heads over 8, 56.7 us (4.75 TB/s, a large copy 4.9); 64
// sequences of up to 8100 keys, 32 over 4, 75.7 us (3.8 TB/s); one behind 517, 9.0 us, and four sequences of eight tokens with heads of
// 256 under a window 15.6 us: dependent loads -- rows, page, bytes --, two steps a wave one behind the other, and the joining, not bytes.
//
// The eight-bit values are exact in f16.  Rows and weights are split into two f16 each (22 bits), so the sums are those of f32
// rows to about 2^-22.  Up to eight rows both parts go through one product: the first parts in columns 0-7, what they miss in
// 8-15.
#include "attn_few.inc"

// The pieces of the rows of attn_many joined, a work-group 256 / (hd / 4) rows: 4 hd bytes a row and piece, read once.  grid (row blocks x sequences x kv heads, row groups)
//   ws: per (block of rows_of rows of a sequence and kv head) nsplit pieces.
extern "C" __global__ __launch_bounds__(256) void attn_join(const float* __restrict__ ws, int nsplit, int rows_of, int blocks, int hd, const int* __restrict__ rows,
                                                            const int* __restrict__ lens, int most_len, int T, int max_rows, int heads, int kvh,
                                                            float* __restrict__ out, int ldo, int o_off) {
  const int sh = blockIdx.x / blocks, blk = blockIdx.x - sh * blocks, s = sh / kvh, h = sh - s * kvh, G = heads / kvh;
  const Seq sq = seq_of(rows, lens, s, T, max_rows, most_len);
  const int per = 1024 / hd, rr = blockIdx.y * per + threadIdx.x / (hd / 4), d = threadIdx.x % (hd / 4) * 4;
  const int r = blk * rows_of + rr;
  if (rr >= rows_of || r >= sq.n * G) return;
  const size_t piece = (size_t)piece_of(rows_of, hd);
  const float* at = ws + (size_t)blockIdx.x * nsplit * piece;
  const float2* mt = (const float2*)(at + (size_t)rows_of * hd) + rr;
  float top = NOTHING;
#pragma unroll 8
  for (int z = 0; z < nsplit; ++z) top = fmaxf(top, mt[z * piece / 2].x);
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  float l = 0.0f;
#pragma unroll 8
  for (int z = 0; z < nsplit; ++z) {
    const float2 ml = mt[z * piece / 2];
    const float f = exp2_f(ml.x - top);
    const float4 v = *(const float4*)(at + z * piece + (size_t)rr * hd + d);
    l = fmaf(ml.y, f, l);
    o.x = fmaf(v.x, f, o.x); o.y = fmaf(v.y, f, o.y); o.z = fmaf(v.z, f, o.z); o.w = fmaf(v.w, f, o.w);
  }
  const int i = r / G;
  float* to = out + (size_t)(sq.r0 + i) * ldo + o_off + (h * G + r - i * G) * hd + d;
  const float f = l == 0.0f ? 0.0f : 1.0f / l;
  if (l == 0.0f) o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  to[0] = o.x * f; to[1] = o.y * f; to[2] = o.z * f; to[3] = o.w * f;
}

// -DFINE=1: blocks of one or two tokens, a scale for each key; 0: a scale for each four
#define FEW(HD, RT, PACK, FINE, W, F)                                                                                                                              \
  extern "C" __global__ __launch_bounds__(256, W) void attn_few__HD##HD##_RT##RT##_PACK##PACK##_FINE##FINE##_FORM##F(                                             \
      const float* q, int ldq, int q_off, const int8_t* kq, const int8_t* vq, const float* ks, const float* vs, int pages, int ps, int bs, const int* rows,     \
      const int* lens, const int* table, int ldt, int T, int max_rows, int heads, int kvh, float* out, int ldo, int o_off, float scale, float cap2, int window, \
      const float* slopes, const int* prefix, const int* first, float* ws, unsigned* counts, int nsplit, int least, int vec) {                                  \
    few_body<HD, RT, PACK, FINE, (F & 1) != 0, (F & 2) != 0>(q, ldq, q_off, kq, vq, ks, vs, pages, ps, bs, rows, lens, table, ldt, T, max_rows, heads, kvh,     \
                                                             out, ldo, o_off, scale, cap2, window, slopes, prefix, first, ws, counts, nsplit, least, vec);      \
  }
#define FEW4(HD, RT, PACK, FINE, W) FEW(HD, RT, PACK, FINE, W, 0) FEW(HD, RT, PACK, FINE, W, 1) FEW(HD, RT, PACK, FINE, W, 2) FEW(HD, RT, PACK, FINE, W, 3)
// W, WF: waves a SIMD that the registers are held to (WF: with a scale for each key)
#define FEWF(HD, RT, PACK, W, WF) FEW4(HD, RT, PACK, 0, W) FEW4(HD, RT, PACK, 1, WF)
FEWF(64, 1, 1, 4, 4)
FEWF(64, 1, 0, 4, 3)
FEWF(64, 2, 0, 3, 2)
FEWF(128, 1, 1, 3, 3)
FEWF(128, 1, 0, 3, 2)
FEWF(128, 2, 0, 2, 1)
FEWF(256, 1, 1, 2, 2)   // (two row tiles of 256 values do not fit a wave's registers: such rows go to attn_many)
FEWF(256, 1, 0, 2, 1)
