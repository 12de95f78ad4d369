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
// The eight-bit values are exact in f16.  Rows and weights are split into two f16 each (22 bits), so the sums are those of f32
// rows to about 2^-22.  Up to eight rows both parts go through one product: the first parts in columns 0-7, what they miss in
// 8-15.
#include "attn.h"

template <int HD> struct Step {   // 32 keys of a lane: keys in two tiles of 16, bytes 64 j + 16 g of key m; values, HD / 16 bytes of 8 tokens
  uint4 k[2][HD / 64];
  uint32_t v[8][HD / 64];
  float ks[2][4], vs[2][4];
};

template <int HD, int RT, bool PACK, bool CAP, bool BIAS>
__device__ inline void few_body(const float* __restrict__ q, int ldq, int q_off, const int8_t* __restrict__ kq, const int8_t* __restrict__ vq,
                                const float* __restrict__ ks, const float* __restrict__ vs, int pages, int ps, int bs, const int* __restrict__ rows,
                                const int* __restrict__ lens, const int* __restrict__ table, int ldt, int T, int max_rows, int heads, int kvh, float* __restrict__ out,
                                int ldo, int o_off, float scale, float cap2, int window, const float* __restrict__ slopes, const int* __restrict__ prefix,
                                const int* __restrict__ first, float* __restrict__ ws, int nsplit, int vec) {
  constexpr int ROWS = PACK ? 8 : 16 * RT, KS = HD / 32, DT = HD / 16;
  constexpr float LOG2E = 1.4426950408889634f;
  __shared__ float sm_m[4][ROWS], sm_l[4][ROWS];
  __shared__ float sm_o[4][ROWS][HD + 4];
  const int s = blockIdx.x / kvh, h = blockIdx.x - s * kvh, G = heads / kvh;
  const Seq sq = seq_of(rows, lens, s, T, max_rows, ldt << ps);
  const int M = min(sq.n * G, ROWS);
  if (M <= 0) return;
  const int wave = wave_id(), lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4, pm = (1 << ps) - 1;
  table += (size_t)s * ldt;

  // ---- the rows: a column's interval of keys, its two f16 parts (of the value times 2^e: the largest at most 2^11)
  int lo[RT], hi[RT], pos[RT];
  float slope[RT];
  float x[RT][KS][8];
  uint32_t big = 0;
  int all_lo = 0x7FFFFFFF, all_hi = 0;
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const int r = PACK ? (m & 7) : t * 16 + m, i = min(r, M - 1) / G, hq = h * G + min(r, M - 1) - i * G;
    pos[t] = sq.p0 + i;
    sees(pos[t], sq.len, window, prefix ? prefix[s] : 0, first ? first[sq.r0 + i] : 0, lo[t], hi[t]);
    if (r >= M) hi[t] = lo[t] = 0;
    slope[t] = BIAS ? slopes[hq] * LOG2E : 0.0f;
    if (lo[t] < hi[t]) { all_lo = min(all_lo, lo[t]); all_hi = max(all_hi, hi[t]); }
    const float* src = q + (size_t)(sq.r0 + i) * ldq + q_off + hq * HD;
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      const float* a = src + (k >> 1) * 64 + g * 16 + (k & 1) * 8;
      if (vec) {
        const float4 u = *(const float4*)a, w = *(const float4*)(a + 4);
        x[t][k][0] = u.x; x[t][k][1] = u.y; x[t][k][2] = u.z; x[t][k][3] = u.w;
        x[t][k][4] = w.x; x[t][k][5] = w.y; x[t][k][6] = w.z; x[t][k][7] = w.w;
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[t][k][e] = a[e];
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t b = __float_as_uint(x[t][k][e]) & 0x7FFFFFFFu;
        if (b < 0x7F800000u) big = max(big, b);
      }
    }
  }
#pragma unroll
  for (int o = 1; o < 64; o *= 2) {
    big = max(big, (uint32_t)__shfl_xor((int)big, o));
    all_lo = min(all_lo, __shfl_xor(all_lo, o));
    all_hi = max(all_hi, __shfl_xor(all_hi, o));
  }
  const int e2 = min(max(137 - (int)(big >> 23), -100), 100);   // (the largest to 2^10 ... 2^11)
  const float up = __uint_as_float((uint32_t)(127 + e2) << 23), down = __uint_as_float((uint32_t)(127 - e2) << 23);
  const float kfac = (CAP ? 2.0f * LOG2E * LOG2E / cap2 : LOG2E) * scale * down;   // (cap2 = cap log2 e)
  h8 qh[RT][KS], ql[RT][PACK ? 1 : KS];
#pragma unroll
  for (int t = 0; t < RT; ++t)
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      h8 a, b;
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        h2 u, w;
        split2(x[t][k][e] * up, x[t][k][e + 1] * up, u, w);
        a[e] = u.x; a[e + 1] = u.y; b[e] = w.x; b[e + 1] = w.y;
      }
      if (PACK) {
        qh[t][k] = m < 8 ? a : b;
      } else {
        qh[t][k] = a;
        ql[t][k] = b;
      }
    }

  // ---- this work-group's steps of 32 keys
  const int base = all_lo & -32, steps = all_lo < all_hi ? (all_hi - base + 31) >> 5 : 0;
  const int share = (steps + nsplit - 1) / nsplit, z0 = blockIdx.y * share, z1 = min(z0 + share, steps);

  auto page_of = [&](int st, int tile) {
    const int p = base + st * 32 + tile * 16;
    return st < z1 && p < sq.len ? table[p >> ps] : -1;
  };
  auto load = [&](Step<HD>& d, int st, int p0, int p1) {
#pragma unroll
    for (int tile = 0; tile < 2; ++tile) {
      const int pg = tile ? p1 : p0;
      const size_t row = (size_t)((uint32_t)pg < (uint32_t)pages ? pg : 0) * kvh + h;
      const int o = (base + st * 32 + tile * 16) & pm;
      const int8_t* kr = kq + ((row << ps) + o) * HD;
      const int8_t* vr = vq + ((row << ps) + o) * HD;
#pragma unroll
      for (int j = 0; j < HD / 64; ++j) d.k[tile][j] = *(const uint4*)(kr + m * HD + j * 64 + g * 16);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int8_t* a = vr + (g * 4 + r) * HD + m * DT;
        if (HD == 64) d.v[tile * 4 + r][0] = *(const uint32_t*)a;
        if (HD == 128) { const uint2 u = *(const uint2*)a; d.v[tile * 4 + r][0] = u.x; d.v[tile * 4 + r][HD / 64 - 1] = u.y; }
        if (HD == 256) { const uint4 u = *(const uint4*)a; d.v[tile * 4 + r][0] = u.x; d.v[tile * 4 + r][HD / 256] = u.y; d.v[tile * 4 + r][HD / 128] = u.z; d.v[tile * 4 + r][HD / 64 - 1] = u.w; }
      }
      const float* kp = ks + (row << (ps - bs));
      const float* vp = vs + (row << (ps - bs));
      const int o4 = o + g * 4;
      if (bs >= 2) {
        const float a = kp[o4 >> bs], b = vp[o4 >> bs];
#pragma unroll
        for (int r = 0; r < 4; ++r) { d.ks[tile][r] = a; d.vs[tile][r] = b; }
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r) { d.ks[tile][r] = kp[(o4 + r) >> bs]; d.vs[tile][r] = vp[(o4 + r) >> bs]; }
      }
    }
  };

  f4 acc[RT][DT];
  float ref[RT], sum[RT], carry = -60.0f;
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    ref[t] = NOTHING;
    sum[t] = 0.0f;
#pragma unroll
    for (int i = 0; i < DT; ++i) acc[t][i] = f4{0, 0, 0, 0};
  }
  Step<HD> now, nxt;
  int st = z0 + wave;
  int pa = page_of(st, 0), pb = page_of(st, 1), na = page_of(st + 4, 0), nb = page_of(st + 4, 1);
  if (st < z1) load(now, st, pa, pb);
  for (; st < z1; st += 4) {
    const int fa = page_of(st + 8, 0), fb = page_of(st + 8, 1);
    if (st + 4 < z1) load(nxt, st + 4, na, nb);
    // scores
    float t8[RT][8], iv[8];
#pragma unroll
    for (int tile = 0; tile < 2; ++tile) {
      f4 sc[RT];
#pragma unroll
      for (int t = 0; t < RT; ++t) sc[t] = f4{0, 0, 0, 0};
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const uint4 u = now.k[tile][k >> 1];
        const h8 a = k & 1 ? cvt8(u.z, u.w) : cvt8(u.x, u.y);
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          sc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, qh[t][k], sc[t], 0, 0, 0);
          if (!PACK) sc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, ql[t][PACK ? 0 : k], sc[t], 0, 0, 0);
        }
      }
      const bool there = (uint32_t)(tile ? pb : pa) < (uint32_t)pages;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float kf = now.ks[tile][r] * kfac;
        float lv;
        value_scale(now.vs[tile][r], carry, lv, iv[tile * 4 + r]);
        const int j = base + st * 32 + tile * 16 + g * 4 + r;
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          float v = sc[t][r];
          if (PACK) v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x128, 0xF, 0xF, true));   // (its other part, eight columns on)
          v = CAP ? capped<true>(v * kf, cap2) + lv : fmaf(v, kf, lv);
          if (BIAS) v = fmaf(-slope[t], fabsf((float)(pos[t] - j)), v);
          t8[t][tile * 4 + r] = there && j >= lo[t] && j < hi[t] ? v : -INFINITY;
        }
      }
    }
    // weights
    h8 ph[RT], pl[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      float top = fmaxf(fmaxf(fmaxf(t8[t][0], t8[t][1]), fmaxf(t8[t][2], t8[t][3])), fmaxf(fmaxf(t8[t][4], t8[t][5]), fmaxf(t8[t][6], t8[t][7])));
      if (__any(top > ref[t] + PASSES)) {
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        const float to = top > ref[t] + PASSES ? top - SETS : ref[t];
        const float f = exp2_f(ref[t] - to);
        ref[t] = to;
        sum[t] *= f;
#pragma unroll
        for (int i = 0; i < DT; ++i) acc[t][i] *= f;
      }
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const float a = exp2_f(t8[t][e] - ref[t]), b = exp2_f(t8[t][e + 1] - ref[t]);
        sum[t] = fmaf(a, iv[e], sum[t]);
        sum[t] = fmaf(b, iv[e + 1], sum[t]);
        h2 u, w;
        split2(a, b, u, w);
        if (PACK) {
          const h2 c = m < 8 ? u : w;
          ph[t][e] = c.x; ph[t][e + 1] = c.y;
        } else {
          ph[t][e] = u.x; ph[t][e + 1] = u.y;
          pl[t][e] = w.x; pl[t][e + 1] = w.y;
        }
      }
    }
    // values
#pragma unroll
    for (int w = 0; w < HD / 64; ++w) {
      h2 a[4][2], b[4][2];
      cvt4x4(now.v[0][w], now.v[1][w], now.v[2][w], now.v[3][w], a);
      cvt4x4(now.v[4][w], now.v[5][w], now.v[6][w], now.v[7][w], b);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const h8 f = {a[i][0].x, a[i][0].y, a[i][1].x, a[i][1].y, b[i][0].x, b[i][0].y, b[i][1].x, b[i][1].y};
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          acc[t][w * 4 + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f, ph[t], acc[t][w * 4 + i], 0, 0, 0);
          if (!PACK) acc[t][w * 4 + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f, pl[t], acc[t][w * 4 + i], 0, 0, 0);
        }
      }
    }
    now = nxt;
    pa = na; pb = nb; na = fa; nb = fb;
  }

  // ---- the waves' parts together.  A lane has values (4 g + r) DT + i of its row.
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    float l = sum[t];
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    const int r = PACK ? m : t * 16 + m;
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        float v = acc[t][i][c];
        if (PACK) v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x128, 0xF, 0xF, true));
        acc[t][i][c] = v;
      }
    if (!PACK || m < 8) {
      if (g == 0) {
        sm_m[wave][r] = ref[t];
        sm_l[wave][r] = l;
      }
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int i = 0; i < DT; i += 4)
          *(float4*)&sm_o[wave][r][(g * 4 + c) * DT + i] = make_float4(acc[t][i][c], acc[t][i + 1][c], acc[t][i + 2][c], acc[t][i + 3][c]);
    }
  }
  __syncthreads();
  for (int u = threadIdx.x; u < M * HD; u += 256) {
    const int r = u / HD, d = u - r * HD;
    const float top = fmaxf(fmaxf(sm_m[0][r], sm_m[1][r]), fmaxf(sm_m[2][r], sm_m[3][r]));
    float o = 0.0f, l = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = exp2_f(sm_m[w][r] - top);
      o = fmaf(sm_o[w][r][d], f, o);
      l = fmaf(sm_l[w][r], f, l);
    }
    if (nsplit == 1) {
      const int i = r / G;
      out[(size_t)(sq.r0 + i) * ldo + o_off + (h * G + r - i * G) * HD + d] = l == 0.0f ? 0.0f : o / l;
    } else {   // (pieces: the sums of each row, then its reference and its sum of weights)
      float* to = ws + ((size_t)blockIdx.x * nsplit + blockIdx.y) * ROWS * (HD + 2);
      to[r * HD + d] = o;
      if (d == 0) {
        to[ROWS * HD + r] = top;
        to[ROWS * HD + ROWS + r] = l;
      }
    }
  }
}

// The pieces of a row joined.  grid (row blocks x sequences x kv heads, rows of a block), local 64 .. 256 = HD.
//   ws: per (block of `rows_of` rows of a sequence and kv head) nsplit pieces of rows_of x (hd + 2).
extern "C" __global__ __launch_bounds__(256) void attn_join(const float* __restrict__ ws, int nsplit, int rows_of, int blocks, int hd, const int* __restrict__ rows,
                                                            const int* __restrict__ lens, int most_len, int T, int max_rows, int heads, int kvh,
                                                            float* __restrict__ out, int ldo, int o_off) {
  const int sh = blockIdx.x / blocks, blk = blockIdx.x - sh * blocks, s = sh / kvh, h = sh - s * kvh, G = heads / kvh;
  const Seq sq = seq_of(rows, lens, s, T, max_rows, most_len);
  const int per = 256 / hd, rr = blockIdx.y * per + threadIdx.x / hd, d = threadIdx.x % hd;
  const int r = blk * rows_of + rr;
  if (rr >= rows_of || r >= sq.n * G) return;
  const size_t piece = (size_t)rows_of * (hd + 2);
  const float* at = ws + (size_t)blockIdx.x * nsplit * piece;
  float top = NOTHING;
  for (int z = 0; z < nsplit; ++z) top = fmaxf(top, at[z * piece + (size_t)rows_of * hd + rr]);
  float o = 0.0f, l = 0.0f;
  for (int z = 0; z < nsplit; ++z) {
    const float f = exp2_f(at[z * piece + (size_t)rows_of * hd + rr] - top);
    l = fmaf(at[z * piece + (size_t)rows_of * (hd + 1) + rr], f, l);
    o = fmaf(at[z * piece + (size_t)rr * hd + d], f, o);
  }
  const int i = r / G;
  out[(size_t)(sq.r0 + i) * ldo + o_off + (h * G + r - i * G) * hd + d] = l == 0.0f ? 0.0f : o / l;
}

#define FEW(HD, RT, PACK, F)                                                                                                                                    \
  extern "C" __global__ __launch_bounds__(256) void attn_few__HD##HD##_RT##RT##_PACK##PACK##_FORM##F(                                                          \
      const float* q, int ldq, int q_off, const int8_t* kq, const int8_t* vq, const float* ks, const float* vs, int pages, int ps, int bs, const int* rows,     \
      const int* lens, const int* table, int ldt, int T, int max_rows, int heads, int kvh, float* out, int ldo, int o_off, float scale, float cap2, int window, \
      const float* slopes, const int* prefix, const int* first, float* ws, int nsplit, int vec) {                                                               \
    few_body<HD, RT, PACK, (F & 1) != 0, (F & 2) != 0>(q, ldq, q_off, kq, vq, ks, vs, pages, ps, bs, rows, lens, table, ldt, T, max_rows, heads, kvh, out, ldo, \
                                                       o_off, scale, cap2, window, slopes, prefix, first, ws, nsplit, vec);                                     \
  }
#define FEWS(HD, F) FEW(HD, 1, 1, F) FEW(HD, 1, 0, F) FEW(HD, 2, 0, F)
#define FEWF(HD) FEWS(HD, 0) FEWS(HD, 1) FEWS(HD, 2) FEWS(HD, 3)
FEWF(64)
FEWF(128)
FEWF(256)
