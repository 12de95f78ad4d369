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
#include "attn.h"

// A piece of some rows: sums [rows][HD], then each row's reference and its sum of weights [rows][2].
__device__ constexpr int piece_of(int rows, int hd) { return rows * (hd + 2); }
// The other half of a row's value, eight columns on.
__device__ inline float plus_8(float v) { return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x128, 0xF, 0xF, true)); }

template <int HD, int RT, bool PACK, bool FINE, bool CAP, bool BIAS>
__device__ inline void few_body(const float* __restrict__ q, int ldq, int q_off, const int8_t* __restrict__ kq, const int8_t* __restrict__ vq,
                                const float* __restrict__ ks, const float* __restrict__ vs, int pages, int ps, int bs, const int* __restrict__ rows,
                                const int* __restrict__ lens, const int* __restrict__ table, int ldt, int T, int max_rows, int heads, int kvh, float* __restrict__ out,
                                int ldo, int o_off, float scale, float cap2, int window, const float* __restrict__ slopes, const int* __restrict__ prefix,
                                const int* __restrict__ first, float* __restrict__ ws, unsigned* __restrict__ counts, int nsplit, int least, int vec) {
  constexpr int ROWS = PACK ? 8 : 16 * RT, KS = HD / 32, DT = HD / 16;
  constexpr float LOG2E = 1.4426950408889634f;
  __shared__ float sm_m[4][ROWS], sm_l[4][ROWS];
  __shared__ float sm_o[4][ROWS][HD + 4];
  const int s = blockIdx.x / kvh, h = blockIdx.x - s * kvh, G = heads / kvh;
  const Seq sq = seq_of(rows, lens, s, T, max_rows, ldt << ps);
  const int M = min(sq.n * G, ROWS);
  if (M <= 0) return;
  const int wave = wave_id(), lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4, pm = (1 << ps) - 1, pre = prefix ? prefix[s] : 0;
  table += (size_t)s * ldt;

  // ---- the rows' intervals of keys, and this work-group's steps of 32 keys.  (Without documents the first row's interval begins
  // first and the last row's ends last.)
  int lo[RT], hi[RT], pos[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const int r = PACK ? (m & 7) : t * 16 + m, i = min(r, M - 1) / G;
    pos[t] = sq.p0 + i;
    sees(pos[t], sq.len, window, pre, first ? first[sq.r0 + i] : 0, lo[t], hi[t]);
    if (r >= M) hi[t] = lo[t] = 0;
  }
  // lo_max, hi_min: what all rows see, where every one sees something.
  int all_lo, all_hi, lo_max, hi_min;
  sees(sq.p0, sq.len, window, pre, 0, all_lo, hi_min);
  sees(sq.p0 + (M - 1) / G, sq.len, window, pre, 0, lo_max, all_hi);
  if (first) {
    all_lo = 0x7FFFFFFF;
    all_hi = 0;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      if (lo[t] < hi[t]) { all_lo = min(all_lo, lo[t]); all_hi = max(all_hi, hi[t]); }
      lo_max = max(lo_max, lo[t]);
    }
#pragma unroll
    for (int o = 1; o < 16; o *= 2) {
      all_lo = min(all_lo, __shfl_xor(all_lo, o));
      all_hi = max(all_hi, __shfl_xor(all_hi, o));
      lo_max = max(lo_max, __shfl_xor(lo_max, o));
    }
    lo_max = __builtin_amdgcn_readfirstlane(lo_max);
    all_lo = __builtin_amdgcn_readfirstlane(all_lo);
    all_hi = __builtin_amdgcn_readfirstlane(all_hi);
  }
  const attn::Span span = attn::span_of(all_lo, all_hi, 32);
  const attn::Part part = attn::part_of(span.steps, nsplit, least, blockIdx.y);
  const int base = span.base, z0 = part.z0, z1 = part.z1;

  // (of keys behind the last: some entry of the table -- no row sees them.  Nothing is done with an entry here, so that a lookup is
  //  not waited for before the bytes are asked for)
  auto page_of = [&](int st, int tile) { return table[attn::entry_of(base + st * 32 + tile * 16, ps, ldt)]; };
  // A lane's part of 32 keys: keys in two tiles of 16, bytes 64 j + 16 g of key m; values, HD / 16 bytes of 8 tokens; a scale for
  // each of four keys or, in longer blocks, for all.  Keys are asked for again as soon as the scores are made of them, values once
  // they are in the sums: half a step's work and the other waves' hide the way, and the registers of one step suffice.
  constexpr int NS = FINE ? 4 : 1;
  uint4 kb[2][HD / 64];
  uint32_t vb[8][HD / 64];
  float ksb[2][NS], vsb[2][NS];
  auto row_at = [&](int pg) { return (size_t)((uint32_t)pg < (uint32_t)pages ? pg : 0) * kvh + h; };
  auto load_keys = [&](int st, const int (&pg)[2]) {
#pragma unroll
    for (int tile = 0; tile < 2; ++tile) {
      const size_t row = row_at(pg[tile]);
      const int o = (base + st * 32 + tile * 16) & pm, o4 = o + g * 4;
      const int8_t* kr = kq + ((row << ps) + o) * HD;
#pragma unroll
      for (int j = 0; j < HD / 64; ++j) kb[tile][j] = *(const uint4*)(kr + m * HD + j * 64 + g * 16);
      const float* kp = ks + (row << (ps - bs));
      const float* vp = vs + (row << (ps - bs));
#pragma unroll
      for (int r = 0; r < NS; ++r) { ksb[tile][r] = kp[(o4 + r) >> bs]; vsb[tile][r] = vp[(o4 + r) >> bs]; }
    }
  };
  auto load_values = [&](int st, const int (&pg)[2]) {
#pragma unroll
    for (int tile = 0; tile < 2; ++tile) {
      const int8_t* vr = vq + ((row_at(pg[tile]) << ps) + ((base + st * 32 + tile * 16) & pm)) * HD;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int8_t* a = vr + (g * 4 + r) * HD + m * DT;
        if (HD == 64) vb[tile * 4 + r][0] = *(const uint32_t*)a;
        if (HD == 128) { const uint2 u = *(const uint2*)a; vb[tile * 4 + r][0] = u.x; vb[tile * 4 + r][HD / 64 - 1] = u.y; }
        if (HD == 256) { const uint4 u = *(const uint4*)a; vb[tile * 4 + r][0] = u.x; vb[tile * 4 + r][HD / 256] = u.y; vb[tile * 4 + r][HD / 128] = u.z; vb[tile * 4 + r][HD / 64 - 1] = u.w; }
      }
    }
  };
  int st = z0 + wave, pg[2] = {page_of(st, 0), page_of(st, 1)}, pn[2] = {page_of(st + 4, 0), page_of(st + 4, 1)};
  if (st < z1) {
    load_keys(st, pg);
    load_values(st, pg);
  }

  // ---- the rows in two f16 parts each, times 2^e (a row's largest value to 2^10 ... 2^11), while the first keys come
  const float one = opaque_one();
  float slope[RT], kfac[RT];
  h8 qh[RT][KS], ql[RT][PACK ? 1 : KS];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const int r = min(PACK ? (m & 7) : t * 16 + m, M - 1), i = r / G, hq = h * G + r - i * G;
    slope[t] = BIAS ? slopes[hq] * LOG2E : 0.0f;
    const float* src = q + (size_t)(sq.r0 + i) * ldq + q_off + hq * HD;
    float x[KS][8];
    float big = 0.0f;
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      const float* a = src + (k >> 1) * 64 + g * 16 + (k & 1) * 8;
      if (vec) {
        const float4 u = *(const float4*)a, w = *(const float4*)(a + 4);
        x[k][0] = u.x; x[k][1] = u.y; x[k][2] = u.z; x[k][3] = u.w;
        x[k][4] = w.x; x[k][5] = w.y; x[k][6] = w.z; x[k][7] = w.w;
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[k][e] = a[e];
      }
    }
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
      for (int e = 0; e < 8; ++e) big = fmaxf(big, fabsf(x[k][e]));
    big = fmaxf(big, __shfl_xor(big, 16));
    big = fmaxf(big, __shfl_xor(big, 32));
    const int e2 = min(max(137 - (int)(__float_as_uint(big) >> 23), -118), 126);   // (2^e2 and 2^-e2 are normal numbers)
    const float up = __uint_as_float((uint32_t)(127 + e2) << 23), down = __uint_as_float((uint32_t)(127 - e2) << 23);
    kfac[t] = (CAP ? LOG2E / cap2 : LOG2E) * scale * down;   // (cap2 = cap log2 e)
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      h8 a, b;
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        h2 u, w;
        split2(x[k][e] * up, x[k][e + 1] * up, one, u, w);
        a[e] = u.x; a[e + 1] = u.y; b[e] = w.x; b[e + 1] = w.y;
      }
      if (PACK) {
        qh[t][k] = m < 8 ? a : b;
      } else {
        qh[t][k] = a;
        ql[t][k] = b;
      }
    }
  }

  f4 acc[RT][DT];
  float ref[RT], sum[RT], low = LOW;
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    ref[t] = NOTHING;
    sum[t] = 0.0f;
#pragma unroll
    for (int i = 0; i < DT; ++i) acc[t][i] = f4{0, 0, 0, 0};
  }
  for (; st < z1; st += 4) {
    const int pf[2] = {page_of(st + 8, 0), page_of(st + 8, 1)};   // (two steps ahead)
    const bool more = st + 4 < z1;
    // scores
    float t8[RT][8], iv[8];
#pragma unroll
    for (int tile = 0; tile < 2; ++tile) {
      f4 sc[RT];
#pragma unroll
      for (int t = 0; t < RT; ++t) sc[t] = f4{0, 0, 0, 0};
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const uint4 u = kb[tile][k >> 1];
        const h8 a = k & 1 ? cvt8(u.z, u.w) : cvt8(u.x, u.y);
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          sc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, qh[t][k], sc[t], 0, 0, 0);
          if (!PACK) sc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, ql[t][PACK ? 0 : k], sc[t], 0, 0, 0);
        }
      }
      float kv[4], lv[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if (FINE || r == 0) {
          kv[r] = ksb[tile][FINE ? r : 0];
          value_scale(vsb[tile][FINE ? r : 0], low, lv[r], iv[tile * 4 + r]);
        } else {
          kv[r] = kv[0]; lv[r] = lv[0]; iv[tile * 4 + r] = iv[tile * 4];
        }
      }
      const int j0 = base + st * 32 + tile * 16;
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        float v[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          v[r] = PACK ? plus_8(sc[t][r]) : sc[t][r];
          v[r] = CAP ? v[r] * (kv[r] * kfac[t]) : fmaf(v[r], kv[r] * kfac[t], lv[r]);
        }
        if (CAP) cap_scores(v, cap2);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if (CAP) v[r] += lv[r];
          if (BIAS) v[r] = fmaf(-slope[t], fabsf((float)(pos[t] - (j0 + g * 4 + r))), v[r]);
          t8[t][tile * 4 + r] = v[r];
        }
      }
      const bool there = (uint32_t)pg[tile] < (uint32_t)pages;
      if (!there || j0 < lo_max || j0 + 16 > hi_min) {
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int j = j0 + g * 4 + r;
            t8[t][tile * 4 + r] = there && j >= lo[t] && j < hi[t] ? t8[t][tile * 4 + r] : -INFINITY;
          }
      }
    }
    if (more) load_keys(st + 4, pn);
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
      float part = 0.0f;   // (the row's sum is rounded once a step, like the sums of values, not once a key)
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const float a = exp2_f(t8[t][e] - ref[t]), b = exp2_f(t8[t][e + 1] - ref[t]);
        part = fmaf(a, iv[e], part);
        part = fmaf(b, iv[e + 1], part);
        h2 u, w;
        split2(a, b, one, u, w);
        if (PACK) {
          const h2 c = m < 8 ? u : w;
          ph[t][e] = c.x; ph[t][e + 1] = c.y;
        } else {
          ph[t][e] = u.x; ph[t][e + 1] = u.y;
          pl[t][e] = w.x; pl[t][e + 1] = w.y;
        }
      }
      sum[t] += part;
    }
    // values
#pragma unroll
    for (int w = 0; w < HD / 64; ++w) {
      h2 a[4][2], b[4][2];
      cvt4x4(vb[0][w], vb[1][w], vb[2][w], vb[3][w], a);
      cvt4x4(vb[4][w], vb[5][w], vb[6][w], vb[7][w], b);
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
    if (more) load_values(st + 4, pn);
    pg[0] = pn[0]; pg[1] = pn[1];
    pn[0] = pf[0]; pn[1] = pf[1];
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
      for (int c = 0; c < 4; ++c)
        if (PACK) acc[t][i][c] = plus_8(acc[t][i][c]);
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
  constexpr int PIECE = piece_of(ROWS, HD);
  const Shared pieces(ws + (size_t)blockIdx.x * nsplit * PIECE);   // (the host keeps a row block's pieces below 2^31 bytes)
  auto put = [&](int r, int d, float4 o, float l) {   // a row's sums over its sum of weights
    const int i = r / G;
    float* to = out + (size_t)(sq.r0 + i) * ldo + o_off + (h * G + r - i * G) * HD + d;
    const float f = l == 0.0f ? 0.0f : 1.0f / l;
    if (l == 0.0f) o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    to[0] = o.x * f; to[1] = o.y * f; to[2] = o.z * f; to[3] = o.w * f;
  };
  for (int u = threadIdx.x; u < M * (HD / 4); u += 256) {
    const int r = u / (HD / 4), d = (u - r * (HD / 4)) * 4;
    const float top = fmaxf(fmaxf(sm_m[0][r], sm_m[1][r]), fmaxf(sm_m[2][r], sm_m[3][r]));
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float l = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = exp2_f(sm_m[w][r] - top);
      const float4 v = *(const float4*)&sm_o[w][r][d];
      o.x = fmaf(v.x, f, o.x); o.y = fmaf(v.y, f, o.y); o.z = fmaf(v.z, f, o.z); o.w = fmaf(v.w, f, o.w);
      l = fmaf(sm_l[w][r], f, l);
    }
    if (nsplit == 1) {
      put(r, d, o, l);
    } else {   // (past this XCD's L2: another's work-group reads it)
      pieces.put4(blockIdx.y * PIECE + r * HD + d, o);
      if (d == 0) pieces.put2(blockIdx.y * PIECE + ROWS * HD + 2 * r, top, l);
    }
  }
  if (nsplit == 1) return;
  // ---- the last work-group of these rows to come here joins all pieces, in their order
  if (!last_of(counts + blockIdx.x, nsplit)) return;
  constexpr int U = (ROWS * HD / 4 + 255) / 256, B = U >= 4 ? 6 : 16 / U;   // four values each of U rows a thread, B pieces' loads on the way at once
  float4 o[U];
  float l[U], top[U];
  int ur[U], ud[U];
#pragma unroll
  for (int k = 0; k < U; ++k) {
    const int u = k * 256 + threadIdx.x;
    ur[k] = min(u / (HD / 4), M - 1);
    ud[k] = (u % (HD / 4)) * 4;
    o[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    l[k] = 0.0f;
    top[k] = NOTHING;
  }
  for (int z = 0; z < nsplit; z += B) {
    float4 v[B][U];
    float2 ml[B][U];
#pragma unroll
    for (int i = 0; i < B; ++i)
#pragma unroll
      for (int k = 0; k < U; ++k) {   // (past the last piece: the last again, of no weight)
        const int at = min(z + i, nsplit - 1) * PIECE;
        v[i][k] = pieces.get4(at + ur[k] * HD + ud[k]);
        ml[i][k] = pieces.get2(at + ROWS * HD + 2 * ur[k]);
      }
#pragma unroll
    for (int k = 0; k < U; ++k) {
      float t = top[k];
#pragma unroll
      for (int i = 0; i < B; ++i) t = fmaxf(t, ml[i][k].x);
      const float f0 = exp2_f(top[k] - t);
      o[k].x *= f0; o[k].y *= f0; o[k].z *= f0; o[k].w *= f0;
      l[k] *= f0;
      top[k] = t;
#pragma unroll
      for (int i = 0; i < B; ++i) {
        const float f = z + i < nsplit ? exp2_f(ml[i][k].x - t) : 0.0f;
        l[k] = fmaf(ml[i][k].y, f, l[k]);
        o[k].x = fmaf(v[i][k].x, f, o[k].x); o[k].y = fmaf(v[i][k].y, f, o[k].y); o[k].z = fmaf(v[i][k].z, f, o[k].z); o[k].w = fmaf(v[i][k].w, f, o[k].w);
      }
    }
  }
#pragma unroll
  for (int k = 0; k < U; ++k)
    if (k * 256 + threadIdx.x < M * (HD / 4)) put(ur[k], ud[k], o[k], l[k]);
}

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
