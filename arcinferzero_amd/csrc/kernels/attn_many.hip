// "attn" module: attention of many rows over the 8-bit cache -- prompts and chunks behind a context.
//
// Per kv head the rows are the sequence's tokens times the query heads that share it (row = token * group + head), 128 to a
// work-group, 32 to a wave.  KT keys at a time are brought into LDS as f16 -- the eight-bit values exactly, converted once for
// the four waves --, the keys as they lie, the values with tokens and columns exchanged; the next tile's bytes are on their
// way meanwhile.
//
//   S^T = K Q^T   32 x 32 x 16 products, A = 32 keys from LDS, B = 32 rows held in registers: a lane has 16 keys' scores of one row
//   O^T += V^T P^T  B = the weights just as the scores' product left them (a lane's keys of a slot of 16 are 4 h + 0..3 and
//                  8 + 4 h + 0..3, so the values' tokens lie in that order in LDS): no weight goes through LDS
//
// A row's maximum and sum are its lane's own, but for the two halves of the wave, which meet only where the reference is set
// anew.  Rows and weights are split into two f16 (22 bits of the f32 value; the sums are those of f32 rows to about 2^-22), so
// the matrix pipe does twice the products of plain f16 rows; it is what bounds the kernel.
#include "attn.h"

template <int HD, int KT, bool FINE, bool CAP, bool BIAS>
__device__ inline void many_body(const float* __restrict__ q, int ldq, int q_off, const int8_t* __restrict__ kq, const int8_t* __restrict__ vq,
                                 const float* __restrict__ ks, const float* __restrict__ vs, int pages, int ps, int bs, const int* __restrict__ rows,
                                 const int* __restrict__ lens, const int* __restrict__ table, int ldt, int T, int max_rows, int heads, int kvh,
                                 float* __restrict__ out, int ldo, int o_off, float scale, float cap2, int window, const float* __restrict__ slopes,
                                 const int* __restrict__ prefix, const int* __restrict__ first, float* __restrict__ ws, int nsplit, int tiles, int vec) {
  constexpr int BM = 128, KSTEPS = HD / 16, DT = HD / 32, NT = KT / 32;
  constexpr int TPK = 256 / KT, KB = HD / TPK;          // threads a key's row, bytes each
  constexpr int TPV = 1024 / KT, VB = HD / TPV;         // threads four tokens' values, bytes each and token
  constexpr int KLD = HD + 8, VLD = KT + 8;             // (rows 16 bytes longer: neighbouring rows four banks on)
  constexpr float LOG2E = 1.4426950408889634f;
  __shared__ _Float16 sk[2][KT * KLD], sv[2][HD * VLD];
  // scales: of each key, or of each 32 keys that share one (kf: the score's factor; lv, iv: value_scale)
  constexpr int NS = FINE ? KT : NT;
  __shared__ float skf[2][NS], slv[2][NS], siv[2][NS];
  __shared__ int red[4][3];

  const int sh = blockIdx.x / tiles, tile = tiles - 1 - (blockIdx.x - sh * tiles), s = sh / kvh, h = sh - s * kvh, G = heads / kvh;
  const Seq sq = seq_of(rows, lens, s, T, max_rows, ldt << ps);
  const int M = sq.n * G;   // (the host holds max_rows * heads below 2^31)
  if (tile * BM >= M) return;
  const int wave = wave_id(), lane = threadIdx.x & 63, c = lane & 31, hf = lane >> 5, pm = (1 << ps) - 1;
  table += (size_t)s * ldt;

  // ---- this lane's row
  const int r = tile * BM + wave * 32 + c, rr = min(r, M - 1), i = rr / G, hq = h * G + rr - i * G, pos = sq.p0 + i;
  int lo, hi;
  sees(pos, sq.len, window, prefix ? prefix[s] : 0, first ? first[sq.r0 + i] : 0, lo, hi);
  if (r >= M) hi = lo = 0;
  const float slope = BIAS ? slopes[hq] * LOG2E : 0.0f;
  uint32_t big = 0;
  float x[KSTEPS][8];
  {
    const float* src = q + (size_t)(sq.r0 + i) * ldq + q_off + hq * HD + hf * 8;
#pragma unroll
    for (int k = 0; k < KSTEPS; ++k) {
      const float* a = src + k * 16;
      if (vec) {
        const float4 u = *(const float4*)a, w = *(const float4*)(a + 4);
        x[k][0] = u.x; x[k][1] = u.y; x[k][2] = u.z; x[k][3] = u.w;
        x[k][4] = w.x; x[k][5] = w.y; x[k][6] = w.z; x[k][7] = w.w;
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[k][e] = a[e];
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t b = __float_as_uint(x[k][e]) & 0x7FFFFFFFu;
        if (b < 0x7F800000u) big = max(big, b);
      }
    }
  }
  // (rows that see nothing take no part in the wave's range)
  int lo_min = lo < hi ? lo : 0x7FFFFFFF, lo_max = lo < hi ? lo : 0, hi_min = lo < hi ? hi : 0x7FFFFFFF, hi_max = lo < hi ? hi : 0;
  int blind = lo < hi ? 0 : 1;
#pragma unroll
  for (int o = 1; o < 64; o *= 2) {
    big = max(big, (uint32_t)__shfl_xor((int)big, o));
    lo_min = min(lo_min, __shfl_xor(lo_min, o));
    lo_max = max(lo_max, __shfl_xor(lo_max, o));
    hi_min = min(hi_min, __shfl_xor(hi_min, o));
    hi_max = max(hi_max, __shfl_xor(hi_max, o));
    blind |= __shfl_xor(blind, o);
  }
  if (blind) hi_min = 0;   // (a row without keys: every tile goes through the masks)
  lo_min = __builtin_amdgcn_readfirstlane(lo_min); lo_max = __builtin_amdgcn_readfirstlane(lo_max);
  hi_min = __builtin_amdgcn_readfirstlane(hi_min); hi_max = __builtin_amdgcn_readfirstlane(hi_max);
  if (lane == 0) {
    red[wave][0] = (int)big; red[wave][1] = lo_min; red[wave][2] = hi_max;
  }
  __syncthreads();
  big = max(max((uint32_t)red[0][0], (uint32_t)red[1][0]), max((uint32_t)red[2][0], (uint32_t)red[3][0]));
  const int all_lo = __builtin_amdgcn_readfirstlane(min(min(red[0][1], red[1][1]), min(red[2][1], red[3][1])));
  const int all_hi = __builtin_amdgcn_readfirstlane(max(max(red[0][2], red[1][2]), max(red[2][2], red[3][2])));
  const int e2 = min(max(137 - (int)(big >> 23), -100), 100);   // (the largest of the work-group's rows to 2^10 ... 2^11)
  const float up = __uint_as_float((uint32_t)(127 + e2) << 23), down = __uint_as_float((uint32_t)(127 - e2) << 23);
  const float kfac = (CAP ? 2.0f * LOG2E * LOG2E / cap2 : LOG2E) * scale * down;   // (cap2 = cap log2 e)
  const float one = opaque_one();
  h8 qh[KSTEPS], ql[KSTEPS];
#pragma unroll
  for (int k = 0; k < KSTEPS; ++k)
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      h2 a, b;
      split2(x[k][e] * up, x[k][e + 1] * up, one, a, b);
      qh[k][e] = a.x; qh[k][e + 1] = a.y; ql[k][e] = b.x; ql[k][e + 1] = b.y;
    }

  // ---- this work-group's tiles of keys
  const int base = all_lo & -KT, steps = all_lo < all_hi ? (all_hi - base + KT - 1) / KT : 0;
  const int share = (steps + nsplit - 1) / nsplit, z0 = blockIdx.y * share, z1 = min(z0 + share, steps);

  // this thread's key and its bytes 16 kc, 16 (kc + TPK), ...; its four tokens and VB bytes of each.  (Threads side by side write
  // side by side in LDS: a key's 16-byte pieces dealt out in turn, the tokens of one column.)
  const int tk = threadIdx.x / TPK, kc = threadIdx.x % TPK * 16;
  const int tv = threadIdx.x % (KT / 4) * 4, vc = threadIdx.x / (KT / 4) * VB;
  const int vpos = (tv & ~15) + ((tv >> 2 & 1) << 3) + ((tv >> 3 & 1) << 2);   // where they lie in LDS
  const int ts = FINE ? threadIdx.x & (KT - 1) : (threadIdx.x & (NT - 1)) * 32;  // ... and the key whose scales it brings
  auto page_at = [&](int st, int t) {
    const int p = base + st * KT + t;
    const int pg = table[min(p >> ps, ldt - 1)];
    return st < z1 && p < sq.len ? pg : -1;
  };
  auto row_at = [&](int pg) { return (size_t)((uint32_t)pg < (uint32_t)pages ? pg : 0) * kvh + h; };
  uint4 kr[KB / 16];
  uint32_t vr[4][VB / 4];
  float rks = 0.0f, rvs = 0.0f;
  auto load = [&](int st, int pk, int pv, int pc) {
    const int t0 = base + st * KT;
    const int8_t* a = kq + ((row_at(pk) << ps) + ((t0 + tk) & pm)) * HD + kc;
#pragma unroll
    for (int b = 0; b < KB / 16; ++b) kr[b] = *(const uint4*)(a + 16 * TPK * b);
    const int8_t* v = vq + ((row_at(pv) << ps) + ((t0 + tv) & pm)) * HD + vc;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      if (VB == 4) vr[t][0] = *(const uint32_t*)(v + t * HD);
      if (VB == 8) { const uint2 u = *(const uint2*)(v + t * HD); vr[t][0] = u.x; vr[t][VB / 8] = u.y; }
      if (VB == 16) { const uint4 u = *(const uint4*)(v + t * HD); vr[t][0] = u.x; vr[t][VB / 16] = u.y; vr[t][VB / 8] = u.z; vr[t][VB / 4 - 1] = u.w; }
    }
    if (threadIdx.x < NS) {
      const size_t d = (row_at(pc) << (ps - bs)) + (((t0 + ts) & pm) >> bs);
      rks = ks[d];
      rvs = vs[d];
    }
  };
  float carry = -60.0f;
  auto store = [&](int buf, int pc) {
    _Float16* a = &sk[buf][tk * KLD + kc];
#pragma unroll
    for (int b = 0; b < KB / 16; ++b) {
      *(h8*)(a + 16 * TPK * b) = cvt8(kr[b].x, kr[b].y);
      *(h8*)(a + 16 * TPK * b + 8) = cvt8(kr[b].z, kr[b].w);
    }
#pragma unroll
    for (int w = 0; w < VB / 4; ++w) {
      h2 p[4][2];
      cvt4x4(vr[0][w], vr[1][w], vr[2][w], vr[3][w], p);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        uint2 u;
        __builtin_memcpy(&u.x, &p[e][0], 4);
        __builtin_memcpy(&u.y, &p[e][1], 4);
        *(uint2*)&sv[buf][(vc + 4 * w + e) * VLD + vpos] = u;
      }
    }
    if (threadIdx.x < NS) {   // (a token of no page: weight 0 whatever its score)
      float lv, iv;
      value_scale(rvs, carry, lv, iv);
      const bool there = (uint32_t)pc < (uint32_t)pages;
      skf[buf][threadIdx.x] = there ? rks * kfac : 0.0f;
      slv[buf][threadIdx.x] = there ? lv : -INFINITY;
      siv[buf][threadIdx.x] = there ? iv : 1.0f;
    }
  };

  f16v acc[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[d][e] = 0.0f;
  // (a row's weights are 2^(score - ref); before the first score that it sees ref is 0 and any score sets it)
  float ref = 0.0f, limit = NOTHING, sum = 0.0f;

  int pk = page_at(z0, tk), pv = page_at(z0, tv), pc = page_at(z0, ts);
  if (z0 < z1) {
    load(z0, pk, pv, pc);
    store(0, pc);
  }
  pk = page_at(z0 + 1, tk); pv = page_at(z0 + 1, tv); pc = page_at(z0 + 1, ts);
  __syncthreads();
  for (int st = z0; st < z1; ++st) {
    const int buf = (st - z0) & 1;
    const bool more = st + 1 < z1;
    const int pc1 = pc;
    if (more) load(st + 1, pk, pv, pc);
    pk = page_at(st + 2, tk); pv = page_at(st + 2, tv); pc = page_at(st + 2, ts);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int j0 = base + st * KT + nt * 32;
      if (j0 >= hi_max || j0 + 32 <= lo_min) continue;   // (of no row of the wave)
      f16v sc;
#pragma unroll
      for (int e = 0; e < 16; ++e) sc[e] = 0.0f;
      const _Float16* kp = &sk[buf][(nt * 32 + c) * KLD + hf * 8];
#pragma unroll
      for (int k = 0; k < KSTEPS; ++k) {
        const h8 a = *(const h8*)(kp + k * 16);
        sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, qh[k], sc, 0, 0, 0);
        sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, ql[k], sc, 0, 0, 0);
      }
      // (register e of the product: key 8 (e / 4) + 4 hf + e % 4)
      float kf1 = 0.0f, lv1 = 0.0f, iv1 = 0.0f;
      if (!FINE) { kf1 = skf[buf][nt]; lv1 = slv[buf][nt] - ref; iv1 = siv[buf][nt]; }
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const int j4 = nt * 32 + 8 * b + 4 * hf;
        f4 kf = {kf1, kf1, kf1, kf1}, lv = {lv1, lv1, lv1, lv1};
        if (FINE) {
          kf = *(const f4*)&skf[buf][j4];
          lv = *(const f4*)&slv[buf][j4];
#pragma unroll
          for (int e = 0; e < 4; ++e) lv[e] -= ref;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float v = sc[4 * b + e];
          sc[4 * b + e] = CAP ? capped<true>(v * kf[e], cap2) + lv[e] : fmaf(v, kf[e], lv[e]);
          if (BIAS) sc[4 * b + e] = fmaf(-slope, fabsf((float)(pos - (base + st * KT + j4 + e))), sc[4 * b + e]);
        }
      }
      if (j0 < lo_max || j0 + 32 > hi_min) {
        const int a = lo - (j0 + 4 * hf), z = hi - (j0 + 4 * hf);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int j = 8 * (e >> 2) + (e & 3);
          sc[e] = j >= a && j < z ? sc[e] : -INFINITY;
        }
      }
      float top = fmaxf(sc[0], sc[1]);
#pragma unroll
      for (int e = 2; e < 16; e += 2) top = fmaxf(fmaxf(top, sc[e]), sc[e + 1]);
      if (__any(top > limit)) {
        top = fmaxf(top, __shfl_xor(top, 32));
        const bool anew = top > limit;
        const float by = anew ? top - SETS : 0.0f;
        const float f = limit > NOTHING ? exp2_f(-by) : 1.0f;   // (nothing summed yet)
        ref += by;
        limit = anew ? PASSES : limit;
        sum *= f;
#pragma unroll
        for (int d = 0; d < DT; ++d) acc[d] *= f;
#pragma unroll
        for (int e = 0; e < 16; ++e) sc[e] -= by;
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) {   // 16 keys
        h8 ph, pl;
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          f4 iv = {iv1, iv1, iv1, iv1};
          if (FINE) iv = *(const f4*)&siv[buf][nt * 32 + 16 * k + 8 * b + 4 * hf];
#pragma unroll
          for (int e = 0; e < 4; e += 2) {
            const float u = exp2_f(sc[8 * k + 4 * b + e]), w = exp2_f(sc[8 * k + 4 * b + e + 1]);
            sum = fmaf(u, iv[e], sum);
            sum = fmaf(w, iv[e + 1], sum);
            h2 a, l;
            split2(u, w, one, a, l);
            ph[4 * b + e] = a.x; ph[4 * b + e + 1] = a.y; pl[4 * b + e] = l.x; pl[4 * b + e + 1] = l.y;
          }
        }
        const _Float16* vp = &sv[buf][c * VLD + nt * 32 + 16 * k + hf * 8];
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          const h8 a = *(const h8*)(vp + d * 32 * VLD);
          acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, ph, acc[d], 0, 0, 0);
          acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, pl, acc[d], 0, 0, 0);
        }
      }
    }
    if (more) store(buf ^ 1, pc1);
    __syncthreads();
  }

  sum += __shfl_xor(sum, 32);
  if (limit == NOTHING) ref = NOTHING;
  if (r >= M) return;
  if (nsplit == 1) {
    float* to = out + (size_t)(sq.r0 + i) * ldo + o_off + hq * HD;
    const float f = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        float* at = to + d * 32 + 8 * b + 4 * hf;
        const float4 o = sum == 0.0f ? make_float4(0.0f, 0.0f, 0.0f, 0.0f)
                                     : make_float4(acc[d][4 * b] * f, acc[d][4 * b + 1] * f, acc[d][4 * b + 2] * f, acc[d][4 * b + 3] * f);
        if (vec & 2) {
          *(float4*)at = o;
        } else {
          at[0] = o.x; at[1] = o.y; at[2] = o.z; at[3] = o.w;
        }
      }
  } else {   // (pieces: the sums of each row, then its reference and its sum of weights)
    float* to = ws + ((size_t)(sh * tiles + tile) * nsplit + blockIdx.y) * BM * (HD + 2);
    const int row = wave * 32 + c;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        float* at = to + row * HD + d * 32 + 8 * b + 4 * hf;
        *(float4*)at = make_float4(acc[d][4 * b], acc[d][4 * b + 1], acc[d][4 * b + 2], acc[d][4 * b + 3]);
      }
    if (hf == 0) {
      to[BM * HD + 2 * row] = ref;
      to[BM * HD + 2 * row + 1] = sum;
    }
  }
}

// grid (tiles of the most rows x sequences x kv heads, pieces), local 256; vec: bit 0 the rows, bit 1 the output in 16-byte pieces
// -DFINE=1: blocks of less than 32 tokens
#define MANY(HD, KT, W, FINE, F)                                                                                                                                \
  extern "C" __global__ __launch_bounds__(256, W) void attn_many__HD##HD##_FINE##FINE##_FORM##F(                                                                \
      const float* q, int ldq, int q_off, const int8_t* kq, const int8_t* vq, const float* ks, const float* vs, int pages, int ps, int bs, const int* rows,     \
      const int* lens, const int* table, int ldt, int T, int max_rows, int heads, int kvh, float* out, int ldo, int o_off, float scale, float cap2, int window, \
      const float* slopes, const int* prefix, const int* first, float* ws, int nsplit, int tiles, int vec) {                                                    \
    many_body<HD, KT, FINE, (F & 1) != 0, (F & 2) != 0>(q, ldq, q_off, kq, vq, ks, vs, pages, ps, bs, rows, lens, table, ldt, T, max_rows, heads, kvh, out,     \
                                                        ldo, o_off, scale, cap2, window, slopes, prefix, first, ws, nsplit, tiles, vec);                        \
  }
#define MANYF(HD, KT, W, FINE) MANY(HD, KT, W, FINE, 0) MANY(HD, KT, W, FINE, 1) MANY(HD, KT, W, FINE, 2) MANY(HD, KT, W, FINE, 3)
MANYF(64, 64, 2, 0)
MANYF(64, 64, 2, 1)
MANYF(128, 64, 2, 0)
MANYF(128, 64, 2, 1)
MANYF(256, 32, 1, 0)
MANYF(256, 32, 1, 1)
