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
// anew.  Rows and weights are split into two f16 (22 bits of the f32 value, a row on its own power of two; the sums are those of f32
// rows to about 2^-22), so the matrix pipe does twice the products of plain f16 rows: most of the time of long prompts.
//
// Measured, 32 query heads over 8 of 128 values: 8192 rows behind 808 keys, causal, 1109 - 1172 us by the card = 562 - 593 TFLOP/s of
// attention, 1124 - 1186 of products (a large f16 matrix product of the library: 1211).  The matrix pipe is busy 62 % of 2.05 million
// cycles, which makes about 1.85 GHz: like the library's product the launch runs below the card's highest clock, and the third of
// the cycles in which no product is under way (a tile's meeting, weights that are not done when they are wanted) costs less time
// than it would at that.  On the way there: 2000 us with the tiles' rows 8 and 16 bytes apart in the same banks (conflicts in 64 %
// of the LDS's cycles, now 0.3 %); 1303 with the rows that see the most keys first; 1141 with no wait for a page's number inside the
// loop; the last 7 to 10 with keys and values as global loads (through pointers of no known address space they counted among
// the LDS reads, and every operand was waited for with them).
// Rows of several documents (1333 rows, 40 heads): 67 us, the matrix pipe busy 22 %: most tiles are one document's end.
// Spills, all before and behind the loop: 4 and 8 registers of heads of 256 with a scale for each few keys and a cap, 9 of eight waves with
// a distance.
#include "attn.h"

// Nothing is moved across by the compiler.
__device__ inline void turn() { __builtin_amdgcn_sched_barrier(0); }
// Worked out here, not where it is used.
__device__ inline void stay(h8 (&a)[2], h8 (&b)[2]) { asm volatile("" : "+v"(a[0]), "+v"(a[1]), "+v"(b[0]), "+v"(b[1])); }

template <int HD, int KT, int NW, bool FINE, bool CAP, bool BIAS>
__device__ inline void many_body(const float* __restrict__ q, int ldq, int q_off, const int8_t* __restrict__ kq, const int8_t* __restrict__ vq,
                                 const float* __restrict__ ks, const float* __restrict__ vs, int pages, int ps, int bs, const int* __restrict__ rows,
                                 const int* __restrict__ lens, const int* __restrict__ table, int ldt, int T, int max_rows, int heads, int kvh,
                                 float* __restrict__ out, int ldo, int o_off, float scale, float cap2, int window, const float* __restrict__ slopes,
                                 const int* __restrict__ prefix, const int* __restrict__ first, float* __restrict__ ws, int nsplit, int tiles, int vec) {
  constexpr int BM = 32 * NW, THREADS = 64 * NW, KSTEPS = HD / 16, DT = HD / 32, NT = KT / 32;
  constexpr int TPK = THREADS / KT, KB = HD / TPK;      // threads a key's row, bytes each
  constexpr int TPV = 4 * THREADS / KT, VB = HD / TPV;  // threads four tokens' values, bytes each and token
  // 128 values: what the rows' first f16 miss stays in LDS (32 registers; with them there the loop's would not fit two waves a SIMD)
  constexpr bool QLDS = NW == 8;
  constexpr int KLD = HD + 8, VLD = KT + 8;             // (rows 16 bytes longer: neighbouring rows four banks on)
  constexpr float LOG2E = 1.4426950408889634f;
  // (the rows on their way in, and out, pass through the tiles' place: SLD floats a row of the wave's 32, 64 columns at a time)
  constexpr int SLD = 68;
  struct Tiles { _Float16 k[2][KT * KLD], v[2][HD * VLD]; };
  static_assert(sizeof(Tiles) >= NW * 32 * SLD * 4, "the rows pass through the tiles' place");
  __shared__ __attribute__((aligned(16))) Tiles tl2;
  auto& sk = tl2.k;
  auto& sv = tl2.v;
  // scales: of each key, or of each 32 keys that share one (kf: the keys'; lv, iv: value_scale)
  constexpr int NS = FINE ? KT : NT;
  __shared__ float skf[2][NS], slv[2][NS], siv[2][NS];
  __shared__ int red[NW][2];
  __shared__ _Float16 sq_lo[QLDS ? NW * 32 * KLD : 1];

  // (the rows that see the most keys first, of all heads; the heads in turn, so that with 8 of them each XCD's L2 holds one's cache)
  const int pairs = gridDim.x / tiles, sh = blockIdx.x % pairs, tile = tiles - 1 - blockIdx.x / pairs, s = sh / kvh, h = sh - s * kvh, G = heads / kvh;
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
  // (rows that see nothing take no part in the wave's range)
  int lo_min = lo < hi ? lo : 0x7FFFFFFF, lo_max = lo < hi ? lo : 0, hi_min = lo < hi ? hi : 0x7FFFFFFF, hi_max = lo < hi ? hi : 0;
  int blind = lo < hi ? 0 : 1;
#pragma unroll
  for (int o = 1; o < 64; o *= 2) {
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
    red[wave][0] = lo_min; red[wave][1] = hi_max;
  }
  __syncthreads();
  int all_lo = red[0][0], all_hi = red[0][1];
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    all_lo = min(all_lo, red[w][0]);
    all_hi = max(all_hi, red[w][1]);
  }
  all_lo = __builtin_amdgcn_readfirstlane(all_lo);
  all_hi = __builtin_amdgcn_readfirstlane(all_hi);

  // ---- this work-group's tiles of keys
  const attn::Span span = attn::span_of(all_lo, all_hi, KT);
  const int base = span.base;
  const attn::Part part = attn::part_of(span.steps, nsplit, 1, blockIdx.y);
  const int z0 = part.z0, z1 = part.z1;

  // this thread's key and its bytes 16 kc, 16 (kc + TPK), ...; its four tokens and VB bytes of each.  (Threads side by side write
  // side by side in LDS: a key's 16-byte pieces dealt out in turn, the tokens of one column.)
  const int tk = threadIdx.x / TPK, kc = threadIdx.x % TPK * 16;
  const int tv = threadIdx.x % (KT / 4) * 4, vc = threadIdx.x / (KT / 4) * VB;
  const int vpos = (tv & ~15) + ((tv >> 2 & 1) << 3) + ((tv >> 3 & 1) << 2);   // where they lie in LDS
  const int ts = FINE ? threadIdx.x & (KT - 1) : (threadIdx.x & (NT - 1)) * 32;  // ... and the key whose scales it brings
  // Where a tile's bytes are: page * (bytes of a page of all heads) + the tile's place in the page (0 where pages are smaller than a
  // tile) + the thread's own.  With pages of a tile and more all threads have the same page (at.k).  Every address lies in the cache,
  // also that of a tile behind the last, which is asked for and not used.
  const bool whole = (1 << ps) >= KT;
  const uint32_t page_bytes = (uint32_t)(kvh << ps) * HD, page_scales = (uint32_t)(kvh << (ps - bs)) * 4;
  const char* const kmine = (const char*)kq + ((size_t)h << ps) * HD + ((tk & pm) * HD + kc);
  const char* const vmine = (const char*)vq + ((size_t)h << ps) * HD + ((tv & pm) * HD + vc);
  const size_t smine = (((size_t)h << (ps - bs)) + ((ts & pm) >> bs)) * 4;
  // (of a key behind the last: some entry of the table -- no row sees it.  Nothing is done with the entry here: a lookup is not
  //  waited for until the next tile's bytes are asked for)
  auto page_at = [&](int st, int t) { return table[attn::entry_of(base + st * KT + t, ps, ldt)]; };
  auto valid = [&](int pg) { return (uint32_t)pg < (uint32_t)pages ? (uint32_t)pg : 0u; };
  struct Pages { int k, v, c; };
  Pages at = {0, 0, 0};
  uint4 kr[KB / 16];
  uint32_t vr[4][VB / 4];
  float rks = 0.0f, rvs = 0.0f;
  size_t ka, va, sa;   // (from kmine, vmine, ks and vs on)
  auto address = [&](int st) {
    const uint32_t in = (uint32_t)((base + st * KT) & pm);
    const int pv = whole ? at.k : at.v, pc = whole ? at.k : at.c;
    ka = (size_t)valid(at.k) * page_bytes + in * HD;
    va = (size_t)valid(pv) * page_bytes + in * HD;
    sa = smine + ((size_t)valid(pc) * page_scales + (in >> bs) * 4);
    return pc;
  };
  auto load = [&](int part) {   // (four parts)
    if (part == 0) {
#pragma unroll
      for (int b = 0; b < KB / 16; ++b) kr[b] = *(const uint4*)(kmine + ka + 16 * TPK * b);
    } else if (part < 3) {
#pragma unroll
      for (int t = 2 * part - 2; t < 2 * part; ++t) {
        const char* v = vmine + va + t * HD;
        if (VB == 4) vr[t][0] = *(const uint32_t*)v;
        if (VB == 8) { const uint2 u = *(const uint2*)v; vr[t][0] = u.x; vr[t][VB / 8] = u.y; }
        if (VB == 16) { const uint4 u = *(const uint4*)v; vr[t][0] = u.x; vr[t][VB / 16] = u.y; vr[t][VB / 8] = u.z; vr[t][VB / 4 - 1] = u.w; }
      }
    } else {
      rks = *(const float*)((const char*)ks + sa);
      rvs = *(const float*)((const char*)vs + sa);
    }
  };
  // (looked up through vector memory, also where all threads have the same page: a wait for a scalar load among the LDS reads
  //  would be a wait for all of them)
  int zero;
  asm("v_mov_b32 %0, 0" : "=v"(zero));
  const int tl = whole ? zero : tk;
  auto look = [&](int st) {   // (with whole pages the other two are left alone: writing them would wait for all loads on the way)
    at.k = page_at(st, tl);
    if (!whole) {
      at.v = page_at(st, tv);
      at.c = page_at(st, ts);
    }
  };
  // (the first tile's way is begun before the rows': they come together)
  look(z0);
  int pc0 = 0;

  // The rows come, and go, 64 columns at a time through LDS: four rows' 256 bytes a load, where a lane's own 16 bytes of 32 rows
  // would be 64 places.  A lane moves 16 bytes of rows 4 n + lane / 16.
  float* const pass = (float*)&tl2 + wave * 32 * SLD;
  const int quarter = lane >> 4, col = (lane & 15) * 4;
  auto of_row = [&](long v, int n) { return (long)__shfl((long long)v, n * 4 + quarter); };
  float big = 0.0f;
  float x[KSTEPS][8];
  {
    const long from = (long)(sq.r0 + i) * ldq + q_off + hq * HD;
#pragma unroll
    for (int cc = 0; cc < HD / 64; ++cc) {
      float4 u[8];
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        const float* a = q + of_row(from, n) + cc * 64 + col;
        u[n] = vec & 1 ? *(const float4*)a : make_float4(a[0], a[1], a[2], a[3]);
      }
      if (cc == 0 && z0 < z1) {
        pc0 = address(z0);
#pragma unroll
        for (int part = 0; part < 4; ++part) load(part);
        look(z0 + 1);
      }
#pragma unroll
      for (int n = 0; n < 8; ++n) *(float4*)&pass[(n * 4 + quarter) * SLD + col] = u[n];
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");   // (among the wave's lanes)
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float4 a = *(const float4*)&pass[c * SLD + k * 16 + hf * 8], b = *(const float4*)&pass[c * SLD + k * 16 + hf * 8 + 4];
        float (&y)[8] = x[cc * 4 + k];
        y[0] = a.x; y[1] = a.y; y[2] = a.z; y[3] = a.w; y[4] = b.x; y[5] = b.y; y[6] = b.z; y[7] = b.w;
#pragma unroll
        for (int e = 0; e < 8; ++e) big = fmaxf(big, fabsf(y[e]));
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
      __builtin_amdgcn_wave_barrier();
    }
  }
  __syncthreads();   // (all rows have passed through the tiles' place)
  // (the row's largest to 2^10 ... 2^11: the lane's own power of two, so that a row's bits do not hang on the rows beside it)
  big = fmaxf(big, __shfl_xor(big, 32));
  const int e2 = min(max(137 - (int)(__float_as_uint(big) >> 23), -118), 126);   // (2^e2 and 2^-e2 are normal numbers)
  const float up = __uint_as_float((uint32_t)(127 + e2) << 23), down = __uint_as_float((uint32_t)(127 - e2) << 23);
  const float kfac = (CAP ? LOG2E / cap2 : LOG2E) * scale * down;   // (cap2 = cap log2 e)
  const float one = opaque_one();
  h8 qh[KSTEPS], ql[QLDS ? 1 : KSTEPS];
  _Float16* const mine = &sq_lo[QLDS ? (wave * 32 + c) * KLD + hf * 8 : 0];
#pragma unroll
  for (int k = 0; k < KSTEPS; ++k) {
    h8 lo8;
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      h2 a, b;
      split2(x[k][e] * up, x[k][e + 1] * up, one, a, b);
      qh[k][e] = a.x; qh[k][e + 1] = a.y; lo8[e] = b.x; lo8[e + 1] = b.y;
    }
    if (QLDS) *(h8*)(mine + k * 16) = lo8;
    else ql[QLDS ? 0 : k] = lo8;
  }

  // (the bytes are waited for here: what is done with them in two branches is not brought in front of both)
  auto arrive = [&] {
#pragma unroll
    for (int b = 0; b < KB / 16; ++b) asm volatile("" : "+v"(kr[b].x), "+v"(kr[b].y), "+v"(kr[b].z), "+v"(kr[b].w));
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int w = 0; w < VB / 4; ++w) asm volatile("" : "+v"(vr[t][w]));
  };
  float low = LOW;
  // ... to LDS in UNITS parts: half a key's 16 bytes each, then two columns of the four tokens each
  constexpr int KU = KB / 8, UNITS = KU + VB / 2;
  auto store = [&](int buf, int u) {
    if (u < KU) {
      // (eight threads side by side on a key's row: four write their second half while the others write their first)
      const uint4 r = kr[u / 2];
      const bool second = (u & 1) != (TPK > 4 && (threadIdx.x & 4));
      *(h8*)&sk[buf][tk * KLD + kc + 16 * TPK * (u / 2) + (second ? 8 : 0)] = cvt8(second ? r.z : r.x, second ? r.w : r.y);
      return;
    }
    const int w = (u - KU) / 2, e = (u - KU) & 1;
    h2 p[2][2];
    cvt4x2(vr[0][w], vr[1][w], vr[2][w], vr[3][w], e, p);
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      uint2 o;
      __builtin_memcpy(&o.x, &p[x][0], 4);
      __builtin_memcpy(&o.y, &p[x][1], 4);
      *(uint2*)&sv[buf][(vc + 4 * w + 2 * e + x) * VLD + vpos] = o;
    }
  };
  auto store_scales = [&](int buf, int pc) {
    if (threadIdx.x < NS) {   // (a token of no page: weight 0 whatever its score)
      float lv, iv;
      value_scale(rvs, low, lv, iv);
      const bool there = (uint32_t)pc < (uint32_t)pages;
      skf[buf][threadIdx.x] = there ? rks : 0.0f;
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

  if (z0 < z1) {
#pragma unroll
    for (int u = 0; u < UNITS; ++u) store(0, u);
    store_scales(0, pc0);
  }
  __syncthreads();
  for (int st = z0; st < z1; ++st) {
    const int buf = (st - z0) & 1;
    int pc1 = address(st + 1);
    asm volatile("" : "+v"(ka), "+v"(va), "+v"(sa), "+v"(pc1));   // (worked out from the lookups of the turn before: they are here now)
    // The tile in parts of 32 keys.  The matrix pipe takes 32 cycles for a product, in which the wave can issue eight other
    // instructions; so while one part's scores are made the weights of the part before are worked out, among its sums the next
    // part's weights, among the last sums the next tile's way to LDS -- two products and their share of the other work at a time,
    // in just this order (turn), the operand of a product read from LDS two turns ahead.
    const int j0 = base + st * KT;
    const bool work = j0 < hi_max && j0 + KT > lo_min;   // (else of no row of the wave)
    auto scores = [&](int nt, f16v& sc, auto beside) {
      const _Float16* kp = &sk[buf][(nt * 32 + c) * KLD + hf * 8];
      h8 a[2] = {*(const h8*)kp, *(const h8*)(kp + 16)}, b[2];
      if (QLDS) { b[0] = *(const h8*)mine; b[1] = *(const h8*)(mine + 16); }
#pragma unroll
      for (int e = 0; e < 16; ++e) sc[e] = 0.0f;
      turn();
#pragma unroll
      for (int k = 0; k < KSTEPS; ++k) {
        sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[k % 2], qh[k], sc, 0, 0, 0);
        sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[k % 2], QLDS ? b[k % 2] : ql[QLDS ? 0 : k], sc, 0, 0, 0);
        if (k + 2 < KSTEPS) {
          a[k % 2] = *(const h8*)(kp + (k + 2) * 16);
          if (QLDS) b[k % 2] = *(const h8*)(mine + (k + 2) * 16);
        }
        beside(k);
        turn();
      }
    };
    // (register e of the product: key 8 (e / 4) + 4 hf + e % 4)
    auto against = [&](int nt, f16v& sc, int pos) {   // the scores against the reference; the largest
      const int jn = j0 + nt * 32;
      float kf1 = 0.0f, lv1 = 0.0f;
      if (!FINE) { kf1 = skf[buf][nt] * kfac; lv1 = slv[buf][nt] - ref; }
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const int j4 = nt * 32 + 8 * b + 4 * hf;
        f4 kf = {kf1, kf1, kf1, kf1}, lv = {lv1, lv1, lv1, lv1};
        if (FINE) {
          kf = *(const f4*)&skf[buf][j4] * kfac;
          lv = *(const f4*)&slv[buf][j4];
#pragma unroll
          for (int e = 0; e < 4; ++e) lv[e] -= ref;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          sc[4 * b + e] = CAP ? sc[4 * b + e] * kf[e] : fmaf(sc[4 * b + e], kf[e], lv[e]);
          if (CAP) continue;
          if (BIAS) sc[4 * b + e] = fmaf(-slope, fabsf((float)(pos - (j0 + j4 + e))), sc[4 * b + e]);
        }
      }
      if (CAP) {
        float v[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = sc[e];
        cap_scores(v, cap2);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int j4 = nt * 32 + 8 * (e >> 2) + 4 * hf;
          sc[e] = v[e] + (FINE ? slv[buf][j4 + (e & 3)] - ref : lv1);
          if (BIAS) sc[e] = fmaf(-slope, fabsf((float)(pos - (j0 + j4 + (e & 3)))), sc[e]);
        }
      }
      if (jn < lo_max || jn + 32 > hi_min) {
        const int a = lo - (jn + 4 * hf), z = hi - (jn + 4 * hf);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int j = 8 * (e >> 2) + (e & 3);
          sc[e] = j >= a && j < z ? sc[e] : -INFINITY;
        }
      }
      float top = fmaxf(sc[0], sc[1]);
#pragma unroll
      for (int e = 2; e < 16; e += 2) top = fmaxf(fmaxf(top, sc[e]), sc[e + 1]);
      return top;
    };
    auto refer = [&](int nt, f16v& sc) {
      float top = against(nt, sc, pos);
      if (__any(top > limit)) {
        top = fmaxf(top, __shfl_xor(top, 32));
        const bool seen = limit > NOTHING;
        const float old = ref;
        // (Scores against a reference far below them are rounded to its distance, 2^-19 of an octave within 64 octaves of it.  Where a
        //  row is further off its scores are made again, against 0 as the first ones are.  With a cap the distance is two of it at
        //  most, and a score's error more than this.)
        const bool far = !CAP && seen && top > 56.0f;
        if (!CAP && __builtin_expect(__any(far), 0)) {
          const _Float16* kp = &sk[buf][(nt * 32 + c) * KLD + hf * 8];
#pragma unroll
          for (int e = 0; e < 16; ++e) sc[e] = 0.0f;
#pragma unroll
          for (int k = 0; k < KSTEPS; ++k) {
            const h8 a = *(const h8*)(kp + k * 16);
            sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, qh[k], sc, 0, 0, 0);
            sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, QLDS ? *(const h8*)(mine + k * 16) : ql[QLDS ? 0 : k], sc, 0, 0, 0);
            turn();
          }
          ref = far ? 0.0f : ref;
          limit = far ? NOTHING : limit;
          int p = pos;
          asm volatile("" : "+v"(p));   // (the distances worked out again: they do not fit beside the scores)
          top = against(nt, sc, p);
          top = fmaxf(top, __shfl_xor(top, 32));
        }
        const bool anew = top > limit;
        const float by = anew ? floorf(top) - SETS : 0.0f;   // (whole octaves: weights already made are brought along exactly)
        ref += by;
        const float f = seen ? exp2_f(old - ref) : 1.0f;   // (else nothing summed yet)
        limit = anew ? PASSES : limit;
        sum *= f;
#pragma unroll
        for (int d = 0; d < DT; ++d) acc[d] *= f;
#pragma unroll
        for (int e = 0; e < 16; ++e) sc[e] -= by;
        return f;
      }
      return 1.0f;
    };
    // Two weights of a part (of eight pairs); their sum apart from the row's: that is rounded once a part, like the sums of values, not
    // once a key, where it would lose what is 2^-25 of it however many keys there are.
    auto weigh = [&](int nt, const f16v& sc, int p, float iv1, h8 (&ph)[2], h8 (&pl)[2], float& part) {
      float2 iv;
      if (FINE) iv = *(const float2*)&siv[buf][nt * 32 + 8 * (p / 2) + 4 * hf + 2 * (p & 1)];
      else iv.x = iv.y = iv1;
      const float u = exp2_f(sc[2 * p]), w = exp2_f(sc[2 * p + 1]);
      part = p == 0 ? u * iv.x : fmaf(u, iv.x, part);
      part = fmaf(w, iv.y, part);
      h2 a, l;
      split2(u, w, one, a, l);
      const int k = p / 4, e = p % 4 * 2;
      ph[k][e] = a.x; ph[k][e + 1] = a.y; pl[k][e] = l.x; pl[k][e + 1] = l.y;
    };
    constexpr int SUMS = 2 * DT;
    auto add = [&](int nt, const h8 (&ph)[2], const h8 (&pl)[2], auto beside) {
      const _Float16* vp = &sv[buf][c * VLD + nt * 32 + hf * 8];
      auto at = [&](int i) { return *(const h8*)(vp + 16 * (i / DT) + (i % DT) * 32 * VLD); };
      h8 a[2] = {at(0), at(1)};
      turn();
#pragma unroll
      for (int i = 0; i < SUMS; ++i) {
        const int k = i / DT, d = i % DT;
        acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[i % 2], ph[k], acc[d], 0, 0, 0);
        acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[i % 2], pl[k], acc[d], 0, 0, 0);
        if (i + 2 < SUMS) a[i % 2] = at(i + 2);
        beside(i);
        turn();
      }
    };
    auto store_some = [&](int i) {   // (behind the last tile: bytes of the one before, which nobody reads)
#pragma unroll
      for (int u = i * UNITS / SUMS; u < (i + 1) * UNITS / SUMS; ++u) store(buf ^ 1, u);
    };
    if (work) {
      f16v s0, s1;
      h8 ph0[2], pl0[2], ph1[2], pl1[2];
      const float iv0 = FINE ? 0.0f : siv[buf][0], iv1 = FINE ? 0.0f : siv[buf][NT - 1];
      float sum0 = 0.0f, sum1 = 0.0f;
      scores(0, s0, [&](int k) {   // (the next tile's bytes, then the lookup for the one behind it)
        if (k < 4) load(k);
        if (k == 3) look(st + 2);
      });
      refer(0, s0);
      if (NT == 2) {
        scores(1, s1, [&](int k) {
#pragma unroll
          for (int p = k * 8 / KSTEPS; p < (k + 1) * 8 / KSTEPS; ++p) weigh(0, s0, p, iv0, ph0, pl0, sum0);
        });
        stay(ph0, pl0);
        sum += sum0;
        // (A reference set anew here lowers the first part's weights too, which are not in the sums yet.  2^-25 and less is 0 in f16,
        //  where a weight of 2^15 times it still is 2^-10: by 2^-24 first, then by the rest.  Both f16 are rounded by 2^-25 at most,
        //  together what a split cuts off.  Split anew from their f32 values, rows with a distance, whose reference moves with every
        //  tile, took 10 % longer.)
        const float f = refer(1, s1);
        if (__any(f != 1.0f)) {
          const _Float16 f1 = (_Float16)fmaxf(f, 0x1p-24f);
#pragma unroll
          for (int k = 0; k < 2; ++k) { ph0[k] *= f1; pl0[k] *= f1; }
          if (__any(f < 0x1p-24f)) {
            const _Float16 f2 = (_Float16)fminf(f * 0x1p24f, 1.0f);
#pragma unroll
            for (int k = 0; k < 2; ++k) { ph0[k] *= f2; pl0[k] *= f2; }
          }
        }
        add(0, ph0, pl0, [&](int i) {
#pragma unroll
          for (int p = i * 8 / SUMS; p < (i + 1) * 8 / SUMS; ++p) weigh(1, s1, p, iv1, ph1, pl1, sum1);
        });
        sum += sum1;
        arrive();
        add(1, ph1, pl1, store_some);
      } else {
#pragma unroll
        for (int p = 0; p < 8; ++p) weigh(0, s0, p, iv0, ph0, pl0, sum0);
        sum += sum0;
        arrive();
        add(0, ph0, pl0, store_some);
      }
    } else {
#pragma unroll
      for (int part = 0; part < 4; ++part) load(part);
      look(st + 2);
      arrive();
#pragma unroll
      for (int u = 0; u < UNITS; ++u) store(buf ^ 1, u);
    }
    store_scales(buf ^ 1, pc1);
    __syncthreads();
  }

  sum += __shfl_xor(sum, 32);
  if (limit == NOTHING) ref = NOTHING;
  // (pieces: the sums of each row, then its reference and its sum of weights)
  float* const piece = nsplit == 1 ? nullptr : ws + ((size_t)(sh * tiles + tile) * nsplit + blockIdx.y) * BM * (HD + 2);
  if (piece && r < M && hf == 0) {
    piece[BM * HD + 2 * (wave * 32 + c)] = ref;
    piece[BM * HD + 2 * (wave * 32 + c) + 1] = sum;
  }
  const float f = piece ? 1.0f : sum == 0.0f ? 0.0f : 1.0f / sum;
  float* const to = piece ? piece : out;
  const long place = r >= M ? -1 : piece ? (long)(wave * 32 + c) * HD : (long)(sq.r0 + i) * ldo + o_off + hq * HD;
  const bool whole16 = piece || (vec & 2);
  for (int cc = 0; cc < HD / 64; ++cc) {
#pragma unroll
    for (int d = 0; d < DT; ++d)
      if (d / 2 == cc) {
#pragma unroll
        for (int b = 0; b < 4; ++b)
          *(float4*)&pass[c * SLD + (d & 1) * 32 + 8 * b + 4 * hf] =
              sum == 0.0f ? make_float4(0.0f, 0.0f, 0.0f, 0.0f)
                          : make_float4(acc[d][4 * b] * f, acc[d][4 * b + 1] * f, acc[d][4 * b + 2] * f, acc[d][4 * b + 3] * f);
      }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      const long o = of_row(place, n);
      const float4 v = *(const float4*)&pass[(n * 4 + quarter) * SLD + col];
      if (o >= 0) {
        float* at = to + o + cc * 64 + col;
        if (whole16) {
          *(float4*)at = v;
        } else {
          at[0] = v.x; at[1] = v.y; at[2] = v.z; at[3] = v.w;
        }
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
    __builtin_amdgcn_wave_barrier();
  }
}

// -DFINE=1: blocks of less than 32 tokens; -DW8: work-groups of eight waves, 256 rows, one a compute unit: a tile is staged once for
// twice the rows (for blocks of 32 tokens and more: with a scale for each key its loop does not fit the registers)
#define MANY(NAME, HD, KT, NW, W, FINE, F)                                                                                                                      \
  extern "C" __global__ __launch_bounds__(64 * NW, W) void NAME(                                                                                                \
      const float* q, int ldq, int q_off, const int8_t* kq, const int8_t* vq, const float* ks, const float* vs, int pages, int ps, int bs, const int* rows,     \
      const int* lens, const int* table, int ldt, int T, int max_rows, int heads, int kvh, float* out, int ldo, int o_off, float scale, float cap2, int window, \
      const float* slopes, const int* prefix, const int* first, float* ws, int nsplit, int tiles, int vec) {                                                    \
    many_body<HD, KT, NW, FINE, (F & 1) != 0, (F & 2) != 0>(q, ldq, q_off, kq, vq, ks, vs, pages, ps, bs, rows, lens, table, ldt, T, max_rows, heads, kvh, out, \
                                                            ldo, o_off, scale, cap2, window, slopes, prefix, first, ws, nsplit, tiles, vec);                    \
  }
#define MANY4(HD, KT, NW, W, FINE, S)                              \
  MANY(attn_many__HD##HD##_FINE##FINE##_FORM0##S, HD, KT, NW, W, FINE, 0) \
  MANY(attn_many__HD##HD##_FINE##FINE##_FORM1##S, HD, KT, NW, W, FINE, 1) \
  MANY(attn_many__HD##HD##_FINE##FINE##_FORM2##S, HD, KT, NW, W, FINE, 2) \
  MANY(attn_many__HD##HD##_FINE##FINE##_FORM3##S, HD, KT, NW, W, FINE, 3)
MANY4(64, 64, 4, 2, 0, )
MANY4(64, 64, 4, 2, 1, )
MANY4(128, 32, 4, 2, 0, )
MANY4(128, 32, 4, 2, 1, )
MANY4(128, 64, 8, 2, 0, _W81)
MANY4(256, 32, 4, 1, 0, )
MANY4(256, 32, 4, 1, 1, )
