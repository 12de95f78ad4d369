// "attn" module: rows of keys and values into the 8-bit cache, and back.
//
// A block of `block` tokens of one head shares a scale.  Where new rows fall into it:
//   top = max |x| over its new rows;  d = max(d_old, top / 127), d_old only if the block holds older tokens;  i = 1 / d (0 below
//   2^-120: such a block is zeros);  q = rte(x * i), held to +-127;  where d > d_old the older tokens' values become
//   rte(q * (d_old * i)).
// Each step is one f32 operation, so the stored bytes are defined to the last bit.  A row with an infinity or a NaN makes the
// block's scale NaN: everything read from the block is NaN until a row is written at the block's first position again.
//
// Mapping: a work-group has a tile of whole blocks (tile tokens, a power of two) of one head of one sequence, so no two
// work-groups touch a block and the result does not depend on their order.  hd / 4 threads take a row, four values each.
// Bound: 4 bytes of HBM read and one written a value; the rows stay in registers between the largest value and the rounding where a
// tile is at most eight rows a thread, else the second look at them comes from the L2.
// Measured: 8192 tokens x 8 heads x 128 values, columns of rows of 24 KB, written in 33.8 us from memory (2.5 TB/s), 19.6 us (4.3 TB/s) where
// the rows are still in the 256 MB behind the L2s, as those of a product just made are; read back behind that in 16.8 us (5.0
// TB/s); 48 tokens of as many sequences, 8 heads, 6.0 and 8.0 us, of which a launch and the chain row count -> page -> value are most.
#include "attn.h"

// NP passes of a tile are held in registers, so that a tile of that size is read once and all its loads are on their way at once;
// larger ones (long blocks) are read again from the L2.
template <int HD>
__device__ inline void kv_write_body(const float* __restrict__ x, int ld, int off, int8_t* __restrict__ q, float* __restrict__ d, int pages, int heads, int ps,
                                     int bs, const int* __restrict__ table, int ldt, const Seq& sq, int tile, int vec) {
  constexpr int TPR = HD / 4, RPP = 256 / TPR, NP = 8, CHUNK = RPP * NP;   // threads a row, rows a pass
  __shared__ uint32_t top[256];
  __shared__ float inv[256], ratio[256];
  __shared__ int page[256];   // a page for each 16 tokens at most
  const int h = blockIdx.z >> 1, lane = threadIdx.x % TPR, r0 = threadIdx.x / TPR, pm = (1 << ps) - 1;
  // (rows whose positions lie below 0 have no place)
  const int from = max(sq.p0, 0), to = sq.p0 + sq.n;
  const int t0 = attn::tile_at(from, to, tile, blockIdx.x), block = 1 << bs, nb = (tile + block - 1) >> bs, end = min(t0 + tile, to);
  if (t0 < 0) return;
  const int ntab = ((end - 1) >> ps) - (t0 >> ps) + 1;   // (at most tile / 16 + 1)
  for (int b = threadIdx.x; b < ntab; b += 256) page[b] = table[(t0 >> ps) + b];
  for (int b = threadIdx.x; b < nb; b += 256) top[b] = 0;
  float4 v[NP];
  auto load = [&](int c) {   // the rows of pass NP c ... that are new
#pragma unroll
    for (int k = 0; k < NP; ++k) {
      const int p = t0 + c * CHUNK + k * RPP + r0;
      v[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (p >= from && p < end) {
        const float* s = x + (size_t)(sq.r0 + p - sq.p0) * ld + off + h * HD + lane * 4;
        v[k] = vec ? *(const float4*)s : make_float4(s[0], s[1], s[2], s[3]);
      }
    }
  };
  const int chunks = (tile + CHUNK - 1) / CHUNK;
  load(0);
  __syncthreads();
  for (int c = 0; c < chunks; ++c) {
    if (c) load(c);
#pragma unroll
    for (int k = 0; k < NP; ++k) {
      // (sign off, the order of the words is that of the magnitudes, with infinity and NaN on top)
      uint32_t m = max(max(__float_as_uint(v[k].x) & 0x7FFFFFFFu, __float_as_uint(v[k].y) & 0x7FFFFFFFu),
                       max(__float_as_uint(v[k].z) & 0x7FFFFFFFu, __float_as_uint(v[k].w) & 0x7FFFFFFFu));
#pragma unroll
      for (int o = 1; o < TPR; o *= 2) m = max(m, (uint32_t)__shfl_xor((int)m, o));
      const int r = c * CHUNK + k * RPP + r0;
      if (lane == 0 && t0 + r >= from && t0 + r < end) atomicMax(&top[r >> bs], m);
    }
  }
  __syncthreads();
  const int old0 = from & -block;   // the first block's beginning: [old0, from) are older tokens
  auto row_of = [&](int p) {        // of a position's page: below 0 where that is none
    const int pg = page[(p >> ps) - (t0 >> ps)];
    return (uint32_t)pg < (uint32_t)pages ? (long)pg * heads + h : -1L;
  };
  for (int b = threadIdx.x; b < nb; b += 256) {
    const int p = t0 + (b << bs);
    inv[b] = 0.0f;
    ratio[b] = -1.0f;   // (nothing to do)
    if (p + block <= from || p >= end) continue;
    const long row = row_of(p);
    if (row < 0) continue;
    float* at = d + ((size_t)row << (ps - bs)) + ((p & pm) >> bs);
    const float now = top[b] >= 0x7F800000u ? __uint_as_float(0x7FC00000u) : __uint_as_float(top[b]) / 127.0f;
    const float was = p < from ? *at : 0.0f;
    const float s = was != was || now != now ? __uint_as_float(0x7FC00000u) : fmaxf(was, now);
    const float i = s >= 0x1p-120f ? 1.0f / s : 0.0f;
    inv[b] = i;
    if (s > was && p < from) ratio[b] = was * i;
    *at = s;
  }
  __syncthreads();
  auto byte = [](float v) { return (uint32_t)(int)fminf(fmaxf(__builtin_rintf(v), -127.0f), 127.0f) & 255u; };
  for (int c = 0; c < chunks; ++c) {
    if (chunks > 1) load(c);
#pragma unroll
    for (int k = 0; k < NP; ++k) {
      const int r = c * CHUNK + k * RPP + r0, p = t0 + r;
      if (p < from || p >= end) continue;
      const long row = row_of(p);
      const float i = inv[r >> bs];
      // (times 0 is a value's sign and zero; a block whose scale is NaN gets zeros)
      const uint32_t w = i > 0.0f ? byte(v[k].x * i) | byte(v[k].y * i) << 8 | byte(v[k].z * i) << 16 | byte(v[k].w * i) << 24 : 0u;
      if (row >= 0) ((uint32_t*)(q + (((size_t)row << ps) + (p & pm)) * HD))[lane] = w;
    }
  }
  // the older tokens of the first block, where its scale has grown
  const int b0 = max(old0, t0);
  if (b0 < from) {
    const float f = ratio[(b0 - t0) >> bs];
    const long row = row_of(b0);
    if (f >= 0.0f && row >= 0)
      for (int p = b0 + r0; p < from; p += RPP) {
        uint32_t* at = (uint32_t*)(q + (((size_t)row << ps) + (p & pm)) * HD) + lane;
        const uint32_t w = *at;
        uint32_t o = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) o |= byte((float)(int8_t)(w >> 8 * k) * f) << 8 * k;
        *at = o;
      }
  }
}

// grid (tiles of the most rows, sequences, 2 heads): even z the keys, odd the values.
template <int HD>
__device__ inline void kv_write_any(const float* k, int ldk, int k_off, const float* v, int ldv, int v_off, int8_t* kq, int8_t* vq, float* ks, float* vs, int pages,
                                    int heads, int ps, int bs, const int* rows, const int* lens, const int* table, int ldt, int T, int max_rows, int tile,
                                    int vec) {
  const int s = blockIdx.y;
  const Seq sq = seq_of(rows, lens, s, T, max_rows, ldt << ps);
  const bool second = blockIdx.z & 1;
  kv_write_body<HD>(second ? v : k, second ? ldv : ldk, second ? v_off : k_off, second ? vq : kq, second ? vs : ks, pages, heads, ps, bs, table + (size_t)s * ldt, ldt, sq,
                    tile, vec);
}
#define KV_WRITE(HD)                                                                                                                                          \
  extern "C" __global__ __launch_bounds__(256) void kv_write__HD##HD(const float* k, int ldk, int k_off, const float* v, int ldv, int v_off, int8_t* kq,      \
                                                                     int8_t* vq, float* ks, float* vs, int pages, int heads, int ps, int bs, const int* rows, \
                                                                     const int* lens, const int* table, int ldt, int T, int max_rows, int tile, int vec) {    \
    kv_write_any<HD>(k, ldk, k_off, v, ldv, v_off, kq, vq, ks, vs, pages, heads, ps, bs, rows, lens, table, ldt, T, max_rows, tile, vec);                     \
  }
KV_WRITE(64)
KV_WRITE(128)
KV_WRITE(256)

// Back to f32: rows of positions len - n + i.  A page that is none reads as zeros.  grid (ceil(max_rows / per), sequences, 2), a
// work-group `per` rows, a thread four values at a time, four times with all its loads on their way.
extern "C" __global__ __launch_bounds__(256) void kv_read(float* k, int ldk, int k_off, float* v, int ldv, int v_off, const int8_t* __restrict__ kq,
                                                          const int8_t* __restrict__ vq, const float* __restrict__ ks, const float* __restrict__ vs, int pages, int heads,
                                                          int hd, int ps, int bs, const int* __restrict__ rows, const int* __restrict__ lens,
                                                          const int* __restrict__ table, int ldt, int T, int max_rows, int per, int vec) {
  constexpr int N = 4;
  const int s = blockIdx.y, second = blockIdx.z;
  const Seq sq = seq_of(rows, lens, s, T, max_rows, ldt << ps);
  const int8_t* q = second ? vq : kq;
  const float* d = second ? vs : ks;
  float* out = second ? v : k;
  const int ld = second ? ldv : ldk, off = second ? v_off : k_off, w = heads * hd / 4, mask = (1 << ps) - 1;
  const int i0 = blockIdx.x * per, n = min(per, sq.n - i0);
  table += (size_t)s * ldt;
  for (int u0 = threadIdx.x; u0 < n * w; u0 += 256 * N) {
    int i[N], c[N], pg[N];
    uint32_t b[N];
    float f[N];
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const int u = min(u0 + 256 * e, n * w - 1);
      i[e] = u / w;
      c[e] = u - i[e] * w;
      pg[e] = table[max(sq.p0 + i0 + i[e], 0) >> ps];
    }
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const int p = max(sq.p0 + i0 + i[e], 0), h = 4 * c[e] / hd;
      const bool there = (uint32_t)pg[e] < (uint32_t)pages;
      const size_t row = (size_t)(there ? pg[e] : 0) * heads + h;
      b[e] = *(const uint32_t*)(q + ((row << ps) + (p & mask)) * hd + (4 * c[e] - h * hd));
      f[e] = d[(row << (ps - bs)) + ((p & mask) >> bs)];
      if (!there) { b[e] = 0; f[e] = 0.0f; }
    }
#pragma unroll
    for (int e = 0; e < N; ++e) {
      if (u0 + 256 * e >= n * w || sq.p0 + i0 + i[e] < 0) continue;
      const float4 o = make_float4((float)(int8_t)b[e] * f[e], (float)(int8_t)(b[e] >> 8) * f[e], (float)(int8_t)(b[e] >> 16) * f[e], (float)(int8_t)(b[e] >> 24) * f[e]);
      float* to = out + (size_t)(sq.r0 + i0 + i[e]) * ld + off + 4 * c[e];
      if (vec) {
        *(float4*)to = o;
      } else {
        to[0] = o.x; to[1] = o.y; to[2] = o.z; to[3] = o.w;
      }
    }
  }
}
