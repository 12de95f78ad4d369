// What the attention block's kernels share: a batch's sequences, the cache in pages, eight-bit values as f16.
//
// Batch: rows [rows[s], rows[s + 1]) of the row buffers are the newest positions of sequence s, of which len[s] are in the
// cache with them; row i of the sequence has position len - n + i.  table[s][p >> log2(page)] is the page of position p.
// Cache: values int8 [pages][heads][page][hd], a scale f32 for each block of tokens and head [pages][heads][page / block];
// value = int8 * scale.  (A page's rows of one head are contiguous: what a work-group reads or writes is whole runs of 128
// bytes and more, and a token is appended without moving another.)
//
// Everything that comes from device memory -- rows, lengths, pages -- is held to the buffers before it addresses anything: rows
// to [0, T], lengths to the table, and a page outside the cache holds no tokens.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "attn_index.h"

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef float f16v __attribute__((ext_vector_type(16)));

using attn::Seq;
using attn::sees;
__device__ inline Seq seq_of(const int* __restrict__ rows, const int* __restrict__ lens, int s, int T, int max_rows, int most_len) {
  return attn::seq_at(rows[s], rows[s + 1], lens[s], T, max_rows, most_len);
}
__device__ inline int wave_id() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

__device__ inline float exp2_f(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ inline uint32_t perm(uint32_t hi, uint32_t lo, uint32_t sel) { return __builtin_amdgcn_perm(hi, lo, sel); }
// Eight-bit values as f16, exactly: with the sign bit turned over a byte is v + 128, behind 0x64 it is the f16 1024 + 128 + v.
__device__ inline h2 biased(uint32_t u) {
  h2 h;
  __builtin_memcpy(&h, &u, 4);
  return h - h2{(_Float16)1152.0f, (_Float16)1152.0f};
}
__device__ inline void cvt4(uint32_t w, h2& a, h2& b) {
  w ^= 0x80808080u;
  a = biased(perm(0x64646464u, w, 0x04010400u));
  b = biased(perm(0x64646464u, w, 0x04030402u));
}
__device__ inline h8 cvt8(uint32_t w0, uint32_t w1) {
  h2 a, b, c, d;
  cvt4(w0, a, b);
  cvt4(w1, c, d);
  return h8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}
// Four values of each of four tokens, token-major, to pairs of tokens for each value: p[v][0] = tokens 0 and 1, p[v][1] = 2 and 3.
__device__ inline void cvt4x4(uint32_t t0, uint32_t t1, uint32_t t2, uint32_t t3, h2 (&p)[4][2]) {
  t0 ^= 0x80808080u; t1 ^= 0x80808080u; t2 ^= 0x80808080u; t3 ^= 0x80808080u;
  const uint32_t a01 = perm(t1, t0, 0x05010400u), a23 = perm(t1, t0, 0x07030602u);
  const uint32_t b01 = perm(t3, t2, 0x05010400u), b23 = perm(t3, t2, 0x07030602u);
  p[0][0] = biased(perm(0x64646464u, a01, 0x04010400u));
  p[1][0] = biased(perm(0x64646464u, a01, 0x04030402u));
  p[2][0] = biased(perm(0x64646464u, a23, 0x04010400u));
  p[3][0] = biased(perm(0x64646464u, a23, 0x04030402u));
  p[0][1] = biased(perm(0x64646464u, b01, 0x04010400u));
  p[1][1] = biased(perm(0x64646464u, b01, 0x04030402u));
  p[2][1] = biased(perm(0x64646464u, b23, 0x04010400u));
  p[3][1] = biased(perm(0x64646464u, b23, 0x04030402u));
}
// ... of values 2 e and 2 e + 1 alone: p[v][0] = tokens 0 and 1, p[v][1] = 2 and 3.
__device__ inline void cvt4x2(uint32_t t0, uint32_t t1, uint32_t t2, uint32_t t3, int e, h2 (&p)[2][2]) {
  const uint32_t a = perm(t1, t0, e ? 0x07030602u : 0x05010400u) ^ 0x80808080u, b = perm(t3, t2, e ? 0x07030602u : 0x05010400u) ^ 0x80808080u;
  p[0][0] = biased(perm(0x64646464u, a, 0x04010400u));
  p[1][0] = biased(perm(0x64646464u, a, 0x04030402u));
  p[0][1] = biased(perm(0x64646464u, b, 0x04010400u));
  p[1][1] = biased(perm(0x64646464u, b, 0x04030402u));
}
// An f32 pair as two f16 pairs whose sum has 22 bits of it: the first truncated, the second what it misses.  `one` is 1.0 that the
// compiler does not know (opaque_one): the difference is then one instruction that takes the f16 as it is, not two.
__device__ inline float opaque_one() {
  float one;
  asm("v_mov_b32 %0, 1.0" : "=v"(one));
  return one;
}
__device__ inline void split2(float a, float b, float one, h2& hi, h2& lo) {
  auto h = __builtin_amdgcn_cvt_pkrtz(a, b);
  const float ra = fmaf(a, one, -(float)h[0]), rb = fmaf(b, one, -(float)h[1]);
  auto l = __builtin_amdgcn_cvt_pkrtz(ra, rb);
  __builtin_memcpy(&hi, &h, 4);
  __builtin_memcpy(&lo, &l, 4);
}

// ---- pieces that work-groups on other XCDs, with L2s of their own, write and read within one launch: stores that go through to
// memory (agent scope), waited for; a count of the work-groups that have come so far; loads past the
// caches.  Nothing else of a work-group's stores is read by another, so the L2s need not be written back or emptied (fences of
// agent scope, which do that, took 40 us of a launch of 512 work-groups that streams 270 MB).
struct Shared {
  __amdgpu_buffer_rsrc_t at;
  __device__ explicit Shared(float* p) : at(__builtin_amdgcn_make_buffer_rsrc(p, 0, -1, 0x00027000)) {}
  // (offsets in floats; 16: the agent's scope)
  __device__ void put4(int i, float4 v) const {
    u4 u;
    __builtin_memcpy(&u, &v, 16);
    __builtin_amdgcn_raw_buffer_store_b128(u, at, i * 4, 0, 16);
  }
  __device__ void put2(int i, float a, float b) const { __builtin_amdgcn_raw_buffer_store_b64(u2{__float_as_uint(a), __float_as_uint(b)}, at, i * 4, 0, 16); }
  __device__ float4 get4(int i) const {
    const u4 u = __builtin_amdgcn_raw_buffer_load_b128(at, i * 4, 0, 16);
    return make_float4(__uint_as_float(u.x), __uint_as_float(u.y), __uint_as_float(u.z), __uint_as_float(u.w));
  }
  __device__ float2 get2(int i) const {
    const u2 u = __builtin_amdgcn_raw_buffer_load_b64(at, i * 4, 0, 16);
    return make_float2(__uint_as_float(u.x), __uint_as_float(u.y));
  }
};
// True in the work-group that is the last of n to come here; the count is 0 again behind it.
__device__ inline bool last_of(unsigned* count, unsigned n) {
  __shared__ unsigned seen;
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
  __builtin_amdgcn_s_waitcnt(0);   // (this wave's stores have reached memory)
  __syncthreads();
  if (threadIdx.x == 0) {
    seen = __hip_atomic_fetch_add(count, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (seen == n - 1) __hip_atomic_store(count, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
  return seen == n - 1;
}

// ---- a score's form
// N scores over their cap, y, to cap tanh(y) log2(e) (cap2 = cap log2(e)).  Up to 1 as y times a quotient of polynomials (the continued
// fraction y / (1 + y^2 / (3 + y^2 / (5 + ...))) cut off behind its 9: 6e-8 of the value), so that a score's error is relative to the
// score; beyond as 1 - 2 / (1 + e^(2 y)), whose error is one of the cap (there an eighth of 2^-22 of it).
template <int N>
__device__ inline void cap_scores(float (&v)[N], float cap2) {
  auto near = [&](float y) {
    const float z = y * y;
    return (cap2 * y) * fmaf(z, z + 105.0f, 945.0f) * __builtin_amdgcn_rcpf(fmaf(z, fmaf(z, 15.0f, 420.0f), 945.0f));
  };
  float most = 0.0f;
#pragma unroll
  for (int e = 0; e < N; ++e) most = fmaxf(most, fabsf(v[e]));
  if (!__any(most >= 1.0f)) {
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = near(v[e]);
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float far = fmaf(-2.0f * cap2, __builtin_amdgcn_rcpf(1.0f + exp2_f(v[e] * 2.8853900817779268f)), cap2);
      v[e] = fabsf(v[e]) >= 1.0f ? far : near(v[e]);
    }
  }
}
// The scales' part in a score.  A weight is carried as w = p * vs (p = e^(s - reference), vs the scale of the token's values), as
// 2^(s log2(e) + log2(vs) - reference): the product with the scale costs no instruction of its own, the weights stay within a
// fixed range whatever the scales are, and the softmax's sum is the sum of w / vs.  A block of zeros (a scale below
// 2^-120) takes the smallest scale that this thread has met, 2^-60 at most, instead -- its values are zeros whatever it is: with a scale
// above the others' its weights could set the reference and leave the others' f16 nothing, with a smaller one they are small, and
// count in the sum alone, in f32.  A scale that is no number makes the score none, and its weight nothing where it is masked.
// Range of the sum: w <= 2^15 and 1 / vs.  Scales below 2^-97 are taken as 2^-97 (the values, below 127 * 2^-97 then, miss by at most that):
// 2^-97 leaves room for 2^15 keys of the largest weights, 2^21 of such as the reference is set for (with 2^-119 two of them overflow
// it), and a key beside others of scale 1 counts down to 2^-37 of their weight (with 2^-119 to 2^-15).  At the other end, with scales
// of 2^105 w / vs is a normal number down to 2^-29 of the largest weight.
__device__ inline void value_scale(float vs, float& low, float& lv, float& iv) {
  const bool number = vs == vs, holds = vs >= 0x1p-120f;
  const float s = fmaxf(vs, 0x1p-97f), l = __builtin_amdgcn_logf(s), r = __builtin_amdgcn_rcpf(s);
  low = holds ? fminf(low, l) : low;
  lv = holds ? l : number ? low : vs;
  iv = holds ? r : number ? exp2_f(-low) : 1.0f;
}
constexpr float LOW = -60.0f;
// The weights' reference is lowered so that the largest is at least 2^8 when it is set (2^8 for few rows, below 2^9 for many, whose
// reference moves by whole octaves); it is set anew once one would pass 2^15 (f16 ends at 2^16).  With the second f16 of the split,
// cut off at 2^-24, a weight keeps an absolute error of 2^-24, 2^-32 of the largest.
constexpr float SETS = 8.0f, PASSES = 15.0f;
constexpr float NOTHING = -0x1.fffffep127f;   // the reference before the first visible score: below every finite one
