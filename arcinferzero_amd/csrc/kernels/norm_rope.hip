// "attn" module: norms of queries and keys, a head at a time, with the rotation by positions in the same pass.
//
//   n = x / sqrt(mean(x^2) + eps) * w  over the head's values, w the queries' weights for the first heads and the keys' for the rest;
//   y = n turned by the row's position (rope.hip: pairs, axes, angles), what lies behind the pairs as it is.
//
// Squares, their sums, the mean and its root are 64-bit, so that no finite head overflows or vanishes on the way; n is rounded to f32 twice, behind the root and
// behind the weight.  (With f32
// squares and the root's reciprocal in f32 the launches took the same: 777 tokens of 24 heads of 256 values 11.1 - 11.4 and 11.1 - 11.5 us, 8192 of 40 of
// 128 63.3 and 63.3.)
// Bound: 8 bytes of HBM a value.  A head's values stay in the registers of 8 to 64 lanes between the sum and the rotation, eight a lane (and
// four behind the pairs), so x is read once; a work-group takes all heads of some tokens, whose sines and cosines it works out once, as it
// brings the weights into LDS once.  Heads whose pairs are no multiple of four (of two, where neighbours) or longer ones go value by value,
// a wave each, and read x twice.
// Measured, 40 heads of 128 values (what rotation alone takes): 8192 tokens 63 us = 5.3 TB/s (63), 2500 23.6 (22), 777 10 (9), 256 4.8 (4.2), one 3.2 (3.0).
// Behind the launch itself short ones wait for HBM once and for the lanes' sums; four values brought in under a lane's condition, value by value, took
// 8192 tokens to 71 us, weights not held in LDS 777 to 12.  Value by value (29 pairs): 8192 tokens 158 us, 2.1 TB/s, 777 23, one 4.0.
#include "attn.h"
#include "turn.h"

constexpr int CS = 512;   // sines and cosines of a work-group's tokens
constexpr int WS = 768;   // a head's weights (64 lanes, twelve values each)

// 1 / sqrt(sum / hd + eps), to 2^-40 (the instruction's 2^-24 and one step); a head of zeros without eps stays zeros, and the finite values of
// one with an infinity are 0
__device__ inline double inverse_root(double sum, double per, float eps) {
  const double v = fma(sum, per, (double)eps), y = __builtin_amdgcn_rsq(v);
  return v == 0.0 || v == __builtin_inf() ? 0.0 : y * fma(-0.5 * v * y, y, 1.5);
}
__device__ inline float normed(float x, double f, float w) { return (float)((double)x * f) * w; }
__device__ inline void sines(float2* cs, const int* __restrict__ pos, int ld_pos, const uint64_t* __restrict__ tab, int pairs, int axes, float mscale, int t0, int nt) {
  const int* axis = (const int*)(tab + pairs);
  for (int i = threadIdx.x; i < nt * pairs; i += 256) {
    const int t = i / pairs, j = i - t * pairs;
    const int p = pos[(size_t)min(axis[j], axes - 1) * ld_pos + t0 + t];
    const float2 v = cos_sin((uint64_t)(int64_t)p * tab[j]);
    cs[i] = make_float2(v.x * mscale, v.y * mscale);
  }
}

// The sum of v over L lanes side by side, in each of them.  (Behind a step all lanes of a group have its sum, so that a row turned round
// brings another group's.)
template <int DPP>
__device__ inline double moved(double v) {
  const long long b = __double_as_longlong(v);
  const int lo = __builtin_amdgcn_update_dpp(0, (int)b, DPP, 0xF, 0xF, true), hi = __builtin_amdgcn_update_dpp(0, (int)(b >> 32), DPP, 0xF, 0xF, true);
  return __longlong_as_double((long long)(((unsigned long long)(unsigned)hi << 32) | (unsigned)lo));
}
__device__ inline double sum_of(double v, int L) {
  if (L > 1) v += moved<0xB1>(v);    // lanes 1, 0, 3, 2
  if (L > 2) v += moved<0x4E>(v);    // 2, 3, 0, 1
  if (L > 4) v += moved<0x141>(v);   // eight lanes turned round
  if (L > 8) v += moved<0x140>(v);   // sixteen
  if (L > 16) v += __shfl_xor(v, 16);
  if (L > 32) v += __shfl_xor(v, 32);
  return v;
}

// A head on L lanes (a power of two up to 64), four values at a time: columns ca and cb -- the halves of four pairs, or four neighbours each -- and cr behind
// the pairs.  x and y may be the same rows: a head is read before it is written, by its own lanes.
template <bool NB>
__device__ inline void norm_rope_lanes(const float* x, int ldx, int x_off, float* y, int ldy, int y_off, const float* __restrict__ wq, const float* __restrict__ wk, float eps,
                                       const int* __restrict__ pos, int ld_pos, const uint64_t* __restrict__ tab, int pairs, int axes, float mscale, int T, int nq, int heads,
                                       int hd, int tpw, int per, int L) {
  __shared__ __attribute__((aligned(16))) float2 cs[CS];
  __shared__ __attribute__((aligned(16))) float sw[2][WS];
  const int t0 = blockIdx.x * tpw, nt = min(tpw, T - t0), h0 = blockIdx.y * per, nh = min(per, heads - h0), units = nt * nh;
  const int lane = threadIdx.x & (L - 1), step = 256 / L;
  const int ca = 4 * lane, cb = NB ? ca + 4 * L : pairs + ca, cr = 2 * pairs + ca;
  const bool ha = ca < (NB ? hd : pairs), hb = NB ? cb < hd : ha, hr = !NB && cr < hd;
  const bool some_rest = 2 * pairs < hd;
  float4 a, b, r = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  auto load = [&](int u) {
    const int t = u / nh, h = u - t * nh;
    const float* src = x + (size_t)(t0 + t) * ldx + x_off + (size_t)(h0 + h) * hd;
    a = *(const float4*)(src + (ha ? ca : 0));   // (a lane without such columns: the head's first, which it does not count)
    b = *(const float4*)(src + (hb ? cb : 0));
    if (!NB && some_rest) r = *(const float4*)(src + (hr ? cr : 0));
  };
  int u = threadIdx.x / L;
  if (u < units) load(u);
  for (int i = threadIdx.x; i < hd; i += 256) {
    sw[0][i] = wq ? wq[i] : 1.0f;
    sw[1][i] = wk ? wk[i] : 1.0f;
  }
  sines(cs, pos, ld_pos, tab, pairs, axes, mscale, t0, nt);
  __syncthreads();
  const double per_value = 1.0 / hd;
  // (all lanes of a head go round together: L divides 64)
  for (; u < units; u += step) {
    const int t = u / nh, h = h0 + u - t * nh;
    double sum = 0.0;
    auto square = [&](const float4& v) {
      sum = fma((double)v.x, (double)v.x, sum);
      sum = fma((double)v.y, (double)v.y, sum);
      sum = fma((double)v.z, (double)v.z, sum);
      sum = fma((double)v.w, (double)v.w, sum);
    };
    if (ha) square(a);
    if (hb) square(b);
    if (hr) square(r);
    const double f = inverse_root(sum_of(sum, L), per_value, eps);
    auto times = [&](const float4& v) { return make_float4((float)(v.x * f), (float)(v.y * f), (float)(v.z * f), (float)(v.w * f)); };
    float4 na = times(a), nb = times(b), nr = times(r);
    const float* w = sw[h < nq ? 0 : 1];
    auto weigh = [&](float4& v, int c, bool has) {
      const float4 k = *(const float4*)(w + (has ? c : 0));
      v = make_float4(v.x * k.x, v.y * k.y, v.z * k.z, v.w * k.w);
    };
    weigh(na, ca, ha);
    weigh(nb, cb, hb);
    if (!NB) weigh(nr, cr, hr);
    if (u + step < units) load(u + step);
    float* dst = y + (size_t)(t0 + t) * ldy + y_off + (size_t)h * hd;
    const float2* c = cs + t * pairs;
    if (NB) {
      auto turned = [&](const float4& v, int col) {   // (pairs is a multiple of two)
        if (col >= 2 * pairs) return v;
        const float4 k = *(const float4*)(c + col / 2);
        return make_float4(v.x * k.x - v.y * k.y, v.x * k.y + v.y * k.x, v.z * k.z - v.w * k.w, v.z * k.w + v.w * k.z);
      };
      if (ha) *(float4*)(dst + ca) = turned(na, ca);
      if (hb) *(float4*)(dst + cb) = turned(nb, cb);
    } else {
      if (ha) {   // (pairs is a multiple of four)
        const float4 k = *(const float4*)(c + ca), l = *(const float4*)(c + ca + 2);
        *(float4*)(dst + ca) = make_float4(na.x * k.x - nb.x * k.y, na.y * k.z - nb.y * k.w, na.z * l.x - nb.z * l.y, na.w * l.z - nb.w * l.w);
        *(float4*)(dst + cb) = make_float4(na.x * k.y + nb.x * k.x, na.y * k.w + nb.y * k.z, na.z * l.y + nb.z * l.x, na.w * l.w + nb.w * l.z);
      }
      if (hr) *(float4*)(dst + cr) = nr;
    }
  }
}

// tab: as rope's.  grid ceil(T / tpw) x ceil(heads / per): tpw tokens and `per` heads to a work-group (one token, or all heads).  heads: queries and
// keys together, the first nq of them queries.  -DFORM: 0 halves, 1 neighbours, 2 value by value.
#define NORM_ROPE(F, BODY)                                                                                                                                       \
  extern "C" __global__ __launch_bounds__(256) void norm_rope__FORM##F(const float* x, int ldx, int x_off, float* y, int ldy, int y_off, const float* wq,       \
                                                                       const float* wk, float eps, const int* pos, int ld_pos, const uint64_t* tab, int pairs,  \
                                                                       int axes, int neighbours, float mscale, int T, int nq, int heads, int hd, int tpw,       \
                                                                       int per, int L) {                                                                        \
    BODY;                                                                                                                                                       \
  }
NORM_ROPE(0, norm_rope_lanes<false>(x, ldx, x_off, y, ldy, y_off, wq, wk, eps, pos, ld_pos, tab, pairs, axes, mscale, T, nq, heads, hd, tpw, per, L))
NORM_ROPE(1, norm_rope_lanes<true>(x, ldx, x_off, y, ldy, y_off, wq, wk, eps, pos, ld_pos, tab, pairs, axes, mscale, T, nq, heads, hd, tpw, per, L))

__device__ inline void norm_rope_values(const float* x, int ldx, int x_off, float* y, int ldy, int y_off, const float* __restrict__ wq, const float* __restrict__ wk, float eps,
                                        const int* __restrict__ pos, int ld_pos, const uint64_t* __restrict__ tab, int pairs, int axes, int neighbours, float mscale, int T,
                                        int nq, int heads, int hd, int tpw, int per) {
  __shared__ float2 cs[CS];
  const int t0 = blockIdx.x * tpw, nt = min(tpw, T - t0), h0 = blockIdx.y * per, nh = min(per, heads - h0), units = nt * nh;
  sines(cs, pos, ld_pos, tab, pairs, axes, mscale, t0, nt);
  __syncthreads();
  const int lane = threadIdx.x & 63;
  for (int u = wave_id(); u < units; u += 4) {
    const int t = u / nh, h = h0 + u - t * nh;
    const float* src = x + (size_t)(t0 + t) * ldx + x_off + (size_t)h * hd;
    float* dst = y + (size_t)(t0 + t) * ldy + y_off + (size_t)h * hd;
    const float* w = h < nq ? wq : wk;
    double sum = 0.0;
    for (int i = lane; i < hd; i += 64) sum = fma((double)src[i], (double)src[i], sum);
    const double f = inverse_root(sum_of(sum, 64), 1.0 / hd, eps);
    for (int i = lane; i < pairs; i += 64) {   // (a lane reads and writes its own pairs: x may be y)
      const int m = neighbours ? 2 * i : i, n = neighbours ? 2 * i + 1 : i + pairs;
      const float a = normed(src[m], f, w ? w[m] : 1.0f), b = normed(src[n], f, w ? w[n] : 1.0f);
      const float2 c = cs[t * pairs + i];
      dst[m] = a * c.x - b * c.y;
      dst[n] = a * c.y + b * c.x;
    }
    for (int i = 2 * pairs + lane; i < hd; i += 64) dst[i] = normed(src[i], f, w ? w[i] : 1.0f);
  }
}
NORM_ROPE(2, norm_rope_values(x, ldx, x_off, y, ldy, y_off, wq, wk, eps, pos, ld_pos, tab, pairs, axes, neighbours, mscale, T, nq, heads, hd, tpw, per))
