// "attn" module: rotary positions.
//
// Pair i of a head is turned by the angle pos[axis_i][t] * freq_i:  (a, b) -> (a cos - b sin, a sin + b cos) * mscale.
// A pair is (x[i], x[i + pairs]) or (x[2 i], x[2 i + 1]); what lies behind the pairs is copied.
//
// Angles: a position of 10^6 times a frequency of 1 has no correct digit of its sine left after an f32 product.  freq / 2 pi is
// kept as a 64-bit fraction of a turn instead, and position * fraction modulo 2^64 is the angle in turns, exact to 2^-64 times
// the position -- three integer products, whatever the position.  Its top two bits are the quadrant, the rest an angle of at
// most pi / 4 for the Taylor series of sine (to x^9, truncation 2e-9) and cosine (to x^10, 1e-10).
//
// Bound: 8 bytes of HBM a value; a work-group turns the heads of one token, whose sines and cosines it works out once into LDS (a head
// to a work-group would work them out again for each).  A token of few heads does not fill its work-group: 8192 tokens of 5 heads of 64
// values 8.4 us, 2.5 TB/s, of 10 of 128 15.2 us, 5.5 TB/s; several tokens a work-group were not tried.  Pairs that are no multiple of
// four (of two, where neighbours) go value by value, a division each.
// Measured (launches back to back): 4096 tokens x 48 heads x 128 values on three axes 38.9 us, 5.2 TB/s (a large copy: 4.9), 31
// where the rows are still in the 256 MB behind the L2s; 777
// tokens, half of each head turned, neighbours 6.5 us, 4.4 TB/s; one token 3.9 us, a launch's own time.
#include "attn.h"
#include "turn.h"

// tab: pairs words of 64 bits (the fractions), then `pairs` ints (the axes).  grid (T, ceil(heads / per)), local 256.
// vec: every offset and stride is a multiple of four values and every address of 16 bytes.
extern "C" __global__ __launch_bounds__(256) void rope(const float* x, int ldx, int x_off, float* y, int ldy, int y_off,
                                                       const int* __restrict__ pos, int ld_pos, const uint64_t* __restrict__ tab, int pairs, int axes,
                                                       int neighbours, float mscale, int heads, int hd, int per, int vec) {
  __shared__ float2 cs[512];
  const int t = blockIdx.x, h0 = blockIdx.y * per, nh = min(per, heads - h0);
  const int* axis = (const int*)(tab + pairs);
  const float* src = x + (size_t)t * ldx + x_off + (size_t)h0 * hd;
  float* dst = y + (size_t)t * ldy + y_off + (size_t)h0 * hd;
  for (int i = threadIdx.x; i < pairs; i += 256) {
    const int p = pos[(size_t)min(axis[i], axes - 1) * ld_pos + t];
    const float2 v = cos_sin((uint64_t)(int64_t)p * tab[i]);
    cs[i] = make_float2(v.x * mscale, v.y * mscale);
  }
  __syncthreads();
  const int rest = hd - 2 * pairs;
  if (vec && !neighbours && pairs % 4 == 0) {
    const int per_head = pairs / 4;
    for (int u = threadIdx.x; u < nh * per_head; u += 256) {
      const int h = u / per_head, i = (u - h * per_head) * 4;
      const float4 a = *(const float4*)(src + (size_t)h * hd + i), b = *(const float4*)(src + (size_t)h * hd + i + pairs);
      const float2 c0 = cs[i], c1 = cs[i + 1], c2 = cs[i + 2], c3 = cs[i + 3];
      *(float4*)(dst + (size_t)h * hd + i) =
          make_float4(a.x * c0.x - b.x * c0.y, a.y * c1.x - b.y * c1.y, a.z * c2.x - b.z * c2.y, a.w * c3.x - b.w * c3.y);
      *(float4*)(dst + (size_t)h * hd + i + pairs) =
          make_float4(a.x * c0.y + b.x * c0.x, a.y * c1.y + b.y * c1.x, a.z * c2.y + b.z * c2.x, a.w * c3.y + b.w * c3.x);
    }
  } else if (vec && neighbours && pairs % 2 == 0) {
    const int per_head = pairs / 2;
    for (int u = threadIdx.x; u < nh * per_head; u += 256) {
      const int h = u / per_head, i = (u - h * per_head) * 2;
      const float4 a = *(const float4*)(src + (size_t)h * hd + 2 * i);
      const float2 c0 = cs[i], c1 = cs[i + 1];
      *(float4*)(dst + (size_t)h * hd + 2 * i) =
          make_float4(a.x * c0.x - a.y * c0.y, a.x * c0.y + a.y * c0.x, a.z * c1.x - a.w * c1.y, a.z * c1.y + a.w * c1.x);
    }
  } else {
    for (int u = threadIdx.x; u < nh * pairs; u += 256) {
      const int h = u / pairs, i = u - h * pairs;
      const size_t at = (size_t)h * hd + (neighbours ? 2 * i : i), bt = at + (neighbours ? 1 : pairs);
      const float a = src[at], b = src[bt];
      const float2 c = cs[i];
      dst[at] = a * c.x - b * c.y;
      dst[bt] = a * c.y + b * c.x;
    }
  }
  if (rest > 0 && src != dst) {
    if (vec && rest % 4 == 0) {
      const int per_head = rest / 4;
      for (int u = threadIdx.x; u < nh * per_head; u += 256) {
        const int h = u / per_head;
        const size_t at = (size_t)h * hd + 2 * pairs + (u - h * per_head) * 4;
        *(float4*)(dst + at) = *(const float4*)(src + at);
      }
    } else {
      for (int u = threadIdx.x; u < nh * rest; u += 256) {
        const int h = u / rest;
        const size_t at = (size_t)h * hd + 2 * pairs + (u - h * rest);
        dst[at] = src[at];
      }
    }
  }
}
