// The sine and cosine of a position's angle, kept as a 64-bit fraction of a turn (rope.hip says why).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

// (cos, sin) of turns / 2^64 of a turn
__device__ inline float2 cos_sin(uint64_t turns) {
  const uint32_t t = (uint32_t)(turns >> 32);
  const uint32_t q = (t + 0x20000000u) >> 30;
  const float x = (float)(int32_t)(t - (q << 30)) * (6.283185307179586f / 4294967296.0f);
  const float z = x * x;
  const float s = x * fmaf(z, fmaf(z, fmaf(z, fmaf(z, 1.0f / 362880.0f, -1.0f / 5040.0f), 1.0f / 120.0f), -1.0f / 6.0f), 1.0f);
  const float c = fmaf(z, fmaf(z, fmaf(z, fmaf(z, fmaf(z, -1.0f / 3628800.0f, 1.0f / 40320.0f), -1.0f / 720.0f), 1.0f / 24.0f), -0.5f), 1.0f);
  const float cc = q & 1 ? s : c, ss = q & 1 ? c : s;
  return make_float2(q == 1 || q == 2 ? -cc : cc, q == 2 || q == 3 ? -ss : ss);
}
