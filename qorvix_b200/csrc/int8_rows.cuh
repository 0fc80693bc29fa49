// Rows in 8-bit integers: q_k = round(127 x_k / top), ties to the even one, and the scale top / 127, with top = max_k |x_k|.
//   top 0:           scale 0, q 0
//   top not finite:  scale NaN, q 0 (every product with the row is NaN, as it is in floating arithmetic)
// The quotient is the exact one: q does not depend on how a kernel forms it.  In float32 it is off by at most 2^-23 of itself, under
// 2e-5; only where it comes out nearer than 1e-4 to the border between two numbers is it decided in float64, where 127 |x| and
// (n + 1/2) top are both exact (31 and 32 bits).  What is rounded has then lost half a step of 1/127 of the row's largest entry, no more.
#pragma once
#include "common.cuh"

struct Int8Scale {
  float top, pre, inv;        // the largest magnitude and the entries times `pre`, a power of two that keeps 127 / top in range
  float scale;
  bool live;                  // false: all q are 0
};

__device__ __forceinline__ Int8Scale int8_scale(float top) {
  Int8Scale s;
  s.live = top > 0.f && top < __int_as_float(0x7f800000);
  s.scale = __fdiv_rn(top, 127.f);
  if (!(top < __int_as_float(0x7f800000))) s.scale = __int_as_float(0x7fffffff);
  s.pre = top < 0x1p-60f ? 0x1p64f : top > 0x1p60f ? 0x1p-64f : 1.f;
  s.top = top * s.pre;        // exact: entries that fall below the normal range are under 2^-60 of top
  s.inv = s.live ? __fdiv_rn(127.f, s.top) : 0.f;
  return s;
}

// The row's entry x (times s.pre), whose quotient v is next to a border.
__device__ __noinline__ float int8_border(float x, float v, float top) {
  const float lo = floorf(fabsf(v));
  const double a = 127.0 * (double)fabsf(x), h = ((double)lo + 0.5) * (double)top;
  const float r = a > h || (a == h && ((int)lo & 1)) ? lo + 1.f : lo;
  return copysignf(r, x);
}

__device__ __forceinline__ int int8_of(float x, const Int8Scale& s) {
  x *= s.pre;
  const float v = x * s.inv;
  float r = rintf(v);
  if (fabsf(v - r) > 0.4999f) r = int8_border(x, v, s.top);
  return s.live ? (int)r : 0;
}

__device__ __forceinline__ uint32_t int8_pack4(int a, int b, int c, int d) {
  return (uint32_t)(a & 255) | (uint32_t)(b & 255) << 8 | (uint32_t)(c & 255) << 16 | (uint32_t)d << 24;
}

// The largest of the magnitudes `bits` (of finite and infinite numbers and NaN alike: as unsigned numbers they are ordered, NaN on top),
// over the block.
__device__ __forceinline__ float int8_block_top(uint32_t bits, uint32_t* red /* >= 33 */) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nwarp = (blockDim.x + 31) >> 5;
  bits = __reduce_max_sync(0xffffffffu, bits);
  __syncthreads();
  if (lane == 0) red[warp] = bits;
  __syncthreads();
  uint32_t t = lane < nwarp ? red[lane] : 0u;
  return __uint_as_float(__reduce_max_sync(0xffffffffu, t));
}
