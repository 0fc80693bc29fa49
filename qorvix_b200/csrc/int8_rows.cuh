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

// Entries of a row as bytes, N of them (a multiple of 4) packed in words.  t = v + 1.5 2^23 holds round(v) in its low bits; v - round(v) says
// how near the border lies, and the whole group is looked at once.
template <int N>
__device__ __forceinline__ void int8_pack(const float (&x)[N], const Int8Scale& s, uint32_t (&out)[N / 4]) {
  constexpr float MAGIC = 12582912.f;
  float t[N], far = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float xi = x[i] * s.pre;
    t[i] = fmaf(xi, s.inv, MAGIC);
    far = fmaxf(far, fabsf(fmaf(xi, s.inv, MAGIC - t[i])));
  }
  if (far > 0.4999f) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float xi = x[i] * s.pre, v = xi * s.inv;
      if (fabsf(fmaf(xi, s.inv, MAGIC - t[i])) > 0.4999f) t[i] = MAGIC + int8_border(xi, v, s.top);
    }
  }
#pragma unroll
  for (int i = 0; i < N; i += 4) {
    const uint32_t lo = __byte_perm(__float_as_uint(t[i]), __float_as_uint(t[i + 1]), 0x0040);
    const uint32_t hi = __byte_perm(__float_as_uint(t[i + 2]), __float_as_uint(t[i + 3]), 0x0040);
    out[i / 4] = s.live ? __byte_perm(lo, hi, 0x5410) : 0u;
  }
}

// The largest magnitude's bits: of finite and infinite numbers and NaN alike, ordered as unsigned numbers, NaN on top.
__device__ __forceinline__ uint32_t int8_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// The largest of `bits` over the block's threads, as a float.
__device__ __forceinline__ float int8_block_top(uint32_t bits, uint32_t* red /* >= 32 */) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nwarp = (blockDim.x + 31) >> 5;
  bits = __reduce_max_sync(0xffffffffu, bits);
  if (nwarp == 1) return __uint_as_float(bits);
  __syncthreads();
  if (lane == 0) red[warp] = bits;
  __syncthreads();
  return __uint_as_float(__reduce_max_sync(0xffffffffu, lane < nwarp ? red[lane] : 0u));
}
