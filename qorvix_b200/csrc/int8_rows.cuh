// Rows in 8-bit integers: q_k = round(127 x_k / top), ties to the even one, and the scale top / 127, with top = max_k |x_k|.
//   top 0:           scale 0, q 0
//   top not finite:  scale NaN, q 0 (every product with the row is NaN, as it is in floating arithmetic)
// The quotient is the exact one: q does not depend on how a kernel forms it.  v = x * (127 / top) in float32 is off by at most 2^-21.4 of itself
// (2^-22 for the quotient of two steps' error that a thread works out for itself, half a step for it as a number, half for the product).
//   bfloat16 entries: 127 x / top = a / b with whole a up to 127 * 255 and b up to 255, times a power of two; where it is not a half-integer it
//     differs from every one by 2^-17 of itself or more.  So v rounded to 20 bits (half a step is 2^-21 of it or more, 2^-20 at most) is a
//     half-integer just where the quotient is one, and lies on the quotient's side of it elsewhere.  No entry needs a second look (one in 200 lies on a border; looking at those cost half
//     the time of a pass).
//   float32 entries: where v comes out nearer than 1e-4 to a border, the exact products decide.
// What is rounded has then lost half a step of 1/127 of the row's largest entry, no more.
#pragma once
#include "common.cuh"
#include <atomic>

struct Int8Scale {
  float top, pre, inv;        // the largest magnitude and the entries times `pre`, a power of two that keeps 127 / top in range
  bool live;                  // false: all q are 0
};

__device__ __forceinline__ Int8Scale int8_scale(float top) {
  Int8Scale s;
  s.live = top > 0.f && top < __int_as_float(0x7f800000);
  s.pre = top < 0x1p-60f ? 0x1p64f : top > 0x1p60f ? 0x1p-64f : 1.f;
  s.top = top * s.pre;        // exact: entries that fall below the normal range are under 2^-60 of top
  s.inv = s.live ? __fdividef(127.f, s.top) : 0.f;
  return s;
}
// What is kept beside the row: top / 127, of which the row's entries are whole multiples.
__device__ __forceinline__ float int8_step(float top) {
  return top < __int_as_float(0x7f800000) ? __fdiv_rn(top, 127.f) : __int_as_float(0x7fffffff);
}

// The row's entry x (times s.pre), whose quotient lies next to the border on the side d of the number r that t = r + 1.5 2^23 holds: whether it
// goes to r or to the next number on that side, as t.  With m = r +- 1/2, 127 x and m top differ by less than 2^-12 of themselves (by 1e-4 of a
// quotient of 1/2 or more); with p = m top rounded, both 127 x - p (fewer than 2^20 units of x's last place) and what p was rounded by come out of
// a multiply-add exactly, so their order is that of the two products.
__device__ __forceinline__ float int8_border(float x, float t, float d, float top) {
  const float m = (t - 12582912.f) + copysignf(0.5f, d);
  const float p = m * top, off = fmaf(m, top, -p), a = fmaf(127.f, x, -p);
  const bool beyond = d > 0.f ? a > off : a < off;
  return beyond || (a == off && (__float_as_uint(t) & 1u)) ? t + copysignf(1.f, d) : t;
}

// Two operations an instruction, each half rounded as the one it stands for.
union FloatPair { float2 f; unsigned long long u; };
__device__ __forceinline__ float2 fma_pair(float2 a, float2 b, float2 c) {
  FloatPair x{a}, y{b}, z{c}, r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.u) : "l"(x.u), "l"(y.u), "l"(z.u));
  return r.f;
}
__device__ __forceinline__ float2 mul_pair(float2 a, float2 b) {
  FloatPair x{a}, y{b}, r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.u) : "l"(x.u), "l"(y.u));
  return r.f;
}
__device__ __forceinline__ float2 add_pair(float2 a, float2 b) {
  FloatPair x{a}, y{b}, r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.u) : "l"(x.u), "l"(y.u));
  return r.f;
}

// Entries of a row as bytes, N of them (a multiple of 4) packed in words; BF16: they are bfloat16 numbers.  t = v + 1.5 2^23 holds round(v) in
// its low bits.  The instructions of this function are what bounds passes over many rows.
template <bool BF16, int N>
__device__ __forceinline__ void int8_pack(float (&x)[N], const Int8Scale& s, uint32_t (&out)[N / 4]) {
  constexpr float MAGIC = 12582912.f;
  if (!s.live) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) out[i] = 0u;
    return;
  }
  if (s.pre != 1.f) {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] *= s.pre;
  }
  float t[N], far = 0.f;
  const float2 inv = make_float2(s.inv, s.inv), magic = make_float2(MAGIC, MAGIC), minus = make_float2(-1.f, -1.f), split = make_float2(17.f, 17.f);
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    float2 v = make_float2(x[i], x[i + 1]), r;
    if (BF16) {
      v = mul_pair(v, inv);
      const float2 p = mul_pair(v, split);           // p - (p - v): v rounded to 20 bits
      r = add_pair(fma_pair(fma_pair(v, minus, p), minus, p), magic);
    } else {
      r = fma_pair(v, inv, magic);
      const float2 d = fma_pair(v, inv, fma_pair(r, minus, magic));
      far = fmaxf(far, fmaxf(fabsf(d.x), fabsf(d.y)));
    }
    t[i] = r.x;
    t[i + 1] = r.y;
  }
  if (!BF16 && far > 0.4999f) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float d = fmaf(x[i], s.inv, MAGIC - t[i]);
      if (fabsf(d) > 0.4999f) t[i] = int8_border(x[i], t[i], d, s.top);
    }
  }
#pragma unroll
  for (int i = 0; i < N; i += 4) {
    const uint32_t lo = __byte_perm(__float_as_uint(t[i]), __float_as_uint(t[i + 1]), 0x0040);
    const uint32_t hi = __byte_perm(__float_as_uint(t[i + 2]), __float_as_uint(t[i + 3]), 0x0040);
    out[i / 4] = __byte_perm(lo, hi, 0x5410);
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

// Streaming multiprocessors of the current device.
static inline int device_sms() {
  static std::atomic<int> known[64];
  int dev = 0, v = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 148;
  if (dev >= 0 && dev < 64 && (v = known[dev].load(std::memory_order_relaxed)) > 0) return v;
  if (cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || v <= 0) v = 148;
  if (dev >= 0 && dev < 64) known[dev].store(v, std::memory_order_relaxed);
  return v;
}
