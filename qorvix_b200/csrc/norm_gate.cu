// What lies between two sublayers, in one pass over the float32 residual stream: the norm on the sublayer's output y, its gate, its
// residual scale, the sum, and the norm the next sublayer reads; and rows in 8 bits for the products that follow.
//
//   z = y / rms(y) * w_post          (w_post null: y itself)
//   z = z * sigmoid(g + b)           (g null: no gate; b null: no bias)
//   z = z * s                        (s null: no scale)
//   stream' = stream + z             (y null: stream' = stream)
//   rows = stream' / rms(stream') * w_next, in float32, bfloat16 or 8 bits with a scale a row (w_next null: stream' itself)
//
// rms(v) = sqrt(mean(v^2) + eps).  Sums and everything between are float32.  A row's bits depend on the row and its operands alone, not on how
// many rows there are: which kernel takes them goes by their number, so all kernels form the same sums in the same order (row_total) and
// the same root.  8-bit rows are those of the bfloat16 rows, so that they do not depend on whether this pass or qv_quantize_rows made them.
#include "int8_rows.cuh"
#include "per_device.h"
#include "tc_common.cuh"
#include <type_traits>

namespace {

// ---------------------------------------------------------------- the pass between two sublayers
struct NormGateArgs {
  const float* stream;
  float* into;
  const void* y;
  const float* w_post;
  const void* gate;
  const float* gate_bias;
  const float* scale;
  const float* w_next;
  void* out;                 // rows; null: none
  float* out_scale;          // 8-bit rows
  long long ld_y, ld_gate, ld_out;
  int d;
  float inv_d;               // 1 / d
  float eps_post, eps_next;
};

// Four neighbouring entries.
template <typename T> struct Four;
template <> struct Four<float> {
  static __device__ __forceinline__ float4 load(const float* p) { return *(const float4*)p; }
  static __device__ __forceinline__ void store(float* p, float4 v) { *(float4*)p = v; }
};
template <> struct Four<bf16> {
  static __device__ __forceinline__ float4 load(const bf16* p) {
    const uint2 w = *(const uint2*)p;
    return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16), __uint_as_float(w.y & 0xffff0000u));
  }
  static __device__ __forceinline__ void store(bf16* p, float4 v) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
    *(uint2*)p = make_uint2(*(const uint32_t*)&a, *(const uint32_t*)&b);
  }
};
// The same of a row that ends at d, from pointers of any alignment.
template <typename T, bool ALIGNED> __device__ __forceinline__ float4 load_four(const T* p, int i, int d) {
  if (ALIGNED) return Four<T>::load(p + i);
  return make_float4(to_f(p[i]), i + 1 < d ? to_f(p[i + 1]) : 0.f, i + 2 < d ? to_f(p[i + 2]) : 0.f, i + 3 < d ? to_f(p[i + 3]) : 0.f);
}
template <typename T, bool ALIGNED> __device__ __forceinline__ void store_four(T* p, int i, int d, float4 v) {
  if (ALIGNED) { Four<T>::store(p + i, v); return; }
  p[i] = from_f<T>(v.x);
  if (i + 1 < d) p[i + 1] = from_f<T>(v.y);
  if (i + 2 < d) p[i + 2] = from_f<T>(v.z);
  if (i + 3 < d) p[i + 3] = from_f<T>(v.w);
}
// Arithmetic on two entries an instruction: over many rows the instructions are what bounds the pass next to memory.
__device__ __forceinline__ float2 lo2(float4 v) { return make_float2(v.x, v.y); }
__device__ __forceinline__ float2 hi2(float4 v) { return make_float2(v.z, v.w); }
__device__ __forceinline__ float4 both(float2 a, float2 b) { return make_float4(a.x, a.y, b.x, b.y); }
__device__ __forceinline__ float4 mul(float4 a, float4 b) { return both(mul_pair(lo2(a), lo2(b)), mul_pair(hi2(a), hi2(b))); }
__device__ __forceinline__ float4 mul(float4 a, float b) { return mul(a, make_float4(b, b, b, b)); }
__device__ __forceinline__ float4 fma(float4 a, float4 b, float4 c) { return both(fma_pair(lo2(a), lo2(b), lo2(c)), fma_pair(hi2(a), hi2(b), hi2(c))); }
__device__ __forceinline__ float4 add(float4 a, float b) { return both(add_pair(lo2(a), make_float2(b, b)), add_pair(hi2(a), make_float2(b, b))); }
__device__ __forceinline__ void add_squares(float2& s, float4 v) { s = fma_pair(hi2(v), hi2(v), fma_pair(lo2(v), lo2(v), s)); }
__device__ __forceinline__ float4 add(float4 a, float4 b) { return both(add_pair(lo2(a), lo2(b)), add_pair(hi2(a), hi2(b))); }
__device__ __forceinline__ float exp2_of(float v) { float r; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v)); return r; }
__device__ __forceinline__ float one_over(float v) { float r; asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v)); return r; }
// sigmoid(x) = 1 / (1 + exp(-x)), x = g + b rounded once, which moves it by |x| / 2 steps of 2^-23 at most; 0 from 2^-126 down.  float32 y: the accurate
// exponential, within a few steps.  bfloat16 y: 2^(-log2(e) x), whose argument's roundings move it by as many as |x| steps more, under 2^-16 of itself
// where it is not 0; y itself has lost up to 2^-9.  (us, 8,192 rows of 4,096, bfloat16 y and gate, 8-bit rows: 86, with the accurate exponential 96.)
template <typename TY> __device__ __forceinline__ float4 sigmoid_of(float4 g, float4 bias) {
  float4 x = add(g, bias), e;
  if (std::is_same<TY, float>::value) {
    e = make_float4(expf(-x.x), expf(-x.y), expf(-x.z), expf(-x.w));
  } else {
    x = mul(x, -1.4426950408889634f);
    e = make_float4(exp2_of(x.x), exp2_of(x.y), exp2_of(x.z), exp2_of(x.w));
  }
  e = add(e, 1.f);
  return make_float4(one_over(e.x), one_over(e.y), one_over(e.z), one_over(e.w));
}

// Sum over the block, the same in every thread; its order depends on the block's size alone.
__device__ __forceinline__ float block_total(float v, float* red /* >= 32 */) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nwarp = (blockDim.x + 31) >> 5;
  v = warp_sum(v);
  if (nwarp == 1) return v;
  __syncthreads();
  if (lane == 0) red[warp] = v;
  __syncthreads();
  return warp_sum(lane < nwarp ? red[lane] : 0.f);
}

// The sum of a row's squares, the same in every thread, for rows of up to 2,048 groups of four: `sums` threads add up the groups g, g + sums,
// ... in turn, then comes the tree over them.  FOURS 4: a thread holds just these groups.  FOURS 1: a thread a group; the groups meet in shared memory
// (`room`), where the first `sums` threads find theirs.  us, rows of 4,096 with a post norm and a gate, a thread a group: 1 row 2.9, 64 rows 3.8, as
// with a tree over the threads' own sums, which is another order; four groups a thread whatever the number of rows: 4.2 and 6.8.
__host__ __device__ __forceinline__ int sums_of(int fours) { return (fours + 127) / 128 * 32; }
template <int FOURS> __device__ __forceinline__ float row_total(const float4 (&v)[FOURS], int fours, float4* room, float* red /* >= 32 */) {
  float2 s = make_float2(0.f, 0.f);
  if (FOURS > 1) {
#pragma unroll
    for (int k = 0; k < FOURS; ++k) add_squares(s, v[k]);
    return block_total(s.x + s.y, red);
  }
  const int sums = sums_of(fours), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  room[threadIdx.x] = v[0];
  __syncthreads();
  if (threadIdx.x < sums) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (threadIdx.x + k * sums < fours) add_squares(s, room[threadIdx.x + k * sums]);
    const float t = warp_sum(s.x + s.y);
    if (lane == 0) red[warp] = t;
  }
  __syncthreads();
  return warp_sum(lane < sums / 32 ? red[lane] : 0.f);
}
__device__ __forceinline__ float one_over_rms(float total, float inv_d, float eps) { return rsqrtf(fmaf(total, inv_d, eps)); }

// What the row-wide operands hold beside one group of four: post is the norm's weight times the scale, bias the gate's; ones (a
// bias: zeros) stand for what there is not, which changes no bit.
struct Beside { float4 post, bias; };
struct NoGate {};                                            // in the place of the gate's type
__device__ __forceinline__ float4 four_of(float v) { return make_float4(v, v, v, v); }
template <typename TG, bool ALIGNED> __device__ __forceinline__ Beside beside(const NormGateArgs& a, int i) {
  Beside w;
  w.post = a.w_post ? load_four<float, ALIGNED>(a.w_post, i, a.d) : four_of(1.f);
  if (a.scale) w.post = mul(w.post, load_four<float, ALIGNED>(a.scale, i, a.d));
  if constexpr (!std::is_same<TG, NoGate>::value) w.bias = a.gate_bias ? load_four<float, ALIGNED>(a.gate_bias, i, a.d) : four_of(0.f);
  return w;
}
template <typename TG, bool ALIGNED> __device__ __forceinline__ float4 load_gate(const TG* g, int i, int d) {
  if constexpr (std::is_same<TG, NoGate>::value) return make_float4(0.f, 0.f, 0.f, 0.f);
  else return load_four<TG, ALIGNED>(g, i, d);
}
// The new stream's entries: x + z (times 1 / rms(y), and the norm's weight times the scale) (times the gate).
template <typename TY, typename TG> __device__ __forceinline__ float4 new_stream(float4 x, float4 z, float4 g, float inv_rms, const Beside& w) {
  z = mul(z, inv_rms);
  if constexpr (!std::is_same<TG, NoGate>::value) z = mul(z, sigmoid_of<TY>(g, w.bias));
  return fma(z, w.post, x);
}
__device__ __forceinline__ float4 rounded(float4 v) {
  return make_float4(to_f(from_f<bf16>(v.x)), to_f(from_f<bf16>(v.y)), to_f(from_f<bf16>(v.z)), to_f(from_f<bf16>(v.w)));
}
__device__ __forceinline__ uint32_t larger(uint32_t top, float4 v) { return max(top, max(max(int8_bits(v.x), int8_bits(v.y)), max(int8_bits(v.z), int8_bits(v.w)))); }
__device__ __forceinline__ void put_int8(int8_t* o, int i, int d, float4 v, const Int8Scale& s) {
  float f[4] = {v.x, v.y, v.z, v.w};
  uint32_t w[1];
  int8_pack<true, 4>(f, s, w);
  if (i + 4 <= d) { *(uint32_t*)(o + i) = w[0]; return; }
  for (int k = 0; i + k < d; ++k) o[i + k] = (int8_t)(w[0] >> (8 * k));
}

// A block a row, FOURS groups of four entries a thread, in registers from the first load to the last store: each operand is read once and all
// loads of a row are in flight together (two sums over the row lie between them and the stores).  LONG: rows longer than four groups of
// 512 threads, of which the new stream is read back from where this thread stored it.
// OUT: 0 float32 rows, 1 bfloat16, 2 8-bit.
template <typename TY, typename TG, int OUT, int FOURS, bool ALIGNED, bool LONG>
__global__ void __launch_bounds__(FOURS == 4 ? 512 : 1024) norm_gate_kernel(const NormGateArgs a) {
  __shared__ float red[32];
  __shared__ float4 room[FOURS == 1 && !LONG ? 1024 : 1];
  pdl_wait();
  pdl_launch_dependents();
  const int t = blockIdx.x, d = a.d, fours = (d + 3) / 4, step = blockDim.x * 4;
  const float* sr = a.stream + (size_t)t * d;
  float* so = a.into + (size_t)t * d;
  const TY* yr = a.y ? (const TY*)a.y + (size_t)t * a.ld_y : nullptr;
  const TG* gr = (const TG*)a.gate + (std::is_same<TG, NoGate>::value ? 0 : (size_t)t * a.ld_gate);
  float4 x[FOURS], z[FOURS], g[FOURS];
  const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
  float4 next_of_one = zero;
  float post = 1.f, total = 0.f;                     // total: of the new stream's squares
  const bool stores = yr != nullptr || so != sr;
  if (LONG) {
    if (yr && a.w_post) {
      float2 ss = make_float2(0.f, 0.f);
      for (int i = threadIdx.x * 4; i < d; i += step) add_squares(ss, load_four<TY, ALIGNED>(yr, i, d));
      post = one_over_rms(block_total(ss.x + ss.y, red), a.inv_d, a.eps_post);
    }
    float2 s2 = make_float2(0.f, 0.f);
    for (int i = threadIdx.x * 4; i < d; i += step) {
      float4 v = load_four<float, ALIGNED>(sr, i, d);
      if (yr) v = new_stream<TY, TG>(v, load_four<TY, ALIGNED>(yr, i, d), load_gate<TG, ALIGNED>(gr, i, d), post, beside<TG, ALIGNED>(a, i));
      if (stores) store_four<float, ALIGNED>(so, i, d, v);
      add_squares(s2, v);
    }
    total = block_total(s2.x + s2.y, red);
  } else {
#pragma unroll
    for (int k = 0; k < FOURS; ++k) {
      const int i = threadIdx.x * 4 + k * step;
      const bool in = i < d;
      z[k] = in && yr ? load_four<TY, ALIGNED>(yr, i, d) : zero;
      x[k] = in ? load_four<float, ALIGNED>(sr, i, d) : zero;
      g[k] = in ? load_gate<TG, ALIGNED>(gr, i, d) : zero;
    }
    Beside w[FOURS];                                 // of one group: on its way with the row, ahead of the sum
    float4 w_next = zero;
    if (FOURS == 1 && threadIdx.x * 4 < d) {
      w[0] = beside<TG, ALIGNED>(a, threadIdx.x * 4);
      if (a.w_next) w_next = load_four<float, ALIGNED>(a.w_next, threadIdx.x * 4, d);
    }
    next_of_one = w_next;
    if (yr && a.w_post) post = one_over_rms(row_total(z, fours, room, red), a.inv_d, a.eps_post);
#pragma unroll
    for (int k = 0; k < FOURS; ++k) {
      const int i = threadIdx.x * 4 + k * step;
      if (i < d) {
        if (yr) x[k] = new_stream<TY, TG>(x[k], z[k], g[k], post, FOURS == 1 ? w[0] : beside<TG, ALIGNED>(a, i));
        if (stores) store_four<float, ALIGNED>(so, i, d, x[k]);
      }
    }
    if (a.out && a.w_next) total = row_total(x, fours, room, red);
  }
  if (!a.out) return;
  const float next = a.w_next ? one_over_rms(total, a.inv_d, a.eps_next) : 1.f;
  auto row = [&](int i, float4 v) {
    return a.w_next ? mul(mul(v, next), FOURS == 1 && !LONG ? next_of_one : load_four<float, ALIGNED>(a.w_next, i, d)) : v;
  };
  const float* nr = stores ? so : sr;
  if (OUT != 2) {
    typedef typename std::conditional<OUT == 0, float, bf16>::type TO;
    TO* o = (TO*)a.out + (size_t)t * a.ld_out;
    if (LONG) {
      for (int i = threadIdx.x * 4; i < d; i += step) store_four<TO, ALIGNED>(o, i, d, row(i, load_four<float, ALIGNED>(nr, i, d)));
    } else {
#pragma unroll
      for (int k = 0; k < FOURS; ++k) {
        const int i = threadIdx.x * 4 + k * step;
        if (i < d) store_four<TO, ALIGNED>(o, i, d, row(i, x[k]));
      }
    }
    return;
  }
  uint32_t top = 0;
  if (LONG) {
    for (int i = threadIdx.x * 4; i < d; i += step) top = larger(top, rounded(row(i, load_four<float, ALIGNED>(nr, i, d))));
  } else {
#pragma unroll
    for (int k = 0; k < FOURS; ++k) {
      const int i = threadIdx.x * 4 + k * step;
      if (i < d) {
        x[k] = rounded(row(i, x[k]));
        top = larger(top, x[k]);
      }
    }
  }
  const float most = int8_block_top(top, (uint32_t*)red);
  const Int8Scale s = int8_scale(most);
  if (threadIdx.x == 0) a.out_scale[t] = int8_step(most);
  int8_t* o = (int8_t*)a.out + (size_t)t * a.ld_out;
  if (LONG) {
    for (int i = threadIdx.x * 4; i < d; i += step) put_int8(o, i, d, rounded(row(i, load_four<float, ALIGNED>(nr, i, d))), s);
  } else {
#pragma unroll
    for (int k = 0; k < FOURS; ++k) {
      const int i = threadIdx.x * 4 + k * step;
      if (i < d) put_int8(o, i, d, x[k], s);
    }
  }
}

// Many rows: memory bounds the pass, and the instructions nearly do, so an SM should never be without loads on the way and a thread should have
// little to do beside its entries.  As many blocks as the SMs hold walk over the rows; the row ahead of the one that a block works on comes
// into shared memory by bulk copies, a ring of `stages` of them (two; one where a row of three float32 operands fills the block's share), and
// the weights, which all rows share, stay in registers.  A row then costs two sums over the block (a barrier each) and its arithmetic, two
// entries an instruction.  Every row of every operand on 16 bytes and a multiple of them, rows of up to FOURS groups of THREADS threads, as many
// blocks on an SM as make 640 threads (768 with no gate and no 8-bit rows, which need fewer registers): one block's sums and stores run beside
// another's.
// us, 2,048 rows of 5,120, bfloat16 y and gate, captured calls over 300 MB in turn: bfloat16 rows 30.0 (4.9 TB/s), 8-bit rows 31.3; 8,192 rows of 4,096
// without a gate 69.0 and 62.4, 2,048 rows of 2,048 15.3 and 17.4.  Beside two groups a thread and scalar arithmetic, over less memory: 27.9 and 27.9, so
// 26.8 and 34.5 (8,192 rows of 4,096: 66.8 and 61.7, so 68.2 and 86.3; 2,048 rows of 2,048: 12.9 and 14.8, so 15.5 and 19.5); 53 with a block a row, which
// waits for its loads and its sums in turn.
// Two stages or six: 39.9 and 43.2 for rows of 8,192.
__device__ __forceinline__ float block_total_of(float v, float* red /* >= 32; read by all since this row's or the last row's barrier */) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nwarp = blockDim.x >> 5;
  v = warp_sum(v);
  if (lane == 0) red[warp] = v;
  __syncthreads();
  return warp_sum(lane < nwarp ? red[lane] : 0.f);
}
template <typename TG, int OUT> constexpr __host__ __device__ int rows_threads() { return std::is_same<TG, NoGate>::value && OUT != 2 ? 768 : 640; }   // on an SM
template <typename TY, typename TG, int OUT, int FOURS, int THREADS>
__global__ void __launch_bounds__(THREADS, rows_threads<TG, OUT>() / THREADS) norm_gate_rows_kernel(const NormGateArgs a, int T, int stages, int* err) {
  extern __shared__ __align__(128) uint8_t ring[];           // [stages][stream row | y row | gate row]
  __shared__ float red[4][32];                               // of the first sum, the second in rows of either parity, the maximum
  __shared__ uint64_t full[8];
  const int d = a.d, n4 = d / 4, step = blockDim.x;
  const bool has_y = a.y != nullptr, has_post = has_y && a.w_post, has_next = a.w_next != nullptr;
  const uint32_t x_bytes = d * 4, y_bytes = has_y ? d * (uint32_t)sizeof(TY) : 0, g_bytes = std::is_same<TG, NoGate>::value ? 0 : d * (uint32_t)sizeof(TG);
  const uint32_t stage_bytes = x_bytes + y_bytes + g_bytes;
  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) mbar_init(&full[s], 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  __syncthreads();
  pdl_launch_dependents();
  pdl_wait();
  auto fetch = [&](int t, int s) {                           // by thread 0
    uint8_t* dst = ring + s * stage_bytes;
    mbar_expect_tx(&full[s], stage_bytes);
    bulk_load_1d(dst, a.stream + (size_t)t * d, &full[s], x_bytes);
    if (y_bytes) bulk_load_1d(dst + x_bytes, (const TY*)a.y + (size_t)t * a.ld_y, &full[s], y_bytes);
    if (g_bytes) bulk_load_1d(dst + x_bytes + y_bytes, (const TG*)a.gate + (size_t)t * a.ld_gate, &full[s], g_bytes);
  };
  if (threadIdx.x == 0)
    for (int s = 0; s < stages; ++s)
      if (blockIdx.x + s * gridDim.x < T) fetch(blockIdx.x + s * gridDim.x, s);
  const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
  Beside w[FOURS];
  float4 wn[FOURS];
#pragma unroll
  for (int k = 0; k < FOURS; ++k) {
    const int i = threadIdx.x + k * step;
    w[k] = i < n4 ? beside<TG, true>(a, 4 * i) : Beside{zero, zero};
    wn[k] = i < n4 && has_next ? ((const float4*)a.w_next)[i] : four_of(1.f);
  }
  const bool stores = has_y || a.into != a.stream;
  typedef typename std::conditional<OUT == 0, float, typename std::conditional<OUT == 1, bf16, int8_t>::type>::type TO;
  float* into = a.into + (size_t)blockIdx.x * d + 4 * threadIdx.x;
  TO* out = (TO*)a.out + (size_t)blockIdx.x * a.ld_out + 4 * threadIdx.x;
  const size_t into_step = (size_t)gridDim.x * d, out_step = (size_t)gridDim.x * a.ld_out;
  bool ok = true;                                            // false: a wait gave up; the rest of this block's rows say nothing, and the error word does
  int s = 0, odd = 0;
  uint32_t parity = 0;
  for (int t = blockIdx.x; t < T; t += gridDim.x, into += into_step, out += out_step, odd ^= 1) {
    const uint8_t* row = ring + s * stage_bytes + 16 * threadIdx.x;
    const TY* y = (const TY*)(ring + s * stage_bytes + x_bytes) + 4 * threadIdx.x;
    const TG* g = (const TG*)(ring + s * stage_bytes + x_bytes + y_bytes) + 4 * (std::is_same<TG, NoGate>::value ? 0 : threadIdx.x);
    if (ok && !mbar_wait(&full[s], parity, err, 71)) {
      ok = false;
      if (threadIdx.x == 0)                                  // no copy outlives the block: the ones behind this have been asked for as well
        for (int n = s + 1; n < s + stages && t + (long long)(n - s) * gridDim.x < T; ++n) mbar_wait(&full[n % stages], parity ^ (n >= stages), err, 71);
    }
    float post = 1.f;
    float2 s2 = make_float2(0.f, 0.f);
    if (has_post) {
      float2 ss = make_float2(0.f, 0.f);
#pragma unroll
      for (int k = 0; k < FOURS; ++k)
        if (threadIdx.x + k * step < n4) add_squares(ss, Four<TY>::load(y + 4 * k * step));
      post = one_over_rms(block_total_of(ss.x + ss.y, red[0]), a.inv_d, a.eps_post);
    }
    float4 v[FOURS];
#pragma unroll
    for (int k = 0; k < FOURS; ++k) {
      v[k] = zero;
      if (threadIdx.x + k * step < n4) {
        v[k] = *(const float4*)(row + 16 * k * step);
        if (has_y) v[k] = new_stream<TY, TG>(v[k], Four<TY>::load(y + 4 * k * step), load_gate<TG, true>(g, 4 * k * step, d), post, w[k]);
        add_squares(s2, v[k]);
        if (stores) *(float4*)(into + 4 * k * step) = v[k];
      }
    }
    const float total = block_total_of(s2.x + s2.y, red[1 + odd]), next = has_next ? one_over_rms(total, a.inv_d, a.eps_next) : 1.f;
    if (threadIdx.x == 0 && ok && t + (long long)stages * gridDim.x < T) fetch(t + stages * gridDim.x, s);      // (behind the barrier: the row has been read)
    if (++s == stages) s = 0, parity ^= 1;
    if (!a.out) continue;
    uint32_t tops = 0;                                       // of the entries' 16 bits, two at a time
    uint2 h[FOURS];
#pragma unroll
    for (int k = 0; k < FOURS; ++k) {
      if (threadIdx.x + k * step < n4) {
        v[k] = mul(mul(v[k], next), wn[k]);
        if constexpr (OUT != 2) Four<TO>::store(out + 4 * k * step, v[k]);
        if constexpr (OUT == 2) {
          Four<bf16>::store((bf16*)&h[k], v[k]);
          tops = __vmaxu2(tops, __vmaxu2(h[k].x & 0x7fff7fffu, h[k].y & 0x7fff7fffu));
        }
      }
    }
    if constexpr (OUT == 2) {
      const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nwarp = blockDim.x >> 5;
      const uint32_t top = __reduce_max_sync(0xffffffffu, max(tops << 16, tops & 0xffff0000u));
      if (lane == 0) red[3][warp] = __uint_as_float(top);
      __syncthreads();
      const float most = __uint_as_float(__reduce_max_sync(0xffffffffu, lane < nwarp ? __float_as_uint(red[3][lane]) : 0u));
      const Int8Scale q = int8_scale(most);
      if (threadIdx.x == 0) a.out_scale[t] = int8_step(most);
#pragma unroll
      for (int k = 0; k < FOURS; ++k) {
        if (threadIdx.x + k * step < n4) {
          const float4 r = Four<bf16>::load((const bf16*)&h[k]);
          float f[4] = {r.x, r.y, r.z, r.w};
          uint32_t word[1];
          int8_pack<true, 4>(f, q, word);
          *(uint32_t*)(out + 4 * k * step) = word[0];
        }
      }
    }
  }
}

template <typename TY, typename TG, int OUT, int FOURS, int THREADS>
int launch_norm_gate_rows(const NormGateArgs& a, int T, int sms, int* err, cudaStream_t st) {
  static PerDevice devices;
  constexpr int ROOM = 216 * 1024;
  auto kernel = norm_gate_rows_kernel<TY, TG, OUT, FOURS, THREADS>;
  const int rc = qv_allow_smem(kernel, ROOM, devices);
  if (rc) return rc;
  static_assert(FOURS == 4, "sums_of");
  const int threads = sums_of(a.d / 4);
  constexpr int ON_SM = rows_threads<TG, OUT>();
  const int on_sm = ON_SM / threads > 10 ? 10 : ON_SM / threads, blocks = sms * on_sm;      // a stage is 192 bytes a thread at most: on_sm of them find room
  const size_t stage = (size_t)a.d * (4 + (a.y ? sizeof(TY) : 0) + (std::is_same<TG, NoGate>::value ? 0 : sizeof(TG)));
  int stages = (int)((size_t)ROOM / on_sm / stage);
  stages = stages > 2 ? 2 : stages;
  return qv_launch(kernel, dim3(T < blocks ? T : blocks), dim3(threads), stages * stage, st, a, T, stages, err);
}

template <typename TY, typename TG, int OUT, bool ALIGNED>
int launch_norm_gate(const NormGateArgs& a, int T, int* err, cudaStream_t st) {
  const int fours = (a.d + 3) / 4, sms = device_sms();
  // whole 16-byte pieces in every row that a bulk copy brings
  const bool pieces = ((uintptr_t)a.y & 15) == 0 && ((uintptr_t)a.gate & 15) == 0 && (a.d * sizeof(TY)) % 16 == 0 && (!a.gate || ((a.d * sizeof(TG)) % 16 == 0 && (a.ld_gate * sizeof(TG)) % 16 == 0)) &&
                      (a.ld_y * sizeof(TY)) % 16 == 0;
  // A block a row up to two rows an SM, where all rows are asked for at once; above, blocks that walk over rows.  us, a block a row / blocks that walk:
  // bfloat16 y and 8-bit rows, no gate, 150 rows of 2,048 3.0 / 3.3, 600 rows 6.1 / 5.0, 900 rows of 4,096 13.8 / 10.6; with a post norm and a float32 gate,
  // bfloat16 rows, 150 rows of 2,048 3.8 / 5.8, 600 rows 8.7 / 7.8, 900 rows of 4,096 22.1 / 16.8.  The number at which they are equal falls with the rows'
  // length (with a gate 1,000 rows of 1,024, 500 of 2,048, 150 of 4,096): 297 to 600 rows of 1,024 lose some 2 us by this rule.
  if (ALIGNED && pieces && T > 2 * sms && a.d <= 8192)
    return fours <= 256    ? launch_norm_gate_rows<TY, TG, OUT, 4, 64>(a, T, sms, err, st)
           : fours <= 640  ? launch_norm_gate_rows<TY, TG, OUT, 4, 160>(a, T, sms, err, st)
           : fours <= 1280 ? launch_norm_gate_rows<TY, TG, OUT, 4, 320>(a, T, sms, err, st)
                           : launch_norm_gate_rows<TY, TG, OUT, 4, 512>(a, T, sms, err, st);
#define NORM_GATE_LAUNCH(FOURS, LONG, THREADS) return qv_launch(norm_gate_kernel<TY, TG, OUT, FOURS, ALIGNED, LONG>, dim3(T), dim3(THREADS), 0, st, a)
  if (fours > 2048) NORM_GATE_LAUNCH(1, true, 1024);
  if (T <= 2 * sms && fours <= 1024) NORM_GATE_LAUNCH(1, false, (fours + 31) / 32 * 32);
  NORM_GATE_LAUNCH(4, false, sums_of(fours));
#undef NORM_GATE_LAUNCH
}

}  // namespace

// The pass at the head of this file.  stream, into [T, d] float32 contiguous (the same, or apart from each other); out_kind: 0 float32, 1 bfloat16,
// 2 8-bit rows with out_scale.
extern "C" int qv_norm_gate_add(const float* stream, float* into, const void* y, long long ld_y, int y_dt, const float* w_post, float eps_post,
                                const void* gate, long long ld_gate, int gate_dt, const float* gate_bias, const float* scale, const float* w_next,
                                float eps_next, void* out, long long ld_out, int out_kind, float* out_scale, int T, int d, int* err, void* cuda_stream) {
  if (T <= 0 || d <= 0) return 0;
  if ((out_kind == 2) != (out_scale != nullptr) || out_kind < 0 || out_kind > 2) return QV_ERR_UNSUPPORTED;
  NormGateArgs a;
  a.stream = stream; a.into = into; a.y = y; a.w_post = w_post; a.gate = gate; a.gate_bias = gate_bias; a.scale = scale; a.w_next = w_next;
  a.out = out; a.out_scale = out_scale; a.ld_y = ld_y; a.ld_gate = ld_gate; a.ld_out = ld_out; a.d = d; a.inv_d = 1.0f / (float)d; a.eps_post = eps_post; a.eps_next = eps_next;
  cudaStream_t st = (cudaStream_t)cuda_stream;
  const size_t ysz = y_dt == QV_DT_F32 ? 4 : 2, gsz = gate_dt == QV_DT_F32 ? 4 : 2;
  const uintptr_t wide = (uintptr_t)stream | (uintptr_t)into | (uintptr_t)w_post | (uintptr_t)gate_bias | (uintptr_t)scale | (uintptr_t)w_next;
  const size_t osz = out_kind == 0 ? 4 : out_kind == 1 ? 2 : 1;
  // groups of four on their own alignment (16 bytes of float32, 8 of bfloat16) in every operand
  const bool aligned = d % 4 == 0 && (wide & 15) == 0 && ((uintptr_t)y & (4 * ysz - 1)) == 0 && ld_y % 4 == 0 && ((uintptr_t)gate & (4 * gsz - 1)) == 0 &&
                       ld_gate % 4 == 0 && ((uintptr_t)out & (4 * osz - 1)) == 0 && ld_out % 4 == 0;
  if (out_kind == 2 && (((uintptr_t)out & 3) || (ld_out & 3))) return QV_ERR_UNSUPPORTED;
#define NORM_GATE_AS(TY, TG, OUT) return aligned ? launch_norm_gate<TY, TG, OUT, true>(a, T, err, st) : launch_norm_gate<TY, TG, OUT, false>(a, T, err, st)
#define NORM_GATE(TY, TG)                        \
  do {                                           \
    if (out_kind == 0) NORM_GATE_AS(TY, TG, 0);  \
    if (out_kind == 1) NORM_GATE_AS(TY, TG, 1);  \
    NORM_GATE_AS(TY, TG, 2);                     \
  } while (0)
  if (y_dt == QV_DT_F32 && !gate) NORM_GATE(float, NoGate);
  if (y_dt == QV_DT_BF16 && !gate) NORM_GATE(bf16, NoGate);
  if (y_dt == QV_DT_F32 && gate_dt == QV_DT_F32) NORM_GATE(float, float);
  if (y_dt == QV_DT_F32 && gate_dt == QV_DT_BF16) NORM_GATE(float, bf16);
  if (y_dt == QV_DT_BF16 && gate_dt == QV_DT_F32) NORM_GATE(bf16, float);
  if (y_dt == QV_DT_BF16 && gate_dt == QV_DT_BF16) NORM_GATE(bf16, bf16);
#undef NORM_GATE
#undef NORM_GATE_AS
  return QV_ERR_UNSUPPORTED;
}
