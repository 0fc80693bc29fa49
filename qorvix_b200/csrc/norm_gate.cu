// What lies between two sublayers, in one pass over the float32 residual stream: the norm on the sublayer's output y, its gate, its
// residual scale, the sum, and the norm the next sublayer reads; and rows in 8 bits for the products that follow.
//
//   z = y / rms(y) * w_post          (w_post null: y itself)
//   z = z * sigmoid(g + b)           (g null: no gate; b null: no bias)
//   z = z * s                        (s null: no scale)
//   stream' = stream + z             (y null: stream' = stream)
//   rows = stream' / rms(stream') * w_next, in float32, bfloat16 or 8 bits with a scale a row (w_next null: stream' itself)
//
// rms(v) = sqrt(mean(v^2) + eps).  Sums and everything between are float32.  8-bit rows are those of the bfloat16 rows, so that they do
// not depend on whether this pass or qv_quantize_rows made them.
#include "int8_rows.cuh"
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
__device__ __forceinline__ float sigmoid_of(float v) { return 1.0f / (1.0f + __expf(-v)); }
__device__ __forceinline__ float square_sum(float4 v) { return (v.x * v.x + v.y * v.y) + (v.z * v.z + v.w * v.w); }
__device__ __forceinline__ float4 mul(float4 a, float4 b) { return make_float4(a.x * b.x, a.y * b.y, a.z * b.z, a.w * b.w); }
__device__ __forceinline__ float4 mul(float4 a, float b) { return make_float4(a.x * b, a.y * b, a.z * b, a.w * b); }

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

// A block a row, FOURS groups of four entries a thread, in registers from the first load to the last store: each operand is read once and all
// loads of a row are in flight together (two sums over the row lie between them and the stores).  LONG: rows longer than four groups of
// 512 threads, of which the new stream is read back from where this thread stored it.
// OUT: 0 float32 rows, 1 bfloat16, 2 8-bit.
template <typename TY, typename TG, int OUT, int FOURS, bool ALIGNED, bool LONG>
__global__ void __launch_bounds__(FOURS == 4 ? 512 : 1024) norm_gate_kernel(const NormGateArgs a) {
  __shared__ float red[32];
  pdl_wait();
  pdl_launch_dependents();
  const int t = blockIdx.x, d = a.d, step = blockDim.x * 4;
  const float* sr = a.stream + (size_t)t * d;
  float* so = a.into + (size_t)t * d;
  const TY* yr = a.y ? (const TY*)a.y + (size_t)t * a.ld_y : nullptr;
  const TG* gr = a.gate ? (const TG*)a.gate + (size_t)t * a.ld_gate : nullptr;
  float4 x[FOURS], z[FOURS], g[FOURS];
  const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
  float post = 1.f, s2 = 0.f;
  // the new stream's entries from what was read
  auto add = [&](int i, float4 x, float4 z, float4 g) {
    if (!yr) return x;
    if (a.w_post) z = mul(mul(z, post), load_four<float, ALIGNED>(a.w_post, i, d));
    if (gr) {
      if (a.gate_bias) {
        const float4 b = load_four<float, ALIGNED>(a.gate_bias, i, d);
        g = make_float4(g.x + b.x, g.y + b.y, g.z + b.z, g.w + b.w);
      }
      z = mul(z, make_float4(sigmoid_of(g.x), sigmoid_of(g.y), sigmoid_of(g.z), sigmoid_of(g.w)));
    }
    if (a.scale) z = mul(z, load_four<float, ALIGNED>(a.scale, i, d));
    return make_float4(x.x + z.x, x.y + z.y, x.z + z.z, x.w + z.w);
  };
  const bool stores = yr != nullptr || so != sr;
  if (LONG) {
    if (yr && a.w_post) {
      float ss = 0.f;
      for (int i = threadIdx.x * 4; i < d; i += step) ss += square_sum(load_four<TY, ALIGNED>(yr, i, d));
      post = 1.0f / sqrtf(block_total(ss, red) / (float)d + a.eps_post);
    }
    for (int i = threadIdx.x * 4; i < d; i += step) {
      const float4 v = add(i, load_four<float, ALIGNED>(sr, i, d), yr ? load_four<TY, ALIGNED>(yr, i, d) : zero, gr ? load_four<TG, ALIGNED>(gr, i, d) : zero);
      if (stores) store_four<float, ALIGNED>(so, i, d, v);
      s2 += square_sum(v);
    }
  } else {
#pragma unroll
    for (int k = 0; k < FOURS; ++k) {
      const int i = threadIdx.x * 4 + k * step;
      const bool in = i < d;
      z[k] = in && yr ? load_four<TY, ALIGNED>(yr, i, d) : zero;
      x[k] = in ? load_four<float, ALIGNED>(sr, i, d) : zero;
      g[k] = in && gr ? load_four<TG, ALIGNED>(gr, i, d) : zero;
    }
    if (yr && a.w_post) {
      float ss = 0.f;
#pragma unroll
      for (int k = 0; k < FOURS; ++k) ss += square_sum(z[k]);
      post = 1.0f / sqrtf(block_total(ss, red) / (float)d + a.eps_post);
    }
#pragma unroll
    for (int k = 0; k < FOURS; ++k) {
      const int i = threadIdx.x * 4 + k * step;
      if (i < d) {
        x[k] = add(i, x[k], z[k], g[k]);
        if (stores) store_four<float, ALIGNED>(so, i, d, x[k]);
        s2 += square_sum(x[k]);
      }
    }
  }
  if (!a.out) return;
  const float next = a.w_next ? 1.0f / sqrtf(block_total(s2, red) / (float)d + a.eps_next) : 1.f;
  auto row = [&](int i, float4 v) { return a.w_next ? mul(mul(v, next), load_four<float, ALIGNED>(a.w_next, i, d)) : v; };
  auto rounded = [&](float4 v) {
    return make_float4(to_f(from_f<bf16>(v.x)), to_f(from_f<bf16>(v.y)), to_f(from_f<bf16>(v.z)), to_f(from_f<bf16>(v.w)));
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
  auto larger = [&](float4 v) { top = max(top, max(max(int8_bits(v.x), int8_bits(v.y)), max(int8_bits(v.z), int8_bits(v.w)))); };
  if (LONG) {
    for (int i = threadIdx.x * 4; i < d; i += step) larger(rounded(row(i, load_four<float, ALIGNED>(nr, i, d))));
  } else {
#pragma unroll
    for (int k = 0; k < FOURS; ++k) {
      const int i = threadIdx.x * 4 + k * step;
      if (i < d) {
        x[k] = rounded(row(i, x[k]));
        larger(x[k]);
      }
    }
  }
  const Int8Scale s = int8_scale(int8_block_top(top, (uint32_t*)red));
  if (threadIdx.x == 0) a.out_scale[t] = s.scale;
  int8_t* o = (int8_t*)a.out + (size_t)t * a.ld_out;
  auto put = [&](int i, float4 v) {
    float f[4] = {v.x, v.y, v.z, v.w};
    uint32_t w[1];
    int8_pack<true, 4>(f, s, w);
    if (i + 4 <= d) { *(uint32_t*)(o + i) = w[0]; return; }
    for (int k = 0; i + k < d; ++k) o[i + k] = (int8_t)(w[0] >> (8 * k));
  };
  if (LONG) {
    for (int i = threadIdx.x * 4; i < d; i += step) put(i, rounded(row(i, load_four<float, ALIGNED>(nr, i, d))));
  } else {
#pragma unroll
    for (int k = 0; k < FOURS; ++k) {
      const int i = threadIdx.x * 4 + k * step;
      if (i < d) put(i, x[k]);
    }
  }
}

template <typename TY, typename TG, int OUT, bool ALIGNED>
int launch_norm_gate(const NormGateArgs& a, int T, cudaStream_t st) {
  const int fours = (a.d + 3) / 4;
#define NORM_GATE_LAUNCH(FOURS, LONG, THREADS) return qv_launch(norm_gate_kernel<TY, TG, OUT, FOURS, ALIGNED, LONG>, dim3(T), dim3(THREADS), 0, st, a)
  if (fours > 2048) NORM_GATE_LAUNCH(1, true, 1024);
  if (T <= 296 && fours <= 1024) NORM_GATE_LAUNCH(1, false, (fours + 31) / 32 * 32);
  if (fours <= 512) NORM_GATE_LAUNCH(2, false, (fours + 63) / 64 * 32);
  NORM_GATE_LAUNCH(4, false, (fours + 127) / 128 * 32);
#undef NORM_GATE_LAUNCH
}

}  // namespace

// The pass at the head of this file.  stream, into [T, d] float32 contiguous (the same, or apart from each other); out_kind: 0 float32, 1 bfloat16,
// 2 8-bit rows with out_scale.
extern "C" int qv_norm_gate_add(const float* stream, float* into, const void* y, long long ld_y, int y_dt, const float* w_post, float eps_post,
                                const void* gate, long long ld_gate, int gate_dt, const float* gate_bias, const float* scale, const float* w_next,
                                float eps_next, void* out, long long ld_out, int out_kind, float* out_scale, int T, int d, void* cuda_stream) {
  if (T <= 0 || d <= 0) return 0;
  if ((out_kind == 2) != (out_scale != nullptr) || out_kind < 0 || out_kind > 2) return QV_ERR_UNSUPPORTED;
  NormGateArgs a;
  a.stream = stream; a.into = into; a.y = y; a.w_post = w_post; a.gate = gate; a.gate_bias = gate_bias; a.scale = scale; a.w_next = w_next;
  a.out = out; a.out_scale = out_scale; a.ld_y = ld_y; a.ld_gate = ld_gate; a.ld_out = ld_out; a.d = d; a.eps_post = eps_post; a.eps_next = eps_next;
  cudaStream_t st = (cudaStream_t)cuda_stream;
  const size_t ysz = y_dt == QV_DT_F32 ? 4 : 2, gsz = gate_dt == QV_DT_F32 ? 4 : 2;
  const uintptr_t wide = (uintptr_t)stream | (uintptr_t)into | (uintptr_t)w_post | (uintptr_t)gate_bias | (uintptr_t)scale | (uintptr_t)w_next;
  const size_t osz = out_kind == 0 ? 4 : out_kind == 1 ? 2 : 1;
  // groups of four on their own alignment (16 bytes of float32, 8 of bfloat16) in every operand
  const bool aligned = d % 4 == 0 && (wide & 15) == 0 && ((uintptr_t)y & (4 * ysz - 1)) == 0 && ld_y % 4 == 0 && ((uintptr_t)gate & (4 * gsz - 1)) == 0 &&
                       ld_gate % 4 == 0 && ((uintptr_t)out & (4 * osz - 1)) == 0 && ld_out % 4 == 0;
  if (out_kind == 2 && (((uintptr_t)out & 3) || (ld_out & 3))) return QV_ERR_UNSUPPORTED;
#define NORM_GATE_AS(TY, TG, OUT) return aligned ? launch_norm_gate<TY, TG, OUT, true>(a, T, st) : launch_norm_gate<TY, TG, OUT, false>(a, T, st)
#define NORM_GATE(TY, TG)                        \
  do {                                           \
    if (out_kind == 0) NORM_GATE_AS(TY, TG, 0);  \
    if (out_kind == 1) NORM_GATE_AS(TY, TG, 1);  \
    NORM_GATE_AS(TY, TG, 2);                     \
  } while (0)
  if (y_dt == QV_DT_F32 && gate_dt == QV_DT_F32) NORM_GATE(float, float);
  if (y_dt == QV_DT_F32 && gate_dt == QV_DT_BF16) NORM_GATE(float, bf16);
  if (y_dt == QV_DT_BF16 && gate_dt == QV_DT_F32) NORM_GATE(bf16, float);
  if (y_dt == QV_DT_BF16 && gate_dt == QV_DT_BF16) NORM_GATE(bf16, bf16);
#undef NORM_GATE
#undef NORM_GATE_AS
  return QV_ERR_UNSUPPORTED;
}
