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
#include "per_device.h"

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

// OUT: 0 float32 rows, 1 bfloat16, 2 8-bit.
template <typename TY, typename TG, int OUT>
__global__ void __launch_bounds__(256) norm_gate_kernel(const NormGateArgs a) {
  extern __shared__ float xs[];                              // the row of the new stream
  __shared__ float red[33];
  pdl_wait();
  pdl_launch_dependents();
  const int t = blockIdx.x, d = a.d;
  const float* sr = a.stream + (size_t)t * d;
  float* so = a.into + (size_t)t * d;
  const TY* yr = a.y ? (const TY*)a.y + (size_t)t * a.ld_y : nullptr;
  const TG* gr = a.gate ? (const TG*)a.gate + (size_t)t * a.ld_gate : nullptr;
  float post = 1.f;
  if (yr && a.w_post) {
    float ss = 0.f;
    for (int i = threadIdx.x; i < d; i += blockDim.x) { const float v = to_f(yr[i]); ss = fmaf(v, v, ss); }
    post = 1.0f / sqrtf(block_sum(ss, red) / (float)d + a.eps_post);
  }
  float s2 = 0.f;
  for (int i = threadIdx.x; i < d; i += blockDim.x) {
    float x = sr[i];
    if (yr) {
      float z = to_f(yr[i]);
      if (a.w_post) z = z * post * a.w_post[i];
      if (gr) z = z / (1.0f + expf(-(to_f(gr[i]) + (a.gate_bias ? a.gate_bias[i] : 0.f))));
      if (a.scale) z *= a.scale[i];
      x += z;
      so[i] = x;
    } else if (so != sr) {
      so[i] = x;
    }
    xs[i] = x;
    s2 = fmaf(x, x, s2);
  }
  if (!a.out) return;
  const float next = a.w_next ? 1.0f / sqrtf(block_sum(s2, red) / (float)d + a.eps_next) : 1.f;
  uint32_t top = 0;
  for (int i = threadIdx.x; i < d; i += blockDim.x) {        // every thread reads back what it wrote itself
    const float v = a.w_next ? xs[i] * next * a.w_next[i] : xs[i];
    if (OUT == 0) ((float*)a.out)[(size_t)t * a.ld_out + i] = v;
    if (OUT == 1) ((bf16*)a.out)[(size_t)t * a.ld_out + i] = __float2bfloat16_rn(v);
    if (OUT == 2) {
      const float h = __bfloat162float(__float2bfloat16_rn(v));
      xs[i] = h;
      const uint32_t b = __float_as_uint(h) & 0x7fffffffu;
      top = b > top ? b : top;
    }
  }
  if (OUT == 2) {
    const Int8Scale s = int8_scale(int8_block_top(top, (uint32_t*)red));
    if (threadIdx.x == 0) a.out_scale[t] = s.scale;
    int8_t* o = (int8_t*)a.out + (size_t)t * a.ld_out;
    for (int i = threadIdx.x; i < d; i += blockDim.x) o[i] = (int8_t)int8_of(xs[i], s);
  }
}

template <typename TY, typename TG, int OUT>
int launch_norm_gate(const NormGateArgs& a, int T, cudaStream_t st) {
  const size_t smem = (size_t)a.d * sizeof(float);
  if (smem > 200 * 1024) return QV_ERR_TOO_LARGE;
  auto kernel = norm_gate_kernel<TY, TG, OUT>;
  if (smem > 48 * 1024) {
    static PerDevice devices;
    const int rc = qv_allow_smem(kernel, 200 * 1024, devices);
    if (rc) return rc;
  }
  return qv_launch(kernel, dim3(T), dim3(256), smem, st, a);
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
#define NORM_GATE(TY, TG)                                                          \
  do {                                                                             \
    if (out_kind == 0) return launch_norm_gate<TY, TG, 0>(a, T, st);               \
    if (out_kind == 1) return launch_norm_gate<TY, TG, 1>(a, T, st);               \
    return launch_norm_gate<TY, TG, 2>(a, T, st);                                  \
  } while (0)
  if (y_dt == QV_DT_F32 && gate_dt == QV_DT_F32) NORM_GATE(float, float);
  if (y_dt == QV_DT_F32 && gate_dt == QV_DT_BF16) NORM_GATE(float, bf16);
  if (y_dt == QV_DT_BF16 && gate_dt == QV_DT_F32) NORM_GATE(bf16, float);
  if (y_dt == QV_DT_BF16 && gate_dt == QV_DT_BF16) NORM_GATE(bf16, bf16);
#undef NORM_GATE
  return QV_ERR_UNSUPPORTED;
}
