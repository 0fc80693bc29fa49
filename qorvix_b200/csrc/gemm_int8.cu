// Products of 8-bit integers on the 5th-generation tensor cores (sm_100a): rows x of 8-bit integers with a scale each (int8_rows.cuh) times a
// matrix of such rows, one an output channel,
//   out[t, n] = (sum_k x[t, k] w[n, k]) * x_scale[t] * w_scale[n]
// The sum is whole: int32 accumulators in tensor memory (tcgen05.mma kind::i8), exact for K up to 131,071 whatever the order, so results
// do not depend on how the work is cut.  Forms: the sums as they are; a gated product, whose matrix alternates 16 gate rows and the 16 up
// rows of the same features; and either of them grouped by expert, where a table of tiles says which rows an expert's matrix multiplies.
//
// The matrix is packed in 16 KB tiles of 128 rows x 128 k, the shared-memory image the product reads (128-byte rows, 16-byte chunk c of
// row r at chunk c ^ (r % 8)), zero where the matrix ends.  It is the 128-row operand and the token rows are the narrow one, so that a
// thread of the epilogue holds one channel of many tokens, rows are padded to 16 only, and dense and grouped products are one kernel.
//
// One CTA per SM walks over items (a tile of rows, a block of 128 channels):
//   warp 0      weights by contiguous bulk copies, rows by TMA, through a ring of STAGES
//   warp 1      tcgen05.mma, accumulators double-buffered in tensor memory
//   warps 2..5  epilogue of the item before: scales, activation, stores
// Every wait is bounded; one that gives up records a code and the CTA winds down.
#include "int8_rows.cuh"
#include "per_device.h"
#include "tc_common.cuh"

#define QK 128                        // k entries of a stage: 128 bytes, one swizzle span
#define W_TILE_BYTES (BM * QK)

namespace {

// Instruction descriptor, kind::i8: D int32, A and B signed 8-bit, both K-major, 128 x n.
__device__ __forceinline__ uint32_t umma_idesc_i8(int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(BM >> 4) << 24);
}
__device__ __forceinline__ void umma_i8(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate) : "memory");
}

struct Int8Args {
  void* out;
  const float* x_scale;
  const uint8_t* w;                   // packed: [experts][NT][KT] tiles
  const float* w_scale;               // [experts][N]
  const int* tiles;                   // grouped: (expert or -1, first row, rows) of each tile of rows; null: dense
  int experts;
  int* err;
  long long ld_out;
  int rows, row_tiles, bn;            // dense: rows in all, tiles of them, rows of a tile (a multiple of 16); grouped: row_tiles is the table's length
  int box;                            // rows of a TMA box
  int N, K;
  GluAct glu;
};

// Dense items: tiles of rows fastest within bands of BAND of them, so that the CTAs at work share few weights and the rows of a band, which
// stay in L2; grouped: channels fastest, so that they share a tile's rows.
#define BAND 16
struct Item { int e, row0, rows, fb; };
__device__ __forceinline__ Item item_at(const Int8Args& p, int item, int NT) {
  Item it;
  if (p.tiles) {
    const int t = item / NT;
    it.fb = item - t * NT;
    it.e = p.tiles[3 * t]; it.row0 = p.tiles[3 * t + 1]; it.rows = p.tiles[3 * t + 2];
    if (it.rows > p.bn) it.rows = p.bn;              // (a table that was made for other tiles or other rows reads and writes nothing outside)
    if (it.rows > p.rows - it.row0) it.rows = p.rows - it.row0;
    if (it.e >= p.experts || it.row0 < 0 || it.rows <= 0) it.e = -1;
    return it;
  }
  const int band = item / (BAND * NT), in = item - band * BAND * NT;
  const int wide = p.row_tiles - band * BAND < BAND ? p.row_tiles - band * BAND : BAND;
  it.fb = in / wide;
  it.e = 0;
  it.row0 = (band * BAND + in - it.fb * wide) * p.bn;
  it.rows = p.rows - it.row0 < p.bn ? p.rows - it.row0 : p.bn;
  return it;
}


// The gated activations (see GluAct) as g / (1 + exp(-a)) * u: the tanh form of GELU too, 1 + tanh(x) = 2 / (1 + exp(-2 x)), which loses
// nothing where tanh is near -1.  Where the result is rounded to bfloat16 the fast exponential and quotient serve: their error, a few
// steps of 2^-23, vanishes in the rounding.
template <typename TO> __device__ __forceinline__ float gated(float g, float u, const GluAct& a) {
  float arg = g;
  if (a.kind == 1) arg = 1.5957691216057308f * fmaf(0.044715f * g * g, g, g);
  if (a.kind == 2) {
    g = fminf(g, a.limit);
    u = fminf(fmaxf(u, -a.limit), a.limit) + 1.f;
    arg = a.slope * g;
  }
  if (sizeof(TO) == 2) return __fdividef(g, 1.f + __expf(-arg)) * u;
  return g / (1.f + expf(-arg)) * u;
}

// GLU: a gated product.  TO: the output's type.  RT: rows of a tile at most.
template <bool GLU, typename TO, int RT, int STAGES>
__global__ void __launch_bounds__(192) int8_product_kernel(const __grid_constant__ CUtensorMap map_x, const Int8Args p) {
  extern __shared__ uint8_t smem_raw[];
  constexpr int STAGE_BYTES = W_TILE_BYTES + RT * QK;
  constexpr int TMEM_COLS = 2 * RT < 32 ? 32 : 2 * RT;
  uint8_t* ring = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  float* scales = (float*)(ring + STAGES * STAGE_BYTES);       // [4 warps][RT]: the rows' scales
  uint64_t* full = (uint64_t*)(scales + 4 * RT);
  uint64_t* empty = full + STAGES;
  uint64_t* acc_full = empty + STAGES;               // [2]
  uint64_t* acc_empty = acc_full + 2;                // [2]
  uint32_t* tmem_slot = (uint32_t*)(acc_empty + 2);
  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
    for (int b = 0; b < 2; ++b) { mbar_init(&acc_full[b], 1); mbar_init(&acc_empty[b], 128); }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(TMEM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_launch_dependents();
  pdl_wait();                                        // the rows, the tile table and the output belong to the kernels ahead until here
  const int NT = (p.N + BM - 1) / BM, KT = (p.K + QK - 1) / QK;
  const int items = p.row_tiles * NT;

  if (warp == 0) {
    const bool leader = elect_one();
    int it = 0;
    bool ok = true;
    for (int item = blockIdx.x; ok && item < items; item += gridDim.x) {
      const Item w = item_at(p, item, NT);
      if (w.e < 0) break;
      const int boxes = (w.rows + p.box - 1) / p.box;
      const uint8_t* src = p.w + ((size_t)w.e * NT + w.fb) * KT * W_TILE_BYTES;
      for (int kb = 0; kb < KT; ++kb, ++it) {
        const int s = it % STAGES;
        if (!mbar_wait(&empty[s], ((it / STAGES) & 1) ^ 1, p.err, 61)) { ok = false; break; }
        if (leader) {
          uint8_t* dst = ring + s * STAGE_BYTES;
          mbar_expect_tx(&full[s], W_TILE_BYTES + boxes * p.box * QK);
          bulk_load_1d(dst, src + (size_t)kb * W_TILE_BYTES, &full[s], W_TILE_BYTES);
          for (int x = 0; x < boxes; ++x) tma_load_2d(dst + W_TILE_BYTES + x * p.box * QK, &map_x, &full[s], kb * QK, w.row0 + x * p.box);
        }
        __syncwarp();
      }
    }
    // after a wait that gave up: the copies in flight land before the CTA's shared memory goes to another
    if (!ok)
      for (int i = it < STAGES ? 0 : it - STAGES; i < it; ++i) mbar_wait(&full[i % STAGES], (i / STAGES) & 1, p.err, 65);
  } else if (warp == 1) {
    const bool leader = elect_one();                 // the whole warp walks the loop and waits, an elected lane issues
    int it = 0, local = 0;
    bool ok = true;
    for (int item = blockIdx.x; ok && item < items; item += gridDim.x, ++local) {
      const Item w = item_at(p, item, NT);
      if (w.e < 0) break;
      const uint32_t idesc = umma_idesc_i8((w.rows + 15) & ~15);
      const int b = local & 1;
      ok = mbar_wait(&acc_empty[b], ((local >> 1) & 1) ^ 1, p.err, 64);
      if (!ok) break;
      tc_fence_after();
      const uint32_t d_tmem = tmem_base + (uint32_t)(b * RT);
      for (int kb = 0; kb < KT; ++kb, ++it) {
        const int s = it % STAGES;
        ok = mbar_wait(&full[s], (it / STAGES) & 1, p.err, 62);
        if (!ok) break;
        tc_fence_after();
        const uint32_t a_addr = smem_u32(ring + s * STAGE_BYTES);
        const uint64_t da = umma_desc(a_addr), db = umma_desc(a_addr + W_TILE_BYTES);
        if (leader) {
#pragma unroll
          for (int kk = 0; kk < QK / 32; ++kk)       // 32 entries of k a product: 32 bytes, 2 descriptor units
            umma_i8(d_tmem, da + 2 * kk, db + 2 * kk, idesc, (kb > 0 || kk > 0) ? 1u : 0u);
          umma_commit(&empty[s]);
        }
        __syncwarp();
      }
      if (leader) umma_commit(&acc_full[b]);
      __syncwarp();
    }
  } else {
    const int q = warp & 3;                          // tensor memory lanes 32 q .. + 31
    float* xs = scales + q * RT;
    int local = 0;
    for (int item = blockIdx.x; item < items; item += gridDim.x, ++local) {
      const Item w = item_at(p, item, NT);
      if (w.e < 0) break;
      const int ch = w.fb * BM + q * 32 + lane;      // this thread's channel
      const float ws = ch < p.N ? p.w_scale[(size_t)w.e * p.N + ch] : 0.f;
      __syncwarp();
#pragma unroll
      for (int i = 0; i < RT; i += 32)
        if (i + lane < RT) xs[i + lane] = i + lane < w.rows ? p.x_scale[w.row0 + i + lane] : 0.f;
      __syncwarp();
      const int b = local & 1;
      if (!__all_sync(0xffffffffu, mbar_wait(&acc_full[b], (local >> 1) & 1, p.err, 63))) break;     // (the MMA warp then gives up too)
      tc_fence_after();
      const uint32_t taddr = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(b * RT);
      const int feat = GLU ? w.fb * 64 + q * 16 + (lane & 15) : ch;
      const bool there = GLU ? 2 * feat < p.N : ch < p.N;
      TO* out = (TO*)p.out + (size_t)w.row0 * p.ld_out + feat;
#pragma unroll 1
      for (int c0 = 0; c0 < w.rows; c0 += 16) {
        uint32_t r[16];
        tmem_ld16(taddr + c0, r);
        tmem_wait_ld();
        float v[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] = (float)(int)r[j] * xs[c0 + j] * ws;
        if (GLU) {
          // a lane of the lower half gives its gate value of the odd row for the up value of the even row
          const int up = lane >> 4;
#pragma unroll
          for (int j = 0; j < 16; j += 2) {
            const float got = __shfl_xor_sync(0xffffffffu, up ? v[j] : v[j + 1], 16);
            const float g = up ? got : v[j], u = up ? v[j + 1] : got;
            const int row = c0 + j + up;
            if (row < w.rows && there) out[(size_t)row * p.ld_out] = from_f<TO>(gated<TO>(g, u, p.glu));
          }
        } else if (there) {
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (c0 + j < w.rows) out[(size_t)(c0 + j) * p.ld_out] = from_f<TO>(v[j]);
        }
        __syncwarp();
      }
      tc_fence_before();
      mbar_arrive(&acc_empty[b]);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS) : "memory");
  }
}

// ---------------------------------------------------------------- rows in 8 bits
// One read and one write of the row are all it cannot do without, so a row stays in registers between its maximum and its rounding: VECS
// pieces of 16 bytes a thread, all asked for at once.  A row has a block of its own, whose size goes by the row's length; rows longer than
// VECS pieces of 1,024 threads are read twice (LONG).  ALIGNED: pieces lie on 16 bytes; else their entries are read one by one.
template <typename T> struct Piece { static constexpr int N = 16 / (int)sizeof(T); };
template <typename T, bool ALIGNED>
__device__ __forceinline__ void load_piece(float (&f)[Piece<T>::N], const T* x, int k, int K) {
  constexpr int N = Piece<T>::N;
  if (ALIGNED && k + N <= K) {
    const uint4 v = *(const uint4*)(x + k);
    const T* e = (const T*)&v;
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = to_f(e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = k + i < K ? to_f(x[k + i]) : 0.f;
  }
}
template <int N>
__device__ __forceinline__ void store_piece(int8_t* q, const float (&f)[N], const Int8Scale& s, int k, int K) {
  uint32_t w[N / 4];
  int8_pack<N>(f, s, w);
  if (k + N <= K) {
    if (N == 8) *(uint2*)(q + k) = make_uint2(w[0], w[N / 4 - 1]);
    else *(uint32_t*)(q + k) = w[0];
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (k + i < K) q[k + i] = (int8_t)(w[i / 4] >> (8 * (i & 3)));
  }
}

template <typename T, int VECS, bool ALIGNED, bool LONG>
__global__ void __launch_bounds__(1024) quantize_rows_kernel(int8_t* __restrict__ q, long long ld_q, float* __restrict__ scale, const T* __restrict__ x,
                                                             long long ld_x, const int* __restrict__ row_idx, int rows_in, int K) {
  constexpr int N = Piece<T>::N;
  __shared__ uint32_t red[32];
  pdl_wait();
  pdl_launch_dependents();
  const int r = blockIdx.x, step = blockDim.x * N;
  const int src = row_idx ? row_idx[r] : r;
  const bool there = (unsigned)src < (unsigned)rows_in;      // an index outside the rows: a row of zeros
  const T* xr = x + (size_t)(there ? src : 0) * ld_x;
  const int n = there ? K : 0;
  int8_t* o = q + (size_t)r * ld_q;
  float f[VECS][N];
  uint32_t top = 0;
  if (LONG) {
    for (int k = threadIdx.x * N; k < n; k += step) {
      load_piece<T, ALIGNED>(f[0], xr, k, n);
#pragma unroll
      for (int i = 0; i < N; ++i) top = max(top, int8_bits(f[0][i]));
    }
  } else {
#pragma unroll
    for (int v = 0; v < VECS; ++v) load_piece<T, ALIGNED>(f[v], xr, threadIdx.x * N + v * step, n);
#pragma unroll
    for (int v = 0; v < VECS; ++v)
#pragma unroll
      for (int i = 0; i < N; ++i) top = max(top, int8_bits(f[v][i]));
  }
  const Int8Scale s = int8_scale(int8_block_top(top, red));
  if (threadIdx.x == 0) scale[r] = s.scale;
  if (LONG) {
    for (int k = threadIdx.x * N; k < K; k += step) {
      load_piece<T, ALIGNED>(f[0], xr, k, n);
      store_piece<N>(o, f[0], s, k, K);
    }
  } else {
#pragma unroll
    for (int v = 0; v < VECS; ++v)
      if (threadIdx.x * N + v * step < K) store_piece<N>(o, f[v], s, threadIdx.x * N + v * step, K);
  }
}

// ---------------------------------------------------------------- packing
// values [E][N][K] (row stride ld, matrix stride N * ld) -> [E][NT][KT] tiles.  Any K, any alignment: it runs once a matrix.
__global__ void __launch_bounds__(256) pack_int8_kernel(uint4* __restrict__ out, const int8_t* __restrict__ values, long long ld, int N, int K, int NT, int KT) {
  const size_t tile = ((size_t)blockIdx.z * NT + blockIdx.y) * KT + blockIdx.x;
  const int8_t* src = values + (size_t)blockIdx.z * N * ld;
  for (int i = threadIdx.x; i < BM * 8; i += blockDim.x) {
    const int r = i >> 3, c = i & 7, n = blockIdx.y * BM + r, k0 = blockIdx.x * QK + c * 16;
    uint32_t v[4] = {0u, 0u, 0u, 0u};
    if (n < N)
      for (int k = 0; k < 16 && k0 + k < K; ++k) v[k >> 2] |= (uint32_t)(uint8_t)src[(size_t)n * ld + k0 + k] << (8 * (k & 3));
    out[tile * (BM * 8) + r * 8 + (c ^ (r & 7))] = make_uint4(v[0], v[1], v[2], v[3]);
  }
}

// ---------------------------------------------------------------- host side
int sms_of_device() {
  static std::atomic<int> known[64];
  int dev = 0, v = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 148;
  if (dev >= 0 && dev < 64 && (v = known[dev].load(std::memory_order_relaxed)) > 0) return v;
  if (cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || v <= 0) v = 148;
  if (dev >= 0 && dev < 64) known[dev].store(v, std::memory_order_relaxed);
  return v;
}

// Rows of 8-bit integers [rows, K], row stride ld bytes; box = 128 k x box_rows, 128-byte swizzle, zeros outside.
bool make_map_i8(CUtensorMap* map, const void* ptr, long long rows, int K, long long ld, int box_rows) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)ld};
  cuuint32_t box[2] = {QK, (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, (void*)ptr, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <bool GLU, typename TO, int RT, int STAGES>
int launch_product(const CUtensorMap& map, const Int8Args& p, cudaStream_t st) {
  constexpr int smem = STAGES * (W_TILE_BYTES + RT * QK) + 4 * RT * 4 + 1024 + 256;
  static PerDevice devices;
  auto kernel = int8_product_kernel<GLU, TO, RT, STAGES>;
  const int rc = qv_allow_smem(kernel, smem, devices);
  if (rc) return rc;
  const long long items = (long long)p.row_tiles * ((p.N + BM - 1) / BM);
  if (items > 0x40000000LL) return QV_ERR_TOO_LARGE;
  const int sms = sms_of_device();
  return qv_launch(kernel, dim3((unsigned)(items < sms ? items : sms)), dim3(192), (size_t)smem, st, map, p);
}

template <int RT, int STAGES>
int launch_product_as(const CUtensorMap& map, const Int8Args& p, bool glu, int out_dt, cudaStream_t st) {
  if (glu) return out_dt == QV_DT_BF16 ? launch_product<true, bf16, RT, STAGES>(map, p, st) : launch_product<true, float, RT, STAGES>(map, p, st);
  return out_dt == QV_DT_BF16 ? launch_product<false, bf16, RT, STAGES>(map, p, st) : launch_product<false, float, RT, STAGES>(map, p, st);
}

#define INT8_MAX_K 131071             // 128 * 128 * K stays below 2^31

}  // namespace

extern "C" long long qv_int8_packed_bytes(int E, int N, int K) {
  return (long long)E * ((N + BM - 1) / BM) * ((K + QK - 1) / QK) * W_TILE_BYTES;
}

extern "C" int qv_pack_int8(void* out, const int8_t* values, long long ld, int E, int N, int K, void* stream) {
  if (E <= 0 || N <= 0 || K <= 0 || ld < K || ((uintptr_t)out & 15)) return QV_ERR_UNSUPPORTED;
  const int NT = (N + BM - 1) / BM, KT = (K + QK - 1) / QK;
  if (E > 65535 || NT > 65535 || K > INT8_MAX_K) return QV_ERR_TOO_LARGE;
  pack_int8_kernel<<<dim3(KT, NT, E), 256, 0, (cudaStream_t)stream>>>((uint4*)out, values, ld, N, K, NT, KT);
  return qv_launch_status();
}

// q [T, K] (row stride ld_q, a multiple of 16, on 16 bytes) and scale [T] of the rows of x (row stride ld_x, rows_in of them), row r from
// row_idx[r] where row_idx is given.
extern "C" int qv_quantize_rows(int8_t* q, long long ld_q, float* scale, const void* x, long long ld_x, int x_dt, const int* row_idx, int rows_in, int T, int K,
                                void* stream) {
  if (T <= 0) return 0;
  if (K <= 0 || ld_q < K || ((uintptr_t)q & 15) || (ld_q & 15) || ld_x < K || (!row_idx && rows_in < T)) return QV_ERR_UNSUPPORTED;
  cudaStream_t st = (cudaStream_t)stream;
#define QUANTIZE(VECS, ALIGNED, LONG, THREADS)                                                                                                          \
  return qv_launch(quantize_rows_kernel<TX, VECS, ALIGNED, LONG>, dim3(T), dim3(THREADS), 0, st, q, ld_q, scale, (const TX*)x, ld_x, row_idx, rows_in, K)
#define QUANTIZE_AS(ALIGNED)                                                             \
  do {                                                                                   \
    if (pieces > 4096) QUANTIZE(1, ALIGNED, true, 1024);                                 \
    if (few && pieces <= 1024) QUANTIZE(1, ALIGNED, false, (pieces + 31) / 32 * 32);     \
    if (pieces <= 512) QUANTIZE(2, ALIGNED, false, (pieces + 63) / 64 * 32);             \
    QUANTIZE(4, ALIGNED, false, (pieces + 127) / 128 * 32);                              \
  } while (0)
  QV_DISPATCH_DT(x_dt, TX, {
    const int pieces = (K + Piece<TX>::N - 1) / Piece<TX>::N;
    const bool few = T <= 2 * sms_of_device();
    if (((uintptr_t)x & 15) == 0 && (ld_x * sizeof(TX)) % 16 == 0) QUANTIZE_AS(true);
    QUANTIZE_AS(false);
  });
#undef QUANTIZE_AS
#undef QUANTIZE
}

// out [rows, N] (act < 0) or [rows, N / 2] (a gated product, act a GluAct kind; N a multiple of 32) of x [rows, K] (8-bit, row stride ld_x, a multiple
// of 16) with x_scale [rows], and a packed matrix with w_scale [N].  tiles null: dense.  Else the table of max_tiles tiles of at most tile_rows
// rows (32, 64, 128 or 256), and w, w_scale hold E matrices; rows that no tile lists are left as they were.
extern "C" int qv_gemm_int8(void* out, long long ld_out, int out_dt, const int8_t* x, long long ld_x, const float* x_scale, const void* w, const float* w_scale,
                            int rows, int N, int K, int E, const int* tiles, int max_tiles, int tile_rows, int act, float limit, float slope, int* err,
                            void* stream) {
  if (rows <= 0 || N <= 0) return 0;
  const bool glu = act >= 0;
  if (K <= 0 || (ld_x & 15) || ld_x < K || (((uintptr_t)x | (uintptr_t)w) & 15) || act > 2 || (glu && (N & 31))) return QV_ERR_UNSUPPORTED;
  if (out_dt != QV_DT_BF16 && out_dt != QV_DT_F32) return QV_ERR_UNSUPPORTED;
  if (K > INT8_MAX_K) return QV_ERR_TOO_LARGE;
  Int8Args p;
  p.out = out; p.x_scale = x_scale; p.w = (const uint8_t*)w; p.w_scale = w_scale; p.tiles = tiles; p.err = err; p.ld_out = ld_out;
  p.rows = rows; p.N = N; p.K = K; p.experts = E;
  p.glu = {glu ? act : 0, limit, slope};
  int rt;
  if (tiles) {
    if (max_tiles <= 0) return 0;
    rt = tile_rows; p.box = 32; p.bn = tile_rows; p.row_tiles = max_tiles;
  } else {
    p.bn = rows < 256 ? (rows + 15) & ~15 : 256;
    rt = p.bn <= 32 ? 32 : p.bn <= 64 ? 64 : p.bn <= 128 ? 128 : 256;
    p.box = p.bn; p.row_tiles = (rows + p.bn - 1) / p.bn;
  }
  CUtensorMap map;
  if (!make_map_i8(&map, x, rows, K, ld_x, p.box)) return QV_ERR_UNSUPPORTED;
  cudaStream_t st = (cudaStream_t)stream;
  if (rt == 32) return launch_product_as<32, 10>(map, p, glu, out_dt, st);
  if (rt == 64) return launch_product_as<64, 8>(map, p, glu, out_dt, st);
  if (rt == 128) return launch_product_as<128, 6>(map, p, glu, out_dt, st);
  if (rt == 256) return launch_product_as<256, 4>(map, p, glu, out_dt, st);
  return QV_ERR_UNSUPPORTED;
}

// The same for rows of float32 or bfloat16 (dense): they are quantized into q (row stride ld_q) and q_scale first.
extern "C" int qv_linear_int8(void* out, long long ld_out, int out_dt, const void* x, long long ld_x, int x_dt, int8_t* q, long long ld_q, float* q_scale,
                              const void* w, const float* w_scale, int rows, int N, int K, int act, float limit, float slope, int* err, void* stream) {
  const int rc = qv_quantize_rows(q, ld_q, q_scale, x, ld_x, x_dt, nullptr, rows, rows, K, stream);
  if (rc) return rc;
  return qv_gemm_int8(out, ld_out, out_dt, q, ld_q, q_scale, w, w_scale, rows, N, K, 1, nullptr, 0, 0, act, limit, slope, err, stream);
}
