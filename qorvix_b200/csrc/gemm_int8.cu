// Products of 8-bit integers on the 5th-generation tensor cores (sm_100a): rows x of 8-bit integers with a scale each (int8_rows.cuh) times a
// matrix of such rows, one an output channel,
//   out[t, n] = (sum_k x[t, k] w[n, k]) * x_scale[t] * w_scale[n]
// The sum is whole: int32 accumulators in tensor memory (tcgen05.mma kind::i8), exact for K up to 131,071 whatever the order, so results
// do not depend on how the work is cut.  Forms: the sums as they are; a gated product, whose matrix alternates 16 gate rows and the 16 up
// rows of the same features; and either of them grouped by expert, where a table of tiles says which rows an expert's matrix multiplies.
//
// The matrix is packed in 16 KB tiles of 128 rows x 128 k, the shared-memory image the product reads (128-byte rows, 16-byte chunk c of
// row r at chunk c ^ (r % 8)), zero where the matrix ends.  It is the 128-row operand and the token rows are the narrow one, so that a
// thread of the epilogue holds one channel of many tokens, few rows cost little padding (to 16, of pairs of SMs to 32), and dense and grouped
// products are one kernel.
//
// Every wait is bounded; one that gives up records a code and the CTA winds down.
#include "int8_rows.cuh"
#include "per_device.h"
#include "tc_common.cuh"
#include <type_traits>

#define QK 128                        // k entries of a stage: 128 bytes, one swizzle span
#define W_TILE_BYTES (BM * QK)

namespace {

// Instruction descriptor, kind::i8: D int32, A and B signed 8-bit, both K-major, m x n.
__device__ __forceinline__ uint32_t umma_idesc_i8(int m, int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
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
  int splits, kb_per_split;           // few rows: CTAs that share a block of channels, and the k blocks of each
  int mine_shift;                     // and, as a power of two, the columns of which each adds up the sums
  const void* x;                      // few rows that the kernel itself puts into 8 bits: the rows, their stride, whether pieces lie on 16 bytes
  long long ld_x;
  int aligned;
  GluAct glu;
};

// Dense items: tiles of rows fastest within bands of BAND of them, so that the CTAs at work share few weights and the rows of a band, which
// stay in L2; grouped: channels fastest, so that they share a tile's rows.
#define BAND 16
struct Item { int e, row0, rows, fb; };
// What the table says of an item (nothing for a dense product).
struct Entry { int e, row0, rows; };
__device__ __forceinline__ Entry entry_of(const Int8Args& p, int item, int items, int NT) {
  Entry n = {-1, 0, 0};
  if (p.tiles && item < items) {
    const int* t = p.tiles + 3 * (item / NT);
    n.e = t[0]; n.row0 = t[1]; n.rows = t[2];
  }
  return n;
}
__device__ __forceinline__ Item item_at(const Int8Args& p, const Entry& n, int item, int NT) {
  Item it;
  if (p.tiles) {
    it.fb = item % NT;
    it.e = n.e; it.row0 = n.row0; it.rows = n.rows;
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

// The items of a pair, first, first + pairs, ..., as a warp walks over them: lane l holds the entry of item base + l * pairs, `left` says which of the
// 32 are still to come.  Entries without an expert or rows are passed over; what comes next is known without a trip to memory, but for one in
// 32 items (a trip an item, an item ahead: the same times).
struct Walk { Entry n; int base; unsigned left; };
__device__ __forceinline__ void look(const Int8Args& p, Walk& w, int items, int pairs, int NT) {
  const int mine = w.base + pairs * (int)(threadIdx.x & 31);           // (items are 2^30 at most)
  bool there = mine < items;
  if (p.tiles) {
    w.n = entry_of(p, mine, items, NT);
    there = there && item_at(p, w.n, mine, NT).e >= 0;
  }
  w.left = __ballot_sync(0xffffffffu, there);
}
__device__ __forceinline__ Item next_item(const Int8Args& p, Walk& w, int items, int pairs, int NT) {       // e -1: there are no more
  while (!w.left) {
    w.base += 32 * pairs;
    if (w.base >= items) return {-1, 0, 0, 0};
    look(p, w, items, pairs, NT);
  }
  const int from = __ffs(w.left) - 1;
  w.left &= w.left - 1;
  Entry n = {-1, 0, 0};
  if (p.tiles) {
    n.e = __shfl_sync(0xffffffffu, w.n.e, from);
    n.row0 = __shfl_sync(0xffffffffu, w.n.row0, from);
    n.rows = __shfl_sync(0xffffffffu, w.n.rows, from);
  }
  return item_at(p, n, w.base + pairs * from, NT);
}

// The gated activations (see GluAct) as g / (1 + exp(-a)) * u: the tanh form of GELU too, 1 + tanh(x) = 2 / (1 + exp(-2 x)), which loses
// nothing where tanh is near -1.  Where the result is rounded to bfloat16 the fast exponential and quotient serve.  The exponential is off by a few
// steps of 2^-23 and, its argument being scaled to base 2, by |a| of them: under 2^-16 of itself where it is not 0, against the rounding's 2^-9.
// It is taken of -|a|: it then has no overflow, and the quotient, whose divisor must stay below 2^126, gates as far down as the smallest exponentials
// (in -103 < a < -87 these have few bits, and 0 below).
template <typename TO> __device__ __forceinline__ float gated(float g, float u, const GluAct& a) {
  float arg = g;
  if (a.kind == 1) arg = 1.5957691216057308f * fmaf(0.044715f * g * g, g, g);
  if (a.kind == 2) {
    g = at_most(g, a.limit);
    u = at_most(at_least(u, -a.limit), a.limit) + 1.f;
    arg = a.slope * g;
  }
  if (sizeof(TO) == 2) {
    const float e = __expf(-fabsf(arg));
    return __fdividef(arg < 0.f ? g * e : g, 1.f + e) * u;
  }
  return g / (1.f + expf(-arg)) * u;
}

// ---------------------------------------------------------------- many rows, and rows grouped by expert
// Two CTAs of a cluster, on neighbouring SMs, work on 256 channels x up to 256 rows: each holds 128 channels of the matrix and half of the
// rows in its shared memory, and one instruction (cta_group::2) multiplies all channels with all rows, so an SM takes in 32 KB for the products
// that it would have to take in 48 KB for by itself.  What an SM takes in sets the pace of such a kernel, not the products.  The pairs
// walk over items (a tile of rows, a block of 256 channels):
//   warp 0      weights and rows by TMA through a ring of STAGES; both CTAs' copies report to the first CTA's barrier
//   warp 1      of the first CTA: tcgen05.mma, accumulators double-buffered in tensor memory
//   warps 2..17 epilogue of the item before: scales, activation, stores; up to four warps share the channels of a quarter of tensor memory
//               and take groups of 32 rows in turn.  An item's scales are on their way while the one before is worked on.
// GLU: a gated product.  TO: the output's type.  RT: rows of a tile at most (a multiple of 32).
__host__ __device__ constexpr int pair_epilogue(int RT) { return RT >= 128 ? 16 : RT / 8; }        // its warps: one for 32 rows of a quarter's channels, up to 16
__device__ __forceinline__ uint32_t of_first(const void* p) {      // the address of the same variable in the cluster's first CTA
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(smem_u32(p)));
  return a;
}
__device__ __forceinline__ void tma_load_pair(void* dst, const CUtensorMap* map, uint32_t bar, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
      ::"r"(smem_u32(dst)), "l"((uint64_t)map), "r"(bar), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void umma_i8_pair(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void commit_pair(uint64_t* bar) {       // arrives on the barrier of both CTAs when the products issued so far are done
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)), "h"((uint16_t)3) : "memory");
}

template <bool GLU, typename TO, int RT, int STAGES>
__global__ void __launch_bounds__(64 + 32 * pair_epilogue(RT)) int8_pair_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                                                                 const Int8Args p) {
  extern __shared__ uint8_t smem_raw[];
  constexpr int STAGE_BYTES = W_TILE_BYTES + RT / 2 * QK;
  constexpr int TMEM_COLS = 2 * RT;
  uint8_t* ring = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  constexpr int EPILOGUE = pair_epilogue(RT), TURNS = EPILOGUE / 4, SCALES = RT < 32 * TURNS ? 32 : RT / TURNS;
  float* scales = (float*)(ring + STAGES * STAGE_BYTES);       // [warps][SCALES]: the scales of the rows that a warp takes
  uint64_t* full = (uint64_t*)(scales + EPILOGUE * SCALES);
  uint64_t* empty = full + STAGES;
  uint64_t* acc_full = empty + STAGES;               // [2]
  uint64_t* acc_empty = acc_full + 2;                // [2]
  uint32_t* tmem_slot = (uint32_t*)(acc_empty + 2);
  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const int rank = blockIdx.x & 1;                   // within the pair
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
    for (int b = 0; b < 2; ++b) { mbar_init(&acc_full[b], 1); mbar_init(&acc_empty[b], 2 * EPILOGUE); }      // the epilogue's warps of either CTA
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(TMEM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  asm volatile("barrier.cluster.arrive.release;" ::: "memory");    // the other CTA's barriers are set up
  asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_launch_dependents();
  pdl_wait();                                        // the rows, the tile table and the output belong to the kernels ahead until here
  const int NT = (p.N + BM - 1) / BM, NP = (NT + 1) / 2, KT = (p.K + QK - 1) / QK;
  const int items = p.row_tiles * NP, first = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  Walk walk = {{-1, 0, 0}, first, 0u};
  look(p, walk, items, pairs, NP);

  if (warp == 0) {
    const bool leader = elect_one();
    int it = 0;
    bool ok = true;
    while (ok) {
      const Item w = next_item(p, walk, items, pairs, NP);
      if (w.e < 0) break;
      const int half = ((w.rows + 31) & ~31) >> 1;             // rows of either CTA
      const int boxes = (half + p.box - 1) / p.box;
      const int block = 2 * w.fb + rank < NT ? 2 * w.fb + rank : NT - 1;       // (a last block without a second half: its sums go nowhere)
      const int w_row = ((w.e * NT + block) * KT) * BM, x_row = w.row0 + rank * half;
      for (int kb = 0; kb < KT; ++kb, ++it) {
        const int s = it % STAGES;
        if (!mbar_wait(&empty[s], ((it / STAGES) & 1) ^ 1, p.err, 61)) { ok = false; break; }
        if (leader) {
          uint8_t* dst = ring + s * STAGE_BYTES;
          if (rank == 0) mbar_expect_tx(&full[s], 2 * (W_TILE_BYTES + boxes * p.box * QK));
          const uint32_t bar = of_first(&full[s]);
          tma_load_pair(dst, &map_w, bar, 0, w_row + kb * BM);
          for (int x = 0; x < boxes; ++x) tma_load_pair(dst + W_TILE_BYTES + x * p.box * QK, &map_x, bar, kb * QK, x_row + x * p.box);
        }
        __syncwarp();
      }
    }
    // after a wait that gave up: the copies in flight land before either CTA's shared memory goes to another
    if (!ok && rank == 0)
      for (int i = it < STAGES ? 0 : it - STAGES; i < it; ++i) mbar_wait(&full[i % STAGES], (i / STAGES) & 1, p.err, 65);
  } else if (warp == 1) {
    if (rank == 0) {
      const bool leader = elect_one();               // the whole warp walks the loop and waits, an elected lane issues
      int it = 0, local = 0;
      bool ok = true;
      for (; ok; ++local) {
        const Item w = next_item(p, walk, items, pairs, NP);
        if (w.e < 0) break;
        const uint32_t idesc = umma_idesc_i8(2 * BM, (w.rows + 31) & ~31);
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
            for (int kk = 0; kk < QK / 32; ++kk)     // 32 entries of k a product: 32 bytes, 2 descriptor units
              umma_i8_pair(d_tmem, da + 2 * kk, db + 2 * kk, idesc, (kb > 0 || kk > 0) ? 1u : 0u);
            commit_pair(&empty[s]);
          }
          __syncwarp();
        }
        if (leader) commit_pair(&acc_full[b]);
        __syncwarp();
      }
    }
  } else {
    const int q = warp & 3, turn = (warp - 2) >> 2;            // tensor memory lanes 32 q .. + 31; groups of 32 rows: turn, turn + TURNS, ...
    float* xs = scales + (warp - 2) * SCALES;
    const uint32_t done[2] = {of_first(&acc_empty[0]), of_first(&acc_empty[1])};
    float ws = 0.f, rs[SCALES / 32];                           // of the item that comes next: this lane's channel, this lane's rows
    auto fetch = [&](const Item& n) {
      const int ch = (2 * n.fb + rank) * BM + q * 32 + lane;
      ws = n.e >= 0 && ch < p.N ? p.w_scale[(size_t)n.e * p.N + ch] : 0.f;
#pragma unroll
      for (int i = 0; i < SCALES / 32; ++i) {
        const int row = (i * TURNS + turn) * 32 + lane;
        rs[i] = n.e >= 0 && row < n.rows ? p.x_scale[n.row0 + row] : 0.f;
      }
    };
    Item w = next_item(p, walk, items, pairs, NP);
    fetch(w);
    for (int local = 0; w.e >= 0; ++local) {
      const int ch0 = (2 * w.fb + rank) * BM + q * 32;         // this warp's channels
      const float w_scale = ws;
      __syncwarp();
#pragma unroll
      for (int i = 0; i < SCALES / 32; ++i) xs[i * 32 + lane] = rs[i];
      __syncwarp();
      const Item now = w;
      w = next_item(p, walk, items, pairs, NP);
      fetch(w);
      const int b = local & 1;
      if (!__all_sync(0xffffffffu, mbar_wait(&acc_full[b], (local >> 1) & 1, p.err, 63))) break;     // (the MMA warp then gives up too)
      tc_fence_after();
      const uint32_t taddr = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(b * RT);
      const int feat = GLU ? (ch0 >> 1) + (lane & 15) : ch0 + lane;
      const bool there = GLU ? 2 * feat < p.N : feat < p.N;
      TO* out = (TO*)p.out + (size_t)now.row0 * p.ld_out + feat;
#pragma unroll 1
      for (int c0 = turn * 32; c0 < now.rows; c0 += 32 * TURNS) {
        uint32_t r[32];
        tmem_ld32(taddr + c0, r);
        float v[32];                                 // the rows' scales, then the scaled sums: all of them ahead of the first store
#pragma unroll
        for (int j = 0; j < 32; j += 4) *(float4*)&v[j] = *(const float4*)(xs + c0 / (32 * TURNS) * 32 + j);
        tmem_wait_ld();
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = (float)(int)r[j] * v[j] * w_scale;
        if (GLU) {
          // a lane of the lower half gives its gate value of the odd row for the up value of the even row
          const int up = lane >> 4;
          TO* o = out + (size_t)(c0 + up) * p.ld_out;
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            const float got = __shfl_xor_sync(0xffffffffu, up ? v[j] : v[j + 1], 16);
            v[j] = gated<TO>(up ? got : v[j], up ? v[j + 1] : got, p.glu);
          }
          const int left = there ? now.rows - c0 - up : 0;       // rows that this lane still has
          if (left >= 31) {
#pragma unroll
            for (int j = 0; j < 32; j += 2, o += 2 * p.ld_out) *o = from_f<TO>(v[j]);
          } else {
#pragma unroll
            for (int j = 0; j < 32; j += 2, o += 2 * p.ld_out)
              if (j < left) *o = from_f<TO>(v[j]);
          }
        } else {
          TO* o = out + (size_t)c0 * p.ld_out;
          const int left = there ? now.rows - c0 : 0;
          if (left >= 32) {
#pragma unroll
            for (int j = 0; j < 32; ++j, o += p.ld_out) *o = from_f<TO>(v[j]);
          } else {
#pragma unroll
            for (int j = 0; j < 32; ++j, o += p.ld_out)
              if (j < left) *o = from_f<TO>(v[j]);
          }
        }
        __syncwarp();
      }
      tc_fence_before();
      __syncwarp();
      // relaxed: what the first CTA waits for is that the reads of tensor memory are complete, and they are, behind tcgen05.wait::ld and the warp's
      // barrier; the arrival orders nothing else.  A release would wait for this warp's stores as well (an item of 256 channels x 256 rows and
      // one k block: 4.7 us instead of 3.7)
      if (lane == 0) asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(done[b]) : "memory");
    }
  }
  tc_fence_before();
  __syncthreads();
  asm volatile("barrier.cluster.arrive.release;" ::: "memory");    // neither CTA's shared or tensor memory is in the other's use any more
  asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS) : "memory");
  }
}

// ---------------------------------------------------------------- pieces of a row: 16 bytes of it
template <typename T> struct Piece { static constexpr int N = 16 / (int)sizeof(T); };
template <typename T, bool ALIGNED> __device__ __forceinline__ uint4 load_piece(const T* x, int k, int K) {
  constexpr int N = Piece<T>::N;
  uint4 v = make_uint4(0u, 0u, 0u, 0u);
  if (ALIGNED && k + N <= K) return *(const uint4*)(x + k);
  T* e = (T*)&v;
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (k + i < K) e[i] = x[k + i];
  return v;
}
// The largest magnitude so far, of bfloat16 a pair of them (their bits are ordered as float32's are).
__device__ __forceinline__ uint32_t larger(uint32_t top, const uint4& v, const float*) {
  constexpr uint32_t M = 0x7fffffffu;
  return max(max(top, max(v.x & M, v.y & M)), max(v.z & M, v.w & M));
}
__device__ __forceinline__ uint32_t larger(uint32_t top, const uint4& v, const bf16*) {
  constexpr uint32_t M = 0x7fff7fffu;
  return __vmaxu2(__vmaxu2(top, __vmaxu2(v.x & M, v.y & M)), __vmaxu2(v.z & M, v.w & M));
}
__device__ __forceinline__ uint32_t top_bits(uint32_t top, const float*) { return top; }
__device__ __forceinline__ uint32_t top_bits(uint32_t top, const bf16*) { return max(top << 16, top & 0xffff0000u); }

// ---------------------------------------------------------------- few rows
// A step of few tokens is bound by the matrix' bytes, so that all SMs have to ask for weights at once, and from the start: a block of 128
// channels is shared along k by the CTAs of a cluster (grid z), each with a ring of its own, and the first weights are asked for before the
// wait for the kernel ahead (a packed matrix lies still: qv_pack_int8 lets no kernel start before its end).  The CTAs hand their int32 sums
// to one another through distributed shared memory: each adds up a share of the columns of all of them, scales and stores these; whole
// sums have no order, so splits change no bit.
// TX void: the rows are in 8 bits already and come with the weights.  Else they are float32 or bfloat16 and every CTA puts its share of them, all
// rows of its k blocks, into 8 bits itself, while its first weights are on their way: eight warps hold the share in registers, the CTAs of the
// cluster tell one another the largest magnitudes that they found, and the rounded entries go to shared memory as the products read them.
// That is a launch less, and mostly behind the weights' latency, as long as a share is small (see rows_inside).
#define FEW_QUANTIZERS 256
#define FEW_PIECES 4                  // 16-byte pieces of the share that a thread holds: 16 KB in all
template <bool GLU, typename TO, typename TX, int BN, int STAGES>
__global__ void __launch_bounds__(std::is_void<TX>::value ? 192 : 64 + FEW_QUANTIZERS) int8_few_kernel(const __grid_constant__ CUtensorMap map_x, const Int8Args p) {
  extern __shared__ uint8_t smem_raw[];
  constexpr bool INSIDE = !std::is_void<TX>::value;
  constexpr int STAGE_BYTES = W_TILE_BYTES + (INSIDE ? 0 : BN * QK);
  constexpr int TMEM_COLS = BN < 32 ? 32 : BN;
  uint8_t* ring = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* rows8 = ring + STAGES * STAGE_BYTES;                // INSIDE: [k blocks of this CTA][BN rows][128], as the products read them
  uint8_t* behind = rows8 + (INSIDE ? p.kb_per_split * BN * QK : 0);
  uint64_t* full = (uint64_t*)behind;
  uint64_t* empty = full + STAGES;
  uint64_t* accum = empty + STAGES;
  uint64_t* rows_there = accum + 1;
  uint32_t* tmem_slot = (uint32_t*)(rows_there + 1);
  __shared__ __align__(16) float xs[BN];                       // the rows' scales
  __shared__ uint32_t tops[BN];                                // INSIDE: the largest magnitudes of this CTA's share of the rows
  __shared__ uint32_t all_tops[4][BN];                         // and those of the cluster's CTAs
  __shared__ Int8Scale row_scale[BN];
  int* sums = (int*)(behind + 256);                            // [splits][columns of this CTA / 4][128 channels][4]: what the cluster hands this CTA
  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const int KT = (p.K + QK - 1) / QK;
  const int split = blockIdx.z, kb0 = split * p.kb_per_split;
  const int num_kb = KT - kb0 < p.kb_per_split ? KT - kb0 : p.kb_per_split;
  const int row0 = blockIdx.y * BN, rows = p.rows - row0 < BN ? p.rows - row0 : BN;
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
    mbar_init(accum, 1);
    mbar_init(rows_there, FEW_QUANTIZERS);
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
  if (p.splits > 1) asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");      // met ahead of the first store into another CTA

  if (warp == 0) {
    const bool leader = elect_one();
    const uint8_t* w = p.w + ((size_t)blockIdx.x * KT + kb0) * W_TILE_BYTES;
    const int pre = num_kb < STAGES ? num_kb : STAGES;
    if (leader)
      for (int kb = 0; kb < pre; ++kb) {
        mbar_expect_tx(&full[kb], STAGE_BYTES);
        bulk_load_1d(ring + kb * STAGE_BYTES, w + (size_t)kb * W_TILE_BYTES, &full[kb], W_TILE_BYTES);
      }
    __syncwarp();
    if (INSIDE && p.splits > 1) {                    // (the two meetings of the cluster's magnitudes)
      asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
      asm volatile("barrier.cluster.arrive.release;" ::: "memory");
      asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
    }
    pdl_wait();                                      // (no bounded wait begins while the kernel ahead is still at work, here or in the warp below)
    if (!INSIDE) {
      if (leader)
        for (int kb = 0; kb < pre; ++kb) tma_load_2d(ring + kb * STAGE_BYTES + W_TILE_BYTES, &map_x, &full[kb], (kb0 + kb) * QK, row0);
      __syncwarp();
    }
    int kb = pre;
    for (; kb < num_kb; ++kb) {
      const int s = kb % STAGES;
      if (!mbar_wait(&empty[s], ((kb / STAGES) & 1) ^ 1, p.err, 61)) break;
      if (leader) {
        uint8_t* dst = ring + s * STAGE_BYTES;
        mbar_expect_tx(&full[s], STAGE_BYTES);
        bulk_load_1d(dst, w + (size_t)kb * W_TILE_BYTES, &full[s], W_TILE_BYTES);
        if (!INSIDE) tma_load_2d(dst + W_TILE_BYTES, &map_x, &full[s], (kb0 + kb) * QK, row0);
      }
      __syncwarp();
    }
    if (kb < num_kb)                                 // gave up: the copies in flight land first
      for (int i = kb < STAGES ? 0 : kb - STAGES; i < kb; ++i) mbar_wait(&full[i % STAGES], (i / STAGES) & 1, p.err, 65);
  } else if (warp == 1) {
    const bool leader = elect_one();
    const uint32_t idesc = umma_idesc_i8(BM, BN);
    if (INSIDE && p.splits > 1) {
      asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
      asm volatile("barrier.cluster.arrive.release;" ::: "memory");
      asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
    }
    pdl_wait();
    const bool there = !INSIDE || mbar_wait(rows_there, 0, p.err, 66);
    for (int kb = 0; there && kb < num_kb; ++kb) {
      const int s = kb % STAGES;
      if (!mbar_wait(&full[s], (kb / STAGES) & 1, p.err, 62)) break;
      tc_fence_after();
      const uint32_t a_addr = smem_u32(ring + s * STAGE_BYTES), b_addr = INSIDE ? smem_u32(rows8 + kb * BN * QK) : a_addr + W_TILE_BYTES;
      const uint64_t da = umma_desc(a_addr), db = umma_desc(b_addr);
      if (leader) {
#pragma unroll
        for (int kk = 0; kk < QK / 32; ++kk) umma_i8(tmem_base, da + 2 * kk, db + 2 * kk, idesc, (kb > 0 || kk > 0) ? 1u : 0u);
        umma_commit(&empty[s]);
      }
      __syncwarp();
    }
    if (leader) umma_commit(accum);
    __syncwarp();
  }
  const int q = warp & 3, ch0 = blockIdx.x * BM + q * 32;
  const int feat = GLU ? (ch0 >> 1) + (lane & 15) : ch0 + lane;
  const bool stores = warp >= 2 && warp < 6;         // the epilogue's warps
  const bool there = stores && (GLU ? 2 * feat < p.N : feat < p.N);
  TO* out = (TO*)p.out + (size_t)row0 * p.ld_out + feat;
  float ws = 0.f;
  // the scaled sums of columns c, c + 1, ... to the output: all lanes of an epilogue warp are here
  auto finish = [&](int c, auto& sum) {
    constexpr int N = sizeof(sum) / 4;
    float v[N];                                      // all of them ahead of the first store
#pragma unroll
    for (int j = 0; j < N; j += 4) *(float4*)&v[j] = *(const float4*)&xs[c + j];
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = (float)(int)sum[j] * v[j] * ws;
    if (GLU) {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float other = __shfl_xor_sync(0xffffffffu, v[j], 16);
        v[j] = gated<TO>(v[j], other, p.glu);        // (of the lower half; the upper half's are not stored)
      }
    }
    TO* o = out + (size_t)c * p.ld_out;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if (c + j < rows && there && (!GLU || lane < 16)) *o = from_f<TO>(v[j]);
      o += p.ld_out;
    }
  };
  bool ok = true;
  if (warp >= 2) {
    pdl_wait();                                      // the rows (or their scales) are the kernel's ahead, and the output may still be in its use
    const int te = threadIdx.x - 64;
    if constexpr (INSIDE) {
      constexpr int N = Piece<TX>::N;
      const TX* x = (const TX*)p.x + (size_t)row0 * p.ld_x;
      if (te < BN) tops[te] = 0u;
      const int per_row = num_kb * (QK / N), pieces = rows * per_row;                          // of the share; a multiple of 16 a row
      const int down = FEW_QUANTIZERS / per_row, on = FEW_QUANTIZERS - down * per_row;         // from a thread's piece to its next: rows, pieces
      uint4 v[FEW_PIECES];
      int row[FEW_PIECES], col[FEW_PIECES];
      row[0] = te / per_row;
      col[0] = te - row[0] * per_row;
#pragma unroll
      for (int u = 0; u < FEW_PIECES; ++u) {
        if (u > 0) {
          col[u] = col[u - 1] + on;
          row[u] = row[u - 1] + down;
          if (col[u] >= per_row) { col[u] -= per_row; ++row[u]; }
        }
        v[u] = make_uint4(0u, 0u, 0u, 0u);
        if (row[u] < rows) {
          const TX* xr = x + (size_t)row[u] * p.ld_x;
          const int k = kb0 * QK + col[u] * N;
          v[u] = p.aligned ? load_piece<TX, true>(xr, k, p.K) : load_piece<TX, false>(xr, k, p.K);
        }
      }
      asm volatile("bar.sync 2, %0;" ::"n"(FEW_QUANTIZERS) : "memory");
#pragma unroll
      for (int u = 0; u < FEW_PIECES; ++u) {
        if (u * FEW_QUANTIZERS >= pieces) break;
        uint32_t top = top_bits(larger(0u, v[u], x), x);
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));         // sixteen lanes are in one row
        if ((lane & 15) == 0 && row[u] < rows) atomicMax(&tops[row[u]], top);
      }
      asm volatile("bar.sync 2, %0;" ::"n"(FEW_QUANTIZERS) : "memory");
      if (p.splits > 1) {
        asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
        if (te < BN * p.splits) {
          uint32_t remote;
          asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_u32(&all_tops[split][te % BN])), "r"(te / BN));
          asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(remote), "r"(tops[te % BN]) : "memory");
        }
        asm volatile("barrier.cluster.arrive.release;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
      }
      if (te < BN) {
        uint32_t top = p.splits > 1 ? 0u : tops[te];
        for (int s = 0; p.splits > 1 && s < p.splits; ++s) top = max(top, all_tops[s][te]);
        row_scale[te] = int8_scale(__uint_as_float(top));
        xs[te] = te < rows ? int8_step(__uint_as_float(top)) : 0.f;
      }
      asm volatile("bar.sync 2, %0;" ::"n"(FEW_QUANTIZERS) : "memory");
#pragma unroll
      for (int u = 0; u < FEW_PIECES; ++u) {
        if (u * FEW_QUANTIZERS >= pieces) break;
        if (row[u] < rows) {
          const TX* e = (const TX*)&v[u];
          float f[N];
#pragma unroll
          for (int m = 0; m < N; ++m) f[m] = to_f(e[m]);
          uint32_t w[N / 4];
          int8_pack<sizeof(TX) == 2, N>(f, row_scale[row[u]], w);
          const int k = col[u] * N;                  // of the share
          uint8_t* at = rows8 + (k / QK) * (BN * QK) + row[u] * QK + ((((k % QK) >> 4) ^ (row[u] & 7)) << 4) + (k & 15);
          if (N == 8) *(uint2*)at = make_uint2(w[0], w[N / 4 - 1]);
          else *(uint32_t*)at = w[0];
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");       // the products read them
      mbar_arrive(rows_there);
    }
    if (stores) {
      if (ch0 + lane < p.N) ws = p.w_scale[ch0 + lane];
      if (!INSIDE && te < BN) xs[te] = te < rows ? p.x_scale[row0 + te] : 0.f;
      asm volatile("bar.sync 1, 128;" ::: "memory");
      ok = __all_sync(0xffffffffu, mbar_wait(accum, 0, p.err, 63));
      tc_fence_after();
    }
  }
  const int shift = p.mine_shift, mine = 1 << shift;           // columns a CTA adds up: 4 or more
  if (!INSIDE && p.splits > 1) asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
  if (stores && ok) {
    const uint32_t taddr = tmem_base + ((uint32_t)(q * 32) << 16);
    const uint32_t to = smem_u32(sums) + (uint32_t)(((split << (shift - 2)) * BM + q * 32 + lane) * 16);
#pragma unroll 1
    for (int c0 = 0; c0 < rows; c0 += 16) {
      uint32_t r[16];
      tmem_ld16(taddr + c0, r);
      tmem_wait_ld();
      if (p.splits == 1) {
        finish(c0, r);
      } else {
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
          const int c = c0 + j;
          if (c < rows) {
            uint32_t remote;
            asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(to + (uint32_t)(((c & (mine - 1)) >> 2) * BM * 16)), "r"(c >> shift));
            asm volatile("st.shared::cluster.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(remote), "r"(r[j]), "r"(r[j + 1]), "r"(r[j + 2]), "r"(r[j + 3]) : "memory");
          }
        }
      }
    }
  }
  tc_fence_before();
  if (p.splits > 1) {
    asm volatile("barrier.cluster.arrive.release;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
    if (stores && ok) {
      const int4* part = (const int4*)sums + q * 32 + lane;
      for (int i = 0; i < mine; i += 4) {
        const int c = (split << shift) + i;
        if (c >= rows) break;
        int t[4] = {0, 0, 0, 0};
#pragma unroll 4
        for (int s = 0; s < p.splits; ++s) {
          const int4 v = part[((s << shift) + i) * (BM / 4)];
          t[0] += v.x; t[1] += v.y; t[2] += v.z; t[3] += v.w;
        }
        finish(c, t);
      }
    }
  }
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS) : "memory");
  }
}

// ---------------------------------------------------------------- rows in 8 bits
// One read and one write of the row are all it cannot do without, so a row stays in registers, as stored, between its maximum and its
// rounding: VECS pieces of 16 bytes a thread, all asked for at once.  A row has a warp (no barrier between its two halves, so that the SM's
// other rows go on: many short rows) or a block; rows longer than VECS pieces of 1,024 threads are read twice (LONG).  ALIGNED: pieces lie
// on 16 bytes; else their entries are read one by one.  BLOCKS: how many the registers are to leave room for on an SM.  What bounds
// it is the instructions and, for many rows, how many are on their way at once: 12,288 rows of 1,408 take 9.9 us (5.2 TB/s) with six pieces a
// thread and 11.1 with eight; 2,048 rows of 14,336 18.1 us (4.9 TB/s) with three blocks an SM and 20.8 with two.
template <typename T> __device__ __forceinline__ void store_piece(int8_t* q, const uint4& v, const Int8Scale& s, int k, int K) {
  constexpr int N = Piece<T>::N;
  float f[N];
  const T* e = (const T*)&v;
#pragma unroll
  for (int i = 0; i < N; ++i) f[i] = to_f(e[i]);
  uint32_t w[N / 4];
  int8_pack<sizeof(T) == 2, N>(f, s, w);
  if (k + N <= K) {
    if (N == 8) *(uint2*)(q + k) = make_uint2(w[0], w[N / 4 - 1]);
    else *(uint32_t*)(q + k) = w[0];
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (k + i < K) q[k + i] = (int8_t)(w[i / 4] >> (8 * (i & 3)));
  }
}

#define QUANTIZE_WARPS 4              // rows of a block whose rows have a warp each
template <typename T, int VECS, bool WARP, int THREADS, int BLOCKS, bool ALIGNED, bool LONG>
__global__ void __launch_bounds__(THREADS, BLOCKS) quantize_rows_kernel(int8_t* __restrict__ q, long long ld_q, float* __restrict__ scale, const T* __restrict__ x,
                                                                       long long ld_x, const int* __restrict__ row_idx, int rows_in, int rows, int K) {
  constexpr int N = Piece<T>::N;
  __shared__ uint32_t red[32];
  pdl_wait();
  pdl_launch_dependents();
  const int r = WARP ? blockIdx.x * QUANTIZE_WARPS + (threadIdx.x >> 5) : blockIdx.x;
  const int at = (WARP ? threadIdx.x & 31 : threadIdx.x) * N, step = (WARP ? 32 : blockDim.x) * N;
  if (WARP && r >= rows) return;
  const int src = row_idx ? row_idx[r] : r;
  const bool there = (unsigned)src < (unsigned)rows_in;      // an index outside the rows: a row of zeros
  const T* xr = x + (size_t)(there ? src : 0) * ld_x;
  const int n = there ? K : 0;
  int8_t* o = q + (size_t)r * ld_q;
  uint4 v[VECS];
  uint32_t top = 0;
  if (LONG) {
    for (int k = at; k < n; k += step) top = larger(top, load_piece<T, ALIGNED>(xr, k, n), xr);
  } else {
#pragma unroll
    for (int i = 0; i < VECS; ++i) v[i] = load_piece<T, ALIGNED>(xr, at + i * step, n);
#pragma unroll
    for (int i = 0; i < VECS; ++i) top = larger(top, v[i], xr);
  }
  top = top_bits(top, xr);
  const float most = WARP ? __uint_as_float(__reduce_max_sync(0xffffffffu, top)) : int8_block_top(top, red);
  const Int8Scale s = int8_scale(most);
  if (at == 0) scale[r] = int8_step(most);
  if (LONG) {
    for (int k = at; k < K; k += step) store_piece<T>(o, load_piece<T, ALIGNED>(xr, k, n), s, k, K);
  } else {
#pragma unroll
    for (int i = 0; i < VECS; ++i)
      if (at + i * step < K) store_piece<T>(o, v[i], s, at + i * step, K);
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

// The packed tiles as rows of 128 bytes, copied as they are.
bool make_map_tiles(CUtensorMap* map, const void* packed, long long tiles) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  cuuint64_t dims[2] = {QK, (cuuint64_t)tiles * BM};
  cuuint64_t strides[1] = {QK};
  cuuint32_t box[2] = {QK, BM};
  cuuint32_t estr[2] = {1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, (void*)packed, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <bool GLU, typename TO, int RT, int STAGES>
int launch_pair(const CUtensorMap& map_x, const CUtensorMap& map_w, const Int8Args& p, cudaStream_t st) {
  constexpr int smem = STAGES * (W_TILE_BYTES + RT / 2 * QK) + (RT < 128 ? 32 * pair_epilogue(RT) : 4 * RT) * 4 + 1024 + 256;
  static_assert(smem <= 227 * 1024, "a CTA's shared memory");
  static PerDevice devices;
  auto kernel = int8_pair_kernel<GLU, TO, RT, STAGES>;
  const int rc = qv_allow_smem(kernel, smem, devices);
  if (rc) return rc;
  const long long items = (long long)p.row_tiles * ((p.N + 2 * BM - 1) / (2 * BM));
  if (items > 0x40000000LL) return QV_ERR_TOO_LARGE;
  const int pairs = device_sms() / 2;
  return qv_launch_cluster(kernel, dim3(2 * (unsigned)(items < pairs ? items : pairs)), dim3(64 + 32 * pair_epilogue(RT)), (size_t)smem, st, dim3(2, 1, 1), map_x, map_w, p);
}

template <int RT, int STAGES>
int launch_pair_as(const CUtensorMap& map_x, const CUtensorMap& map_w, const Int8Args& p, bool glu, int out_dt, cudaStream_t st) {
  if (glu) return out_dt == QV_DT_BF16 ? launch_pair<true, bf16, RT, STAGES>(map_x, map_w, p, st) : launch_pair<true, float, RT, STAGES>(map_x, map_w, p, st);
  return out_dt == QV_DT_BF16 ? launch_pair<false, bf16, RT, STAGES>(map_x, map_w, p, st) : launch_pair<false, float, RT, STAGES>(map_x, map_w, p, st);
}

// How a dense product is cut, by the time that each cut is expected to take: rounds of CTAs or pairs, times the k blocks of one, times what an
// SM takes in for a k block at 88 bytes a ns, plus what comes behind.
//   few rows: tiles of 16, 32 or 64 rows, 1, 2 or 4 CTAs that share a block of channels, two CTAs an SM; a tile's last stores and, with several
//     CTAs, handing over its sums cost some 20 and 15 ns a row.
//   pairs: tiles of a multiple of 32 rows; a k block takes 187 ns up to 64 rows, 235 at 128, 303 at 192 and 387 at 256 (2,048 rows, 28672 x
//     4096); 3.5 us for setting up pairs, and for filling and emptying them.
// Measured, us with their rounding to 8 bits (few as rows / CTAs): 77 rows, 777 x 1001: 16/1 4.9, 16/2 4.7, 32/4 4.6, 64/1 5.9, pairs of 32 6.1; 128
// rows, 4096 x 14336: 32/2 21.9, 64/2 18.8, 64/4 18.9, pairs of 64 26.3; 256 rows, 2048 x 2048: 16/1 7.2, 32/1 7.1, 64/2 8.0, pairs of 64 7.9;
// 512 rows, 1024 x 1024: 32/1 5.4, pairs of 64 6.5; 64 rows, 28672 x 4096: 64/1 28.5, pairs of 64 26.3; 8 rows of it: 16/1 22.1, pairs of 32 24.5.
struct Plan { int few, bn, splits; };
Plan plan_of(int rows, int N, int K, int sms) {
  const long long KT = (K + QK - 1) / QK, blocks = (N + BM - 1) / BM, pairs = sms / 2;
  Plan best = {1, 16, 1};
  long long least = 0x7fffffffffffffffLL;
  for (int bn = 16; bn <= 64; bn *= 2) {
    if (bn > 16 && bn / 2 >= rows) break;
    const long long tiles = (rows + bn - 1) / bn;
    if (tiles > 65535) continue;
    for (int splits = 1; splits <= 4; splits *= 2) {
      const long long ctas = blocks * tiles * splits;
      if (splits > 1 && (ctas > 2 * sms || KT < 2 * splits)) break;
      const long long cost = (ctas + sms - 1) / sms * ((KT + splits - 1) / splits) * (128 + bn) * 145 / 100 + 20 * bn + (splits > 1 ? 800 + 15 * bn : 0);
      if (cost <= least) { least = cost; best = {1, bn, splits}; }
    }
  }
  for (int bn = 32; bn <= 256; bn += 32) {
    if (bn > 32 && bn - 32 >= rows) break;
    const long long items = (rows + bn - 1) / bn * ((N + 2 * BM - 1) / (2 * BM));
    const long long cost = (items + pairs - 1) / pairs * KT * ((bn < 64 ? 64 : bn) + 116) * 104 / 100 + 3500;
    if (cost < least || (!best.few && cost == least)) { least = cost; best = {0, bn, 1}; }
  }
  return best;
}

template <bool GLU, typename TO, typename TX, int BN, int STAGES>
int launch_few(const CUtensorMap& map, Int8Args p, int blocks, int tiles, cudaStream_t st) {
  constexpr bool INSIDE = !std::is_void<TX>::value;
  auto kernel = int8_few_kernel<GLU, TO, TX, BN, STAGES>;
  p.mine_shift = 2;
  while ((p.splits << p.mine_shift) < BN) ++p.mine_shift;
  const int columns = p.splits > 1 ? p.splits << p.mine_shift : 0;
  const size_t smem = STAGES * (W_TILE_BYTES + (INSIDE ? 0 : BN * QK)) + (INSIDE ? p.kb_per_split * BN * QK : 0) + 1024 + 256 + (size_t)columns * BM * 4;
  constexpr size_t most = INSIDE ? 226 * 1024 : STAGES * (W_TILE_BYTES + BN * QK) + 1024 + 256 + (size_t)(BN < 32 ? 32 : BN) * BM * 4;
  static_assert(most <= 227 * 1024, "a CTA's shared memory");
  if (smem > most) return QV_ERR_TOO_LARGE;
  static PerDevice devices;
  const int rc = qv_allow_smem(kernel, most, devices);
  if (rc) return rc;
  return qv_launch_cluster(kernel, dim3(blocks, tiles, p.splits), dim3(INSIDE ? 64 + FEW_QUANTIZERS : 192), smem, st, dim3(1, 1, p.splits), map, p);
}

// k blocks a CTA and whether the CTAs' rings may fill an SM each: where every CTA finds one for itself (clusters of four find 32 places on
// 148 SMs), else two CTAs share an SM.
struct Cut { int splits, kb_per_split; bool one_wave; };
Cut cut_of(const Plan& plan, int rows, int N, int K, int sms) {
  const int blocks = (N + BM - 1) / BM, KT = (K + QK - 1) / QK, tiles = (rows + plan.bn - 1) / plan.bn;
  Cut c = {plan.splits, 0, false};
  c.kb_per_split = (KT + c.splits - 1) / c.splits;
  while ((c.splits - 1) * c.kb_per_split >= KT) c.splits /= 2, c.kb_per_split = (KT + c.splits - 1) / c.splits;      // none without k blocks
  const long long ctas = (long long)blocks * tiles * c.splits;
  c.one_wave = c.splits == 4 ? ctas * 8 <= sms * 7 : ctas <= sms;
  return c;
}

template <typename TX, int BN, int DEEP, int SHALLOW>
int launch_few_as(const CUtensorMap& map, Int8Args p, const Cut& cut, bool glu, int out_dt, cudaStream_t st) {
  const int blocks = (p.N + BM - 1) / BM, tiles = (p.rows + BN - 1) / BN;
  p.splits = cut.splits; p.kb_per_split = cut.kb_per_split;
#define FEW(GLU, TO) return cut.one_wave ? launch_few<GLU, TO, TX, BN, DEEP>(map, p, blocks, tiles, st) : launch_few<GLU, TO, TX, BN, SHALLOW>(map, p, blocks, tiles, st)
  if (glu) {
    if (out_dt == QV_DT_BF16) FEW(true, bf16);
    FEW(true, float);
  }
  if (out_dt == QV_DT_BF16) FEW(false, bf16);
  FEW(false, float);
#undef FEW
}

// Whether the kernel for few rows puts them into 8 bits itself: up to 8 rows, of which a CTA's share is 16 KB at most, with room for it beside a ring
// of eight stages, or of five where two CTAs share an SM.  A call by itself is bound by its launches, of which this saves one (8 rows, 6144 x 4096:
// 16.0 us apart, 10.5 inside); among captured ones, us apart / inside: 1 row, 4096 x 14336 12.7 / 12.6, 4096 x 4096 6.8 / 6.2; 3 rows, 512 x 512 3.8 /
// 3.1; 8 rows, 2048 x 2048 4.7 / 5.0, 4096 x 4096 7.1 / 7.5, 6144 x 4096 7.9 / 8.7; but 4 rows, 4096 x 14336 13.1 / 14.7, 16 rows, 4096 x 4096 7.1 / 9.1.
bool rows_inside(const Plan& plan, const Cut& cut, int rows, int bytes) {
  return plan.few && plan.bn == 16 && rows <= 8 && rows * cut.kb_per_split * QK * bytes <= 16 * 1024 && cut.kb_per_split <= (cut.one_wave ? 32 : 10);
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
#define QUANTIZE(VECS, WARP, MOST, BLOCKS, ALIGNED, LONG, THREADS)                                                                                     \
  return qv_launch(quantize_rows_kernel<TX, VECS, WARP, MOST, BLOCKS, ALIGNED, LONG>, dim3(WARP ? (T + QUANTIZE_WARPS - 1) / QUANTIZE_WARPS : T),      \
                   dim3(THREADS), 0, st, q, ld_q, scale, (const TX*)x, ld_x, row_idx, rows_in, T, K)
#define QUANTIZE_AS(ALIGNED)                                                                                  \
  do {                                                                                                        \
    if (pieces > 4096) QUANTIZE(1, false, 1024, 1, ALIGNED, true, 1024);                                      \
    if (few && pieces <= 1024) QUANTIZE(1, false, 1024, 1, ALIGNED, false, (pieces + 31) / 32 * 32);          \
    if (pieces <= 128) QUANTIZE(4, true, 32 * QUANTIZE_WARPS, 8, ALIGNED, false, 32 * QUANTIZE_WARPS);       \
    if (pieces <= 192) QUANTIZE(6, true, 32 * QUANTIZE_WARPS, 9, ALIGNED, false, 32 * QUANTIZE_WARPS);        \
    if (pieces <= 256) QUANTIZE(8, true, 32 * QUANTIZE_WARPS, 8, ALIGNED, false, 32 * QUANTIZE_WARPS);       \
    if (pieces <= 2048) QUANTIZE(4, false, 512, 3, ALIGNED, false, (pieces + 127) / 128 * 32);                \
    QUANTIZE(4, false, 1024, 1, ALIGNED, false, (pieces + 127) / 128 * 32);                                   \
  } while (0)
  QV_DISPATCH_DT(x_dt, TX, {
    const int pieces = (K + Piece<TX>::N - 1) / Piece<TX>::N;
    // blocks of as many threads as a row has pieces find room at once: us, such a block a row / a warp or fewer threads a row, bfloat16: 8 rows of 2,048
    // 1.48 / 1.98, 296 rows 2.12 / 2.68; 296 rows of 4,096 2.52 / 2.67, 400 rows 3.07 / 2.92
    const bool few = T <= 2 * device_sms();
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
  cudaStream_t st = (cudaStream_t)stream;
  CUtensorMap map, map_w;
  int rt;
  if (tiles) {
    if (max_tiles <= 0) return 0;
    rt = tile_rows; p.bn = tile_rows; p.row_tiles = max_tiles; p.box = tile_rows >= 64 ? 32 : 16;
  } else {
    const int sms = device_sms();
    const Plan plan = plan_of(rows, N, K, sms);
    p.bn = plan.bn;
    if (plan.few) {
      const Cut cut = cut_of(plan, rows, N, K, sms);
      if (!make_map_i8(&map, x, rows, K, ld_x, p.bn)) return QV_ERR_UNSUPPORTED;
      if (p.bn == 16) return launch_few_as<void, 16, 10, 5>(map, p, cut, glu, out_dt, st);
      if (p.bn == 32) return launch_few_as<void, 32, 9, 4>(map, p, cut, glu, out_dt, st);
      return launch_few_as<void, 64, 7, 3>(map, p, cut, glu, out_dt, st);
    }
    rt = p.bn <= 32 ? 32 : p.bn <= 64 ? 64 : p.bn <= 128 ? 128 : 256;
    p.box = p.bn / 2; p.row_tiles = (rows + p.bn - 1) / p.bn;
  }
  const long long w_tiles = (long long)E * ((N + BM - 1) / BM) * ((K + QK - 1) / QK);
  if (w_tiles * BM > 0x7fffffffLL) return QV_ERR_TOO_LARGE;     // rows of the tensor map are counted in 31 bits
  if (!make_map_i8(&map, x, rows, K, ld_x, p.box) || !make_map_tiles(&map_w, w, w_tiles)) return QV_ERR_UNSUPPORTED;
  if (rt == 32) return launch_pair_as<32, 11>(map, map_w, p, glu, out_dt, st);
  if (rt == 64) return launch_pair_as<64, 10>(map, map_w, p, glu, out_dt, st);
  if (rt == 128) return launch_pair_as<128, 8>(map, map_w, p, glu, out_dt, st);
  if (rt == 256) return launch_pair_as<256, 6>(map, map_w, p, glu, out_dt, st);
  return QV_ERR_UNSUPPORTED;
}

// Bytes of room that qv_linear_int8 wants for its rows in 8 bits and their scales (0: none).
extern "C" long long qv_linear_int8_room(int rows, int N, int K, int x_dt) {
  if (rows <= 0 || N <= 0 || K <= 0) return 0;
  const int sms = device_sms();
  const Plan plan = plan_of(rows, N, K, sms);
  if (plan.few && rows_inside(plan, cut_of(plan, rows, N, K, sms), rows, x_dt == QV_DT_F32 ? 4 : 2)) return 0;
  return (long long)rows * ((K + 15) / 16 * 16 + 4);
}

// qv_gemm_int8 for rows of float32 or bfloat16 (dense), which are put into 8 bits first: by the product's kernel itself, or in `room`
// (qv_linear_int8_room bytes on 16), a launch of its own.
extern "C" int qv_linear_int8(void* out, long long ld_out, int out_dt, const void* x, long long ld_x, int x_dt, void* room, const void* w, const float* w_scale,
                              int rows, int N, int K, int act, float limit, float slope, int* err, void* stream) {
  if (rows <= 0 || N <= 0) return 0;
  const bool glu = act >= 0;
  if (K <= 0 || ld_x < K || ((uintptr_t)w & 15) || act > 2 || (glu && (N & 31))) return QV_ERR_UNSUPPORTED;
  if ((out_dt != QV_DT_BF16 && out_dt != QV_DT_F32) || (x_dt != QV_DT_BF16 && x_dt != QV_DT_F32)) return QV_ERR_UNSUPPORTED;
  if (K > INT8_MAX_K) return QV_ERR_TOO_LARGE;
  const int sms = device_sms(), bytes = x_dt == QV_DT_F32 ? 4 : 2;
  const Plan plan = plan_of(rows, N, K, sms);
  const Cut cut = plan.few ? cut_of(plan, rows, N, K, sms) : Cut{};
  if (plan.few && rows_inside(plan, cut, rows, bytes)) {
    Int8Args p = {};
    p.out = out; p.w = (const uint8_t*)w; p.w_scale = w_scale; p.err = err; p.ld_out = ld_out;
    p.rows = rows; p.N = N; p.K = K; p.experts = 1; p.bn = plan.bn;
    p.glu = {glu ? act : 0, limit, slope};
    p.x = x; p.ld_x = ld_x; p.aligned = ((uintptr_t)x & 15) == 0 && (ld_x * bytes) % 16 == 0;
    CUtensorMap none;
    memset(&none, 0, sizeof(none));
    if (x_dt == QV_DT_F32) return launch_few_as<float, 16, 8, 5>(none, p, cut, glu, out_dt, (cudaStream_t)stream);
    return launch_few_as<bf16, 16, 8, 5>(none, p, cut, glu, out_dt, (cudaStream_t)stream);
  }
  if (!room || ((uintptr_t)room & 15)) return QV_ERR_UNSUPPORTED;
  const long long ld_q = (K + 15) / 16 * 16;
  float* scale = (float*)((int8_t*)room + rows * ld_q);
  const int rc = qv_quantize_rows((int8_t*)room, ld_q, scale, x, ld_x, x_dt, nullptr, rows, rows, K, stream);
  if (rc) return rc;
  return qv_gemm_int8(out, ld_out, out_dt, (const int8_t*)room, ld_q, scale, w, w_scale, rows, N, K, 1, nullptr, 0, 0, act, limit, slope, err, stream);
}
