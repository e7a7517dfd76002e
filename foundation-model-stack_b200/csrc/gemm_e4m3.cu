// y[m, n] = sx[m] * sw[n] * sum_k qx[m, k] * qw[n, k] (+ bias[n]): rows and weights of 8 bits (e4m3) with one float32 scale a
// row of either, on the tcgen05 tensor cores of sm_100a (kind::f8f6f4: twice the rate of 16-bit operands, half the bytes).
// The products of two e4m3 values and their sums are float32 in tensor memory; the scales come in once, in the epilogue, so
// that nothing is rounded but the result.  GLU: y = act(gate) * up for weights [gate; up] (fms/modules/feedforward.py:288-297).
//
// Both kernels bring operands in by TMA in boxes of 128 k (128 bytes, 128-byte swizzle) and issue 4 instructions of 32 k on a
// box.  Rows lie `pitch` bytes apart, a multiple of 16, with zeros behind the last value; what lies beyond M, N and the
// pitch is zeros on the way in (TMA) and is not stored on the way out.  Every wait on an mbarrier is bounded: on a time-out the
// block records error 4, skips the rest of its work and still frees its tensor memory.
#include <cuda.h>

#include "common.cuh"

namespace {
constexpr int TILE = 128, TILE_K = 128, UMMA_K = 32, MAX_STAGES = 12;
constexpr int THREADS = 320, EPILOGUE_WARPS = 8, ROWS_THREADS = THREADS + 32;
constexpr int BOX_BYTES = TILE * TILE_K;  // 128 rows of an operand for one step

#include "tcgen05.cuh"
#include "umma_issue.cuh"
#include "quantized.cuh"

// instruction descriptor of kind::f8f6f4: float32 accumulator, e4m3 a and b, both K-major; the shape M x N
__host__ __device__ constexpr uint32_t idesc_e4m3(int m, int n) { return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24); }
// by a whole warp, which gives up as one
__device__ __forceinline__ bool warp_wait(void* bar, uint32_t parity, volatile int* failed) {
  return __all_sync(0xffffffffu, wait_or_abort(bar, parity, failed));
}

struct Epilogue {
  void* out;                  // [M, outputs] bfloat16 or float32 (GLU: bfloat16)
  Bias bias;
  const float *sx, *sw;       // [M], [N]
  int out_f32, glu, act;
  int outputs;                // columns of y: N, or the hidden values of GLU (half of N)
  int tile_n, stages, n_tokens;
  float* scratch;             // [blocks][slots][n_tokens][128], of the second kernel
  int slots;                  // of a block in scratch, or 0: each takes one whole tile
  long scratch_floats;        // for the bounds-checked build
};

// four sums times the scales of their row and columns (+ bias)
__device__ __forceinline__ void scale4(float* v, float sx, const float* scales, const float* biases) {
  const float4 s = *reinterpret_cast<const float4*>(scales);
  float4 b = make_float4(0.f, 0.f, 0.f, 0.f);
  if (biases) b = *reinterpret_cast<const float4*>(biases);
  v[0] = fmaf(v[0], sx * s.x, b.x);
  v[1] = fmaf(v[1], sx * s.y, b.y);
  v[2] = fmaf(v[2], sx * s.z, b.z);
  v[3] = fmaf(v[3], sx * s.w, b.w);
}
// twice 16 columns of this thread's row (lane) of tensor memory: both loads are in flight before the one wait
__device__ __forceinline__ void tmem_load_2x16(uint32_t taddr_a, uint32_t taddr_b, float* va, float* vb) {
  __syncwarp();
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%32];\n"
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%33];\n"
      "tcgen05.wait::ld.sync.aligned;\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
        "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr_a), "r"(taddr_b)
      : "memory");
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    va[i] = __uint_as_float(r[i]);
    vb[i] = __uint_as_float(r[16 + i]);
  }
}
__device__ __forceinline__ void store16(const Epilogue& ep, const float* v, int row, int col0, int M) {
  if (!FMS_IN((size_t)row * ep.outputs + col0, (size_t)M * ep.outputs)) return;
  if (ep.out_f32) {
    float* o = (float*)ep.out + (size_t)row * ep.outputs + col0;
    if (col0 + 16 <= ep.outputs && ep.outputs % 4 == 0) {
#pragma unroll
      for (int j = 0; j < 16; j += 4) *reinterpret_cast<float4*>(o + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (col0 + j < ep.outputs) o[j] = v[j];
    }
    return;
  }
  __nv_bfloat16* o = (__nv_bfloat16*)ep.out + (size_t)row * ep.outputs + col0;
  if (col0 + 16 <= ep.outputs && ep.outputs % 8 == 0) {
#pragma unroll
    for (int j = 0; j < 16; j += 8) {
      uint32_t pk[4];
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        __nv_bfloat162 t = __floats2bfloat162_rn(v[j + 2 * p], v[j + 2 * p + 1]);
        pk[p] = *reinterpret_cast<uint32_t*>(&t);
      }
      *reinterpret_cast<uint4*>(o + j) = make_uint4(pk[0], pk[1], pk[2], pk[3]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (col0 + j < ep.outputs) o[j] = __float2bfloat16_rn(v[j]);
  }
}

// values of neighbouring rows of y, one column
template <int N> __device__ __forceinline__ void store_column(const Epilogue& ep, const float* v, int row0, int col, int M, size_t pitch) {
  const size_t at = (size_t)row0 * pitch + col;
#pragma unroll
  for (int j = 0; j < N; ++j)
    if (row0 + j < M && FMS_IN(at + j * pitch, (size_t)M * pitch)) {
      if (ep.out_f32) ((float*)ep.out)[at + j * pitch] = v[j];
      else ((__nv_bfloat16*)ep.out)[at + j * pitch] = __float2bfloat16_rn(v[j]);
    }
}

// ---- many rows (prefill) --------------------------------------------------------------------------------------------
// Persistent pairs of thread blocks (a cluster of two, cta_group::2): a pair owns a tile of 256 rows of x by TN rows of w, of
// which each block brings 128 rows of x and half the rows of w (GLU: block 0 the gate rows, block 1 the up rows) into its own
// shared memory.  What a multiprocessor takes in, 128 + TN / 2 bytes a k, against 2 * 128 * TN operations is what limits
// tiles without a pair.  Two accumulators: the epilogue of a tile runs under the products of the next.
//   warp 0 TMA, warp 1 (of block 0) the instructions, warps 2-9 the epilogue: 32 rows of this block's 128 and every second
//   16 columns each (with four warps the activation of GLU takes longer than the tile's products)
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1)
    e4m3_pair_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, Epilogue ep, int M,
                     int k_steps, int* __restrict__ error_flag) {
  extern __shared__ unsigned char smem_unaligned[];
  unsigned char* smem = smem_unaligned + (-smem_u32(smem_unaligned) & 1023);
  const int b_rows = ep.tile_n / 2, stage_bytes = BOX_BYTES + b_rows * TILE_K, stages = ep.stages;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + (size_t)stages * stage_bytes);
  uint64_t* empty = full + MAX_STAGES;
  uint64_t* acc_full = empty + MAX_STAGES;  // [2]
  uint64_t* acc_empty = acc_full + 2;       // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  __shared__ int failed_flag;
  __shared__ __align__(16) float col_scales[EPILOGUE_WARPS][128], col_biases[EPILOGUE_WARPS][128];  // of a warp's columns of the tile; GLU: the up rows' behind
  volatile int* failed = &failed_flag;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const bool leader = rank == 0;
  const int tile_n = ep.glu ? ep.tile_n / 2 : ep.tile_n;  // output columns of a tile
  const int tiles_m = (M + 2 * TILE - 1) / (2 * TILE), n_tiles = tiles_m * ((ep.outputs + tile_n - 1) / tile_n);
  const int pair = blockIdx.x / 2, pairs = gridDim.x / 2;

  if (threadIdx.x == 0) {
    failed_flag = 0;
    for (int s = 0; s < MAX_STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&acc_full[a], 1);
      mbar_init(&acc_empty[a], 2 * EPILOGUE_WARPS);  // of either block (used in block 0)
    }
    mbar_fence_init();
  }
  __syncthreads();
  cluster_sync_all();  // the partner runs, and its barriers exist
  if (warp == 1) tmem_alloc_pair(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // and it has its tensor memory
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    if (elect_one()) {
      int it = 0;
      for (int tile = pair; tile < n_tiles && !*failed; tile += pairs) {
        const int m0 = (tile % tiles_m) * 2 * TILE + (int)rank * TILE, n0 = (tile / tiles_m) * tile_n;
        const int w_row = ep.glu ? (leader ? n0 : ep.outputs + n0) : n0 + (int)rank * b_rows;
        for (int i = 0; i < k_steps; ++i, ++it) {
          const int s = it % stages;
          if (!wait_or_abort(&empty[s], ((it / stages) & 1) ^ 1, failed)) break;
          unsigned char* a = smem + (size_t)s * stage_bytes;
          if (leader) mbar_arrive_expect_tx(&full[s], 2 * stage_bytes);  // the bytes of both blocks
          tma_load_2d_pair(a, &map_x, i * TILE_K, m0, &full[s]);
          tma_load_2d_pair(a + BOX_BYTES, &map_w, i * TILE_K, w_row, &full[s]);
        }
      }
    }
  } else if (warp == 1) {
    if (leader && elect_one()) {
      const uint32_t idesc = idesc_e4m3(2 * TILE, ep.tile_n);
      const MatrixDesc base(smem_u32(smem));
      int j = 0, s = 0;
      uint32_t phase = 0;
      for (int tile = pair; tile < n_tiles && !*failed; tile += pairs, ++j) {
        const int acc = j & 1;
        if (!wait_or_abort(&acc_empty[acc], ((j >> 1) & 1) ^ 1, failed)) break;  // both epilogues have read this buffer
        tc_fence_after();
        for (int i = 0; i < k_steps; ++i) {
          if (!quick_wait(&full[s], phase, failed)) break;
          tc_fence_after();
          const uint32_t x = base.lo + (uint32_t)(s * stage_bytes >> 4), w = x + (BOX_BYTES >> 4);
#pragma unroll
          for (int kk = 0; kk < TILE_K / UMMA_K; ++kk)
            issue_e4m3_pair(tmem + acc * 256, x + kk * (UMMA_K >> 4), base.hi, w + kk * (UMMA_K >> 4), idesc, kk > 0 ? 1u : i > 0);
          tc_commit_pair(&empty[s]);
          if (++s == stages) s = 0, phase ^= 1;
        }
        tc_commit_pair(&acc_full[acc]);
      }
    }
  } else {
    const int quarter = warp & 3, half = (warp - 2) >> 2;
    float *scales = col_scales[warp - 2], *biases = col_biases[warp - 2];
    int j = 0;
    for (int tile = pair; tile < n_tiles; tile += pairs, ++j) {
      const int acc = j & 1;
      const int row = (tile % tiles_m) * 2 * TILE + (int)rank * TILE + quarter * 32 + lane, n0 = (tile / tiles_m) * tile_n;
      const float sx = row < M ? ep.sx[row] : 0.f;
      // read from global memory in the loop below they would be waited for 16 columns at a time
      __syncwarp();
      for (int i = lane; i < 128; i += 32) {
        const bool up = ep.glu && i >= 64;
        const int at = up ? i - 64 : i, c = (at >> 4) * 32 + half * 16 + (at & 15);
        const int col = min(n0 + c, ep.outputs - 1) + (up ? ep.outputs : 0);
        scales[i] = ep.sw[col];
        if (ep.bias) biases[i] = ep.bias[col];
      }
      __syncwarp();
      if (!warp_wait(&acc_full[acc], (j >> 1) & 1, failed)) break;
      tc_fence_after();
      const uint32_t taddr = tmem + acc * 256 + ((uint32_t)(quarter * 32) << 16);
      for (int c0 = half * 16; c0 < tile_n; c0 += 32) {  // every lane loads: tensor-memory loads are warp-wide
        float v[16], u[16];
        const int col0 = n0 + c0, at = c0 >> 5 << 4;
        if (ep.glu) tmem_load_2x16(taddr + c0, taddr + tile_n + c0, v, u);
        else tmem_load_16(taddr + c0, v);
        if (row >= M || col0 >= ep.outputs) continue;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          scale4(v + 4 * q, sx, scales + at + 4 * q, ep.bias ? biases + at + 4 * q : nullptr);
          if (ep.glu) {
            scale4(u + 4 * q, sx, scales + 64 + at + 4 * q, ep.bias ? biases + 64 + at + 4 * q : nullptr);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[4 * q + e] = activate(v[4 * q + e], ep.act) * u[4 * q + e];
          }
        }
        store16(ep, v, row, col0, M);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (leader) mbar_arrive(&acc_empty[acc]);
        else mbar_arrive_remote(&acc_empty[acc], 0);
      }
    }
    tc_fence_before();
  }
  __syncthreads();
  cluster_sync_all();  // nothing is sent to a block that has left
  if (threadIdx.x == 0 && *failed && error_flag) atomicExch(error_flag, 4);
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
}

// ---- up to 256 rows (decode) ---------------------------------------------------------------------------------------
// The operands swapped: 128 rows of w fill the instruction's rows and the tokens are its columns (16 to 256), since a product
// of this size is bound by reading w once.  A tile is 128 rows of w (GLU: 64 gate rows and the 64 up rows that belong to them),
// a step of it 128 k.  Many tiles, or short ones: a block takes one whole tile, two blocks a multiprocessor, and stores y.  Few
// tiles (cut_of): every multiprocessor takes an equal run of the steps of all tiles; where a tile's steps fall to several blocks,
// each leaves its sums in a slot of its own in scratch memory, and a second kernel adds them in the order of k; under GLU all
// tiles of such a cut go that way, since a gate and its up value lie in different lanes.  (Clusters that shared a tile and added
// their sums through distributed shared memory: 6,144 x 4,096 by 64 rows 11.8 us, 4,096 x 14,336 17.7 us; so 9.5 and 14.1.)  The
// cut depends on the weights' shape alone, so a row's result does not depend on the rest of the batch.  The first stages'
// boxes of w are asked for before griddepcontrol.wait: weights do not depend on the kernel before.
//   warp 0 the copies of w, warp 10 those of x (one thread for both: 4,096 x 14,336 by 8 rows 14.5 us, 6,144 x 4,096 by 64 10.2; so
//   12.8 and 9.5), warp 1 the instructions, warps 2-9 the epilogue, under the next tile's steps up to 128 tokens
__global__ void __launch_bounds__(ROWS_THREADS, 2) e4m3_rows_kernel(const __grid_constant__ CUtensorMap map_x,
                                                               const __grid_constant__ CUtensorMap map_w, Epilogue ep, int M,
                                                               int tiles, int k_steps, int* __restrict__ error_flag) {
  extern __shared__ unsigned char smem_unaligned[];
  unsigned char* smem = smem_unaligned + (-smem_u32(smem_unaligned) & 1023);
  const int stage_bytes = BOX_BYTES + ep.n_tokens * TILE_K, stages = ep.stages;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + stages * stage_bytes);
  uint64_t* empty = full + MAX_STAGES;
  uint64_t* acc_full = empty + MAX_STAGES;  // [2]
  uint64_t* acc_empty = acc_full + 2;       // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  __shared__ int failed_flag;
  __shared__ float row_scales[256];  // of x: read from global memory they would be waited for at every run of tokens
  volatile int* failed = &failed_flag;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int all = tiles * k_steps, row_step = ep.glu ? TILE / 2 : TILE;
  const int lo = first_step(blockIdx.x, gridDim.x, all), hi = first_step(blockIdx.x + 1, gridDim.x, all);
  const int accs = ep.n_tokens <= 128 ? 2 : 1;
  // a block of one whole tile, beside which others fit, takes no more tensor memory than it needs
  uint32_t tmem_cols = 32;
  while ((int)tmem_cols < ep.n_tokens) tmem_cols *= 2;
  if (ep.slots) tmem_cols = 256;

  if (threadIdx.x == 0) {
    failed_flag = 0;
    for (int s = 0; s < MAX_STAGES; ++s) {
      mbar_init(&full[s], 2);
      mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], EPILOGUE_WARPS);
    }
    mbar_fence_init();
  }
  if (warp == 1) tmem_alloc(tmem_slot, tmem_cols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_launch_dependents();  // a block of the next kernel must not take the tensor memory that this one still needs

  if (warp == 0) {
    if (elect_one()) {  // the weights, which do not depend on the kernel before
      int tile = lo / k_steps, k = lo - tile * k_steps, s = 0;
      uint32_t phase = 1;
      for (int i = lo; i < hi; ++i) {
        if (!quick_wait(&empty[s], phase, failed)) break;
        unsigned char* to = smem + s * stage_bytes;
        mbar_arrive_expect_tx(&full[s], BOX_BYTES);
        tma_load_2d(to, &map_w, k * TILE_K, tile * row_step, &full[s]);
        if (ep.glu) tma_load_2d(to + BOX_BYTES / 2, &map_w, k * TILE_K, ep.outputs + tile * row_step, &full[s]);
        if (++k == k_steps) k = 0, ++tile;
        if (++s == stages) s = 0, phase ^= 1;
      }
    }
  } else if (warp == 2 + EPILOGUE_WARPS) {
    if (elect_one()) {
      pdl_wait();  // x is what the kernel before wrote
      int k = lo % k_steps, s = 0;
      uint32_t phase = 1;
      for (int i = lo; i < hi; ++i) {
        if (!quick_wait(&empty[s], phase, failed)) break;
        mbar_arrive_expect_tx(&full[s], stage_bytes - BOX_BYTES);
        tma_load_2d(smem + s * stage_bytes + BOX_BYTES, &map_x, k * TILE_K, 0, &full[s]);
        if (++k == k_steps) k = 0;
        if (++s == stages) s = 0, phase ^= 1;
      }
    }
  } else if (warp == 1) {
    if (elect_one()) {
      const uint32_t idesc = idesc_e4m3(TILE, ep.n_tokens);
      const MatrixDesc base(smem_u32(smem));
      int k = lo % k_steps, s = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 1;
      for (int i = lo; i < hi; ++i) {
        const bool first = i == lo || k == 0;
        if (first && !quick_wait(&acc_empty[acc], acc_phase, failed)) break;
        if (!quick_wait(&full[s], phase, failed)) break;
        tc_fence_after();
        const uint32_t w = base.lo + (uint32_t)(s * stage_bytes >> 4), x = w + (BOX_BYTES >> 4);
#pragma unroll
        for (int kk = 0; kk < TILE_K / UMMA_K; ++kk)
          issue_e4m3(tmem + acc * 128, w + kk * (UMMA_K >> 4), base.hi, x + kk * (UMMA_K >> 4), idesc, kk > 0 ? 1u : !first);
        tc_commit(&empty[s]);
        if (++k == k_steps) k = 0;
        if (k == 0 || i + 1 == hi) {
          tc_commit(&acc_full[acc]);
          if (++acc == accs) acc = 0, acc_phase ^= 1;
        }
        if (++s == stages) s = 0, phase ^= 1;
      }
    }
  } else {
    pdl_wait();  // these warps read and write what other kernels touch (scales, scratch memory, y)
    for (int t = threadIdx.x - 64; t < ep.n_tokens; t += 32 * EPILOGUE_WARPS) row_scales[t] = t < M ? ep.sx[t] : 0.f;
    asm volatile("bar.sync 1, %0;\n" ::"n"(32 * EPILOGUE_WARPS) : "memory");
    const int quarter = warp & 3, part = (warp - 2) >> 2, row = quarter * 32 + lane;
    // A block of one whole tile under GLU: the sums meet in shared memory, as float32 [128][n_tokens + 4] over the stages (every
    // copy into them has landed and every instruction that read them is done once the accumulator is ready).
    const bool exchange = ep.glu && ep.slots == 0;
    float* sums = reinterpret_cast<float*>(smem);
    const int sums_pitch = ep.n_tokens + 4;
    int acc = 0, segment = 0;
    uint32_t acc_phase = 0;
    for (int i = lo; i < hi; ++segment) {
      const int tile = i / k_steps, k_lo = i - tile * k_steps, k_hi = min(k_steps, hi - tile * k_steps), col = tile * TILE + row;
      const bool whole = !ep.glu && k_lo == 0 && k_hi == k_steps, live = whole && col < ep.outputs;
      const float sw = live ? ep.sw[col] : 0.f, bias = live && ep.bias ? ep.bias[col] : 0.f;
      float* slot = ep.scratch + ((size_t)(ep.slots * blockIdx.x + segment) * ep.n_tokens) * TILE + row;
      if (!warp_wait(&acc_full[acc], acc_phase, failed)) break;
      tc_fence_after();
      for (int c0 = 16 * part; c0 < ep.n_tokens; c0 += 32) {
        float v[16];
        tmem_load_16(tmem + acc * 128 + ((uint32_t)(quarter * 32) << 16) + c0, v);
        if (exchange) {
#pragma unroll
          for (int j = 0; j < 16; j += 4)
            *reinterpret_cast<float4*>(sums + row * sums_pitch + c0 + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
        } else if (!whole) {
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (FMS_IN(slot + (c0 + j) * TILE - ep.scratch, max(ep.scratch_floats, 1L))) slot[(size_t)(c0 + j) * TILE] = v[j];
        } else if (live) {
#pragma unroll
          for (int j = 0; j < 16; ++j) v[j] = fmaf(v[j], row_scales[c0 + j] * sw, bias);
          store_column<16>(ep, v, c0, col, M, ep.outputs);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_empty[acc]);
      if (++acc == accs) acc = 0, acc_phase ^= 1;
      i += k_hi - k_lo;
    }
    if (exchange) {
      asm volatile("bar.sync 1, %0;\n" ::"n"(32 * EPILOGUE_WARPS) : "memory");
      const int e = threadIdx.x - 64, r = e & 63, col = blockIdx.x * (TILE / 2) + r;
      if (col < ep.outputs && !*failed) {
        const float sw = ep.sw[col], su = ep.sw[ep.outputs + col];
        const float bias = ep.bias ? ep.bias[col] : 0.f;
        const float bias_up = ep.bias ? ep.bias[ep.outputs + col] : 0.f;
        for (int t = 4 * (e >> 6); t < ep.n_tokens; t += 16) {
          const float4 g = *reinterpret_cast<const float4*>(sums + r * sums_pitch + t);
          const float4 u = *reinterpret_cast<const float4*>(sums + (TILE / 2 + r) * sums_pitch + t);
          float v[4] = {g.x, g.y, g.z, g.w}, up[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float sx = row_scales[t + j];
            v[j] = activate(fmaf(v[j], sx * sw, bias), ep.act) * fmaf(up[j], sx * su, bias_up);
          }
          store_column<4>(ep, v, t, col, M, ep.outputs);
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && *failed && error_flag) atomicExch(error_flag, 4);
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, tmem_cols);
  }
}

// y of the tiles that several blocks share (GLU: of all) in a cut of equal runs: their sums in the order of k, scales, bias,
// activation.  Block: a tile's columns of y by 4 tokens (GLU: 64 by 8); the slots of four blocks are on their way at a time.
__global__ void __launch_bounds__(TILE) e4m3_join_kernel(Epilogue ep, int M, int k_steps, int blocks, int tiles) {
  pdl_launch_dependents();
  const int all = tiles * k_steps, tile = blockIdx.x, start = tile * k_steps, row_step = ep.glu ? TILE / 2 : TILE;
  const int from = block_of_step(start, blocks, all), to = block_of_step(start + k_steps - 1, blocks, all);
  const int row = (int)threadIdx.x & (row_step - 1), col = tile * row_step + row;
  const int t0 = (blockIdx.y * (TILE / row_step) + (int)threadIdx.x / row_step) * 4;
  if ((!ep.glu && from == to) || col >= ep.outputs || t0 >= M) return;  // some block of some tile goes on, and waits
  // only the first block of a tile can have begun with an earlier one
  const int head = tile - first_step(from, blocks, all) / k_steps;
  const size_t pitch = (size_t)ep.n_tokens * TILE;
  const float sw = ep.sw[col];  // of the weight
  pdl_wait();
  const float bias = ep.bias ? ep.bias[col] : 0.f;  // any tensor: the kernel before the product may have written it
  float sx[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) sx[j] = t0 + j < M ? ep.sx[t0 + j] : 0.f;
  auto sum_of = [&](const float* at) { return FMS_IN(at - ep.scratch, max(ep.scratch_floats, 1L)) ? __ldcg(at) : 0.f; };
  auto total = [&](int r, float* sum) {
    const float* slots = ep.scratch + (size_t)t0 * TILE + r;
    sum[0] = sum[1] = sum[2] = sum[3] = 0.f;
    for (int b = from; b <= to; b += 4) {
      float v[4][4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          v[i][j] = b + i <= to ? sum_of(slots + ((size_t)ep.slots * (b + i) + (b + i == from ? head : 0)) * pitch + j * TILE) : 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) sum[j] += v[i][j];
    }
  };
  float y[4];
  total(row, y);
#pragma unroll
  for (int j = 0; j < 4; ++j) y[j] = fmaf(y[j], sx[j] * sw, bias);
  if (ep.glu) {
    const float su = ep.sw[ep.outputs + col], bias_up = ep.bias ? ep.bias[ep.outputs + col] : 0.f;
    float up[4];
    total(TILE / 2 + row, up);
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = activate(y[j], ep.act) * fmaf(up[j], sx[j] * su, bias_up);
  }
  store_column<4>(ep, y, t0, col, M, ep.outputs);
}

// [rows, pitch] bytes in boxes of `box_rows` rows x 128 bytes with the 128-byte swizzle
int make_byte_map(CUtensorMap* map, const void* base, long rows, long pitch, int box_rows) {
  EncodeTiled enc = encode_tiled();
  if (enc == nullptr) return fms_fail("gemm_e4m3: the driver does not export cuTensorMapEncodeTiled");
  const cuuint64_t dims[2] = {(cuuint64_t)pitch, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)pitch};
  const cuuint32_t box[2] = {TILE_K, (cuuint32_t)box_rows}, elem[2] = {1, 1};
  CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, elem,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fms_fail("gemm_e4m3: cuTensorMapEncodeTiled failed with %d (rows %ld, pitch %ld)", (int)r, rows, pitch);
  return 0;
}

// The width of a pair's tile: the one whose tiles cost least in whole rounds of the pairs.  A tile costs, in one round (2,304 rows, 8 tiles
// a row, k 8,192), 29.8 us at 256 columns, 28.5 at 240, 27.4 at 224, 25.3 at 208, 24.2 at 192, 23.2 at 176, 22.0 at 160, 21.2 at 128 and
// 19.4 at 64: of the widest tile 0.96, 0.92, 0.85, 0.81, 0.78, 0.74, 0.71 and 0.65.  The line below is within 6% of that.  Widths by 16
// are a pair's shapes where both operands come from shared memory; GLU: by 32, so that a half is a multiple of 16.
int choose_tile_n(int tiles_m, int cols, bool glu, int pairs) {
  const int step = glu ? 32 : 16;
  long best_cost = -1;
  int best = 256;
  for (int tn = 256; tn >= 64; tn -= step) {
    const int out = glu ? tn / 2 : tn;
    const long tiles = (long)tiles_m * ((cols + out - 1) / out);
    const long cost = ((tiles + pairs - 1) / pairs) * (tn == 256 ? 10000 : 5600 + 14 * tn);
    if (best_cost < 0 || cost < best_cost) {
      best_cost = cost;
      best = tn;
    }
  }
  return best;
}

// How the second kernel cuts a product; slots 0: a block takes one whole tile, and there is nothing to join.  Equal runs cost the
// second launch and a trip through scratch memory, about what 16 steps of a block cost, and more the more tiles there are.  By
// 64 rows, equal runs against whole tiles, us: 4,096 x 4,096 8.1 : 11.4, 6,144 x 4,096 10.0 : 11.5, 8,192 x 4,096 11.0 : 11.7,
// 6,144 x 2,560 8.3 : 8.3, 8,192 x 2,048 8.4 : 7.5, 12,288 x 4,096 14.1 : 12.6, 28,672 x 4,096 28.7 : 21.7.  That is what the line was
// drawn by; since whole tiles take no more tensor memory than their sums they are ahead on a part of this side of it too: 7.8 : 8.5,
// 9.5 : 9.1, 10.3 : 9.7, 7.8 : 6.5, 8.1 : 6.4, 14.1 : 11.6, and 12,288 x 12,288 30.8 : 27.6.
// A run is 4 steps or more: the sums of 32 blocks of one step each take longer to join than to make.
struct Cut {
  int tiles, k_steps, blocks, slots;
};
Cut cut_of(int outputs, bool glu, long pitch) {
  Cut c;
  const int row_step = glu ? TILE / 2 : TILE, sms = multiprocessors();
  c.tiles = (outputs + row_step - 1) / row_step;
  c.k_steps = (int)((pitch + TILE_K - 1) / TILE_K);
  if (3L * c.tiles >= 2L * sms || (long)c.k_steps * (sms - c.tiles) <= 16L * sms) {
    c.blocks = c.tiles;
    c.slots = 0;
  } else {  // more than 16 steps a tile and fewer tiles than multiprocessors, so more blocks than tiles: a run reaches into two at most
    const long runs = (long)c.tiles * c.k_steps / 4;
    c.blocks = runs < sms ? (int)runs : sms;
    c.slots = 2;
  }
  return c;
}

constexpr int ROWS_MOST = 256;  // rows of x that the second kernel takes
// A block that holds all of the tensor memory takes so much shared memory that no block that wants some fits beside it: one that
// waits for it could be what this one waits for (the partner of a pair, the kernel before).
constexpr size_t PAIR_RING = 200 * 1024, EXTRA = 1024 /* alignment */ + 512 /* barriers */;

int launch(const void* x, const void* w, Epilogue ep, int M, int N, long pitch, long scratch_floats, int* error_flag, cudaStream_t stream) {
  if (pitch <= 0 || pitch % 16 || pitch > 0x7fffff00L) return fms_fail("gemm_e4m3: rows of %ld bytes, a multiple of 16 is wanted", pitch);
  if (((uintptr_t)x | (uintptr_t)w | (uintptr_t)ep.out) & 15) return fms_fail("gemm_e4m3: operands and result must be 16-byte aligned");
  const int k_steps = (int)((pitch + TILE_K - 1) / TILE_K);
  CUtensorMap map_x, map_w;
  static uint64_t rows_allowed = 0, pair_allowed = 0;
  if (M <= ROWS_MOST ? allow_smem("gemm_e4m3", e4m3_rows_kernel, (int)(PAIR_RING + EXTRA), &rows_allowed)
                     : allow_smem("gemm_e4m3", e4m3_pair_kernel, (int)(PAIR_RING + EXTRA), &pair_allowed))
    return 1;
  if (M <= ROWS_MOST) {
    const Cut c = cut_of(ep.outputs, ep.glu != 0, pitch);
    ep.n_tokens = (M + 15) / 16 * 16;
    ep.slots = c.slots;
    ep.scratch_floats = scratch_floats;
    if ((long)c.tiles * c.k_steps > 0x3fffffffL) return fms_fail("gemm_e4m3: %d tiles of %d steps", c.tiles, c.k_steps);
    const long wanted = (long)c.blocks * c.slots * ep.n_tokens * TILE;
    if (scratch_floats < wanted) return fms_fail("gemm_e4m3: %ld floats of scratch memory, %ld are wanted", scratch_floats, wanted);
    // room for two blocks on a multiprocessor where they are as many and the ring stays deep enough
    const size_t ring = ep.n_tokens <= 128 && c.slots == 0 && c.blocks > multiprocessors() ? PAIR_RING / 2 : PAIR_RING;
    ep.stages = min((int)(ring / (BOX_BYTES + ep.n_tokens * TILE_K)), MAX_STAGES);
    if (make_byte_map(&map_x, x, M, pitch, ep.n_tokens) || make_byte_map(&map_w, w, N, pitch, ep.glu ? TILE / 2 : TILE)) return 1;
    fms_launch(e4m3_rows_kernel, dim3(c.blocks), dim3(ROWS_THREADS), ring + EXTRA, stream, map_x, map_w, ep, M, c.tiles, c.k_steps, error_flag);
    if (fms_launch_status("gemm_e4m3")) return 1;
    if (c.slots == 0) return 0;
    const int each = ep.glu ? 8 : 4;
    fms_launch(e4m3_join_kernel, dim3(c.tiles, (ep.n_tokens + each - 1) / each), dim3(TILE), 0, stream, ep, M, c.k_steps, c.blocks, c.tiles);
    return fms_launch_status("gemm_e4m3_join");
  }
  const int pairs = max(multiprocessors() / 2, 1), tiles_m = (M + 2 * TILE - 1) / (2 * TILE);
  ep.tile_n = choose_tile_n(tiles_m, ep.outputs, ep.glu != 0, pairs);
  const int stage_bytes = BOX_BYTES + ep.tile_n / 2 * TILE_K, out = ep.glu ? ep.tile_n / 2 : ep.tile_n;
  ep.stages = min((int)(PAIR_RING / stage_bytes), MAX_STAGES);
  if (make_byte_map(&map_x, x, M, pitch, TILE) || make_byte_map(&map_w, w, N, pitch, ep.tile_n / 2)) return 1;
  const long tiles = (long)((ep.outputs + out - 1) / out) * tiles_m;
  if (tiles > 0x7fffffffL) return fms_fail("gemm_e4m3: %ld tiles", tiles);
  const int busy = (int)(tiles < pairs ? tiles : pairs);
  // A plain launch: the pairs, which want all of the tensor memory, run beside no block of another kernel of the stream.  (Launched
  // while the kernel before was still draining, and asking for its tensor memory ahead of the cluster's barrier, a pair of blocks in a
  // prompt of 8,192 tokens began and never got it.)
  e4m3_pair_kernel<<<dim3(2 * busy), dim3(THREADS), PAIR_RING + EXTRA, stream>>>(map_x, map_w, ep, M, k_steps, error_flag);
  return fms_launch_status("gemm_e4m3");
}
}  // namespace

// Columns of the accumulator of a tile where pairs of thread blocks take M rows; 0: the other kernel does.
FMS_API int fms_e4m3_tile(int M, int N, int glu) {
  if (M <= ROWS_MOST || N <= 0) return 0;
  return choose_tile_n((M + 2 * TILE - 1) / (2 * TILE), glu ? N / 2 : N, glu != 0, max(multiprocessors() / 2, 1));
}

// Floats of scratch memory that the products of M rows with weights of N rows (glu 1: of N / 2 gate and N / 2 up rows) want.
FMS_API long fms_e4m3_scratch(long M, long N, long pitch, long glu) {
  if (M <= 0 || N <= 0 || pitch <= 0 || M > ROWS_MOST) return 0;
  const Cut c = cut_of((int)(glu ? N / 2 : N), glu != 0, pitch);
  return (long)c.blocks * c.slots * ((M + 15) / 16 * 16) * TILE;
}

// y [M, N] (bfloat16, or float32 with out_dtype FMS_F32) of x [M, pitch] and w [N, pitch], e4m3, with sx [M], sw [N] float32 and
// bias [N] bfloat16 or float32, or null.
FMS_API int fms_linear_e4m3(const void* x, const float* sx, const void* w, const float* sw, const void* bias, int bias_dtype, void* y, int out_dtype,
                            int M, int N, long pitch, float* scratch, long scratch_floats, int* error_flag, cudaStream_t stream) {
  if (M <= 0 || N <= 0) return 0;
  if (out_dtype != FMS_F32 && out_dtype != FMS_BF16) return fms_fail("linear_e4m3: out dtype %d", out_dtype);
  Epilogue ep = {};
  ep.out = y;
  ep.bias = {bias, bias_dtype == FMS_F32};
  ep.sx = sx;
  ep.sw = sw;
  ep.out_f32 = out_dtype == FMS_F32;
  ep.outputs = N;
  if (check_bias("linear_e4m3", ep.bias, bias_dtype)) return 1;
  ep.scratch = scratch;
  return launch(x, w, ep, M, N, pitch, scratch_floats, error_flag, stream);
}

// y [M, hidden] bfloat16 = act(gate) * up for w = [gate; up] of 2 hidden rows (sw and bias [2 hidden]).
FMS_API int fms_glu_e4m3(const void* x, const float* sx, const void* w, const float* sw, const void* bias, int bias_dtype, void* y, int M, int hidden,
                         long pitch, int act, float* scratch, long scratch_floats, int* error_flag, cudaStream_t stream) {
  if (M <= 0 || hidden <= 0) return 0;
  if (act < 0 || act > 3) return fms_fail("glu_e4m3: activation %d", act);
  Epilogue ep = {};
  ep.out = y;
  ep.bias = {bias, bias_dtype == FMS_F32};
  ep.sx = sx;
  ep.sw = sw;
  ep.glu = 1;
  ep.act = act;
  ep.outputs = hidden;
  ep.scratch = scratch;
  if (check_bias("glu_e4m3", ep.bias, bias_dtype)) return 1;
  return launch(x, w, ep, M, 2 * hidden, pitch, scratch_floats, error_flag, stream);
}
