// y[m, n] = sum_k x[m, k] * (q[n, k] - z[n, g(k)]) * s[n, g(k)] (+ bias[n]): bfloat16 rows, weights of 4 bits with one bfloat16
// scale and one whole zero point a group of consecutive k.  GLU: act(gate) * up for weights [gate; up].
//
// Layout, made once (kernels/quantized.py, pack_int4).  Weights: blocks of 16 rows x 128 k, 1,024 bytes each, [rows / 16]
// [k / 128][16 rows][4 pieces of 16 bytes]; word w of a row's piece c holds k = 32 w + 8 c .. + 7, value 2 i in bits 4 i and
// value 2 i + 1 in bits 16 + 4 i, so that one shift and one logical operation leave a pair of neighbours in the halves of a
// register; piece c lies at place c ^ (row / 2 % 4), which lets the rows of a warp read a piece from shared memory without
// meeting in a bank.  Groups: [groups][N] words, the scale in the low half and 128 + z, exact in bfloat16, in the high half.
//
// 0x4300 | q is the bfloat16 128 + q; minus 128 + z it is q - z, exact.
//   few rows: mma.sync over q - z, whole numbers, a group's float32 sum times its scale: nothing is rounded but the result.
//   more rows: tcgen05 over (q - z) * s rounded to bfloat16 on its way into the operand, as the bfloat16 weight would be: the
//             tensor cores' sums run over all of k and cannot be scaled group by group.
#include <cuda.h>

#include "common.cuh"

namespace {
#include "tcgen05.cuh"

constexpr int BLOCK_ROWS = 16, BLOCK_K = 128, BLOCK_BYTES = 1024;

__device__ __forceinline__ float activate(float g, int act) {
  switch (act) {
    case 0: return g / (1.f + expf(-g));
    case 1: return 0.5f * g * (1.f + erff(g * 0.70710678118654752f));
    case 2: return 0.5f * g * (1.f + tanhf(0.7978845608028654f * (g + 0.044715f * g * g * g)));
    default: return fmaxf(g, 0.f);
  }
}

// the 8 values of a word as four pairs of bfloat16 q - z
__device__ __forceinline__ void unpack8(uint32_t word, __nv_bfloat162 zero, uint32_t* pairs) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t v = ((word >> (4 * i)) & 0x000f000fu) | 0x43004300u;
    const __nv_bfloat162 d = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&v), zero);
    pairs[i] = *reinterpret_cast<const uint32_t*>(&d);
  }
}
__device__ __forceinline__ __nv_bfloat162 both(uint32_t half) {
  const uint32_t v = __byte_perm(half, half, 0x1010);
  return *reinterpret_cast<const __nv_bfloat162*>(&v);
}

struct Int4Args {
  const __nv_bfloat16* x;     // [M, K]
  const unsigned char* w;     // the packed blocks
  const uint32_t* groups;     // [n_groups, N]
  const __nv_bfloat16* bias;  // [N] or null
  __nv_bfloat16* y;           // [M, outputs]
  int M, N, K, k_blocks, n_groups, group, outputs, act;
};

// ---- up to 16 rows ------------------------------------------------------------------------------------------------------
// Bound by reading the weights once.  A block of 8 warps owns RT tiles of 16 rows of w (GLU: 8 gate rows and the 8 up rows that
// belong to them); the warps take the 128-k blocks in turn and add their sums in shared memory in a fixed order.  A lane
// copies what it needs (its piece of two rows, of the x rows, the groups' words) into a ring that only it reads, D blocks ahead.
// PER: scales a block of 128 k (1: groups of whole blocks; 2: of 64 k; 4: any multiple of 32).
constexpr int WARPS = 8, THREADS = 256;

__device__ __forceinline__ void mma_bf16(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void cp_async16(void* smem, const void* gmem, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(smem_u32(smem)), "l"(gmem), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async4(void* smem, const void* gmem) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;\n" ::"r"(smem_u32(smem)), "l"(gmem) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory"); }

template <int NT, int RT, int PER, bool GLU, int D>
__global__ void __launch_bounds__(THREADS) int4_few_rows_kernel(Int4Args p) {
  constexpr int WL = RT * 2, XL = NT * 4, LOADS = WL + XL, GL = RT * 2 * PER;
  constexpr int TILE_ROWS = GLU ? 8 : 16;
  extern __shared__ uint4 ring[];
  uint32_t* group_ring = reinterpret_cast<uint32_t*>(ring + (size_t)D * LOADS * THREADS);
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;

  const unsigned char* wp[RT][2];
  const uint32_t* gp[RT][2];
#pragma unroll
  for (int t = 0; t < RT; ++t)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = (blockIdx.x * RT + t) * TILE_ROWS + g;
      const int row = min(GLU ? r + h * p.outputs : r + 8 * h, p.N - 1);
      wp[t][h] = p.w + ((size_t)(row / BLOCK_ROWS) * p.k_blocks) * BLOCK_BYTES + (row % BLOCK_ROWS) * 64 + ((c ^ ((row >> 1) & 3)) * 16);
      gp[t][h] = p.groups + row;
    }
  const __nv_bfloat16* xp[NT];
  bool xok[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    xok[j] = j * 8 + g < p.M;
    xp[j] = p.x + (size_t)(xok[j] ? j * 8 + g : 0) * p.K + 8 * c;
  }
  const int mine = p.k_blocks > warp ? (p.k_blocks - warp + WARPS - 1) / WARPS : 0;
  auto issue_w = [&](int i) {
    if (i >= mine) return;
    const int kb = warp + i * WARPS;
    uint4* st = ring + (size_t)(i % D) * LOADS * THREADS + threadIdx.x;
    uint32_t* gs = group_ring + (size_t)(i % D) * GL * THREADS + threadIdx.x;
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        cp_async16(st + (t * 2 + h) * THREADS, wp[t][h] + (size_t)kb * BLOCK_BYTES, true);
#pragma unroll
        for (int u = 0; u < PER; ++u) {
          const int at = min((kb * BLOCK_K + u * (BLOCK_K / PER)) / p.group, p.n_groups - 1);
          cp_async4(gs + ((t * 2 + h) * PER + u) * THREADS, gp[t][h] + (size_t)at * p.N);
        }
      }
  };
  auto issue_x = [&](int i) {
    if (i >= mine) return;
    const int k0 = (warp + i * WARPS) * BLOCK_K;
    uint4* st = ring + ((size_t)(i % D) * LOADS + WL) * THREADS + threadIdx.x;
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int u = 0; u < 4; ++u) {  // K is a multiple of 8: a lane's 8 values are all inside or all outside
        const bool in = xok[j] && k0 + 32 * u + 8 * c < p.K;
        cp_async16(st + (j * 4 + u) * THREADS, xp[j] + (in ? k0 + 32 * u : 0), in);
      }
  };
  float acc[RT][NT][4];
#pragma unroll
  for (int t = 0; t < RT; ++t)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[t][j][e] = 0.f;
#pragma unroll
  for (int i = 0; i < D; ++i) issue_w(i);  // weights: before the wait for the kernel that makes x
  pdl_wait();
#pragma unroll
  for (int i = 0; i < D; ++i) {
    issue_x(i);
    cp_async_commit();  // the first group holds all stages' weights
  }
  for (int i = 0; i < mine; ++i) {
    cp_async_wait<D - 1>();
    const uint4* st = ring + (size_t)(i % D) * LOADS * THREADS + threadIdx.x;
    const uint32_t* gs = group_ring + (size_t)(i % D) * GL * THREADS + threadIdx.x;
    uint4 b[NT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int u = 0; u < 4; ++u) b[j][u] = st[(WL + j * 4 + u) * THREADS];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      const uint4 lo = st[(t * 2) * THREADS], hi = st[(t * 2 + 1) * THREADS];
      const uint32_t wl[4] = {lo.x, lo.y, lo.z, lo.w}, wh[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
      for (int u = 0; u < PER; ++u) {
        const uint32_t gl = gs[((t * 2) * PER + u) * THREADS], gh = gs[((t * 2 + 1) * PER + u) * THREADS];
        const __nv_bfloat162 zl = both(gl >> 16), zh = both(gh >> 16);
        float part[NT][4];
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) part[j][e] = 0.f;
#pragma unroll
        for (int v = u * (4 / PER); v < (u + 1) * (4 / PER); ++v) {
          uint32_t a[4], d[4];
          unpack8(wl[v], zl, a);
          unpack8(wh[v], zh, d);
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            mma_bf16(part[j], a[0], d[0], a[1], d[1], b[j][v].x, b[j][v].y);
            mma_bf16(part[j], a[2], d[2], a[3], d[3], b[j][v].z, b[j][v].w);
          }
        }
        const float sl = __uint_as_float(gl << 16), sh = __uint_as_float(gh << 16);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          acc[t][j][0] = fmaf(part[j][0], sl, acc[t][j][0]);
          acc[t][j][1] = fmaf(part[j][1], sl, acc[t][j][1]);
          acc[t][j][2] = fmaf(part[j][2], sh, acc[t][j][2]);
          acc[t][j][3] = fmaf(part[j][3], sh, acc[t][j][3]);
        }
      }
    }
    issue_w(i + D);  // into the stage just consumed
    issue_x(i + D);
    cp_async_commit();
  }
  cp_async_wait<0>();
  __syncthreads();  // the ring is free: the warps' sums go over it
  float* red = reinterpret_cast<float*>(ring);  // [WARPS][RT * NT][32][4]
#pragma unroll
  for (int t = 0; t < RT; ++t)
#pragma unroll
    for (int j = 0; j < NT; ++j)
      *reinterpret_cast<float4*>(red + ((warp * RT * NT + t * NT + j) * 32 + lane) * 4) =
          make_float4(acc[t][j][0], acc[t][j][1], acc[t][j][2], acc[t][j][3]);
  __syncthreads();
  auto total = [&](int t, int j, int l, int e) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) s += red[((w * RT * NT + t * NT + j) * 32 + l) * 4 + e];
    return s;
  };
  // element e of lane l is (row l / 4 + 8 (e / 2) of the tile, row 2 (l % 4) + e % 2 of x); neighbouring threads take neighbouring rows of w
  constexpr int ITEMS = RT * NT * 8 * TILE_ROWS;
  for (int i = threadIdx.x; i < ITEMS; i += THREADS) {
    const int r = i % TILE_ROWS, t = i / TILE_ROWS % RT, mm = i / (TILE_ROWS * RT), j = mm / 8, m = mm % 8;
    const int col = (blockIdx.x * RT + t) * TILE_ROWS + r, l = (r & 7) * 4 + (m >> 1), e = m & 1;
    if (col >= p.outputs || mm >= p.M) continue;
    float v;
    if (GLU) {
      float gate = total(t, j, l, e), up = total(t, j, l, e + 2);
      if (p.bias) {
        gate += __bfloat162float(p.bias[col]);
        up += __bfloat162float(p.bias[p.outputs + col]);
      }
      v = activate(gate, p.act) * up;
    } else {
      v = total(t, j, l, e + 2 * (r >> 3));
      if (p.bias) v += __bfloat162float(p.bias[col]);
    }
    if (FMS_IN((size_t)mm * p.outputs + col, (size_t)p.M * p.outputs)) p.y[(size_t)mm * p.outputs + col] = __float2bfloat16_rn(v);
  }
}

// Asks for a kernel's shared memory once on every device.
template <typename Kernel> int allow_smem(const char* what, Kernel kernel, int bytes, uint64_t* done) {
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e == cudaSuccess && device < 64 && (*done >> device & 1)) return 0;
  if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return fms_fail("%s: %d bytes of shared memory refused: %s", what, bytes, cudaGetErrorString(e));
  if (device < 64) *done |= 1ull << device;
  return 0;
}

template <int NT, int RT, int PER, bool GLU> int launch_few(const Int4Args& p, cudaStream_t stream) {
  constexpr int STAGE = (RT * 2 + NT * 4) * THREADS * 16 + RT * 2 * PER * THREADS * 4;
  constexpr int D = STAGE * 4 <= 100 * 1024 ? 4 : 3;
  constexpr int RED = WARPS * RT * NT * 32 * 16;
  constexpr int SMEM = STAGE * D > RED ? STAGE * D : RED;
  static_assert(SMEM <= 227 * 1024, "shared memory");
  auto kernel = int4_few_rows_kernel<NT, RT, PER, GLU, D>;
  static uint64_t allowed = 0;
  if (allow_smem("gemm_int4", kernel, SMEM, &allowed)) return 1;
  const int rows = RT * (GLU ? 8 : 16);
  fms_launch(kernel, dim3((p.outputs + rows - 1) / rows), dim3(THREADS), SMEM, stream, p);
  return fms_launch_status("gemm_int4");
}
template <int NT, int RT, bool GLU> int launch_few_per(const Int4Args& p, cudaStream_t stream) {
  if (p.group % 128 == 0 || p.n_groups == 1) return launch_few<NT, RT, 1, GLU>(p, stream);
  return p.group % 64 == 0 ? launch_few<NT, RT, 2, GLU>(p, stream) : launch_few<NT, RT, 4, GLU>(p, stream);
}
template <bool GLU> int few(const Int4Args& p, cudaStream_t stream) {
  // two tiles a block share the rows of x, where that still leaves two blocks a multiprocessor
  const int tiles = (p.outputs + (GLU ? 7 : 15)) / (GLU ? 8 : 16);
  if (p.M <= 8) return tiles >= 592 ? launch_few_per<1, 2, GLU>(p, stream) : launch_few_per<1, 1, GLU>(p, stream);
  return tiles >= 592 ? launch_few_per<2, 2, GLU>(p, stream) : launch_few_per<2, 1, GLU>(p, stream);
}

// ---- more rows ----------------------------------------------------------------------------------------------------------
// The weights fill the instruction's 128 rows, as its A operand in tensor memory, where the threads that unpack them put them: lane =
// row of w, a pair of k a column.  The tokens (16 to 256) are its columns, B, brought by TMA.  So the weights cross shared
// memory once, as 4 bits, and the instruction reads x alone from there.
//   warp 0     per step of 128 k: two 64-k boxes of x and eight 1,024-byte blocks of w, into one of up to 8 stages
//   warp 1     one lane issues 8 instructions (128 x tokens x 16) a step
//   warps 2-9  two groups of four unpack every second step each, a thread a row of w, into the group's half of the operand
//   warps 2-5  then read the accumulator; the ks blocks of a tile (a cluster) add their sums through distributed shared memory
constexpr int ROWS_THREADS = 320, TILE = 128, MAX_STAGES = 8, MAX_KS = 8, A_COLUMNS = 64;

struct RowsArgs {
  Int4Args p;
  int n_tokens, stages, ks, acc_columns, tmem_columns, per;
};

// by a whole warp, which gives up as one
__device__ __forceinline__ bool warp_wait(void* bar, uint32_t parity, volatile int* failed) {
  return __all_sync(0xffffffffu, wait_or_abort(bar, parity, failed));
}
__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t local_addr, uint32_t rank) {
  float4 v;
  asm volatile(
      "{\n.reg .b32 remote;\nmapa.shared::cluster.u32 remote, %4, %5;\nld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [remote];\n}\n"
      : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
      : "r"(local_addr), "r"(rank)
      : "memory");
  return v;
}
__device__ __forceinline__ void tmem_store_pairs(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,"
      "%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};\n" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]),
      "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]),
      "r"(r[31])
      : "memory");
}

__global__ void __launch_bounds__(ROWS_THREADS) int4_rows_kernel(const __grid_constant__ CUtensorMap map_x, RowsArgs a,
                                                                 int* __restrict__ error_flag) {
  extern __shared__ unsigned char smem_unaligned[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(((uintptr_t)smem_unaligned + 1023) & ~(uintptr_t)1023);
  const Int4Args& p = a.p;
  const int x_bytes = a.n_tokens * BLOCK_K * 2, stage_bytes = x_bytes + TILE / BLOCK_ROWS * BLOCK_BYTES, stages = a.stages, ks = a.ks;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + (size_t)stages * stage_bytes);
  uint64_t* empty = full + MAX_STAGES;
  uint64_t* a_full = empty + MAX_STAGES;  // [2]
  uint64_t* a_empty = a_full + 2;         // [2]
  uint64_t* acc_full = a_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_full + 1);
  __shared__ int failed_flag;
  volatile int* failed = &failed_flag;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = ks > 1 ? (int)cluster_rank() : 0;
  const int n0 = blockIdx.y * TILE, m0 = blockIdx.z * a.n_tokens;
  const int per_block = (p.k_blocks + ks - 1) / ks;
  const int step_lo = min(rank * per_block, p.k_blocks), k_steps = min(step_lo + per_block, p.k_blocks) - step_lo;  // may be 0

  if (threadIdx.x == 0) {
    failed_flag = 0;
    for (int s = 0; s < MAX_STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&a_full[i], 4);  // the warps of a group
      mbar_init(&a_empty[i], 1);
    }
    mbar_init(acc_full, 1);
    mbar_fence_init();
  }
  if (warp == 1) tmem_alloc(tmem_slot, a.tmem_columns);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot, tmem_a = tmem + a.acc_columns;
  pdl_launch_dependents();  // now: a block of the next kernel must not take the tensor memory that this one still needs

  if (warp == 0) {
    if (elect_one()) {
      const int row_blocks = min(TILE / BLOCK_ROWS, (p.N + BLOCK_ROWS - 1) / BLOCK_ROWS - n0 / BLOCK_ROWS);
      auto load_w = [&](int i) {
        const int s = i % stages;
        unsigned char* to = smem + (size_t)s * stage_bytes + x_bytes;
        mbar_arrive_expect_tx(&full[s], x_bytes + row_blocks * BLOCK_BYTES);
        for (int b = 0; b < row_blocks; ++b)
          bulk_copy_g2s(to + b * BLOCK_BYTES, p.w + ((size_t)(n0 / BLOCK_ROWS + b) * p.k_blocks + step_lo + i) * BLOCK_BYTES, BLOCK_BYTES, &full[s]);
      };
      auto load_x = [&](int i) {
        const int s = i % stages;
        unsigned char* to = smem + (size_t)s * stage_bytes;
        tma_load_2d(to, &map_x, (step_lo + i) * BLOCK_K, m0, &full[s]);
        tma_load_2d(to + x_bytes / 2, &map_x, (step_lo + i) * BLOCK_K + 64, m0, &full[s]);
      };
      const int early = min(stages, k_steps);
      for (int i = 0; i < early; ++i) load_w(i);  // weights do not depend on the kernel before
      pdl_wait();
      for (int i = 0; i < early; ++i) load_x(i);
      for (int i = early; i < k_steps && !*failed; ++i) {
        if (!wait_or_abort(&empty[i % stages], ((i / stages) & 1) ^ 1, failed)) break;
        load_w(i);
        load_x(i);
      }
    }
  } else if (warp == 1) {
    if (elect_one()) {
      const uint32_t idesc = umma_idesc(TILE, a.n_tokens);
      for (int i = 0; i < k_steps; ++i) {
        const int s = i % stages, half = i & 1;
        if (!wait_or_abort(&full[s], (i / stages) & 1, failed)) break;
        if (!wait_or_abort(&a_full[half], (i >> 1) & 1, failed)) break;
        tc_fence_after();
        const uint32_t b = smem_u32(smem + (size_t)s * stage_bytes);
#pragma unroll
        for (int kk = 0; kk < BLOCK_K / 16; ++kk)
          umma_a_tmem(tmem, tmem_a + half * A_COLUMNS + kk * 8, umma_desc(b + (kk >> 2) * (x_bytes / 2) + (kk & 3) * 32), idesc, i > 0 || kk > 0);
        tc_commit(&empty[s]);
        tc_commit(&a_empty[half]);
      }
      tc_commit(acc_full);
    }
  } else {
    const int group = (warp - 2) >> 2, quarter = warp & 3, row = quarter * 32 + lane;  // a warp reaches the 32 lanes of its number's rest by 4
    const int out_row = min(n0 + row, p.N - 1);
    const uint32_t* words = p.groups + out_row;
    auto group_word = [&](int i, int u) {  // of sub-block u (32 k) of step i
      return words[(size_t)min(((step_lo + i) * BLOCK_K + 32 * u) / p.group, p.n_groups - 1) * p.N];
    };
    uint32_t next[4] = {};
    auto load_words = [&](int i) {
      if (i >= k_steps) return;
      next[0] = group_word(i, 0);
      if (a.per >= 2) next[2] = group_word(i, 2);
      if (a.per == 4) {
        next[1] = group_word(i, 1);
        next[3] = group_word(i, 3);
      }
    };
    load_words(group);
    for (int i = group; i < k_steps; i += 2) {
      const int s = i % stages;
      uint32_t g[4] = {next[0], a.per == 4 ? next[1] : next[0], a.per >= 2 ? next[2] : next[0], 0};
      g[3] = a.per == 4 ? next[3] : g[2];
      load_words(i + 2);
      if (!warp_wait(&full[s], (i / stages) & 1, failed)) break;
      const uint4* at = reinterpret_cast<const uint4*>(smem + (size_t)s * stage_bytes + x_bytes + row * 64);
      uint4 piece[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) piece[c] = at[c ^ ((row >> 1) & 3)];
      if (!warp_wait(&a_empty[group], ((i >> 1) & 1) ^ 1, failed)) break;
      tc_fence_after();
#pragma unroll
      for (int h = 0; h < 2; ++h) {  // 64 k: 32 columns
        uint32_t col[32];
#pragma unroll
        for (int v = 0; v < 2; ++v) {
          const uint32_t gw = g[2 * h + v];
          const __nv_bfloat162 zero = both(gw >> 16), scale = both(gw & 0xffffu);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const uint32_t word = h == 0 ? (v == 0 ? piece[c].x : piece[c].y) : (v == 0 ? piece[c].z : piece[c].w);
            unpack8(word, zero, col + v * 16 + c * 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const __nv_bfloat162 r = __hmul2(*reinterpret_cast<__nv_bfloat162*>(&col[v * 16 + c * 4 + e]), scale);
              col[v * 16 + c * 4 + e] = *reinterpret_cast<const uint32_t*>(&r);
            }
          }
        }
        tmem_store_pairs(tmem_a + group * A_COLUMNS + h * 32 + ((uint32_t)(quarter * 32) << 16), col);
      }
      asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory");
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&a_full[group]);
    }
  }
  // This block's sums as float32 [128][n_tokens + 4] in shared memory, over the stages: every copy into them has landed and
  // every instruction that read them is done once the accumulator is ready.
  float* red = reinterpret_cast<float*>(smem);
  const int red_stride = a.n_tokens + 4;
  if (warp >= 2 && warp < 6) {
    pdl_wait();
    const int quarter = warp & 3, row = quarter * 32 + lane;
    const bool ok = warp_wait(acc_full, 0, failed);
    tc_fence_after();
    for (int c0 = 0; c0 < a.n_tokens; c0 += 16) {
      float v[16];
      if (ok && k_steps > 0) {
        tmem_load_16(tmem + ((uint32_t)(quarter * 32) << 16) + c0, v);
      } else {
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] = 0.f;
      }
#pragma unroll
      for (int j = 0; j < 16; j += 4)
        *reinterpret_cast<float4*>(red + row * red_stride + c0 + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
    }
    tc_fence_before();
  }
  __syncthreads();
  if (ks > 1) cluster_sync_all();
  if (warp >= 2 && !*failed) {  // this block's share of the tokens, four at a time; a thread keeps its row of w
    const int e = threadIdx.x - 64, i = e & 127, share = ((a.n_tokens + ks - 1) / ks + 3) / 4 * 4;
    const int t_hi = min((rank + 1) * share, a.n_tokens), col = n0 + i;
    const uint32_t at0 = smem_u32(red) + (uint32_t)(i * red_stride) * 4u;
    const float bias = p.bias && col < p.N ? __bfloat162float(p.bias[col]) : 0.f;
    for (int t = rank * share + 4 * (e >> 7); t < t_hi; t += 8) {
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
      float4 v[MAX_KS];
#pragma unroll
      for (int r = 0; r < MAX_KS; ++r)
        if (r < ks) v[r] = ks == 1 ? *reinterpret_cast<const float4*>(red + i * red_stride + t) : ld_cluster_f32x4(at0 + 4u * t, (uint32_t)r);
#pragma unroll
      for (int r = 0; r < MAX_KS; ++r)
        if (r < ks) {
          sum[0] += v[r].x; sum[1] += v[r].y; sum[2] += v[r].z; sum[3] += v[r].w;
        }
      if (col >= p.N) continue;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int m = m0 + t + j;
        if (m < p.M && FMS_IN((size_t)m * p.N + col, (size_t)p.M * p.N)) p.y[(size_t)m * p.N + col] = __float2bfloat16_rn(sum[j] + bias);
      }
    }
  }
  if (ks > 1) cluster_sync_all();  // nobody leaves while another block still reads its shared memory
  __syncthreads();
  if (threadIdx.x == 0 && *failed && error_flag) atomicExch(error_flag, 4);
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, a.tmem_columns);
  }
}

int launch_rows(const Int4Args& p, int* error_flag, cudaStream_t stream) {
  constexpr int MOST = 256, EXTRA = 1024 + 512;
  RowsArgs a = {};
  a.p = p;
  a.n_tokens = p.M >= MOST ? MOST : (p.M + 15) / 16 * 16;
  const int tiles = (p.N + TILE - 1) / TILE, chunks = (p.M + a.n_tokens - 1) / a.n_tokens;
  if (tiles > 65535 || chunks > 65535) return fms_fail("gemm_int4: %d by %d tiles", tiles, chunks);
  a.ks = 1;  // blocks that share a tile, as many as leave each 4 steps, up to two a multiprocessor
  while (a.ks < MAX_KS && tiles * chunks * a.ks * 2 <= 320 && p.k_blocks / (a.ks * 2) >= 4) a.ks *= 2;
  const int stage_bytes = a.n_tokens * BLOCK_K * 2 + TILE / BLOCK_ROWS * BLOCK_BYTES;
  const int budget = (a.n_tokens <= 128 && tiles * chunks * a.ks > 148) ? 104 * 1024 : 222 * 1024;
  const size_t red_bytes = (size_t)TILE * (a.n_tokens + 4) * sizeof(float);
  a.stages = min(max(budget / stage_bytes, 2), MAX_STAGES);
  while ((size_t)a.stages * stage_bytes < red_bytes) ++a.stages;
  a.acc_columns = (a.n_tokens + 31) / 32 * 32;
  a.tmem_columns = a.acc_columns + 2 * A_COLUMNS <= 256 ? 256 : 512;
  a.per = (p.group % 128 == 0 || p.n_groups == 1) ? 1 : (p.group % 64 == 0 ? 2 : 4);
  CUtensorMap map_x;
  if (make_map(&map_x, p.x, p.M, p.K, a.n_tokens)) return 1;
  static uint64_t allowed = 0;
  if (allow_smem("gemm_int4", int4_rows_kernel, 225 * 1024, &allowed)) return 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.ks, tiles, chunks);
  cfg.blockDim = dim3(ROWS_THREADS);
  // No more blocks on a multiprocessor than its 512 columns of tensor memory serve: one that waited for columns could be what
  // the holder's cluster waits for.
  const size_t least = a.tmem_columns == 512 ? 200 * 1024 : 78 * 1024, smem = (size_t)a.stages * stage_bytes + EXTRA;
  cfg.dynamicSmemBytes = smem < least ? least : smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = a.ks;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = fms_pdl_enabled() ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, int4_rows_kernel, map_x, a, error_flag);
  if (e != cudaSuccess) return fms_fail("gemm_int4: launch failed: %s", cudaGetErrorString(e));
  return fms_launch_status("gemm_int4");
}

int check(const Int4Args& p) {
  if (p.K <= 0 || p.K % 8) return fms_fail("gemm_int4: %d input channels, a multiple of 8 is wanted", p.K);
  if (p.k_blocks != (p.K + BLOCK_K - 1) / BLOCK_K) return fms_fail("gemm_int4: %d blocks for %d input channels", p.k_blocks, p.K);
  if (p.group <= 0 || p.n_groups != (p.K + p.group - 1) / p.group || (p.n_groups > 1 && p.group % 32))
    return fms_fail("gemm_int4: %d groups of %d for %d input channels", p.n_groups, p.group, p.K);
  if (((uintptr_t)p.x | (uintptr_t)p.w) & 15) return fms_fail("gemm_int4: operands must be 16-byte aligned");
  return 0;
}
constexpr int FEW_ROWS = 16;  // rows of x up to which mma.sync takes the product
}  // namespace

// The most rows of fms_glu_int4.
FMS_API int fms_int4_few_rows() { return FEW_ROWS; }

// y [M, N] bfloat16 of x [M, K] bfloat16, w packed, groups [n_groups, N], bias [N] bfloat16 or null.
FMS_API int fms_linear_int4(const void* x, const void* w, const void* groups, const void* bias, void* y, int M, int N, int K,
                            int k_blocks, int n_groups, int group, int* error_flag, cudaStream_t stream) {
  if (M <= 0 || N <= 0) return 0;
  const Int4Args p = {(const __nv_bfloat16*)x, (const unsigned char*)w, (const uint32_t*)groups, (const __nv_bfloat16*)bias,
                      (__nv_bfloat16*)y, M, N, K, k_blocks, n_groups, group, N, 0};
  if (check(p)) return 1;
  return M <= FEW_ROWS ? few<false>(p, stream) : launch_rows(p, error_flag, stream);
}

// y [M, hidden] = act(gate) * up for w = [gate; up] of 2 hidden rows, up to FEW_ROWS rows of x.
FMS_API int fms_glu_int4(const void* x, const void* w, const void* groups, const void* bias, void* y, int M, int hidden, int K,
                         int k_blocks, int n_groups, int group, int act, cudaStream_t stream) {
  if (M <= 0 || hidden <= 0) return 0;
  if (M > FEW_ROWS || act < 0 || act > 3) return fms_fail("glu_int4: %d rows of x, activation %d", M, act);
  const Int4Args p = {(const __nv_bfloat16*)x, (const unsigned char*)w, (const uint32_t*)groups, (const __nv_bfloat16*)bias,
                      (__nv_bfloat16*)y, M, 2 * hidden, K, k_blocks, n_groups, group, hidden, act};
  if (check(p)) return 1;
  return few<true>(p, stream);
}
