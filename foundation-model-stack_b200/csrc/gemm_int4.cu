// y[m, n] = sum_k x[m, k] * (q[n, k] - z[n, g(k)]) * s[n, g(k)] (+ bias[n]): bfloat16 rows, weights of 4 bits with one bfloat16
// scale and one whole zero point a group of consecutive k.  GLU: act(gate) * up for weights [gate; up].
//
// Layout, made once (kernels/quantized.py, pack_int4): one stream of blocks of 16 rows x 128 k, [rows / 16][k / 128], each
//   1,024 bytes of weights: [16 rows][4 pieces of 16 bytes]; word w of a row's piece c holds k = 32 w + 8 c .. + 7, value 2 i in
//     bits 4 i and value 2 i + 1 in bits 16 + 4 i, so that one shift and one logical operation leave a pair of neighbours in
//     the halves of a register; piece c lies at place c ^ (row / 2 % 4), which lets the rows of a warp read a piece from shared
//     memory without meeting in a bank;
//   PER times 64 bytes (PER 1, 2 or 4, by whether groups are whole blocks, halves or quarters of them): a word a row, the scale in
//     its low half and 128 + z, exact in bfloat16, in its high half.
// So all that a tile needs of a block comes in one copy of neighbouring bytes, and groups cost no index arithmetic.
//
// 0x4300 | q is the bfloat16 128 + q; minus 128 + z it is q - z, exact.
//   few rows: mma.sync over q - z, whole numbers, a group's float32 sum times its scale: nothing is rounded but the result.
//   more rows: tcgen05 over (q - z) * s rounded to bfloat16 on its way into the operand, as a bfloat16 weight would be: the
//             tensor cores' sums run over all of k and cannot be scaled group by group.  What that costs, in the root mean square
//             against 64 bits: 0.0021 to 0.0022 of y, where the result's own rounding to bfloat16 leaves 0.0017.
#include <cuda.h>

#include "common.cuh"

namespace {
#include "tcgen05.cuh"
#include "umma_issue.cuh"
#include "quantized.cuh"

constexpr int BLOCK_ROWS = 16, BLOCK_K = 128, WEIGHT_BYTES = 1024;

// the 8 values of a word as four pairs of bfloat16 q - z
__device__ __forceinline__ void unpack8(uint32_t word, __nv_bfloat162 zero, uint32_t* pairs) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t v;  // (word >> 4 i) & 0x000f000f | 0x43004300 as one logical operation
    asm("lop3.b32 %0, %1, %2, %3, 0xea;\n" : "=r"(v) : "r"(word >> (4 * i)), "r"(0x000f000fu), "r"(0x43004300u));
    const __nv_bfloat162 d = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&v), zero);
    pairs[i] = *reinterpret_cast<const uint32_t*>(&d);
  }
}
// a group's word: 128 + z and the scale, each in both halves of a register
__device__ __forceinline__ __nv_bfloat162 zero_of(uint32_t word) {
  const uint32_t v = __byte_perm(word, word, 0x3232);
  return *reinterpret_cast<const __nv_bfloat162*>(&v);
}
__device__ __forceinline__ __nv_bfloat162 scale_of(uint32_t word) {
  const uint32_t v = __byte_perm(word, word, 0x1010);
  return *reinterpret_cast<const __nv_bfloat162*>(&v);
}

struct Int4Args {
  const __nv_bfloat16* x;     // [M, K]
  const unsigned char* w;     // the packed blocks
  Bias bias;
  __nv_bfloat16* y;           // [M, outputs]
  int M, N, K, k_blocks, per, outputs, act;
  __host__ __device__ int block_bytes() const { return WEIGHT_BYTES + 64 * per; }
  __host__ __device__ int row_blocks() const { return (N + BLOCK_ROWS - 1) / BLOCK_ROWS; }
};

// ---- up to 8 rows -------------------------------------------------------------------------------------------------------
// Bound by reading the weights once, and by the instructions that unpack them.  A thread block, one or two a multiprocessor,
// takes an equal run of tiles, 16 rows of w each (GLU: of gate rows and the up rows that belong to them), as many at a time as it
// has warps; each warp takes an equal run of their 128-k blocks, whatever tiles these belong to, two at most, and leaves a sum of
// each in shared memory; after the one barrier those of a tile are added in the order of k.  A lane loads its pieces of two rows
// of a block straight into registers, AHEAD blocks ahead, as many as 64 registers hold (28,672 x 4,096 by one row with groups of
// 128, 1 / 2 / 3 ahead 14.6 / 14.2 / 16.6 us; of 64 17.0 / 17.1 / 19.7; of 32 18.0 / 20.0 / 24.7); x comes from the first-level cache.
// 28,672 x 4,096 by one row 14.2 us, by eight 15.7, gated 16.1 (tiles shared by the warps of a block one after the other, with a
// barrier each: 17.0, gated 23.5; rings in shared memory fed by bulk copies 22.7; without unpacking 12.6, without that and
// the loads of x 11.2; with half the shifts as wide products 18.0; 16 warps 4 blocks ahead 17.6).
constexpr int FEW_ROWS = 8, FEW_WARPS = 32;

__device__ __forceinline__ void mma_bf16_first(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void mma_bf16(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint4 load_once(const uint4* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ uint32_t load_once(const uint32_t* p) {
  uint32_t v;
  asm volatile("ld.global.nc.L1::no_allocate.u32 %0, [%1];\n" : "=r"(v) : "l"(p));
  return v;
}

template <int PER, bool GLU>
__global__ void __launch_bounds__(32 * FEW_WARPS, 1) int4_few_rows_kernel(Int4Args p, int log_warps, int at_once, int each, int more) {
  constexpr int BYTES = WEIGHT_BYTES + 64 * PER, AHEAD = PER == 1 ? 2 : 1;
  extern __shared__ float4 sums[][2][32];  // of a warp's first and second tile: lane l has rows l / 4 and + 8 by tokens 2 (l % 4) and + 1
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
  const int warps = 1 << log_warps, t_lo = blockIdx.x * each + min((int)blockIdx.x, more), t_hi = t_lo + each + ((int)blockIdx.x < more);
  const int rounds = (t_hi - t_lo + at_once - 1) / at_once, per_round = rounds == 1 ? t_hi - t_lo : (t_hi - t_lo + rounds - 1) / rounds;
  // the lane's pieces of a block (those of rows g and g + 8 lie 512 bytes apart)
  const int piece = g * 64 + (c ^ ((g >> 1) & 3)) * 16, word = WEIGHT_BYTES + g * 4 - piece;
  const size_t to_up = (size_t)(p.outputs / BLOCK_ROWS) * p.k_blocks * BYTES;  // GLU: from a gate block to its up block
  // a lane without a row of x of its own reads the first: its sums are not stored
  const __nv_bfloat16* xp = p.x + (size_t)(g < p.M ? g : 0) * p.K + 8 * c;

  for (int from = t_lo; from < t_hi; from += per_round) {
    const int count = min(per_round, t_hi - from);
    const int gates = count * p.k_blocks, units = GLU ? 2 * gates : gates;  // GLU: all gate blocks, then all up blocks
    // warp w has units [run(w), run(w + 1)), fewer units than warps one each
    auto run = [&](int w) { return units < warps ? min(w, units) : (int)((unsigned)(units * w) >> log_warps); };
    auto warp_of = [&](int unit) { return units < warps ? unit : (int)((((unsigned)(unit + 1) << log_warps) - 1) / (unsigned)units); };
    const int u = run(warp);
    int todo = run(warp + 1) - u;
    const unsigned char* next = p.w + ((size_t)from * p.k_blocks + u) * BYTES + piece;
    if (GLU && u >= gates) next += to_up - (size_t)gates * BYTES;
    int turn = GLU ? gates - u : 0;  // loads until the first of an up block
    uint4 w[AHEAD][2];
    uint32_t gw[AHEAD][2 * PER];
    auto load = [&](int at) {
      if (!FMS_IN(next - piece - p.w + BYTES - 1, (size_t)p.row_blocks() * p.k_blocks * BYTES)) return;
      w[at][0] = load_once(reinterpret_cast<const uint4*>(next));
      w[at][1] = load_once(reinterpret_cast<const uint4*>(next + 512));
#pragma unroll
      for (int i = 0; i < 2 * PER; ++i) gw[at][i] = load_once(reinterpret_cast<const uint32_t*>(next + word + i * 32));
      next += BYTES;
      if (GLU && --turn == 0) next += to_up - (size_t)gates * BYTES;
    };
#pragma unroll
    for (int q = 0; q < AHEAD; ++q)
      if (q < todo) load(q);  // weights: before the wait for the kernel that makes x
    if (from == t_lo) pdl_wait();

    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    int slot = 0, left = p.K - u % p.k_blocks * BLOCK_K;  // values of the tile from this block on
    const uint4* xs = reinterpret_cast<const uint4*>(xp + (p.K - left));
    auto multiply = [&](const uint4* wq, const uint32_t* gq) {
      uint4 b[4];
      auto of_x = [&](int v) { return FMS_IN(xs + 4 * v - reinterpret_cast<const uint4*>(p.x), (size_t)p.M * p.K / 8) ? xs[4 * v] : make_uint4(0, 0, 0, 0); };
      if (left >= BLOCK_K) {
#pragma unroll
        for (int v = 0; v < 4; ++v) b[v] = of_x(v);
      } else {  // K is a multiple of 8: a lane's 8 values are all inside or all outside
#pragma unroll
        for (int v = 0; v < 4; ++v) b[v] = left > 32 * v + 8 * c ? of_x(v) : make_uint4(0, 0, 0, 0);
      }
      const uint32_t wl[4] = {wq[0].x, wq[0].y, wq[0].z, wq[0].w}, wh[4] = {wq[1].x, wq[1].y, wq[1].z, wq[1].w};
#pragma unroll
      for (int h = 0; h < PER; ++h) {
        const uint32_t gl = gq[2 * h], gh = gq[2 * h + 1];
        const __nv_bfloat162 zl = zero_of(gl), zh = zero_of(gh);
        float part[4];
#pragma unroll
        for (int v = h * (4 / PER); v < (h + 1) * (4 / PER); ++v) {
          uint32_t a[4], d[4];
          unpack8(wl[v], zl, a);
          unpack8(wh[v], zh, d);
          if (v == h * (4 / PER)) mma_bf16_first(part, a[0], d[0], a[1], d[1], b[v].x, b[v].y);
          else mma_bf16(part, a[0], d[0], a[1], d[1], b[v].x, b[v].y);
          mma_bf16(part, a[2], d[2], a[3], d[3], b[v].z, b[v].w);
        }
        const float sl = __uint_as_float(gl << 16), sh = __uint_as_float(gh << 16);
        acc[0] = fmaf(part[0], sl, acc[0]);
        acc[1] = fmaf(part[1], sl, acc[1]);
        acc[2] = fmaf(part[2], sh, acc[2]);
        acc[3] = fmaf(part[3], sh, acc[3]);
      }
    };
    while (todo > 0) {
#pragma unroll
      for (int q = 0; q < AHEAD; ++q)
        if (todo > 0) {  // of the whole warp
          multiply(w[q], gw[q]);
          if (todo > AHEAD) load(q);
          --todo;
          left -= BLOCK_K;
          xs += BLOCK_K / 8;
          if (left <= 0 || todo == 0) {  // the tile's last block, or this warp's
            if (FMS_IN(slot, 2)) sums[warp][slot][lane] = make_float4(acc[0], acc[1], acc[2], acc[3]);
            ++slot;
            acc[0] = acc[1] = acc[2] = acc[3] = 0.f;
            left = p.K;
            xs = reinterpret_cast<const uint4*>(xp);
          }
        }
    }
    __syncthreads();
    // thread: a row of x and a column of this round's
    const int log_m = p.M > 4 ? 3 : (p.M > 2 ? 2 : p.M - 1), m = threadIdx.x & ((1 << log_m) - 1);
    for (int local = threadIdx.x >> log_m; local < count * BLOCK_ROWS; local += 32 * warps >> log_m) {
      const int tile = local >> 4, row = local & 15, col = from * BLOCK_ROWS + local;
      if (m >= p.M || col >= p.outputs) continue;
      const int at = ((row & 7) * 4 + (m >> 1)) * 4 + (row >> 3) * 2 + (m & 1);  // of 128
      auto total = [&](int t) {
        const int first = t * p.k_blocks, w_lo = warp_of(first), w_hi = warp_of(first + p.k_blocks - 1);
        if (!FMS_IN(w_lo, warps) || !FMS_IN(w_hi, warps)) return 0.f;
        // only the first warp of a tile can have begun with an earlier one
        float sum = reinterpret_cast<const float*>(sums[w_lo][run(w_lo) < first ? 1 : 0])[at];
#pragma unroll 4
        for (int i = w_lo + 1; i <= w_hi; ++i) sum += reinterpret_cast<const float*>(sums[i][0])[at];
        return sum;
      };
      float v = total(tile);
      if (p.bias) v += p.bias[col];
      if (GLU) {
        float up = total(count + tile);
        if (p.bias) up += p.bias[p.outputs + col];
        v = activate(v, p.act) * up;
      }
      if (FMS_IN((size_t)m * p.outputs + col, (size_t)p.M * p.outputs)) p.y[(size_t)m * p.outputs + col] = __float2bfloat16_rn(v);
    }
    if (rounds > 1) __syncthreads();
  }
}

template <int PER, bool GLU> int launch_few(const Int4Args& p, int warps, int tiles, int grid, cudaStream_t stream) {
  const int smem = 2 * warps * 32 * (int)sizeof(float4);  // 32 KB at most
  fms_launch(int4_few_rows_kernel<PER, GLU>, dim3(grid), dim3(32 * warps), smem, stream, p, warps == 32 ? 5 : 4, GLU ? warps / 2 : warps, tiles / grid, tiles % grid);
  return fms_launch_status("gemm_int4");
}
template <bool GLU> int few(const Int4Args& p, cudaStream_t stream) {
  // 32 warps a multiprocessor, as one thread block or two: by how many blocks of w a warp gets at most (16 : 32 warps in us:
  // 28,672 x 4,096 14.5 : 14.2, 6,144 x 4,096 5.8 : 5.4, 512 x 16,384 7.8 : 6.0, 4,096 x 14,336 9.1 : 9.3, 4,096 x 4,096 4.1 : 4.5)
  const int sms = multiprocessors(), tiles = (p.outputs + BLOCK_ROWS - 1) / BLOCK_ROWS;
  auto most = [&](int warps) {
    const int slots = sms * (FEW_WARPS / warps);
    return ((long)((tiles + slots - 1) / slots) * (GLU ? 2 : 1) * p.k_blocks + warps - 1) / warps;
  };
  const int warps = most(16) <= most(32) ? 16 : 32, slots = sms * (FEW_WARPS / warps), grid = tiles < slots ? tiles : slots;
  // blocks of w that a thread block has in hand at once, times its warps, are counted in 32 bits
  if (p.k_blocks > 0x3fffffff / (FEW_WARPS * FEW_WARPS)) return fms_fail("gemm_int4: %d blocks of k", p.k_blocks);
  return p.per == 1 ? launch_few<1, GLU>(p, warps, tiles, grid, stream)
                    : (p.per == 2 ? launch_few<2, GLU>(p, warps, tiles, grid, stream) : launch_few<4, GLU>(p, warps, tiles, grid, stream));
}

// ---- what the tcgen05 kernels share --------------------------------------------------------------------------------------
// The weights fill the instruction's rows, as its A operand in tensor memory, where the threads that unpack them put them: lane =
// row of w, a pair of k a column.  The tokens are its columns, B, brought by TMA.  So the weights cross shared memory once, as 4
// bits, and the instruction reads x alone from there; a thread's row of w is a column of y, and a warp stores 64 neighbouring bytes.
constexpr int TILE = 128, A_COLUMNS = 64;  // columns of the operand for 128 k

// The packed blocks [row_blocks][k_blocks][bytes], in boxes of the eight row blocks of a tile by one k block: one copy a step (eight
// untiled ones of a block each took 900 cycles)
int make_block_map(CUtensorMap* map, const Int4Args& p) {
  EncodeTiled enc = encode_tiled();
  if (enc == nullptr) return fms_fail("gemm_int4: the driver does not export cuTensorMapEncodeTiled");
  const cuuint64_t bytes = p.block_bytes();
  const cuuint64_t dims[3] = {bytes / 8, (cuuint64_t)p.k_blocks, (cuuint64_t)p.row_blocks()}, strides[2] = {bytes, bytes * p.k_blocks};
  const cuuint32_t box[3] = {(cuuint32_t)bytes / 8, 1, TILE / BLOCK_ROWS}, elem[3] = {1, 1, 1};
  const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT64, 3, const_cast<unsigned char*>(p.w), dims, strides, box, elem,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fms_fail("gemm_int4: cuTensorMapEncodeTiled failed with %d (%d rows, %d k)", (int)r, p.N, p.K);
  return 0;
}
__device__ __forceinline__ void tma_load_3d(void* smem_dst, const CUtensorMap* map, int c0, int c1, int c2, void* bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];\n" ::"r"(
                   smem_u32(smem_dst)),
               "l"(map), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
               : "memory");
}
// by a whole warp, which gives up as one
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* failed) {
  return __all_sync(0xffffffffu, quick_wait(bar, parity, failed));
}
// 32 columns of 32 bits of this thread's lane of tensor memory, written; not waited for
__device__ __forceinline__ void tmem_store_pairs(uint32_t taddr, const uint32_t* r) {
  __syncwarp();
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,"
      "%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};\n" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]),
      "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]),
      "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_stores() {
  __syncwarp();
  asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory");
}
// 64 k of a row as 32 columns: words 2 h and 2 h + 1 of its four pieces, with the groups' words of either
__device__ __forceinline__ void unpack64(const uint2* words, uint32_t group0, uint32_t group1, uint32_t* col) {
#pragma unroll
  for (int v = 0; v < 2; ++v) {
    const uint32_t gw = v ? group1 : group0;
    const __nv_bfloat162 zero = zero_of(gw), scale = scale_of(gw);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      uint32_t* to = col + v * 16 + c * 4;
      unpack8(v ? words[c].y : words[c].x, zero, to);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const __nv_bfloat162 r = __hmul2(*reinterpret_cast<__nv_bfloat162*>(&to[e]), scale);
        to[e] = *reinterpret_cast<const uint32_t*>(&r);
      }
    }
  }
}
// the group's word of sub-block u (32 k) of a row
__device__ __forceinline__ uint32_t group_word(const unsigned char* block, int row16, int u, int per) {
  return reinterpret_cast<const uint32_t*>(block + WEIGHT_BYTES)[(u * per >> 2) * 16 + row16];
}
// A warp's 32 rows of a tile's blocks, 128 k, into 64 columns of tensor memory, of which a warp reaches the 32 lanes of its number's
// rest by 4; done, and in order before what the first lane says next, when it returns.
__device__ __forceinline__ void unpack_row(const unsigned char* blocks, int bytes, int per, int quarter, int lane, uint32_t tmem_a) {
  tc_fence_after();
  const int row = quarter * 32 + lane;
  const uint32_t to = tmem_a + ((uint32_t)(quarter * 32) << 16);
  const unsigned char* block = blocks + (row >> 4) * bytes;
  const uint4* at = reinterpret_cast<const uint4*>(block + (row & 15) * 64);
  uint4 piece[4];
  uint32_t g[4], col[32];
  uint2 words[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    piece[c] = at[c ^ ((row >> 1) & 3)];
    g[c] = group_word(block, row & 15, c, per);
  }
#pragma unroll
  for (int c = 0; c < 4; ++c) words[c] = make_uint2(piece[c].x, piece[c].y);
  unpack64(words, g[0], g[1], col);
  tmem_store_pairs(to, col);
#pragma unroll
  for (int c = 0; c < 4; ++c) words[c] = make_uint2(piece[c].z, piece[c].w);
  unpack64(words, g[2], g[3], col);
  tmem_store_pairs(to + 32, col);
  tmem_wait_stores();
  tc_fence_before();
  __syncwarp();
}
// values of neighbouring rows of y, one column
template <int N> __device__ __forceinline__ void store_column(const Int4Args& p, const float* v, int row0, int col, float bias) {
  const size_t pitch = p.N, at = (size_t)row0 * pitch + col;
#pragma unroll
  for (int j = 0; j < N; ++j)
    if (row0 + j < p.M && FMS_IN(at + j * pitch, (size_t)p.M * pitch)) p.y[at + j * pitch] = __float2bfloat16_rn(v[j] + bias);
}

// ---- 9 to 112 or 256 rows ------------------------------------------------------------------------------------------------------
// One thread block a multiprocessor; each takes an equal run of the steps of all tiles, a step being 128 rows of w by 128 k, so that
// no multiprocessor waits for another's second tile (28,672 rows are 224 tiles for 148).  Where a tile's steps fall to several
// blocks, each leaves its sums in a slot of its own in scratch memory, and a second kernel adds them in the order of k.  The
// cut depends on the weights' shape alone, so among batches of up to 64 rows, and among larger ones, a row's result does not depend on
// the rest of the batch.
//   warp 0      per step one copy, the eight blocks of w, into one of up to 8 stages; warp 22 two 64-k boxes of x beside them
//   warp 1      one lane issues 8 instructions (128 x tokens x 16) a step.  What a step costs is the instructions of these single
//               threads more than the tensor cores (some 700 cycles against 260 at 64 tokens), so up to 64 tokens warp 23 takes every
//               second step, into accumulators of its own that the epilogue adds, and a step's copies are waited for by those who unpack
//               it alone: an issuer sees them by way of the operand's barrier.  (One issuer, one thread for all copies: 4,096 x 14,336
//               by 16 rows 13.6 us, by 64 16.8, 28,672 x 4,096 22.7 and 26.5; so 11.9, 15.8, 19.8, 24.4.  Two issuers for
//               128 tokens leave room for 4 stages of the operand and 4 of copies: 100 rows 18.7 -> 21.9 us.)
//   warps 2-17  up to four groups of four unpack every fourth step each, a thread a row of w, into the next of up to 7 stages of the
//               operand, 64 columns each
//   warps 18-21 the epilogue; two accumulators (of each issuer) up to 64 tokens, so that it runs under the next tile's steps
// No wait may meet a barrier that is a phase behind.  One issuer: steps are used up in order, a group waits for its stage of the operand
// before it waits for a step's copies, and there are no fewer copies' stages than operand's stages and no fewer of these than groups.
// Two: their numbers are multiples of the groups', so that the group of a step has itself waited for the last use of either stage,
// and of the issuers', so that a stage of the operand is always the same issuer's.
// Every wait on an mbarrier is bounded: on a time-out the block records error 4, skips the rest of its work and still frees its
// tensor memory.
constexpr int GROUPS = 4, UNPACK_WARPS = 4 * GROUPS, X_WARP = 6 + UNPACK_WARPS, SECOND_ISSUER = 7 + UNPACK_WARPS,
              ROWS_THREADS = 32 * (UNPACK_WARPS + 8), MAX_STAGES = 8, A_FIRST = 256, MAX_A = 7;

struct RowsArgs {
  Int4Args p;
  int n_tokens, stages, groups, a_stages, issuers, accs, acc_columns;
  float* scratch;  // [2 blocks][n_tokens][128]: a block's first tile, then its last, where it has not all of it
  long scratch_floats;  // for the bounds-checked build
};
__global__ void __launch_bounds__(ROWS_THREADS, 1) int4_rows_kernel(const __grid_constant__ CUtensorMap map_x,
                                                                    const __grid_constant__ CUtensorMap map_w, RowsArgs a,
                                                                    int* __restrict__ error_flag) {
  extern __shared__ unsigned char smem_unaligned[];
  unsigned char* smem = smem_unaligned + (-smem_u32(smem_unaligned) & 1023);
  const Int4Args& p = a.p;
  const int bytes = p.block_bytes(), x_bytes = a.n_tokens * BLOCK_K * 2, stages = a.stages;
  const int stage_bytes = (x_bytes + TILE / BLOCK_ROWS * bytes + 1023) / 1024 * 1024;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + stages * stage_bytes);
  uint64_t* empty = full + MAX_STAGES;
  uint64_t* a_full = empty + MAX_STAGES;  // [MAX_A]
  uint64_t* a_empty = a_full + MAX_A;     // [MAX_A]
  uint64_t* acc_full = a_empty + MAX_A;   // [2]
  uint64_t* acc_empty = acc_full + 2;     // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  __shared__ int failed_flag;
  volatile int* failed = &failed_flag;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int all = (p.N + TILE - 1) / TILE * p.k_blocks;
  const int lo = first_step(blockIdx.x, gridDim.x, all), hi = first_step(blockIdx.x + 1, gridDim.x, all);

  if (threadIdx.x == 0) {
    failed_flag = 0;
    for (int s = 0; s < MAX_STAGES; ++s) {
      mbar_init(&full[s], 2);
      mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < MAX_A; ++i) {
      mbar_init(&a_full[i], 4);  // the warps of a group
      mbar_init(&a_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], a.issuers);
      mbar_init(&acc_empty[i], 4);  // the warps of the epilogue
    }
    mbar_fence_init();
  }
  if (warp == 1) tmem_alloc(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot, tmem_a = tmem + a.accs * a.issuers * a.acc_columns;
  pdl_launch_dependents();  // a block of the next kernel must not take the tensor memory that this one still needs

  if (warp == 0) {
    if (elect_one()) {  // the weights, which do not depend on the kernel before
      int tile = lo / p.k_blocks, k = lo - tile * p.k_blocks, s = 0;
      const int w_bytes = TILE / BLOCK_ROWS * bytes;
      uint32_t phase = 1;
      for (int i = lo; i < hi; ++i) {
        if (!quick_wait(&empty[s], phase, failed)) break;
        mbar_arrive_expect_tx(&full[s], w_bytes);
        tma_load_3d(smem + s * stage_bytes + x_bytes, &map_w, 0, k, tile * (TILE / BLOCK_ROWS), &full[s]);
        if (++k == p.k_blocks) k = 0, ++tile;
        if (++s == stages) s = 0, phase ^= 1;
      }
    }
  } else if (warp == X_WARP) {
    if (elect_one()) {
      pdl_wait();
      int k = lo % p.k_blocks, s = 0;
      uint32_t phase = 1;
      for (int i = lo; i < hi; ++i) {
        if (!quick_wait(&empty[s], phase, failed)) break;
        mbar_arrive_expect_tx(&full[s], x_bytes);
        tma_load_2d(smem + s * stage_bytes, &map_x, k * BLOCK_K, 0, &full[s]);
        tma_load_2d(smem + s * stage_bytes + x_bytes / 2, &map_x, k * BLOCK_K + 64, 0, &full[s]);
        if (++k == p.k_blocks) k = 0;
        if (++s == stages) s = 0, phase ^= 1;
      }
    }
  } else if (warp == 1 || warp == SECOND_ISSUER) {
    const int mine = warp == 1 ? 0 : 1;
    if (mine < a.issuers && elect_one()) {
      const uint32_t idesc = umma_idesc(TILE, a.n_tokens), box = (uint32_t)x_bytes / 2 >> 4;
      const MatrixDesc base(smem_u32(smem));
      int i = lo + mine, s = mine, stage = mine, acc = 0, from = lo;
      uint32_t turn = 0, acc_phase = 1;
      bool ok = true;
      while (from < hi) {
        const int to = min(from - from % p.k_blocks + p.k_blocks, hi);
        const uint32_t d = tmem + (acc * a.issuers + mine) * a.acc_columns;
        if (!quick_wait(&acc_empty[acc], acc_phase, failed)) break;
        for (uint32_t more = 0; i < to; i += a.issuers, more = 1) {
          // the group has seen the step's copies land, x among them
          if (!(ok = quick_wait(&a_full[stage], turn, failed))) break;
          tc_fence_after();
          const uint32_t ta = tmem_a + stage * A_COLUMNS, b = base.lo + (uint32_t)(s * stage_bytes >> 4);
#pragma unroll
          for (int kk = 0; kk < BLOCK_K / 16; ++kk)  // 64 k a box of x, 32 bytes of its rows an instruction
            issue_a_tmem(d, ta + kk * 8, b + (kk & 3) * 2 + (kk < 4 ? 0 : box), base.hi, idesc, kk > 0 ? 1u : more);
          tc_commit(&empty[s]);
          tc_commit(&a_empty[stage]);
          s += a.issuers;
          if (s >= stages) s -= stages;
          stage += a.issuers;
          if (stage >= a.a_stages) stage -= a.a_stages, turn ^= 1;
        }
        if (!ok) break;
        tc_commit(&acc_full[acc]);
        if (++acc == a.accs) acc = 0, acc_phase ^= 1;
        from = to;
      }
    }
  } else if (warp < 2 + UNPACK_WARPS) {
    const int group = (warp - 2) >> 2;
    int s = group, stage = group;  // groups <= a_stages <= stages
    uint32_t phase = 0, turn = 1;
    for (int i = group < a.groups ? lo + group : hi; i < hi; i += a.groups) {
      if (!warp_wait(&a_empty[stage], turn, failed)) break;
      if (!warp_wait(&full[s], phase, failed)) break;
      unpack_row(smem + s * stage_bytes + x_bytes, bytes, p.per, warp & 3, lane, tmem_a + stage * A_COLUMNS);
      if (lane == 0) mbar_arrive(&a_full[stage]);
      s += a.groups;
      if (s >= stages) s -= stages, phase ^= 1;
      stage += a.groups;
      if (stage >= a.a_stages) stage -= a.a_stages, turn ^= 1;
    }
  } else {
    pdl_wait();  // y and the scratch memory may be what the kernel before still uses
    const int quarter = warp & 3, row = quarter * 32 + lane;
    int acc = 0;
    uint32_t acc_phase = 0;
    for (int i = lo; i < hi;) {
      const int tile = i / p.k_blocks, k_lo = i - tile * p.k_blocks, k_hi = min(p.k_blocks, hi - tile * p.k_blocks);
      const int col = tile * TILE + row;
      const bool whole = k_lo == 0 && k_hi == p.k_blocks;
      float* slot = a.scratch + ((size_t)(2 * blockIdx.x + (i == lo ? 0 : 1)) * a.n_tokens) * TILE + row;
      const float bias = whole && p.bias && col < p.N ? p.bias[col] : 0.f;
      if (!warp_wait(&acc_full[acc], acc_phase, failed)) break;
      tc_fence_after();
      for (int c0 = 0; c0 < a.n_tokens; c0 += 16) {
        float v[16];
        const uint32_t at = tmem + acc * a.issuers * a.acc_columns + ((uint32_t)(quarter * 32) << 16) + c0;
        if (k_hi - k_lo == 1) {  // one accumulator alone has sums
          tmem_load_16(at + (a.issuers == 2 && ((i - lo) & 1) ? a.acc_columns : 0), v);
        } else {
          tmem_load_16(at, v);
          if (a.issuers == 2) {
            float second[16];
            tmem_load_16(at + a.acc_columns, second);
#pragma unroll
            for (int j = 0; j < 16; ++j) v[j] += second[j];
          }
        }
        if (whole) {
          if (col < p.N) store_column<16>(p, v, c0, col, bias);
        } else {
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (FMS_IN(slot + (c0 + j) * TILE - a.scratch, max(a.scratch_floats, 1L))) slot[(size_t)(c0 + j) * TILE] = v[j];
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_empty[acc]);
      if (++acc == a.accs) acc = 0, acc_phase ^= 1;
      i += k_hi - k_lo;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && *failed && error_flag) atomicExch(error_flag, 4);
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// y of the tiles that several blocks share: their sums in the order of k, + bias.  Block: a tile's 128 columns of y by 4 tokens; the
// slots of four blocks are on their way at a time (one after another they took 9 us of 23).
__global__ void __launch_bounds__(TILE) int4_join_kernel(RowsArgs a, int blocks) {
  pdl_launch_dependents();
  const Int4Args& p = a.p;
  const int all = (p.N + TILE - 1) / TILE * p.k_blocks, tile = blockIdx.x, start = tile * p.k_blocks;
  const int from = block_of_step(start, blocks, all), to = block_of_step(start + p.k_blocks - 1, blocks, all);
  const int col = tile * TILE + (int)threadIdx.x, t0 = blockIdx.y * 4;
  if (from == to || col >= p.N || t0 >= p.M) return;  // some block of some tile goes on, and waits
  // only the first block of a tile can have begun with an earlier one
  const int head = first_step(from, blocks, all) / p.k_blocks == tile ? 0 : 1;
  const float* slots = a.scratch + (size_t)t0 * TILE + threadIdx.x;
  const size_t pitch = (size_t)a.n_tokens * TILE;
  pdl_wait();
  const float bias = p.bias ? p.bias[col] : 0.f;  // any tensor: the kernel before the product may have written it
  auto sum_of = [&](const float* at) { return FMS_IN(at - a.scratch, max(a.scratch_floats, 1L)) ? __ldcg(at) : 0.f; };
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
  for (int b = from; b <= to; b += 4) {
    float v[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) v[i][j] = b + i <= to ? sum_of(slots + (2 * (b + i) + (b + i == from ? head : 0)) * pitch + j * TILE) : 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) sum[j] += v[i][j];
  }
  store_column<4>(p, sum, t0, col, bias);
}

// A block that holds all of the tensor memory takes so much shared memory that no block that wants some fits beside it: one that
// waits for it could be what this one waits for (the others of a cluster, the kernel before).
constexpr size_t SMEM_LEAST = 200 * 1024, SMEM_MOST = 225 * 1024, EXTRA = 1024 /* alignment */ + 512 /* barriers */;

// The most rows of x that this kernel takes: 256, but 112 where the pairs of the kernel below have a tile each.  This one / that one in
// us, by rows: 28,672 x 4,096 96 31.9 / 32.3, 112 34.5 / 34.3, 128 39.0 / 34.4, 256 70.6 / 57.2; 6,144 x 4,096 128 14.1 / 18.6, 256 21.0 / 19.0;
// 4,096 x 14,336 128 20.7 / 44.9, 256 31.1 / 45.6.
int rows_most(int N) { return (long)N >= 2L * TILE * (multiprocessors() / 2) ? 112 : 256; }
int rows_blocks(int N, int K) {
  const long steps = (long)((N + TILE - 1) / TILE) * ((K + BLOCK_K - 1) / BLOCK_K);
  const int sms = multiprocessors();
  return steps < sms ? (int)steps : sms;
}
long rows_scratch(int M, int N, int K) { return 2L * rows_blocks(N, K) * ((M + 15) / 16 * 16) * TILE; }

int launch_rows(const Int4Args& p, float* scratch, long scratch_floats, int* error_flag, cudaStream_t stream) {
  RowsArgs a = {};
  a.p = p;
  a.n_tokens = (p.M + 15) / 16 * 16;
  a.scratch = scratch;
  a.scratch_floats = scratch_floats;
  const int tiles = (p.N + TILE - 1) / TILE, blocks = rows_blocks(p.N, p.K);
  if ((long)tiles * p.k_blocks > 0x3fffffffL) return fms_fail("gemm_int4: %d tiles of %d blocks", tiles, p.k_blocks);
  if (scratch_floats < rows_scratch(p.M, p.N, p.K)) return fms_fail("gemm_int4: %ld floats of scratch memory, %ld are wanted", scratch_floats, rows_scratch(p.M, p.N, p.K));
  const int stage_bytes = (a.n_tokens * BLOCK_K * 2 + TILE / BLOCK_ROWS * p.block_bytes() + 1023) / 1024 * 1024;
  a.stages = min((int)((SMEM_MOST - EXTRA) / stage_bytes), MAX_STAGES);
  a.acc_columns = (a.n_tokens + 31) / 32 * 32;
  a.accs = a.n_tokens <= 64 ? 2 : 1;
  a.issuers = a.n_tokens <= 64 ? 2 : 1;
  if (a.issuers == 2) {  // 8 stages of copies, or 4
    a.a_stages = a.groups = GROUPS;
    a.stages = a.stages / GROUPS * GROUPS;
  } else {
    a.a_stages = min(min(MAX_A, (512 - a.accs * a.acc_columns) / A_COLUMNS), a.stages);
    a.groups = min(GROUPS, a.a_stages);
  }
  CUtensorMap map_x, map_w;
  if (make_map(&map_x, p.x, p.M, p.K, a.n_tokens) || make_block_map(&map_w, p)) return 1;
  static uint64_t allowed = 0;
  if (allow_smem("gemm_int4", int4_rows_kernel, (int)SMEM_MOST, &allowed)) return 1;
  const size_t smem = (size_t)a.stages * stage_bytes + EXTRA;
  fms_launch(int4_rows_kernel, dim3(blocks), dim3(ROWS_THREADS), smem < SMEM_LEAST ? SMEM_LEAST : smem, stream, map_x, map_w, a, error_flag);
  if (fms_launch_status("gemm_int4")) return 1;
  bool shared = false;  // whether any tile's steps fall to two blocks
  for (int b = 1; b < blocks && !shared; ++b) shared = first_step(b, blocks, tiles * p.k_blocks) % p.k_blocks != 0;
  if (!shared) return 0;
  fms_launch(int4_join_kernel, dim3(tiles, a.n_tokens / 4), dim3(TILE), 0, stream, a, blocks);
  return fms_launch_status("gemm_int4_join");
}

// ---- more rows (prefill) ------------------------------------------------------------------------------------------------
// Persistent pairs of thread blocks (a cluster of two, cta_group::2): a pair owns a tile of 256 rows of w by up to 256 tokens.  Each
// block unpacks its own 128 rows of w into its own tensor memory and brings half of the tokens, so a multiprocessor takes in
// 128 rows of x and 128 half-bytes a k for 2 * 128 * 256 operations.  The accumulator takes half of the 512 columns and four stages
// of the operand the other half: a stage goes round in some 2,400 cycles (barriers, unpacking, the instructions), so that two of
// them, which left room for two accumulators of 192 columns, kept the tensor cores waiting (2,048 x 28,672 x 4,096 454 us; so 412).
// The next tile's first four steps are unpacked under the epilogue.
//   warp 0      per step of 128 k: two 64-k boxes of x, counted on block 0's barrier, and one of eight blocks of w, counted on its own
//   warp 1      (of block 0) issues 8 instructions (256 x tokens x 16) a step
//   warps 2-17  four groups of four unpack every fourth step each: a thread a row of w
//   warps 18-25 the epilogue, a warp a row's 32 lanes and every second 16 tokens
constexpr int PAIR_EPILOGUE = 8, PAIR_THREADS = 64 + 32 * (UNPACK_WARPS + PAIR_EPILOGUE), PAIR_TOKENS = 256;

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(PAIR_THREADS, 1)
    int4_pair_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, RowsArgs a,
                     int* __restrict__ error_flag) {
  extern __shared__ unsigned char smem_unaligned[];
  unsigned char* smem = smem_unaligned + (-smem_u32(smem_unaligned) & 1023);
  const Int4Args& p = a.p;
  const int half_tokens = a.n_tokens / 2, bytes = p.block_bytes(), x_bytes = half_tokens * BLOCK_K * 2, stages = a.stages;
  const int stage_bytes = (x_bytes + TILE / BLOCK_ROWS * bytes + 1023) / 1024 * 1024, k_steps = p.k_blocks;
  uint64_t* x_full = reinterpret_cast<uint64_t*>(smem + stages * stage_bytes);
  uint64_t* w_full = x_full + MAX_STAGES;
  uint64_t* empty = w_full + MAX_STAGES;
  uint64_t* a_full = empty + MAX_STAGES;  // [GROUPS]
  uint64_t* a_empty = a_full + GROUPS;    // [GROUPS]
  uint64_t* acc_full = a_empty + GROUPS;
  uint64_t* acc_empty = acc_full + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 1);
  __shared__ int failed_flag;
  volatile int* failed = &failed_flag;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const bool leader = rank == 0;
  const int tiles_m = (p.M + a.n_tokens - 1) / a.n_tokens, n_tiles = tiles_m * ((p.N + 2 * TILE - 1) / (2 * TILE));
  const int pair = blockIdx.x / 2, pairs = gridDim.x / 2;

  if (threadIdx.x == 0) {
    failed_flag = 0;
    for (int s = 0; s < MAX_STAGES; ++s) {
      mbar_init(&x_full[s], 1);
      mbar_init(&w_full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < GROUPS; ++i) {
      mbar_init(&a_full[i], 8);  // the warps of a group, of either block (used in block 0)
      mbar_init(&a_empty[i], 1);
    }
    mbar_init(acc_full, 1);
    mbar_init(acc_empty, 2 * PAIR_EPILOGUE);  // of either block (used in block 0)
    mbar_fence_init();
  }
  __syncthreads();
  cluster_sync_all();  // the partner runs, and its barriers exist
  if (warp == 1) tmem_alloc_pair(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // and it has its tensor memory
  tc_fence_after();
  const uint32_t tmem = *tmem_slot, tmem_a = tmem + A_FIRST;

  if (warp == 0) {
    if (elect_one()) {
      int it = 0;
      for (int tile = pair; tile < n_tiles && !*failed; tile += pairs) {
        const int m0 = (tile % tiles_m) * a.n_tokens + (int)rank * half_tokens;
        const int block0 = ((tile / tiles_m) * 2 + (int)rank) * (TILE / BLOCK_ROWS);
        for (int i = 0; i < k_steps; ++i, ++it) {
          const int s = it % stages;
          if (!wait_or_abort(&empty[s], ((it / stages) & 1) ^ 1, failed)) break;
          unsigned char* to = smem + s * stage_bytes;
          mbar_arrive_expect_tx(&w_full[s], TILE / BLOCK_ROWS * bytes);
          tma_load_3d(to + x_bytes, &map_w, 0, i, block0, &w_full[s]);
          if (leader) mbar_arrive_expect_tx(&x_full[s], 2 * x_bytes);  // the bytes of both blocks
          tma_load_2d_pair(to, &map_x, i * BLOCK_K, m0, &x_full[s]);
          tma_load_2d_pair(to + x_bytes / 2, &map_x, i * BLOCK_K + 64, m0, &x_full[s]);
        }
      }
    }
  } else if (warp == 1) {
    if (leader && elect_one()) {
      const uint32_t idesc = umma_idesc(2 * TILE, a.n_tokens);
      const MatrixDesc base(smem_u32(smem));
      const uint32_t box = (uint32_t)x_bytes / 2 >> 4;
      int j = 0, s = 0, group = 0;
      uint32_t phase = 0, turn = 0;
      for (int tile = pair; tile < n_tiles && !*failed; tile += pairs, ++j) {
        if (!wait_or_abort(acc_empty, (j & 1) ^ 1, failed)) break;  // both epilogues have read the tile before
        for (int i = 0; i < k_steps; ++i) {
          if (!quick_wait(&x_full[s], phase, failed) || !quick_wait(&a_full[group], turn, failed)) break;
          tc_fence_after();
          const uint32_t ta = tmem_a + group * A_COLUMNS, b = base.lo + (uint32_t)(s * stage_bytes >> 4);
#pragma unroll
          for (int kk = 0; kk < BLOCK_K / 16; ++kk)
            issue_a_tmem_pair(tmem, ta + kk * 8, b + (kk & 3) * 2 + (kk < 4 ? 0 : box), base.hi, idesc, kk > 0 ? 1u : i > 0);
          tc_commit_pair(&empty[s]);
          tc_commit_pair(&a_empty[group]);
          if (++s == stages) s = 0, phase ^= 1;
          if (++group == GROUPS) group = 0, turn ^= 1;
        }
        tc_commit_pair(acc_full);
      }
    }
  } else if (warp < 2 + UNPACK_WARPS) {
    const int group = (warp - 2) >> 2;
    int left = 0;  // steps, over all tiles
    for (int tile = pair; tile < n_tiles; tile += pairs) left += k_steps;
    int s = group;  // there are no fewer stages than groups
    uint32_t phase = 0, turn = 1;
    for (int it = group; it < left; it += GROUPS) {
      // its columns first: see the kernel above
      if (!warp_wait(&a_empty[group], turn, failed)) break;
      if (!warp_wait(&w_full[s], phase, failed)) break;
      unpack_row(smem + s * stage_bytes + x_bytes, bytes, p.per, warp & 3, lane, tmem_a + group * A_COLUMNS);
      if (lane == 0) {
        if (leader) mbar_arrive(&a_full[group]);
        else mbar_arrive_remote(&a_full[group], 0);
      }
      turn ^= 1;
      s += GROUPS;
      if (s >= stages) s -= stages, phase ^= 1;
    }
  } else {
    const int quarter = warp & 3, half = (warp - 2 - UNPACK_WARPS) >> 2;
    int j = 0;
    for (int tile = pair; tile < n_tiles; tile += pairs, ++j) {
      const int m0 = (tile % tiles_m) * a.n_tokens, col = ((tile / tiles_m) * 2 + (int)rank) * TILE + quarter * 32 + lane;
      const float bias = p.bias && col < p.N ? p.bias[col] : 0.f;
      if (!warp_wait(acc_full, j & 1, failed)) break;
      tc_fence_after();
      for (int c0 = 16 * half; c0 < a.n_tokens; c0 += 32) {
        float v[16];
        tmem_load_16(tmem + ((uint32_t)(quarter * 32) << 16) + c0, v);
        if (col < p.N) store_column<16>(p, v, m0 + c0, col, bias);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (leader) mbar_arrive(acc_empty);
        else mbar_arrive_remote(acc_empty, 0);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // nothing is sent to a block that has left
  if (threadIdx.x == 0 && *failed && error_flag) atomicExch(error_flag, 4);
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
}

// Tokens of a pair's tile: the width whose tiles cost least in whole rounds of the pairs; below some 100 tokens a step takes what
// unpacking takes.  A multiple of 32, which the instruction's shapes for a pair with A in tensor memory are.
int pair_tokens(int M, int N) {
  const int pairs = max(multiprocessors() / 2, 1), tiles_n = (N + 2 * TILE - 1) / (2 * TILE);
  long best = -1;
  int tokens = PAIR_TOKENS;
  for (int tn = PAIR_TOKENS; tn >= 96; tn -= 32) {
    const long tiles = (long)tiles_n * ((M + tn - 1) / tn), cost = (tiles + pairs - 1) / pairs * (max(tn, 100) + 24);
    if (best < 0 || cost < best) {
      best = cost;
      tokens = tn;
    }
  }
  return tokens;
}

int launch_pair(const Int4Args& p, int* error_flag, cudaStream_t stream) {
  RowsArgs a = {};
  a.p = p;
  const int pairs = max(multiprocessors() / 2, 1), tiles_n = (p.N + 2 * TILE - 1) / (2 * TILE);
  a.n_tokens = pair_tokens(p.M, p.N);
  const long tiles = (long)tiles_n * ((p.M + a.n_tokens - 1) / a.n_tokens);
  if (tiles > 0x7fffffffL) return fms_fail("gemm_int4: %ld tiles", tiles);
  const int stage_bytes = (a.n_tokens * BLOCK_K + TILE / BLOCK_ROWS * p.block_bytes() + 1023) / 1024 * 1024;
  a.stages = min((int)((SMEM_MOST - EXTRA) / stage_bytes), MAX_STAGES);
  CUtensorMap map_x, map_w;
  if (make_map(&map_x, p.x, p.M, p.K, a.n_tokens / 2) || make_block_map(&map_w, p)) return 1;
  static uint64_t allowed = 0;
  if (allow_smem("gemm_int4", int4_pair_kernel, (int)SMEM_MOST, &allowed)) return 1;
  const size_t smem = (size_t)a.stages * stage_bytes + EXTRA;
  // a plain launch: the pairs, which want all of the tensor memory, run beside no block of another kernel of the stream
  int4_pair_kernel<<<dim3(2 * (int)(tiles < pairs ? tiles : pairs)), dim3(PAIR_THREADS), smem < SMEM_LEAST ? SMEM_LEAST : smem, stream>>>(
      map_x, map_w, a, error_flag);
  return fms_launch_status("gemm_int4");
}

int check(const Int4Args& p) {
  if (p.K <= 0 || p.K % 8) return fms_fail("gemm_int4: %d input channels, a multiple of 8 is wanted", p.K);
  if (p.k_blocks != (p.K + BLOCK_K - 1) / BLOCK_K) return fms_fail("gemm_int4: %d blocks for %d input channels", p.k_blocks, p.K);
  if (p.per != 1 && p.per != 2 && p.per != 4) return fms_fail("gemm_int4: %d scales a block of 128 input channels", p.per);
  if (((uintptr_t)p.x | (uintptr_t)p.w) & 15) return fms_fail("gemm_int4: operands must be 16-byte aligned");
  return 0;
}
}  // namespace

// Rows of x that a tile of fms_linear_int4 has where its pairs of thread blocks take M of them; 0: another kernel does.
FMS_API int fms_linear_int4_tile(int M, int N) { return M <= FEW_ROWS || N <= 0 || M <= rows_most(N) ? 0 : pair_tokens(M, N); }

// Floats of scratch memory that fms_linear_int4 wants.
FMS_API long fms_linear_int4_scratch(long M, long N, long K) { return M <= FEW_ROWS || N <= 0 || K <= 0 || M > rows_most(N) ? 0 : rows_scratch(M, N, K); }

// y [M, N] bfloat16 of x [M, K] bfloat16, w packed with `per` scales a block, bias [N] bfloat16 or float32, or null.
FMS_API int fms_linear_int4(const void* x, const void* w, const void* bias, int bias_dtype, void* y, int M, int N, int K, int k_blocks, int per,
                            float* scratch, long scratch_floats, int* error_flag, cudaStream_t stream) {
  if (M <= 0 || N <= 0) return 0;
  const Int4Args p = {(const __nv_bfloat16*)x, (const unsigned char*)w, {bias, bias_dtype == FMS_F32}, (__nv_bfloat16*)y,
                      M, N, K, k_blocks, per, N, 0};
  if (check(p) || check_bias("gemm_int4", p.bias, bias_dtype)) return 1;
  return M <= FEW_ROWS ? few<false>(p, stream)
                       : (M <= rows_most(N) ? launch_rows(p, scratch, scratch_floats, error_flag, stream) : launch_pair(p, error_flag, stream));
}

// y [M, hidden] = act(gate) * up for w = [gate; up] of 2 hidden rows, hidden a multiple of 16, up to 8 rows of x.
FMS_API int fms_glu_int4(const void* x, const void* w, const void* bias, int bias_dtype, void* y, int M, int hidden, int K, int k_blocks, int per,
                         int act, cudaStream_t stream) {
  if (M <= 0 || hidden <= 0) return 0;
  if (M > FEW_ROWS || hidden % BLOCK_ROWS || act < 0 || act > 3)
    return fms_fail("glu_int4: %d rows of x, %d hidden values, activation %d", M, hidden, act);
  const Int4Args p = {(const __nv_bfloat16*)x, (const unsigned char*)w, {bias, bias_dtype == FMS_F32}, (__nv_bfloat16*)y,
                      M, 2 * hidden, K, k_blocks, per, hidden, act};
  if (check(p) || check_bias("gemm_int4", p.bias, bias_dtype)) return 1;
  return few<true>(p, stream);
}
