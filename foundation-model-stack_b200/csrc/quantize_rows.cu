// Rows to 8 bits (e4m3: 4 bits of exponent, 3 of mantissa, largest value 448) with one float32 scale a row, alone or
// behind the residual sum and RMS norm that make the row:
//   quantize_rows     s = max |x| / 448,  q = e4m3(x * 448 / max |x|)
//   add_rmsnorm       x = residual[src] + delta[src]  (float32; written back unless rows are gathered),
//                     y = x * rsqrt(mean(x^2) + eps) * gain,  s = max |y| / 448,  q = e4m3(y * 448 / max |y|)
//                                                                   (the norm: fms/modules/layernorm.py:56-69)
// e4m3() rounds to the nearest value, ties to even.  A row whose scale would lie below 2^-110 (a row of zeros) gets scale 0
// and zeros.  A finite row whose squares overflow float32 (values beyond some 10^19) is summed again, with 2^-80 of every value, which
// the quotient and the division by the root mean square cancel.  A row with a NaN or an infinity gets a scale that is not finite (NaN behind the norm),
// so that what a product makes of it is not finite either, and the other rows do not see it.
//
// Both are bound by memory: a value is read once (2 or 4 bytes, behind the norm 4 and 2 or 4), the stream written (4) and
// one byte stored.  A thread block owns a row and keeps it in registers, as it was loaded, between the maximum and the rounding,
// so that nothing is read twice.  A thread owns runs of 8 neighbours, 16-byte loads and 8-byte stores.  Rows of a width that is no
// multiple of 8 begin anywhere: their runs are moved forward by up to 3 values to where the rows' own loads are aligned, and a
// warp's lanes hand one another the bytes that make aligned stores (1,100 x 5,001 bfloat16 7.7 us, and behind the norm, float32,
// 21.1; 11.4 and 25.1 with single loads and stores).  Rows of q are `pitch` bytes apart, dim rounded up to 16 with zeros behind the last value, as the products'
// copies want them.
//
// q is what the exact quotient rounds to.  Of bfloat16 rows it is often a tie, and otherwise, a ratio of numbers of 11 and 8 bits,
// at least 2^-13 away from one, so one step of Newton's, whose remainder x * 448 - q0 * max |x| is exact in a fused
// multiply-add, decides it.  Behind the norm the division by the root mean square cancels: with t = x * gain, q is t * 448 / max |t|.
// There, and of float32 rows, the float32 quotient is within a few units of its last place, which decides the rounding but for a
// few values in a million that come out beside the middle of two neighbours; a run of 8 that has one is compared with
// those middles in float64, where t * 448 and a middle times max |t| are exact.
#include <cuda_fp8.h>

#include "common.cuh"

namespace {
constexpr float E4M3_MAX = 448.f;
constexpr float LEAST = 0x1p-110f;  // a scale below is none
constexpr float SHRUNK = 0x1p-80f;   // of a row whose squares overflow: then the sum of up to 2^31 does not

// the larger of two, NaN where either is one
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;\n" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// 8 values of a row as they were loaded
template <typename T> struct Run;
template <> struct Run<float> {
  static constexpr bool EXACT = false;  // 448 times a value has 24 bits at most
  float v[8];
  __device__ __forceinline__ float operator[](int e) const { return v[e]; }
  __device__ __forceinline__ void set(int e, float x) { v[e] = x; }
  __device__ __forceinline__ void load(const float* p) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  }
  static __device__ __forceinline__ bool aligned(const float* p) { return ((uintptr_t)p & 15) == 0; }
  __device__ __forceinline__ void load_halves(const float* p) { load(p); }
};
template <> struct Run<__nv_bfloat16> {
  static constexpr bool EXACT = true;
  uint32_t w[4];
  __device__ __forceinline__ float operator[](int e) const { return __uint_as_float(e & 1 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16); }
  __device__ __forceinline__ void set(int e, __nv_bfloat16 x) {
    const uint32_t h = __bfloat16_as_ushort(x);
    w[e / 2] = e & 1 ? w[e / 2] | (h << 16) : h;
  }
  __device__ __forceinline__ void load(const __nv_bfloat16* p) {
    const uint4 t = *reinterpret_cast<const uint4*>(p);
    w[0] = t.x; w[1] = t.y; w[2] = t.z; w[3] = t.w;
  }
  static __device__ __forceinline__ bool aligned(const __nv_bfloat16* p) { return ((uintptr_t)p & 7) == 0; }
  __device__ __forceinline__ void load_halves(const __nv_bfloat16* p) {
    const uint2 a = reinterpret_cast<const uint2*>(p)[0], b = reinterpret_cast<const uint2*>(p)[1];
    w[0] = a.x; w[1] = a.y; w[2] = b.x; w[3] = b.y;
  }
};
// The place in the row of the first value of this thread's run j, moved forward by `shift` (0 where a run's 8 are NEIGHBOURS that
// begin on a multiple of 8, as dim does)
__device__ __forceinline__ int place(int j, int shift) { return 8 * (int)(threadIdx.x + j * blockDim.x) - shift; }
// the values by which the runs of a row are moved so that 4 of them lie aligned
template <typename T> __device__ __forceinline__ int shift_of(const T* row) { return (int)((uintptr_t)row / sizeof(T)) & 3; }
// zeros outside the row; `left`: the values from its first to the array's last, for the bounds-checked build
template <bool NEIGHBOURS, typename T> __device__ __forceinline__ void load_run(Run<T>& run, const T* row, int j, int shift, int dim, long left) {
  const int c0 = place(j, NEIGHBOURS ? 0 : shift);
  if (NEIGHBOURS) {
    if (c0 < dim && FMS_IN(c0 + 7, left)) {
      run.load(row + c0);
      return;
    }
  } else if (c0 >= 0 && c0 + 8 <= dim && Run<T>::aligned(row + c0) && FMS_IN(c0 + 7, left)) {  // (taking the others as three aligned loads and picking was slower)
    run.load_halves(row + c0);
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) run.set(e, !NEIGHBOURS && c0 + e >= 0 && c0 + e < dim && FMS_IN(c0 + e, left) ? row[c0 + e] : T(0.f));
}
// 8 values as e4m3, nearest and ties to even, beyond 448 to 448
__device__ __forceinline__ uint2 to_e4m3(const float* v) {
  uint32_t h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    h[i] = __nv_cvt_float2_to_fp8x2(make_float2(v[2 * i], v[2 * i + 1]), __NV_SATFINITE, __NV_E4M3);
  return make_uint2(h[0] | (h[1] << 16), h[2] | (h[3] << 16));
}

// zeros outside the row, where zeros times what is not finite are not
template <bool NEIGHBOURS> __device__ __forceinline__ float* ended(float* q, int c0, int dim) {
  if (c0 < 0 || c0 + 8 > dim) {
#pragma unroll
    for (int e = 0; e < 8; ++e) q[e] = c0 + e >= 0 && c0 + e < dim ? q[e] : 0.f;
  }
  return q;
}

// 8 quotients t * 448 / most, t = x (* g), to e4m3 as exact quotients would be, zeros where the row has ended; inv = 448 / most.
// The float32 quotient, three or four roundings away, is off by less than 4 units of its last place.
template <bool NEIGHBOURS, bool GAIN, typename X, typename G>
__device__ __forceinline__ uint2 quotients(const X& x, const G& g, float inv, double most, int c0, int dim) {
  float q[8];
  if (!GAIN && X::EXACT) {  // inv = 448 / most is 0.875 / part, and neither 0.875 x nor part is rounded or out of range
    const float part = (float)most * 0x1p-9f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float q0 = x[e] * inv;
      q[e] = fmaf(fmaf(-q0, part, x[e] * 0.875f), inv * (1.f / 0.875f), q0);
    }
    return to_e4m3(ended<NEIGHBOURS>(q, c0, dim));
  }
  // From 2^-6 on a value is beside a middle where its last 20 bits are within 8 of 2^19; below, the middles are the odd
  // multiples of 2^-10, which 2^-6 more puts where the same test finds them.
  uint32_t beside = ~0u;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    q[e] = (GAIN ? x[e] * g[e] : x[e]) * inv;
    const float m = fabsf(q[e]);
    beside = min(beside, __float_as_uint(m < 0x1p-6f ? m + 0x1p-6f : m) * 4096u - (0x7fff8u << 12));  // the 20 bits, first
  }
  if (beside <= (16u << 12) && most < INFINITY) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float m = fabsf(q[e]);
      const float middle = m >= 0x1p-6f ? __uint_as_float((__float_as_uint(m) & ~0xfffffu) | 0x80000u) : (floorf(m * 512.f) + 0.5f) * 0x1p-9f;
      if (fabsf(m - middle) > middle * 0x1p-18f) continue;
      // |t| * 448 (at most 51 bits) against middle * most (at most 5 + 48)
      const double t = fabs((double)x[e] * (GAIN ? (double)g[e] : 1.0)) * 448.0, at = (double)middle * most;
      const float r = __uint_as_float(__float_as_uint(middle) + (t > at ? 1 : (t < at ? -1 : 0)));
      q[e] = copysignf(r, q[e]);
    }
  }
  return to_e4m3(ended<NEIGHBOURS>(q, c0, dim));
}
// By a whole warp.  A run that is moved by `shift` holds the last bytes of its aligned 8 first: the next lane has the others.
template <bool NEIGHBOURS> __device__ __forceinline__ void store_run(uint8_t* row, uint2 q, int j, int shift, int pitch, long left) {
  const int at = place(j, 0);
  if (NEIGHBOURS || shift == 0) {
    if (at < pitch && FMS_IN(at + 7, left)) *reinterpret_cast<uint2*>(row + at) = q;
    return;
  }
  const uint64_t own = ((uint64_t)q.y << 32) | q.x, next = __shfl_down_sync(0xffffffffu, own, 1);
  const int lane = threadIdx.x & 31, bits = 8 * shift;
  if (lane < 31) {
    if (at < pitch && FMS_IN(at + 7, left)) *reinterpret_cast<uint64_t*>(row + at) = (own >> bits) | (next << (64 - bits));
  } else {
    for (int e = shift; e < 8; ++e)
      if (at + e - shift < pitch && FMS_IN(at + e - shift, left)) row[at + e - shift] = (uint8_t)(own >> (8 * e));
  }
  if (lane == 0 && at > 0)  // what the warp before could not store
    for (int e = 0; e < shift; ++e)
      if (at + e - shift < pitch && FMS_IN(at + e - shift, left)) row[at + e - shift] = (uint8_t)(own >> (8 * e));
}

__device__ __forceinline__ float block_max(float v, float* scratch) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nwarps = blockDim.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
  if (lane == 0) scratch[warp] = v;
  __syncthreads();
  v = lane < nwarps ? scratch[lane] : 0.f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// the largest magnitude of a run, NaN where one is NaN
__device__ __forceinline__ float largest(const Run<float>& r) {
  float m = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) m = max_nan(m, fabsf(r.v[e]));
  return m;
}
__device__ __forceinline__ float largest(const Run<__nv_bfloat16>& r) {
  __nv_bfloat162 m = __habs2(*reinterpret_cast<const __nv_bfloat162*>(&r.w[0]));
#pragma unroll
  for (int i = 1; i < 4; ++i) m = __hmax2_nan(m, __habs2(*reinterpret_cast<const __nv_bfloat162*>(&r.w[i])));
  return max_nan(__low2float(m), __high2float(m));
}

// No pointer of these kernels is __restrict__: what the kernel in front wrote must come through the coherent path, not through the one
// for data that nobody writes while a kernel runs, which this one may begin to do before that one is done.

// RUNS: runs of 8 values that a thread keeps; 0: any width, the row is read a second time.
// What bounds many rows is how many of their bytes are on the way, so registers are kept few: three thread blocks of 448 for rows of
// 14,336 (2,048 of them, bfloat16: 17.9 us, 4.9 TB/s; with two blocks 20.8, with four 19.2 for the registers that spill).
template <typename T, int RUNS, bool NEIGHBOURS>
__global__ void __launch_bounds__(RUNS == 1 ? 1024 : 512, NEIGHBOURS && RUNS == 4 && sizeof(T) == 2 ? 3 : (RUNS != 1 && RUNS != 8 ? 2 : 1))
    quantize_rows_kernel(const T* x, uint8_t* q, float* scales, int dim, int pitch) {
  __shared__ float scratch[32];
  pdl_launch_dependents();
  pdl_wait();
  const T* row = x + (size_t)blockIdx.x * dim;
  uint8_t* out = q + (size_t)blockIdx.x * pitch;
  const long left = (long)(gridDim.x - blockIdx.x) * dim;
  constexpr int KEPT = RUNS > 0 ? RUNS : 1;
  const int runs = RUNS > 0 ? RUNS : (pitch / 8 + !NEIGHBOURS + blockDim.x - 1) / blockDim.x, shift = NEIGHBOURS ? 0 : shift_of(row);
  Run<T> v[KEPT];
  float most = 0.f;
#pragma unroll
  for (int j = 0; j < KEPT; ++j)
    if (RUNS > 0) load_run<NEIGHBOURS>(v[j], row, j, shift, dim, left);
#pragma unroll KEPT
  for (int j = 0; j < runs; ++j) {
    if (RUNS == 0) load_run<NEIGHBOURS>(v[0], row, j, shift, dim, left);
    most = max_nan(most, largest(v[RUNS > 0 ? j : 0]));
  }
  most = block_max(most, scratch);
  const float s = most / E4M3_MAX;
  const bool none = s < LEAST;
  const float inv = none ? 0.f : E4M3_MAX / most;
#pragma unroll KEPT
  for (int j = 0; j < runs; ++j) {
    if (RUNS == 0) load_run<NEIGHBOURS>(v[0], row, j, shift, dim, left);
    const Run<T>& u = v[RUNS > 0 ? j : 0];
    store_run<NEIGHBOURS>(out, quotients<NEIGHBOURS, false>(u, u, inv, most, place(j, shift), dim), j, shift, pitch, (long)(gridDim.x - blockIdx.x) * pitch);
  }
  if (threadIdx.x == 0) scales[blockIdx.x] = none ? 0.f : s;
}

// a float32 and what rounding to it left over: the larger of two magnitudes
struct Pair {
  float hi, lo;
};
__device__ __forceinline__ Pair larger(Pair a, Pair b) { return b.hi > a.hi || (b.hi == a.hi && b.lo > a.lo) ? b : a; }

template <typename T, typename TG, int RUNS, bool NEIGHBOURS>
__global__ void __launch_bounds__(RUNS == 1 ? 1024 : 512, RUNS == 0 || RUNS == 2 ? 2 : 1)
    add_rmsnorm_quantized_kernel(float* residual, const T* delta, const TG* gain, float eps, uint8_t* q, float* scales, const int* rows,
                                 int dim, int pitch, int residual_rows) {
  __shared__ float scratch[3][32];
  constexpr int KEPT = RUNS > 0 ? RUNS : 1;
  const int runs = RUNS > 0 ? RUNS : (pitch / 8 + !NEIGHBOURS + blockDim.x - 1) / blockDim.x;
  Run<float> x[KEPT];
  Run<TG> g[KEPT];
  pdl_launch_dependents();
  pdl_wait();  // any of the tensors, the gain among them, may be what the kernel before writes
  const int src = rows ? rows[blockIdx.x] : blockIdx.x;
  if (!FMS_IN(src, residual_rows)) return;  // the whole block alike
  float* res = residual + (size_t)src * dim;
  const long left = residual_rows > 0 ? (long)(residual_rows - src) * dim : 0;
  const int shift = NEIGHBOURS ? 0 : shift_of(res);
  const T* del = delta ? delta + (size_t)src * dim : nullptr;
  const bool writes = del && rows == nullptr;
  auto add = [&](Run<float>& v, const Run<T>& d) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v.v[e] += d[e];
  };
  if (RUNS > 0) {
    Run<T> d[KEPT];
#pragma unroll
    for (int j = 0; j < KEPT; ++j) load_run<NEIGHBOURS>(x[j], res, j, shift, dim, left);
#pragma unroll
    for (int j = 0; j < KEPT; ++j) load_run<NEIGHBOURS>(g[j], gain, j, shift, dim, dim);
    if (del) {
#pragma unroll
      for (int j = 0; j < KEPT; ++j) load_run<NEIGHBOURS>(d[j], del, j, shift, dim, left);
#pragma unroll
      for (int j = 0; j < KEPT; ++j) add(x[j], d[j]);
    }
  }
  // RUNS 0: a run's sums and gains, read again in every pass
  auto fetch = [&](int j, bool stored) {
    load_run<NEIGHBOURS>(x[0], res, j, shift, dim, left);  // the sum, where this thread has stored it
    load_run<NEIGHBOURS>(g[0], gain, j, shift, dim, dim);
    if (del && !stored) {
      Run<T> d;
      load_run<NEIGHBOURS>(d, del, j, shift, dim, left);
      add(x[0], d);
    }
  };
  auto shrink = [&](Run<float>& v) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v.v[e] *= SHRUNK;
  };
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nwarps = blockDim.x >> 5;
  float ss;
  Pair most;
  bool shrunk = false;  // the whole block alike
#pragma unroll 1
  while (true) {
    ss = 0.f;
    most = {0.f, 0.f};
#pragma unroll KEPT
    for (int j = 0; j < runs; ++j) {
      Run<float>& xs = x[RUNS > 0 ? j : 0];
      Run<TG>& gs = g[RUNS > 0 ? j : 0];
      if (RUNS == 0) fetch(j, shrunk && writes);
      if (writes && !shrunk) {
        const int c0 = place(j, shift);
        if (c0 >= 0 && c0 + 8 <= dim && FMS_IN(c0 + 7, left)) {
          float4* to = reinterpret_cast<float4*>(res + c0);
          to[0] = make_float4(xs.v[0], xs.v[1], xs.v[2], xs.v[3]);
          to[1] = make_float4(xs.v[4], xs.v[5], xs.v[6], xs.v[7]);
        } else if (!NEIGHBOURS) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (c0 + e >= 0 && c0 + e < dim && FMS_IN(c0 + e, left)) res[c0 + e] = xs.v[e];
        }
      }
      if (shrunk) shrink(xs);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        ss += xs[e] * xs[e];
        const float t = xs[e] * gs[e], left = fmaf(xs[e], gs[e], -t);
        most = larger(most, Pair{fabsf(t), t < 0.f ? -left : left});
      }
    }
    auto over_warp = [&]() {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        ss += __shfl_xor_sync(0xffffffffu, ss, o);
        most = larger(most, Pair{__shfl_xor_sync(0xffffffffu, most.hi, o), __shfl_xor_sync(0xffffffffu, most.lo, o)});
      }
    };
    over_warp();
    if (lane == 0) {
      scratch[0][warp] = ss;
      scratch[1][warp] = most.hi;
      scratch[2][warp] = most.lo;
    }
    __syncthreads();
    ss = lane < nwarps ? scratch[0][lane] : 0.f;
    most = lane < nwarps ? Pair{scratch[1][lane], scratch[2][lane]} : Pair{0.f, 0.f};
    over_warp();
    if (ss < INFINITY || shrunk) break;
    shrunk = true;
    __syncthreads();  // scratch is written again
  }

  // a NaN or an infinity in the row leaves `ss` not finite; eps is nothing beside the squares of a row that was shrunk
  const float s = ss < INFINITY ? most.hi * rsqrtf(ss / (float)dim + (shrunk ? 0.f : eps)) / E4M3_MAX : NAN;
  const bool none = s < LEAST || most.hi < LEAST;  // far below, the reciprocal would overflow
  const float inv = none ? 0.f : (s == s ? E4M3_MAX / most.hi : NAN);
  const double exact = (double)most.hi + (double)most.lo;
#pragma unroll KEPT
  for (int j = 0; j < runs; ++j) {
    Run<float>& xs = x[RUNS > 0 ? j : 0];
    Run<TG>& gs = g[RUNS > 0 ? j : 0];
    if (RUNS == 0) {
      fetch(j, writes);
      if (shrunk) shrink(xs);
    }
    store_run<NEIGHBOURS>(q + (size_t)blockIdx.x * pitch, quotients<NEIGHBOURS, true>(xs, gs, inv, exact, place(j, shift), dim), j, shift, pitch,
                          (long)(gridDim.x - blockIdx.x) * pitch);
  }
  if (threadIdx.x == 0) scales[blockIdx.x] = none ? 0.f : s;
}

// The runs of 8 that a thread keeps (0: the row is too wide for registers) and the threads for a row of `runs` of them.  Few
// rows: a thread a run as far as 1,024 go, since only latency counts.  Many: `many` runs a thread, so that more bytes a thread and
// more rows a multiprocessor are on their way (8,192 x 4,096 bfloat16 to e4m3 with 1 / 2 / 4 / 8 runs: 27.5 / 22.8 / 16.9 / 19.8 us;
// behind the norm, whose runs take 12 registers and more, 2,048 x 4,096 with 1 / 2 / 4: 22.4 / 17.3 / 18.4 us; since the gain waits for
// the kernel in front and rows that overflow are summed again, 17.6).
int kept_for(int runs, int n_rows, int many, int most_kept, int* threads) {
  int kept = n_rows <= 296 ? (runs <= 1024 ? 1 : 4) : (runs <= 128 ? 1 : many);
  if (runs > 512 * kept && kept > 1) kept = runs <= 512 * 4 ? 4 : (runs <= 512 * most_kept ? most_kept : 0);
  const int wanted = kept ? (runs + kept - 1) / kept : 512;
  *threads = (wanted + 31) / 32 * 32;
  return kept;
}
bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

template <typename T, int RUNS>
void launch_rows(int threads, bool neighbours, const void* x, uint8_t* q, float* scales, int n_rows, int dim, int pitch, cudaStream_t stream) {
  fms_launch(neighbours ? quantize_rows_kernel<T, RUNS, true> : quantize_rows_kernel<T, RUNS, false>, dim3(n_rows), dim3(threads), 0,
             stream, (const T*)x, q, scales, dim, pitch);
}
template <typename T> int quantize(const void* x, uint8_t* q, float* scales, int n_rows, int dim, int pitch, cudaStream_t stream) {
  int threads;
  const bool neighbours = dim % 8 == 0 && aligned16(x);
  const int kept = kept_for(pitch / 8 + !neighbours, n_rows, 4, 8, &threads);  // a run more for rows that begin anywhere
  (kept == 1 ? launch_rows<T, 1> : kept == 4 ? launch_rows<T, 4> : kept == 8 ? launch_rows<T, 8> : launch_rows<T, 0>)(
      threads, neighbours, x, q, scales, n_rows, dim, pitch, stream);
  return fms_launch_status("quantize_rows");
}

struct NormArgs {
  float* residual;
  const void *delta, *gain;
  float eps;
  uint8_t* q;
  float* scales;
  const int* rows;
  int n_rows, dim, pitch, residual_rows;
};
template <typename T, typename TG, int RUNS> void launch_norm(int threads, bool neighbours, const NormArgs& a, cudaStream_t stream) {
  fms_launch(neighbours ? add_rmsnorm_quantized_kernel<T, TG, RUNS, true> : add_rmsnorm_quantized_kernel<T, TG, RUNS, false>, dim3(a.n_rows),
             dim3(threads), 0, stream, a.residual, (const T*)a.delta, (const TG*)a.gain, a.eps, a.q, a.scales, a.rows, a.dim, a.pitch,
             a.residual_rows);
}
template <typename T, typename TG> int norm(const NormArgs& a, cudaStream_t stream) {
  int threads;
  const bool neighbours = a.dim % 8 == 0 && aligned16(a.residual) && aligned16(a.delta) && aligned16(a.gain);
  const int kept = kept_for(a.pitch / 8 + !neighbours, a.n_rows, 2, 4, &threads);
  (kept == 1 ? launch_norm<T, TG, 1> : kept == 2 ? launch_norm<T, TG, 2> : kept == 4 ? launch_norm<T, TG, 4> : launch_norm<T, TG, 0>)(threads, neighbours, a, stream);
  return fms_launch_status("add_rmsnorm_quantized");
}
}  // namespace

// q [n_rows, pitch] e4m3 and scales [n_rows] of x [n_rows, dim]; pitch: dim rounded up to a multiple of 16, the rest zeros.
FMS_API int fms_quantize_rows(const void* x, int dtype, void* q, float* scales, int n_rows, int dim, int pitch,
                              cudaStream_t stream) {
  if (n_rows <= 0) return 0;
  if (dim <= 0 || pitch % 16 || pitch < dim || pitch - dim > 15) return fms_fail("quantize_rows: dim %d, pitch %d", dim, pitch);
  if (!aligned16(q)) return fms_fail("quantize_rows: the 8-bit rows must be 16-byte aligned");
  FMS_DISPATCH_DTYPE(dtype, T, return quantize<T>(x, (uint8_t*)q, scales, n_rows, dim, pitch, stream));
  return 0;
}

// residual_rows: rows of the residual stream (and of delta), which the entries of `rows` index; used by the
// bounds-checked build only (0: not known)
FMS_API int fms_add_rmsnorm_quantized(float* residual, const void* delta, int delta_dtype, const void* gain, int gain_dtype,
                                      float eps, void* q, float* scales, const int* rows, int n_rows, int dim, int pitch,
                                      int residual_rows, cudaStream_t stream) {
  if (n_rows <= 0) return 0;
  if (dim <= 0 || pitch % 16 || pitch < dim || pitch - dim > 15) return fms_fail("add_rmsnorm_quantized: dim %d, pitch %d", dim, pitch);
  if (!aligned16(q)) return fms_fail("add_rmsnorm_quantized: the 8-bit rows must be 16-byte aligned");
  const NormArgs a = {residual, delta, gain, eps, (uint8_t*)q, scales, rows, n_rows, dim, pitch, residual_rows};
  FMS_DISPATCH_DTYPE(delta_dtype, T, FMS_DISPATCH_DTYPE(gain_dtype, TG, return norm<T, TG>(a, stream)));
  return 0;
}
