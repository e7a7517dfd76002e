// Rows to 8 bits (e4m3: 4 bits of exponent, 3 of mantissa, largest value 448) with one float32 scale a row, alone or
// behind the residual sum and RMS norm that make the row:
//   quantize_rows     s = max |x| / 448,  q = e4m3(x * 448 / max |x|)
//   add_rmsnorm       x = residual[src] + delta[src]  (float32; written back unless rows are gathered),
//                     y = x * rsqrt(mean(x^2) + eps) * gain,  s = max |y| / 448,  q = e4m3(y * 448 / max |y|)
//                                                                   (the norm: fms/modules/layernorm.py:56-69)
// e4m3() rounds to the nearest value, ties to even.  A row whose scale would lie below the smallest normal float32 (a row
// of zeros) gets scale 0 and zeros.  A row with a NaN or an infinity gets a scale that is not finite (NaN behind the norm),
// so that what a product makes of it is not finite either, and the other rows do not see it.
//
// Both are bound by memory: a value is read once (2 or 4 bytes, behind the norm 4 and 2 or 4), the stream written (4) and
// one byte stored.  A thread block owns a row and keeps it in registers between the maximum and the rounding, so that
// nothing is read twice; a thread owns runs of 8 values, 16-byte loads and 8-byte stores.  Rows of q are `pitch` bytes
// apart, dim rounded up to 16 with zeros behind the last value, as the products' copies want them; rows of x whose width is
// no multiple of the load's are read value by value.
//
// q is what the exact quotient rounds to.  Behind the norm the division by the root mean square cancels in it: with t = x * gain it
// is t * 448 / max |t|.  In float32 it comes out within a few units of its last place, which decides the rounding to 4 bits but
// for a few values in a million that come out beside the middle of two neighbours; a run of 8 that has one is compared
// with those middles in float64, where t * 448 and a middle times max |t| are exact.
#include <cuda_fp8.h>

#include "common.cuh"

namespace {
constexpr float E4M3_MAX = 448.f;
constexpr float LEAST = 1.17549435e-38f;  // the smallest normal float32

// the larger of two, NaN where either is one
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;\n" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ void load8(const float* p, float* v) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float* v) {
  const uint4 t = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
// values c0 .. c0 + 7 of a row of `dim`; zeros beyond its end
template <typename T>
__device__ __forceinline__ void load_run(const T* row, int c0, int dim, bool vectors, float* v) {
  if (vectors && c0 + 8 <= dim) {
    load8(row + c0, v);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = c0 + e < dim ? to_f32(row[c0 + e]) : 0.f;
  }
}
__device__ __forceinline__ void store_run(float* row, int c0, int dim, bool vectors, const float* v) {
  if (vectors && c0 + 8 <= dim) {
    reinterpret_cast<float4*>(row + c0)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(row + c0)[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c0 + e < dim) row[c0 + e] = v[e];
  }
}
// 8 values as e4m3, nearest and ties to even, beyond 448 to 448
__device__ __forceinline__ uint2 to_e4m3(const float* v) {
  uint32_t h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    h[i] = __nv_cvt_float2_to_fp8x2(make_float2(v[2 * i], v[2 * i + 1]), __NV_SATFINITE, __NV_E4M3);
  return make_uint2(h[0] | (h[1] << 16), h[2] | (h[3] << 16));
}

// zeros behind a row's last value, whatever the quotients there
__device__ __forceinline__ uint2 ended(uint2 q, int c0, int dim) {
  const int left = dim - c0;
  if (left >= 8) return q;
  const uint64_t v = left <= 0 ? 0ull : (((uint64_t)q.y << 32) | q.x) & (~0ull >> (64 - 8 * left));
  return make_uint2((uint32_t)v, (uint32_t)(v >> 32));
}

// 8 quotients t * 448 / most, t = x (* g), rounded to e4m3 as exact quotients would be; inv = 448 / most in float32.
// q0, four roundings away from the quotient, is off by less than 4 units of its last place (2^-22 of it).
template <bool GAIN> __device__ __forceinline__ uint2 quotients(const float* x, const float* g, float inv, double most) {
  float q[8];
  bool near = false;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    q[e] = (GAIN ? x[e] * g[e] : x[e]) * inv;
    // from 2^-6 on the middles have 4 bits of mantissa and a half; below they lie at odd multiples of 2^-10
    const float m = fabsf(q[e]), steps = m * 512.f;
    const bool beside = m >= 0x1p-6f ? ((__float_as_uint(m) & 0xfffffu) - 0x7fff8u) <= 16u : fabsf(steps - floorf(steps) - 0.5f) < 0x1p-14f;
    near |= beside;
  }
  if (near && most < INFINITY) {
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
  return to_e4m3(q);
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

// RUNS: runs of 8 values that a thread keeps; 0: any width, the row is read a second time.
template <typename T, int RUNS>
__global__ void __launch_bounds__(1024) quantize_rows_kernel(const T* __restrict__ x, uint8_t* __restrict__ q, float* __restrict__ scales, int n_rows,
                                                             int dim, int pitch, int vectors) {
  __shared__ float scratch[32];
  pdl_launch_dependents();
  pdl_wait();
  const T* row = x + (size_t)blockIdx.x * dim;
  uint8_t* out = q + (size_t)blockIdx.x * pitch;
  constexpr int KEPT = RUNS > 0 ? RUNS : 1;
  const int runs = RUNS > 0 ? RUNS : (pitch / 8 + blockDim.x - 1) / blockDim.x;
  float v[KEPT][8], most = 0.f;
#pragma unroll
  for (int j = 0; j < KEPT; ++j)
    if (RUNS > 0) load_run(row, 8 * (threadIdx.x + j * blockDim.x), dim, vectors, v[j]);
#pragma unroll KEPT
  for (int j = 0; j < runs; ++j) {
    if (RUNS == 0) load_run(row, 8 * (threadIdx.x + j * blockDim.x), dim, vectors, v[0]);
    float* u = v[RUNS > 0 ? j : 0];
#pragma unroll
    for (int e = 0; e < 8; ++e) most = max_nan(most, fabsf(u[e]));
  }
  most = block_max(most, scratch);
  const float s = most / E4M3_MAX;
  const bool none = s < LEAST;
  const float inv = none ? 0.f : E4M3_MAX / most;
#pragma unroll KEPT
  for (int j = 0; j < runs; ++j) {
    const int c0 = 8 * (threadIdx.x + j * blockDim.x);
    if (RUNS == 0) load_run(row, c0, dim, vectors, v[0]);
    float* u = v[RUNS > 0 ? j : 0];
    if (c0 < pitch && FMS_IN((size_t)blockIdx.x * pitch + c0 + 7, (size_t)n_rows * pitch))
      *reinterpret_cast<uint2*>(out + c0) = ended(quotients<false>(u, nullptr, inv, most), c0, dim);
  }
  if (threadIdx.x == 0 && FMS_IN(blockIdx.x, n_rows)) scales[blockIdx.x] = none ? 0.f : s;
}

// a float32 and what rounding to it left over: the larger of two magnitudes
struct Pair {
  float hi, lo;
};
__device__ __forceinline__ Pair larger(Pair a, Pair b) { return b.hi > a.hi || (b.hi == a.hi && b.lo > a.lo) ? b : a; }

template <typename T, typename TG, int RUNS>
__global__ void __launch_bounds__(1024) add_rmsnorm_quantized_kernel(float* __restrict__ residual, const T* __restrict__ delta,
                                                                     const TG* __restrict__ gain, float eps,
                                                                      uint8_t* __restrict__ q, float* __restrict__ scales,
                                                                      const int* __restrict__ rows, int n_rows, int dim,
                                                                      int pitch, int residual_rows, int vec_x, int vec_d, int vec_g) {
  __shared__ float scratch[3][32];
  constexpr int KEPT = RUNS > 0 ? RUNS : 1;
  const int runs = RUNS > 0 ? RUNS : (pitch / 8 + blockDim.x - 1) / blockDim.x;
  float x[KEPT][8], g[KEPT][8];
  pdl_launch_dependents();
#pragma unroll
  for (int j = 0; j < KEPT; ++j)  // the gain is a weight: it can be read before the kernel before this one is done
    if (RUNS > 0) load_run(gain, 8 * (threadIdx.x + j * blockDim.x), dim, vec_g, g[j]);
  pdl_wait();
  const int src = rows ? rows[blockIdx.x] : blockIdx.x;
  if (!FMS_IN(src, residual_rows)) return;  // the whole block alike
  float* res = residual + (size_t)src * dim;
  const T* del = delta ? delta + (size_t)src * dim : nullptr;
  auto load_sum = [&](int c0, float* v) {
    load_run(res, c0, dim, vec_x, v);
    if (del) {
      float d[8];
      load_run(del, c0, dim, vec_d, d);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += d[e];
    }
  };
#pragma unroll
  for (int j = 0; j < KEPT; ++j)
    if (RUNS > 0) load_sum(8 * (threadIdx.x + j * blockDim.x), x[j]);
  float ss = 0.f;
  Pair most = {0.f, 0.f};
#pragma unroll KEPT
  for (int j = 0; j < runs; ++j) {
    const int c0 = 8 * (threadIdx.x + j * blockDim.x);
    float *xs = x[RUNS > 0 ? j : 0], *gs = g[RUNS > 0 ? j : 0];
    if (RUNS == 0) {
      load_sum(c0, xs);
      load_run(gain, c0, dim, vec_g, gs);
    }
    if (del && rows == nullptr && c0 < dim) store_run(res, c0, dim, vec_x, xs);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      ss += xs[e] * xs[e];
      const float t = xs[e] * gs[e], left = fmaf(xs[e], gs[e], -t);
      most = larger(most, Pair{fabsf(t), t < 0.f ? -left : left});
    }
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nwarps = blockDim.x >> 5;
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

  // a NaN or an infinity in the row leaves `ss` not finite and the scale NaN (infinity times a root of 0, or NaN)
  const float s = ss < INFINITY ? most.hi * rsqrtf(ss / (float)dim + eps) / E4M3_MAX : NAN;
  const bool none = s < LEAST || most.hi < 0x1p-110f;  // below 2^-110 the reciprocal would overflow
  const float inv = none ? 0.f : (s == s ? E4M3_MAX / most.hi : NAN);
  const double exact = (double)most.hi + (double)most.lo;
#pragma unroll KEPT
  for (int j = 0; j < runs; ++j) {
    const int c0 = 8 * (threadIdx.x + j * blockDim.x);
    float *xs = x[RUNS > 0 ? j : 0], *gs = g[RUNS > 0 ? j : 0];
    if (RUNS == 0) {
      if (del && rows == nullptr) load_run(res, c0, dim, vec_x, xs);  // as this thread has stored it
      else load_sum(c0, xs);
      load_run(gain, c0, dim, vec_g, gs);
    }
    if (c0 < pitch && FMS_IN((size_t)blockIdx.x * pitch + c0 + 7, (size_t)n_rows * pitch))
      *reinterpret_cast<uint2*>(q + (size_t)blockIdx.x * pitch + c0) = ended(quotients<true>(xs, gs, inv, exact), c0, dim);
  }
  if (threadIdx.x == 0) scales[blockIdx.x] = none ? 0.f : s;
}

// Threads for a row of `runs` runs of 8, and the runs that each keeps (0: too wide for registers).  Few rows: a thread a run
// as far as 1,024 go, since only latency counts; many: fewer threads with more runs each, so that more rows are in flight.
int threads_for(int runs, int n_rows, int each, int* kept) {
  int threads = 64;
  while (threads < 1024 && threads * (n_rows <= 296 ? 1 : each) < runs) threads *= 2;
  const int k = (runs + threads - 1) / threads;
  *kept = k <= 2 ? k : (k <= 4 && each == 4 ? 4 : 0);
  return threads;
}
bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

template <typename T, int RUNS>
void launch_rows(int threads, const void* x, uint8_t* q, float* scales, int n_rows, int dim, int pitch, cudaStream_t stream) {
  fms_launch(quantize_rows_kernel<T, RUNS>, dim3(n_rows), dim3(threads), 0, stream, (const T*)x, q, scales, n_rows, dim, pitch,
             (int)(dim % (16 / (int)sizeof(T)) == 0 && aligned16(x)));
}
template <typename T> int quantize(const void* x, uint8_t* q, float* scales, int n_rows, int dim, int pitch, cudaStream_t stream) {
  int kept;
  const int threads = threads_for(pitch / 8, n_rows, 4, &kept);
  (kept == 1 ? launch_rows<T, 1> : kept == 2 ? launch_rows<T, 2> : kept == 4 ? launch_rows<T, 4> : launch_rows<T, 0>)(
      threads, x, q, scales, n_rows, dim, pitch, stream);
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
template <typename T, typename TG, int RUNS> void launch_norm(int threads, const NormArgs& a, cudaStream_t stream) {
  fms_launch(add_rmsnorm_quantized_kernel<T, TG, RUNS>, dim3(a.n_rows), dim3(threads), 0, stream, a.residual, (const T*)a.delta,
             (const TG*)a.gain, a.eps, a.q, a.scales, a.rows, a.n_rows, a.dim, a.pitch, a.residual_rows,
             (int)(a.dim % 4 == 0 && aligned16(a.residual)), (int)(a.dim % (16 / (int)sizeof(T)) == 0 && aligned16(a.delta)),
             (int)(a.dim % (16 / (int)sizeof(TG)) == 0 && aligned16(a.gain)));
}
template <typename T, typename TG> int norm(const NormArgs& a, cudaStream_t stream) {
  int kept;
  const int threads = threads_for(a.pitch / 8, a.n_rows, 2, &kept);
  (kept == 1 ? launch_norm<T, TG, 1> : kept == 2 ? launch_norm<T, TG, 2> : launch_norm<T, TG, 0>)(threads, a, stream);
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
