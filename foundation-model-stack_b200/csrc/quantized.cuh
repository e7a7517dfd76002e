// What the products with quantised weights share.  Included inside the anonymous namespace of the kernels that use it, after common.cuh.
#pragma once

// [N] bfloat16 or float32, or none: added to the float32 sums as it is
struct Bias {
  const void* values;
  int f32;
  __device__ __forceinline__ explicit operator bool() const { return values != nullptr; }
  __device__ __forceinline__ float operator[](int i) const {
    return f32 ? static_cast<const float*>(values)[i] : __bfloat162float(static_cast<const __nv_bfloat16*>(values)[i]);
  }
};
int check_bias(const char* what, const Bias& bias, int dtype) {
  return bias.values && dtype != FMS_F32 && dtype != FMS_BF16 ? fms_fail("%s: bias of dtype code %d", what, dtype) : 0;
}

__device__ __forceinline__ float activate(float g, int act) {
  switch (act) {
    case 0: return g / (1.f + expf(-g));
    case 1: return 0.5f * g * (1.f + erff(g * 0.70710678118654752f));
    case 2: return 0.5f * g * (1.f + tanhf(0.7978845608028654f * (g + 0.044715f * g * g * g)));
    default: return fmaxf(g, 0.f);
  }
}

int multiprocessors() {
  static int sms = 0;
  if (sms == 0) {
    int device = 0;
    cudaGetDevice(&device);
    if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess || sms <= 0) sms = 148;
  }
  return sms;
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

// The run of steps of block b of `blocks`: [first_step(b), first_step(b + 1)); and the block of a step
__host__ __device__ inline int first_step(int b, int blocks, int steps) { return (int)((long)b * steps / blocks); }
__device__ __forceinline__ int block_of_step(int step, int blocks, int steps) { return (int)((((long)step + 1) * blocks - 1) / steps); }
