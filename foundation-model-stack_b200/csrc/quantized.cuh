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
