// What the kernels of the linear layer share: activations and their slopes,
// the epilogue of the forward product, and the entry points of the
// tensor-core translation unit.
#pragma once

#include "vcb_common.cuh"
#include "vcb_types.cuh"

namespace vcb {
namespace lin {

// act(z), in fp32.
__device__ __forceinline__ float act_value(float z, int act) {
  switch (act) {
    case VCB_ACT_RELU: return z < 0.f ? 0.f : z;  // NaN stays
    case VCB_ACT_GELU: return 0.5f * z * (1.f + erff(z * 0.70710678118654752f));
    case VCB_ACT_SILU: return z / (1.f + expf(-z));
    default: return z;
  }
}

// act'(z), in fp32; ReLU's slope at 0 is 0.
__device__ __forceinline__ float act_slope(float z, int act) {
  switch (act) {
    case VCB_ACT_RELU: return z > 0.f ? 1.f : 0.f;
    case VCB_ACT_GELU:
      return 0.5f * (1.f + erff(z * 0.70710678118654752f)) +
             z * expf(-0.5f * z * z) * 0.39894228040143268f;
    case VCB_ACT_SILU: {
      const float g = 1.f / (1.f + expf(-z));
      return g * (1.f + z * (1.f - g));
    }
    default: return 1.f;
  }
}

// dz = dy act'(z); a ReLU that is off passes nothing, not even NaN.
__device__ __forceinline__ float act_grad(float dy, float z, int act) {
  if (act == VCB_ACT_NONE) return dy;
  if (act == VCB_ACT_RELU) return z > 0.f ? dy : 0.f;
  return dy * act_slope(z, act);
}

struct Fwd {
  int M, N, K, type, act;
  long long ldx, ldw, ldr, ldy, ldz;
  const void *x, *w, *bias, *res;
  void *y, *z;
};

struct Bwd {
  int M, N, K, type, act;
  long long lddy, ldx, ldw, ldz, lddx, lddw;
  const void *dy, *x, *w, *z;
  void *dx, *dw, *db;
};

}  // namespace lin
}  // namespace vcb
