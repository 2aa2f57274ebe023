// What the kernels of the linear layer share: activations and their slopes,
// the epilogue of the forward product, and the entry points of the
// tensor-core translation unit.
#pragma once

#include <type_traits>

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

// The same for many values, the choice of act outside of their loop.
template <int ACT, int N>
__device__ __forceinline__ void act_grad_all(float (&dy)[N], const float (&z)[N]) {
#pragma unroll
  for (int k = 0; k < N; ++k) dy[k] = act_grad(dy[k], z[k], ACT);
}

template <int N>
__device__ __forceinline__ void act_grads(float (&dy)[N], const float (&z)[N], int act) {
  switch (act) {
    case VCB_ACT_RELU: act_grad_all<VCB_ACT_RELU>(dy, z); break;
    case VCB_ACT_GELU: act_grad_all<VCB_ACT_GELU>(dy, z); break;
    case VCB_ACT_SILU: act_grad_all<VCB_ACT_SILU>(dy, z); break;
    default: break;
  }
}

// Where a product's rows go and what is done to them on the way.
struct Epilogue {
  void *out, *z;
  const void *bias, *res;
  long long ldo, ldz, ldr;
  int act;
  int vec;  // out, z and res take 4-element vectors
};

inline bool vector_rows(const Epilogue& e, int elem) {
  const auto ok = [&](const void* p, long long ld) {
    return !p || (reinterpret_cast<uintptr_t>(p) % (4 * elem) == 0 && ld % 4 == 0);
  };
  return ok(e.out, e.ldo) && ok(e.z, e.ldz) && ok(e.res, e.ldr);
}

template <int ACT, int N>
__device__ __forceinline__ void act_all(float (&v)[N]) {
#pragma unroll
  for (int c = 0; c < N; ++c) v[c] = act_value(v[c], ACT);
}

// Bias of the columns j .. j + 3.
template <typename T>
__device__ __forceinline__ void bias_at(const Epilogue& e, int J, int j, float (&b)[4]) {
#pragma unroll
  for (int k = 0; k < 4; ++k)
    b[k] = e.bias && j + k < J ? to_f32(static_cast<const T*>(e.bias)[j + k]) : 0.f;
}

// v[c] of lane l: column c of row l.  Afterwards v[4 q + k] is column 4 q + l % 4
// of row (l - l % 4) + k: four lanes have traded 4 x 4 blocks.
template <int N>
__device__ __forceinline__ void transpose4(float (&v)[N], int lane) {
  const bool odd = lane & 1, high = lane & 2;
#pragma unroll
  for (int q = 0; q < N; q += 4) {
#pragma unroll
    for (int k = 0; k < 4; k += 2) {
      const float got = __shfl_xor_sync(0xffffffffu, odd ? v[q + k] : v[q + k + 1], 1);
      if (odd) v[q + k] = got; else v[q + k + 1] = got;
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const float got = __shfl_xor_sync(0xffffffffu, high ? v[q + k] : v[q + k + 2], 2);
      if (high) v[q + k] = got; else v[q + k + 2] = got;
    }
  }
}

// Four elements of a row at column j, as they lie.
template <typename T>
struct Four {
  typename std::conditional<sizeof(T) == 4, float4, uint2>::type raw;
};

// Residuals of the rows i, i + 4, .. (N of them), columns j .. j + 3.  Fetched ahead
// of the chunk that adds them: their way from HBM would otherwise be waited for in
// every chunk.
template <typename T, int N>
struct Residual {
  Four<T> v[N];
  __device__ __forceinline__ void fetch(const Epilogue& e, int I, int J, int i, int j) {
    if (!e.res || j >= J) return;
    const bool vec = e.vec && j + 4 <= J;
#pragma unroll
    for (int q = 0; q < N; ++q) {
      if (i + 4 * q >= I) break;
      const T* at = static_cast<const T*>(e.res) + (i + 4 * q) * e.ldr + j;
      if (vec) {
        v[q].raw = __ldcs(reinterpret_cast<const decltype(v[q].raw)*>(at));
      } else {
        T t[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) t[k] = j + k < J ? at[k] : from_f32<T>(0.f);
        v[q].raw = *reinterpret_cast<const decltype(v[q].raw)*>(t);
      }
    }
  }
  __device__ __forceinline__ void add(float (&out)[4 * N]) const {
#pragma unroll
    for (int q = 0; q < N; ++q) {
      T t[4];
      *reinterpret_cast<decltype(v[q].raw)*>(t) = v[q].raw;
#pragma unroll
      for (int k = 0; k < 4; ++k) out[4 * q + k] += to_f32(t[k]);
    }
  }
};

// Rows i, i + 4, .. (N of them), columns j .. j + 3 of the output: bias,
// pre-activation, act, residual, one rounding.
template <typename T, int N>
__device__ __forceinline__ void emit(const Epilogue& e, int I, int J, int i, int j,
                                     const float (&bias)[4], float (&v)[4 * N],
                                     const Residual<T, N>& res) {
  if (j >= J) return;
  const bool vec = e.vec && j + 4 <= J;
  const auto put = [&](void* base, long long ld) {
#pragma unroll
    for (int q = 0; q < N; ++q) {
      if (i + 4 * q >= I) break;
      T* at = static_cast<T*>(base) + (i + 4 * q) * ld + j;
      if (vec) {
        store4_stream(at, {v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]});
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (j + k < J) at[k] = from_f32<T>(v[4 * q + k]);
      }
    }
  };
#pragma unroll
  for (int c = 0; c < 4 * N; ++c) v[c] += bias[c & 3];
  if (e.z) put(e.z, e.ldz);
  switch (e.act) {
    case VCB_ACT_RELU: act_all<VCB_ACT_RELU>(v); break;
    case VCB_ACT_GELU: act_all<VCB_ACT_GELU>(v); break;
    case VCB_ACT_SILU: act_all<VCB_ACT_SILU>(v); break;
    default: break;
  }
  if (e.res) res.add(v);
  put(e.out, e.ldo);
}

// Residuals of N consecutive rows from i of column j.
template <typename T, int N>
struct ColumnResidual {
  T v[N];
  __device__ __forceinline__ void fetch(const Epilogue& e, int I, int J, int i, int j) {
    if (!e.res || j >= J) return;
    const T* at = static_cast<const T*>(e.res) + i * e.ldr + j;
#pragma unroll
    for (int c = 0; c < N; ++c)
      if (i + c < I) v[c] = __ldcs(at + c * e.ldr);
  }
};

// N consecutive rows from i of column j.
template <typename T, int N>
__device__ __forceinline__ void emit_column(const Epilogue& e, int I, int J, int i, int j,
                                            float bias, float (&v)[N],
                                            const ColumnResidual<T, N>& res) {
  const int n = min(N, I - i);
  if (j >= J || n <= 0) return;
#pragma unroll
  for (int c = 0; c < N; ++c) v[c] += bias;
  if (e.z) {
    T* at = static_cast<T*>(e.z) + i * e.ldz + j;
#pragma unroll
    for (int c = 0; c < N; ++c)
      if (c < n) __stcs(at + c * e.ldz, from_f32<T>(v[c]));
  }
  switch (e.act) {
    case VCB_ACT_RELU: act_all<VCB_ACT_RELU>(v); break;
    case VCB_ACT_GELU: act_all<VCB_ACT_GELU>(v); break;
    case VCB_ACT_SILU: act_all<VCB_ACT_SILU>(v); break;
    default: break;
  }
  T* at = static_cast<T*>(e.out) + i * e.ldo + j;
#pragma unroll
  for (int c = 0; c < N; ++c)
    if (c < n) __stcs(at + c * e.ldo, from_f32<T>(e.res ? v[c] + to_f32(res.v[c]) : v[c]));
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

// Up to kFewRows rows (vcb_linear_rows.cu): M, N, K > 0.
constexpr int kFewRows = 16;
int rows_forward(const Fwd& f, cudaStream_t st);
int rows_backward(const Bwd& b, cudaStream_t st);

// Tensor-core paths (vcb_linear_tc.cu: 16-bit types; vcb_linear_f32.cu).  `bytes`: what they need
// of the workspace; the launch functions take one that large, 16-byte aligned.
bool tc_forward_fits(const Fwd& f);
size_t tc_forward_bytes(int M, int N, int K);
int tc_forward(const Fwd& f, void* ws, cudaStream_t st);
bool tc_backward_fits(const Bwd& b);
size_t tc_backward_bytes(int M, int N, int K, int act, bool rows16);
int tc_backward(const Bwd& b, void* ws, cudaStream_t st);
int tc_path(int M, int N, int K, int product);  // as vcb_linear_path, sizes that fit

bool f32_forward_fits(const Fwd& f);
size_t f32_forward_bytes(int M, int N, int K);
int f32_forward(const Fwd& f, void* ws, cudaStream_t st);
bool f32_backward_fits(const Bwd& b);
size_t f32_backward_bytes(int M, int N, int K);
int f32_backward(const Bwd& b, void* ws, cudaStream_t st);
int f32_path(int M, int N, int K, int product);

}  // namespace lin

}  // namespace vcb
