// Linear layer with its epilogue, and its gradients.
//
//   Z = X W^T + b,  Y = act(Z) + R                 X (M x K), W (N x K)
//   dZ = dY * act'(Z),  dX = dZ W,  dW = dZ^T X,  db = sum_m dZ_m
//
// This file has the kernel for small products and the entry points.  Both
// gradients (and db) of a small layer leave in one launch.
//
// Small products are bound by latency: a 32 x 64 tile per CTA of 512 threads,
// four groups of 128 threads each taking a quarter of every 64-deep step of
// the contraction (16 warps hide each other's loads), added in order at the
// end.  Accumulation is in fp32 whatever the type.
#include "vcb_linear.cuh"

#include <algorithm>

namespace vcb {
namespace lin {
namespace {

constexpr int kTI = 32, kTJ = 64, kTT = 64;  // tile rows, columns, contraction step
constexpr int kGroups = 4, kSmallThreads = 128 * kGroups;
constexpr int kPitchA = kTI + 4, kPitchB = kTJ + 4;

// One product out(i, j) = sum_t A(i, t) B(t, j) of a launch, and where its
// tiles start in the grid.
struct Small {
  int I, J, T;
  const void *a, *a2, *b;  // a2: pre-activation beside the gradient a, or NULL
  long long lda, lda2, ldb;
  int a_t, b_t;  // the contraction index is the contiguous one
  int act;
  void *out, *sum, *z;  // sum: row sums of A (db), or NULL
  long long ldo, ldz, ldr;
  const void *bias, *res;
  int epilogue;  // apply bias, act and res
  int tiles_j, tiles;
};

struct SmallPair {
  Small p[2];
};

template <typename T>
__device__ __forceinline__ float a_value(const Small& s, int i, int t) {
  if (i >= s.I || t >= s.T) return 0.f;
  const long long r = s.a_t ? i : t, c = s.a_t ? t : i;
  const float v = to_f32(static_cast<const T*>(s.a)[r * s.lda + c]);
  if (!s.a2) return v;
  return act_grad(v, to_f32(static_cast<const T*>(s.a2)[r * s.lda2 + c]), s.act);
}

template <typename T>
__device__ __forceinline__ float b_value(const Small& s, int t, int j) {
  if (j >= s.J || t >= s.T) return 0.f;
  const long long at = s.b_t ? static_cast<long long>(j) * s.ldb + t
                             : static_cast<long long>(t) * s.ldb + j;
  return to_f32(static_cast<const T*>(s.b)[at]);
}

template <typename T>
__global__ void __launch_bounds__(kSmallThreads) small_kernel(const __grid_constant__ SmallPair pair) {
  constexpr int kStageA = kTT * kPitchA, kStageB = kTT * kPitchB;
  constexpr int kJoin = (kGroups - 1) * 128 * 16;
  __shared__ float buf[kStageA + kStageB > kJoin ? kStageA + kStageB : kJoin];
  __shared__ float row_sum[kGroups][kTI];
  float *sa = buf, *sb = buf + kStageA;
  const int second = static_cast<int>(blockIdx.x) >= pair.p[0].tiles;
  const Small& s = pair.p[second];
  const int tile = blockIdx.x - (second ? pair.p[0].tiles : 0);
  const int i0 = tile / s.tiles_j * kTI, j0 = tile % s.tiles_j * kTJ;
  const int tid = threadIdx.x, group = tid >> 7, in = tid & 127;
  const int ty = in >> 4, tx = in & 15;
  constexpr int NA = kTI * kTT / kSmallThreads, NB = kTJ * kTT / kSmallThreads;
  float ra[NA], rb[NB];
  // neighbouring threads read neighbouring elements, whichever index they run over
  auto fetch = [&](int t0) {
#pragma unroll
    for (int k = 0; k < NA; ++k) {
      const int e = tid + k * kSmallThreads;
      const int i = s.a_t ? e / kTT : e % kTI, t = s.a_t ? e % kTT : e / kTI;
      ra[k] = a_value<T>(s, i0 + i, t0 + t);
    }
#pragma unroll
    for (int k = 0; k < NB; ++k) {
      const int e = tid + k * kSmallThreads;
      const int j = s.b_t ? e / kTT : e % kTJ, t = s.b_t ? e % kTT : e / kTJ;
      rb[k] = b_value<T>(s, t0 + t, j0 + j);
    }
  };
  float acc[4][4] = {}, rs[4] = {};
  const bool sums = s.sum && j0 == 0 && tx == 0;
  fetch(0);
  for (int t0 = 0; t0 < s.T; t0 += kTT) {
    __syncthreads();
#pragma unroll
    for (int k = 0; k < NA; ++k) {
      const int e = tid + k * kSmallThreads;
      const int i = s.a_t ? e / kTT : e % kTI, t = s.a_t ? e % kTT : e / kTI;
      sa[t * kPitchA + i] = ra[k];
    }
#pragma unroll
    for (int k = 0; k < NB; ++k) {
      const int e = tid + k * kSmallThreads;
      const int j = s.b_t ? e / kTT : e % kTJ, t = s.b_t ? e % kTT : e / kTJ;
      sb[t * kPitchB + j] = rb[k];
    }
    __syncthreads();
    if (t0 + kTT < s.T) fetch(t0 + kTT);
#pragma unroll
    for (int k = 0; k < kTT / kGroups; ++k) {
      const int t = group * (kTT / kGroups) + k;
      const float4 av = *reinterpret_cast<const float4*>(sa + t * kPitchA + ty * 4);
      const float4 bv = *reinterpret_cast<const float4*>(sb + t * kPitchB + tx * 4);
      const float a4[4] = {av.x, av.y, av.z, av.w}, b4[4] = {bv.x, bv.y, bv.z, bv.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(a4[i], b4[j], acc[i][j]);
        if (sums) rs[i] += a4[i];
      }
    }
  }
  __syncthreads();
  if (group > 0) {
#pragma unroll
    for (int i = 0; i < 16; ++i) buf[((group - 1) * 16 + i) * 128 + in] = acc[i >> 2][i & 3];
  }
  if (sums) {
#pragma unroll
    for (int i = 0; i < 4; ++i) row_sum[group][ty * 4 + i] = rs[i];
  }
  __syncthreads();
  if (s.sum && j0 == 0 && tid < kTI && i0 + tid < s.I) {
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < kGroups; ++k) v += row_sum[k][tid];
    static_cast<T*>(s.sum)[i0 + tid] = from_f32<T>(v);
  }
  if (group > 0 || !s.out) return;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const long long r = i0 + ty * 4 + i;
    if (r >= s.I) break;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = j0 + tx * 4 + j;
      if (c >= s.J) break;
      float v = acc[i][j];
#pragma unroll
      for (int k = 0; k < kGroups - 1; ++k) v += buf[(k * 16 + i * 4 + j) * 128 + in];
      if (s.epilogue) {
        if (s.bias) v += to_f32(static_cast<const T*>(s.bias)[c]);
        if (s.z) static_cast<T*>(s.z)[r * s.ldz + c] = from_f32<T>(v);
        v = act_value(v, s.act);
        if (s.res) v += to_f32(static_cast<const T*>(s.res)[r * s.ldr + c]);
      }
      static_cast<T*>(s.out)[r * s.ldo + c] = from_f32<T>(v);
    }
  }
}

int tiles_of(Small& s) {
  if (!s.sum && (!s.out || s.J == 0)) return s.tiles = 0;
  s.tiles_j = s.out ? std::max(1, (s.J + kTJ - 1) / kTJ) : 1;
  const long long n = static_cast<long long>((s.I + kTI - 1) / kTI) * s.tiles_j;
  s.tiles = n > 0x3fffffff ? -1 : static_cast<int>(n);
  return s.tiles;
}

int launch_small(const SmallPair& pair, int type, cudaStream_t st, const char* who) {
  if (pair.p[0].tiles < 0 || pair.p[1].tiles < 0)
    return fail(VCB_ERR_UNSUPPORTED, "%s: too many output tiles", who);
  const unsigned grid = pair.p[0].tiles + pair.p[1].tiles;
  if (grid == 0) return VCB_OK;
  if (type == VCB_F32)
    small_kernel<float><<<grid, kSmallThreads, 0, st>>>(pair);
  else if (type == VCB_BF16)
    small_kernel<__nv_bfloat16><<<grid, kSmallThreads, 0, st>>>(pair);
  else
    small_kernel<__half><<<grid, kSmallThreads, 0, st>>>(pair);
  return check_launch(who);
}

int small_forward(const Fwd& f, cudaStream_t st) {
  SmallPair pair{};
  Small& s = pair.p[0];
  s.I = f.M, s.J = f.N, s.T = f.K;
  s.a = f.x, s.lda = f.ldx, s.a_t = 1;
  s.b = f.w, s.ldb = f.ldw, s.b_t = 1;
  s.act = f.act, s.out = f.y, s.ldo = f.ldy, s.z = f.z, s.ldz = f.ldz;
  s.bias = f.bias, s.res = f.res, s.ldr = f.ldr, s.epilogue = 1;
  tiles_of(s);
  return launch_small(pair, f.type, st, "vcb_linear_forward");
}

int small_backward(const Bwd& b, cudaStream_t st) {
  SmallPair pair{};
  const void* z = b.act == VCB_ACT_NONE ? nullptr : b.z;
  Small& x = pair.p[0];
  x.I = b.M, x.J = b.K, x.T = b.N;
  x.a = b.dy, x.lda = b.lddy, x.a2 = z, x.lda2 = b.ldz, x.a_t = 1, x.act = b.act;
  x.b = b.w, x.ldb = b.ldw, x.b_t = 0;
  x.out = b.dx, x.ldo = b.lddx;
  if (b.dx) tiles_of(x);
  Small& w = pair.p[1];
  w.I = b.N, w.J = b.K, w.T = b.M;
  w.a = b.dy, w.lda = b.lddy, w.a2 = z, w.lda2 = b.ldz, w.a_t = 0, w.act = b.act;
  w.b = b.x, w.ldb = b.ldx, w.b_t = 0;
  w.out = b.dw, w.ldo = b.lddw, w.sum = b.db;
  if (b.dw || b.db) tiles_of(w);
  return launch_small(pair, b.type, st, "vcb_linear_backward");
}

}  // namespace
}  // namespace lin

namespace {
bool misaligned(const void* p, int type) {
  return reinterpret_cast<uintptr_t>(p) % dtype_bytes(type) != 0;
}
}  // namespace
}  // namespace vcb

using namespace vcb;

extern "C" size_t vcb_linear_forward_workspace(int32_t M, int32_t N, int32_t K, int32_t type,
                                               int32_t rows16) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  if (type == VCB_F32) return lin::f32_forward_bytes(M, N, K);
  return rows16 ? 0 : lin::tc_forward_bytes(M, N, K);
}

extern "C" size_t vcb_linear_backward_workspace(int32_t M, int32_t N, int32_t K, int32_t type,
                                                int32_t act, int32_t rows16) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  if (type == VCB_F32) return lin::f32_backward_bytes(M, N, K);
  return lin::tc_backward_bytes(M, N, K, act, rows16);
}

static int check_workspace(const void* ws, size_t have, size_t need, const char* who) {
  if (need == 0 || (ws && have >= need && reinterpret_cast<uintptr_t>(ws) % 16 == 0)) return VCB_OK;
  return fail(VCB_ERR_INVALID, "%s: workspace of %zu bytes, %zu needed", who, have, need);
}

static bool rows16(const void* p, int64_t ld, int type) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * dtype_bytes(type) % 16 == 0;
}

extern "C" int vcb_linear_forward(int32_t M, int32_t N, int32_t K, int32_t type, const void* x,
                                  int64_t ldx, const void* w, int64_t ldw, const void* bias,
                                  int32_t act, const void* residual, int64_t ldr, void* y,
                                  int64_t ldy, void* z, int64_t ldz, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  if (M < 0 || N < 0 || K < 0 || !valid_dtype(type) || act < VCB_ACT_NONE || act > VCB_ACT_SILU ||
      ldx < K || ldw < K || ldy < N || (residual && ldr < N) || (z && ldz < N))
    return fail(VCB_ERR_INVALID, "vcb_linear_forward: M=%d N=%d K=%d type=%d act=%d", M, N, K,
                type, act);
  if (M == 0 || N == 0) return VCB_OK;
  if (!y || (K > 0 && (!x || !w)) || misaligned(x, type) || misaligned(w, type) ||
      misaligned(bias, type) || misaligned(residual, type) || misaligned(y, type) ||
      misaligned(z, type))
    return fail(VCB_ERR_INVALID, "vcb_linear_forward: NULL or misaligned pointer");
  const lin::Fwd f{M, N, K, type, act, ldx, ldw, ldr, ldy, ldz, x, w, bias, residual, y, z};
  const bool f32 = lin::f32_forward_fits(f);
  if (!f32 && !lin::tc_forward_fits(f)) return lin::small_forward(f, static_cast<cudaStream_t>(stream));
  const int rc = check_workspace(workspace, workspace_bytes,
                                 vcb_linear_forward_workspace(
                                     M, N, K, type, rows16(x, ldx, type) && rows16(w, ldw, type)),
                                 "vcb_linear_forward");
  if (rc) return rc;
  return (f32 ? lin::f32_forward : lin::tc_forward)(f, workspace, static_cast<cudaStream_t>(stream));
}

extern "C" int vcb_linear_backward(int32_t M, int32_t N, int32_t K, int32_t type, const void* dy,
                                   int64_t lddy, const void* x, int64_t ldx, const void* w,
                                   int64_t ldw, const void* z, int64_t ldz, int32_t act, void* dx,
                                   int64_t lddx, void* dw, int64_t lddw, void* db, void* workspace,
                                   size_t workspace_bytes, void* stream) {
  if (M < 0 || N < 0 || K < 0 || !valid_dtype(type) || act < VCB_ACT_NONE || act > VCB_ACT_SILU ||
      lddy < N || (dw && (ldx < K || lddw < K)) || (dx && (ldw < K || lddx < K)) ||
      (act != VCB_ACT_NONE && ldz < N))
    return fail(VCB_ERR_INVALID, "vcb_linear_backward: M=%d N=%d K=%d type=%d act=%d", M, N, K,
                type, act);
  const bool inputs = M > 0 && N > 0;
  if ((inputs && (!dy || (act != VCB_ACT_NONE && !z) || (K > 0 && ((dx && !w) || (dw && !x))))) ||
      misaligned(dy, type) || misaligned(x, type) || misaligned(w, type) || misaligned(z, type) ||
      misaligned(dx, type) || misaligned(dw, type) || misaligned(db, type))
    return fail(VCB_ERR_INVALID, "vcb_linear_backward: NULL or misaligned pointer");
  const lin::Bwd b{M, N, K, type, act, lddy, ldx, ldw, ldz, lddx, lddw, dy, x, w, z, dx, dw, db};
  const bool f32 = lin::f32_backward_fits(b);
  if (!f32 && !lin::tc_backward_fits(b)) return lin::small_backward(b, static_cast<cudaStream_t>(stream));
  const int rc = check_workspace(workspace, workspace_bytes,
                                 vcb_linear_backward_workspace(
                                     M, N, K, type, act,
                                     rows16(dy, lddy, type) && rows16(x, ldx, type) &&
                                         rows16(w, ldw, type)),
                                 "vcb_linear_backward");
  if (rc) return rc;
  return (f32 ? lin::f32_backward : lin::tc_backward)(b, workspace,
                                                      static_cast<cudaStream_t>(stream));
}
