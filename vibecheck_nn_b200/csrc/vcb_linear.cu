// Linear layer with its epilogue, and its gradients.
//
//   Z = X W^T + b,  Y = act(Z) + R                 X (M x K), W (N x K)
//   dZ = dY * act'(Z),  dX = dZ W,  dW = dZ^T X,  db = sum_m dZ_m
//
// This file has the kernel for small products and the entry points.  Both
// gradients (and db) of a small layer leave in one launch.
//
// Small products are bound by latency, so a product of few tiles is spread as wide
// as it goes: a 32 x 32 tile per CTA of 256 threads, four groups of 64 threads each
// taking every fourth chunk of every 64-deep step of the contraction, and the contraction cut
// over up to 8 CTAs of a cluster when there are few tiles.  Groups are joined through
// shared memory and CTAs through distributed shared memory, in order.  Operands lie
// in shared memory by row, four entries of the contraction to a 16-byte chunk, chunks
// XOR-ed with the row: writes and reads are free of bank conflicts whichever index of
// the operand is contiguous.  A thread owns rows and columns 8 apart.  Accumulation is
// in fp32 whatever the type.
//
// Measured with cold inputs, launch included: fp32 100 x 256 x 784, both gradients and
// db, 16 us (its bytes take 0.4 us: what is left are the launch, two trips to memory
// in turn and the cluster's join), bf16 2000 x 63 x 63 forward 11 us.
#include <algorithm>
#include <initializer_list>

#include "vcb_linear_tc.cuh"

namespace vcb {
namespace lin {
namespace {

constexpr int kTI = 32, kTJ = 32, kTT = 64;  // tile rows, columns, contraction step
constexpr int kTile = kTI * kTJ;
constexpr int kGroups = 4, kSmallThreads = 64 * kGroups;

// One product out(i, j) = sum_t A(i, t) B(t, j) of a launch, and where its
// tiles start in the grid.
struct Small {
  int I, J, T;
  const void *a, *a2, *b;  // a2: pre-activation beside the gradient a, or NULL
  long long lda, lda2, ldb;
  int a_t, b_t;      // the contraction index is the contiguous one
  int va, vb;        // ... and four of its entries are a vector
  int act;
  void* sum;         // row sums of A (db), or NULL
  Epilogue epi;      // out may be NULL
  int tiles_j, tiles;
  int parts;         // CTAs per tile, each with a part of the contraction; a power of 2
  int clusters;
};

struct SmallPair {
  Small p[2];
  int size;  // of a cluster: the larger number of parts
};

// Entries t .. t + 3 of a row: `step` elements apart, `left` of them exist.  Kept as
// loaded until they are used: a conversion would wait for them, and loads follow.
template <typename T>
struct Quad {
  T e[4];
  __device__ __forceinline__ void load(const T* p, long long step, bool vec, int left) {
    using V = decltype(Four<T>::raw);
    if (vec && left >= 4) {
      *reinterpret_cast<V*>(e) = *reinterpret_cast<const V*>(p);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) e[k] = k < left ? p[k * step] : from_f32<T>(0.f);
    }
  }
  __device__ __forceinline__ void values(float (&v)[4]) const {
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = to_f32(e[k]);
  }
};

__device__ __forceinline__ int chunk_at(int row, int chunk) {
  return row * kTT + ((chunk ^ (row & 7)) << 2);
}

// CTAS per SM: three have fewer registers and shorter loops each.
template <typename T, int CTAS>
__global__ void __launch_bounds__(kSmallThreads, CTAS)
    small_kernel(const __grid_constant__ SmallPair pair) {
  // operands of a step; then the groups' sums; then this CTA's sum of the tile
  __shared__ __align__(16) float buf[(kTI + kTJ) * kTT > kGroups * kTile ? (kTI + kTJ) * kTT
                                                                        : kGroups * kTile];
  __shared__ float row_sum[kTT / 4][kTI], row_mine[kTI];
  float *sa = buf, *sb = buf + kTI * kTT;
  const int cluster = blockIdx.x / pair.size, rank = blockIdx.x % pair.size;
  const int second = cluster >= pair.p[0].clusters;
  const Small& s = pair.p[second];
  const int parts = s.parts, lg = 31 - __clz(parts), part = rank & (parts - 1);
  // a cluster of more CTAs than parts holds several tiles; the last may hold none,
  // whose rows lie beyond I
  const int tile = (cluster - (second ? pair.p[0].clusters : 0)) * (pair.size >> lg) + (rank >> lg);
  const int i0 = tile / s.tiles_j * kTI, j0 = tile % s.tiles_j * kTJ;
  const int tid = threadIdx.x, group = tid >> 6, in = tid & 63, ty = in >> 3, tx = in & 7;
  const int steps = (s.T + kTT - 1) / kTT;
  const int s0 = steps * part >> lg, s1 = i0 < s.I ? steps * (part + 1) >> lg : s0;
  // this thread's two quads of A and of B: lanes run along the contiguous index
  const auto row_of = [&](int contiguous_t, int q) {
    return contiguous_t ? (tid >> 4) + 16 * q : tid & 31;
  };
  const auto chunk_of = [&](int contiguous_t, int q) {
    return contiguous_t ? tid & 15 : (tid >> 5) + 8 * q;
  };
  const long long ta = s.a_t ? 1 : s.lda, ta2 = s.a_t ? 1 : s.lda2, tb = s.b_t ? 1 : s.ldb;
  const T *pa[2], *pa2[2], *pb[2];
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int ra = i0 + row_of(s.a_t, q), ca = (s0 * 16 + chunk_of(s.a_t, q)) * 4;
    const int rb = j0 + row_of(s.b_t, q), cb = (s0 * 16 + chunk_of(s.b_t, q)) * 4;
    pa[q] = static_cast<const T*>(s.a) + (s.a_t ? ra * s.lda : ra) + ca * ta;
    pa2[q] = static_cast<const T*>(s.a2) + (s.a_t ? ra * s.lda2 : ra) + ca * ta2;
    pb[q] = static_cast<const T*>(s.b) + (s.b_t ? rb * s.ldb : rb) + cb * tb;
  }
  Quad<T> qa[2], qz[2], qb[2];
  const auto fetch = [&](int step) {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int la = i0 + row_of(s.a_t, q) < s.I ? s.T - (step * 16 + chunk_of(s.a_t, q)) * 4 : 0;
      qa[q].load(pa[q], ta, s.va, la);
      pa[q] += kTT * ta;
      if (s.a2) {
        qz[q].load(pa2[q], ta2, s.va, la);
        pa2[q] += kTT * ta2;
      }
      qb[q].load(pb[q], tb, s.vb,
                 j0 + row_of(s.b_t, q) < s.J ? s.T - (step * 16 + chunk_of(s.b_t, q)) * 4 : 0);
      pb[q] += kTT * tb;
    }
  };
  float acc[4][4] = {}, rs = 0.f;
  const bool sums = s.sum && j0 == 0;
  if (s0 < s1) fetch(s0);
  for (int step = s0; step < s1; ++step) {
    __syncthreads();
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      float v[4];
      qa[q].values(v);
      if (s.a2) {
        float z[4];
        qz[q].values(z);
        act_grads(v, z, s.act);
      }
      *reinterpret_cast<float4*>(sa + chunk_at(row_of(s.a_t, q), chunk_of(s.a_t, q))) =
          make_float4(v[0], v[1], v[2], v[3]);
      qb[q].values(v);
      *reinterpret_cast<float4*>(sb + chunk_at(row_of(s.b_t, q), chunk_of(s.b_t, q))) =
          make_float4(v[0], v[1], v[2], v[3]);
    }
    __syncthreads();
    if (step + 1 < s1) fetch(step + 1);
    if (sums) {
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const float4 v =
            *reinterpret_cast<const float4*>(sa + chunk_at(tid & 31, (tid >> 5) + 8 * q));
        rs += (v.x + v.y) + (v.z + v.w);
      }
    }
    const int chunks = min(kTT / 4, (s.T - step * kTT + 3) / 4);  // the others are 0
#pragma unroll (CTAS == 2 ? 2 : 1)
    for (int c = group; c < chunks; c += kGroups) {
      // rows 8 apart share their place in the XOR
      const float* at_a = sa + ty * kTT + ((c ^ ty) << 2);
      const float* at_b = sb + tx * kTT + ((c ^ tx) << 2);
      float4 bv[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) bv[k] = *reinterpret_cast<const float4*>(at_b + 8 * kTT * k);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 av = *reinterpret_cast<const float4*>(at_a + 8 * kTT * i);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          acc[i][j] = fmaf(av.x, bv[j].x, acc[i][j]);
          acc[i][j] = fmaf(av.y, bv[j].y, acc[i][j]);
          acc[i][j] = fmaf(av.z, bv[j].z, acc[i][j]);
          acc[i][j] = fmaf(av.w, bv[j].w, acc[i][j]);
        }
      }
    }
  }
  // the four groups' sums, in order
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 16; ++k)
    buf[group * kTile + (ty + 8 * (k >> 2)) * kTJ + tx + 8 * (k & 3)] = acc[k >> 2][k & 3];
  if (sums) row_sum[tid >> 5][tid & 31] = rs;
  __syncthreads();
  constexpr int kEntries = kTile / kSmallThreads;
  float v[kEntries], db = 0.f;
#pragma unroll
  for (int k = 0; k < kEntries; ++k) {
    v[k] = 0.f;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) v[k] += buf[g * kTile + tid + k * kSmallThreads];
  }
  if (sums && tid < kTI) {
#pragma unroll
    for (int k = 0; k < kSmallThreads / 32; ++k) db += row_sum[k][tid];
  }
  const auto put = [&](int e, float value) {
    const int i = i0 + e / kTJ, j = j0 + e % kTJ;
    if (!s.epi.out || i >= s.I || j >= s.J) return;
    float one[1] = {value};
    ColumnResidual<T, 1> res;
    res.fetch(s.epi, s.I, s.J, i, j);
    emit_column<T, 1>(s.epi, s.I, s.J, i, j,
                      s.epi.bias ? to_f32(static_cast<const T*>(s.epi.bias)[j]) : 0.f, one, res);
  };
  if (parts == 1) {
#pragma unroll
    for (int k = 0; k < kEntries; ++k) put(tid + k * kSmallThreads, v[k]);
  } else {
    // the parts in order; each CTA finishes its share of the tile
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kEntries; ++k) buf[tid + k * kSmallThreads] = v[k];
    if (sums && tid < kTI) row_mine[tid] = db;
    cluster_sync();
    const int share = kTile >> lg;
    for (int k = tid; k < share; k += kSmallThreads) {
      const int e = part * share + k;
      float sum = 0.f;
      for (int g = 0; g < parts; ++g)
        sum += peer_f32(map_rank(smem_u32(buf + e), rank - part + g));
      put(e, sum);
    }
    if (sums && part == 0 && tid < kTI) {
      db = 0.f;
      for (int g = 0; g < parts; ++g)
        db += peer_f32(map_rank(smem_u32(row_mine + tid), rank + g));
    }
    cluster_sync();  // no CTA leaves while its sums are read
  }
  if (sums && part == 0 && tid < kTI && i0 + tid < s.I)
    static_cast<T*>(s.sum)[i0 + tid] = from_f32<T>(db);
}

int tiles_of(Small& s) {
  if (!s.sum && (!s.epi.out || s.J == 0)) return s.tiles = 0;
  s.tiles_j = s.epi.out ? std::max(1, (s.J + kTJ - 1) / kTJ) : 1;
  const long long n = static_cast<long long>((s.I + kTI - 1) / kTI) * s.tiles_j;
  s.tiles = n > 0x07ffffff ? -1 : static_cast<int>(n);
  return s.tiles;
}

// Rows of four-element vectors (of the type's size).
bool vectors(const void* p, long long ld, int type) {
  const int b = 4 * dtype_bytes(type);
  return reinterpret_cast<uintptr_t>(p) % b == 0 && ld % 4 == 0;
}

int launch_small(SmallPair& pair, int type, cudaStream_t st, const char* who) {
  for (Small& s : pair.p) {
    if (s.tiles < 0) return fail(VCB_ERR_UNSUPPORTED, "%s: too many output tiles", who);
    s.va = s.a_t && vectors(s.a, s.lda, type) && (!s.a2 || vectors(s.a2, s.lda2, type));
    s.vb = s.b_t && vectors(s.b, s.ldb, type);
    s.parts = 1;
  }
  if (pair.p[0].tiles + pair.p[1].tiles == 0) return VCB_OK;
  // The product whose CTAs have the most steps of the contraction is cut in two, again
  // and again, while those steps are more than an even share of all steps over the
  // SMs' two CTAs each: until then the longest CTA is what is waited for.
  const auto steps = [](const Small& s) {
    return s.tiles ? (s.T + kTT - 1) / kTT / s.parts : 0;
  };
  const long long work = static_cast<long long>(pair.p[0].tiles) * steps(pair.p[0]) +
                         static_cast<long long>(pair.p[1].tiles) * steps(pair.p[1]);
  for (;;) {
    Small& s = pair.p[steps(pair.p[1]) > steps(pair.p[0])];
    if (s.parts == 8 || steps(s) < 2 || 2LL * sm_count() * steps(s) <= work) break;
    s.parts *= 2;
  }
  pair.size = std::max(pair.p[0].parts, pair.p[1].parts);
  long long clusters = 0;
  for (Small& s : pair.p) {
    const int per = pair.size / s.parts;
    clusters += s.clusters = (s.tiles + per - 1) / per;
  }
  // Three CTAs per SM where that holds all of them at once and two do not (fp32 100 x
  // 256 x 784 backward 16.4 us against 18.9), two otherwise (bf16 2000 x 64 x 64
  // backward 20.5 against 22.5).
  const long long ctas = clusters * pair.size;
  const bool three = ctas > 2 * sm_count() && ctas <= 3 * sm_count();
  const auto kernel = type == VCB_F32 ? three ? small_kernel<float, 3> : small_kernel<float, 2>
                      : type == VCB_BF16
                          ? three ? small_kernel<__nv_bfloat16, 3> : small_kernel<__nv_bfloat16, 2>
                          : three ? small_kernel<__half, 3> : small_kernel<__half, 2>;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas));
  cfg.blockDim = dim3(kSmallThreads);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = pair.size;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, pair);
  if (e != cudaSuccess) return cuda_fail(e, who);
  return check_launch(who);
}

int small_forward(const Fwd& f, cudaStream_t st) {
  SmallPair pair{};
  Small& s = pair.p[0];
  s.I = f.M, s.J = f.N, s.T = f.K;
  s.a = f.x, s.lda = f.ldx, s.a_t = 1;
  s.b = f.w, s.ldb = f.ldw, s.b_t = 1;
  s.epi = {f.y, f.z, f.bias, f.res, f.ldy, f.ldz, f.ldr, f.act, 0};
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
  x.epi = {b.dx, nullptr, nullptr, nullptr, b.lddx, 0, 0, VCB_ACT_NONE, 0};
  if (b.dx) tiles_of(x);
  Small& w = pair.p[1];
  w.I = b.N, w.J = b.K, w.T = b.M;
  w.a = b.dy, w.lda = b.lddy, w.a2 = z, w.lda2 = b.ldz, w.a_t = 0, w.act = b.act;
  w.b = b.x, w.ldb = b.ldx, w.b_t = 0;
  w.epi = {b.dw, nullptr, nullptr, nullptr, b.lddw, 0, 0, VCB_ACT_NONE, 0};
  w.sum = b.db;
  if (b.dw || b.db) tiles_of(w);
  return launch_small(pair, b.type, st, "vcb_linear_backward");
}

}  // namespace
}  // namespace lin

namespace {
bool misaligned(const void* p, int type) {
  return reinterpret_cast<uintptr_t>(p) % dtype_bytes(type) != 0;
}
// Which calls take the kernels for few rows (vcb_linear_rows.cu).  Times in us of single
// calls between two events with cold inputs, theirs first.  Forward: fp32 8 x 4096 x 4096 33 against 50, 16 x 1024 x
// 1024 11 against 14, 16 x 2048 x 2048 20 against 35, but 16 x 4096 x 4096 51 against
// 48; bf16 1 x 4096 x 4096 16 against 18, x 4097 18 against 34, 2 x 4096 x 4097 23
// against 35, 4 x 1024 x 1024 8 against 12, but 4 x 4096 x 4096 22 against 18.
// Backward: fp32 16 x 1024 x 1024 25 against 31, 16 x 2048 x 2048 32 against 80, but
// 4 x 60 x 60 13 against 9; bf16 4 x 4096 x 4096 39 against 52, 6 x 1024 x 1024 20
// against 35, but 8 x 1024 x 1024 22 against 20.
bool few_rows_forward(long long M, long long N, long long K, int type) {
  if (M <= 0 || N <= 0 || K <= 0) return false;
  if (type == VCB_F32) return M <= 8 || (M <= lin::kFewRows && N * K <= (1 << 23));
  return M <= 2 || (M <= 8 && M * N * K <= (1 << 23));
}

bool few_rows_backward(long long M, long long N, long long K, int type) {
  if (M <= 0 || N <= 0 || K <= 0) return false;
  if (N * K < (1 << 18)) return M <= 2;
  return M <= 4 || (type == VCB_F32 ? M <= lin::kFewRows : M <= 8 && M * N * K < (1 << 23));
}
}  // namespace
}  // namespace vcb

using namespace vcb;

extern "C" size_t vcb_linear_forward_workspace(int32_t M, int32_t N, int32_t K, int32_t type,
                                               int32_t rows16) {
  if (M <= 0 || N <= 0 || K <= 0 || few_rows_forward(M, N, K, type)) return 0;
  if (type == VCB_F32) return lin::f32_forward_bytes(M, N, K);
  return rows16 ? 0 : lin::tc_forward_bytes(M, N, K);
}

extern "C" size_t vcb_linear_backward_workspace(int32_t M, int32_t N, int32_t K, int32_t type,
                                                int32_t act, int32_t rows16) {
  if (M <= 0 || N <= 0 || K <= 0 || few_rows_backward(M, N, K, type)) return 0;
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
  if (few_rows_forward(M, N, K, type)) return lin::rows_forward(f, static_cast<cudaStream_t>(stream));
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
  if (few_rows_backward(M, N, K, type)) return lin::rows_backward(b, static_cast<cudaStream_t>(stream));
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

extern "C" int vcb_linear_path(int32_t M, int32_t N, int32_t K, int32_t type, int32_t product,
                               int32_t act, int32_t aligned) {
  if (M < 0 || N < 0 || K < 0 || !valid_dtype(type) || product < 0 || product > 2) return -1;
  if (product == 0 ? few_rows_forward(M, N, K, type) : few_rows_backward(M, N, K, type)) return 0;
  // operands whose rows start on 16-byte boundaries, or all of them one element further
  const auto* p = reinterpret_cast<const void*>(static_cast<uintptr_t>(aligned ? 4096 : 4100));
  auto* q = const_cast<void*>(p);
  const auto ld = [&](int n) { return aligned ? (n + 7LL) / 8 * 8 : n + 0LL; };
  const lin::Fwd f{M, N, K, type, act, ld(K), ld(K), 0, ld(N), 0, p, p, nullptr, nullptr, q, nullptr};
  const lin::Bwd b{M, N, K, type, act, ld(N), ld(K), ld(K), ld(N), ld(K), ld(K), p, p, p, p, q, q, q};
  if (type == VCB_F32)
    return (product == 0 ? lin::f32_forward_fits(f) : lin::f32_backward_fits(b))
               ? lin::f32_path(M, N, K, product) : 1;
  return (product == 0 ? lin::tc_forward_fits(f) : lin::tc_backward_fits(b))
             ? lin::tc_path(M, N, K, product) : 1;
}

// Pointers of a packed argument list.
template <typename T = void>
static T* at(int64_t v) {
  return reinterpret_cast<T*>(static_cast<uintptr_t>(v));
}

// Those of the arguments `which` that the entry points take in 32 bits do fit.
static bool in_32_bits(const int64_t* a, std::initializer_list<int> which) {
  for (const int k : which)
    if (a[k] != static_cast<int32_t>(a[k])) return false;
  return true;
}

static int too_large(const char* who) {
  return fail(VCB_ERR_UNSUPPORTED, "%s: a size or code that 32 bits do not hold", who);
}

extern "C" int vcb_linear_forward_packed(const int64_t* a) {
  if (!a) return fail(VCB_ERR_INVALID, "vcb_linear_forward_packed: NULL");
  if (!in_32_bits(a, {0, 1, 2, 3, 9})) return too_large("vcb_linear_forward_packed");
  const auto i = [&](int k) { return static_cast<int32_t>(a[k]); };
  return vcb_linear_forward(i(0), i(1), i(2), i(3), at(a[4]), a[5], at(a[6]), a[7], at(a[8]), i(9),
                            at(a[10]), a[11], at(a[12]), a[13], at(a[14]), a[15], at(a[16]),
                            static_cast<size_t>(a[17]), at(a[18]));
}

extern "C" int vcb_linear_backward_packed(const int64_t* a) {
  if (!a) return fail(VCB_ERR_INVALID, "vcb_linear_backward_packed: NULL");
  if (!in_32_bits(a, {0, 1, 2, 3, 12})) return too_large("vcb_linear_backward_packed");
  const auto i = [&](int k) { return static_cast<int32_t>(a[k]); };
  return vcb_linear_backward(i(0), i(1), i(2), i(3), at(a[4]), a[5], at(a[6]), a[7], at(a[8]), a[9],
                             at(a[10]), a[11], i(12), at(a[13]), a[14], at(a[15]), a[16],
                             at(a[17]), at(a[18]), static_cast<size_t>(a[19]), at(a[20]));
}

extern "C" int vcb_cross_entropy_packed(const int64_t* a) {
  if (!a) return fail(VCB_ERR_INVALID, "vcb_cross_entropy_packed: NULL");
  if (!in_32_bits(a, {0, 1, 2})) return too_large("vcb_cross_entropy_packed");
  const auto i = [&](int k) { return static_cast<int32_t>(a[k]); };
  return vcb_cross_entropy(i(0), i(1), i(2), at(a[3]), a[4], at<const int64_t>(a[5]), a[6],
                           at<float>(a[7]), at(a[8]), a[9], at(a[10]), static_cast<size_t>(a[11]),
                           at(a[12]));
}

extern "C" int vcb_cross_entropy_scaled_packed(const int64_t* a) {
  if (!a) return fail(VCB_ERR_INVALID, "vcb_cross_entropy_scaled_packed: NULL");
  if (!in_32_bits(a, {0, 1, 2})) return too_large("vcb_cross_entropy_scaled_packed");
  const auto i = [&](int k) { return static_cast<int32_t>(a[k]); };
  return vcb_cross_entropy_scaled(i(0), i(1), i(2), at(a[3]), a[4], at<const int64_t>(a[5]), a[6],
                                  at<const float>(a[7]), at<float>(a[8]), at(a[9]), a[10],
                                  at(a[11]), static_cast<size_t>(a[12]), at(a[13]));
}
