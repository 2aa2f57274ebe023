// Softmax cross-entropy with its gradient, in one pass over the logits.
//
//   l_r = log sum_c exp(x_rc) - x_r,y(r),   loss = sum of l_r over the labelled
//   rows / their number n,   g_rc = (softmax(x_r)_c - [c = y(r)]) / n,
//   and 0 in rows whose label is ignore_index.
//
// Bound by HBM: a logit is read once and its gradient written once.  A row is
// cut over the CTAs of a cluster so that a slice (72 KB at most, while eight
// CTAs suffice) stays in shared memory between the two uses and three CTAs
// share an SM: one row is written while others are read.  The running maximum
// and sum of a softmax are kept in fp32 per thread, joined by shuffles and
// then over the cluster's shared memory, always in the same order.  Rows of up
// to 1,024 classes stay in the registers of 8 or 32 lanes.
//
// A row without any class left (all logits -inf) has loss +inf and gradient
// 0.  A label outside [0, C) that is not ignore_index makes its row and the
// loss NaN: nothing is read or written by such an index.
#include <cfloat>

#include <algorithm>

#include "vcb_common.cuh"
#include "vcb_types.cuh"

namespace vcb {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

constexpr int kCountCtas = 64;     // most partial counts of labelled rows
constexpr int kHeader = 128;       // words: partial counts, then the ticket
constexpr int kTicket = kCountCtas;

struct CeArgs {
  int R, C, counts;
  long long ld, ldg, ignore;
  const void* x;
  void* g;
  const long long* y;
  int* header;        // kHeader words: partial counts, ticket
  double* part;       // one partial loss per CTA (per cluster)
  int parts;
  float* loss;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__global__ void __launch_bounds__(1024)
    ce_count_kernel(int R, const long long* __restrict__ y, long long ignore, int* header) {
  __shared__ int sums[32];
  int n = 0;
  for (long long r = blockIdx.x * 1024LL + threadIdx.x; r < R; r += gridDim.x * 1024LL)
    n += y[r] != ignore;
  n = __reduce_add_sync(0xffffffffu, n);
  if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = n;
  __syncthreads();
  if (threadIdx.x < 32) {
    n = __reduce_add_sync(0xffffffffu, sums[threadIdx.x]);
    if (threadIdx.x == 0) {
      header[blockIdx.x] = n;
      if (blockIdx.x == 0) header[kTicket] = 0;
    }
  }
}

// 1 / max(1, labelled rows).  A launch of one CTA (parts == 1 and counts == 0)
// counts its few rows by itself.
__device__ __forceinline__ float inv_count(const CeArgs& a) {
  int n = 0;
  if (a.counts == 0) {
    for (int i = threadIdx.x & 31; i < a.R; i += 32) n += a.y[i] != a.ignore;
  } else {
    for (int i = threadIdx.x & 31; i < a.counts; i += 32) n += a.header[i];
  }
  n = __reduce_add_sync(0xffffffffu, n);
  return 1.f / static_cast<float>(max(n, 1));
}

// Joins two (maximum, sum of exp(x - maximum)) pairs.
__device__ __forceinline__ void join(float& m, float& s, float m2, float s2) {
  const float t = fmaxf(m, m2);
  s = s * ex2((m - t) * kLog2e) + s2 * ex2((m2 - t) * kLog2e);
  m = t;
}

// Loss of a row from its maximum, sum and label's logit.
__device__ __forceinline__ float row_loss(float m, float s, float xy) {
  return s == 0.f ? INFINITY : logf(s) - (xy - m);
}

// Takes this CTA's (cluster's) partial loss; the last one adds all up in
// order.  Called by every thread; only thread 0's value counts.
__device__ void finish(const CeArgs& a, int part, double value, float inv) {
  __shared__ int last;
  __shared__ double sums[32];
  if (a.counts == 0) {
    if (threadIdx.x == 0) *a.loss = static_cast<float>(value * inv);
    return;
  }
  if (threadIdx.x == 0) {
    a.part[part] = value;
    __threadfence();
    last = atomicAdd(a.header + kTicket, 1) == a.parts - 1;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  double t = 0.0;
  for (int i = threadIdx.x; i < a.parts; i += blockDim.x) t += __ldcg(a.part + i);
#pragma unroll
  for (int k = 16; k; k >>= 1) t += __shfl_xor_sync(0xffffffffu, t, k);
  if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = t;
  __syncthreads();
  if (threadIdx.x == 0) {
    t = 0.0;
    for (unsigned w = 0; w < blockDim.x / 32; ++w) t += sums[w];
    *a.loss = static_cast<float>(t * inv);
  }
}

// ---- rows in registers: G lanes per row, PER logits per lane ----
template <typename T, int G, int PER>
__global__ void __launch_bounds__(256) ce_small_kernel(const CeArgs a) {
  constexpr int kRows = 256 / G;  // rows of a CTA per step
  const int lane = threadIdx.x % G, sub = threadIdx.x / G;
  const float inv = inv_count(a);
  double total = 0.0;
  for (long long r0 = static_cast<long long>(blockIdx.x) * kRows; r0 < a.R;
       r0 += static_cast<long long>(gridDim.x) * kRows) {
    const long long r = r0 + sub;
    const bool row = r < a.R;
    const long long label = row ? a.y[r] : a.ignore;
    const bool live = label != a.ignore;
    const bool bad = live && (label < 0 || label >= a.C);
    const T* x = static_cast<const T*>(a.x) + r * a.ld;
    T* g = static_cast<T*>(a.g) + r * a.ldg;
    float v[PER];
    float m = -FLT_MAX;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int c = lane + G * i;
      v[i] = live && c < a.C ? to_f32(x[c]) : -INFINITY;
      m = fmaxf(m, v[i]);
    }
#pragma unroll
    for (int k = G / 2; k; k >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, k));
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const float xi = v[i];
      v[i] = ex2((xi - m) * kLog2e);
      s += v[i];
    }
#pragma unroll
    for (int k = G / 2; k; k >>= 1) s += __shfl_xor_sync(0xffffffffu, s, k);
    if (row) {
      const float f = bad ? NAN : live && s != 0.f ? inv / s : 0.f;
      const float one = live && s != 0.f ? inv : 0.f;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int c = lane + G * i;
        if (c < a.C) g[c] = from_f32<T>(c == label ? v[i] * f - one : v[i] * f);
      }
    }
    if (live && lane == 0) total += bad ? NAN : row_loss(m, s, to_f32(x[label]));
  }
  // rows of the CTA, in order
  __shared__ double rows[kRows];
  if (lane == 0) rows[sub] = total;
  __syncthreads();
  if (threadIdx.x == 0) {
    total = 0.0;
    for (int i = 0; i < kRows; ++i) total += rows[i];
  }
  finish(a, blockIdx.x, total, inv);
}

// ---- a row per cluster, slices in shared memory ----
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_barrier() {
  asm volatile(
      "barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::
          : "memory");
}
__device__ __forceinline__ float2 peer_pair(const float2* mine, uint32_t rank) {
  uint32_t at = static_cast<uint32_t>(__cvta_generic_to_shared(mine)), there;
  float2 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(at), "r"(rank));
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];"
               : "=f"(v.x), "=f"(v.y)
               : "r"(there)
               : "memory");
  return v;
}

template <typename T>
__device__ __forceinline__ void unpack(const uint4& q, float (&v)[16 / sizeof(T)]) {
  T e[16 / sizeof(T)];
  *reinterpret_cast<uint4*>(e) = q;
#pragma unroll
  for (int i = 0; i < static_cast<int>(16 / sizeof(T)); ++i) v[i] = to_f32(e[i]);
}

// One cluster per row.  The row's 16-byte vectors are dealt over the CTAs;
// elements before the first and after the last vector (fewer than a vector
// each) belong to the first and the last CTA, one thread each.  STAGED: the
// slice stays in shared memory; otherwise it is read again.
template <typename T, bool STAGED>
__global__ void __launch_bounds__(512) ce_row_kernel(const CeArgs a) {
  constexpr int VE = 16 / sizeof(T);
  extern __shared__ __align__(16) uint4 slice[];
  __shared__ float2 warp_pair[16], mine;
  const int tid = threadIdx.x, nt = blockDim.x;
  const uint32_t rank = cluster_rank(), size = cluster_size();
  const long long r = blockIdx.x / size;
  const float inv = inv_count(a);
  const T* x = static_cast<const T*>(a.x) + r * a.ld;
  T* g = static_cast<T*>(a.g) + r * a.ldg;
  const long long label = a.y[r];
  const int head0 = static_cast<int>((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / sizeof(T);
  const int head = min(head0, a.C);
  const int vecs = (a.C - head) / VE;
  const int tail = a.C - head - vecs * VE;
  const int v0 = static_cast<int>(static_cast<long long>(vecs) * rank / size);
  const int v1 = static_cast<int>(static_cast<long long>(vecs) * (rank + 1) / size);
  // this thread's edge element, or -1
  int edge = -1;
  if (rank == 0 && tid < head) edge = tid;
  if (rank == size - 1 && tid >= 32 && tid < 32 + tail) edge = head + vecs * VE + tid - 32;
  const bool whole = (reinterpret_cast<uintptr_t>(g + head) & 15) == 0;
  const uint4* xv = reinterpret_cast<const uint4*>(x + head);
  double value = 0.0;
  if (label == a.ignore || label < 0 || label >= a.C) {
    const T fill = from_f32<T>(label == a.ignore ? 0.f : NAN);
    if (whole) {
      T e[VE];
#pragma unroll
      for (int i = 0; i < VE; ++i) e[i] = fill;
      const uint4 q = *reinterpret_cast<const uint4*>(e);
      for (int v = v0 + tid; v < v1; v += nt) reinterpret_cast<uint4*>(g + head)[v] = q;
    } else {
      for (int c = head + v0 * VE + tid; c < head + v1 * VE; c += nt) g[c] = fill;
    }
    if (edge >= 0) g[edge] = fill;
    if (label != a.ignore) value = NAN;
  } else {
    const float xe = edge >= 0 ? to_f32(x[edge]) : -INFINITY;
    float m = fmaxf(-FLT_MAX, xe), s = ex2((xe - m) * kLog2e);
    constexpr int U = 4;  // loads in flight
    for (int b = v0 + tid; b < v1; b += U * nt) {
      uint4 q[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (b + u * nt < v1) q[u] = xv[b + u * nt];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (b + u * nt < v1) {
          if (STAGED) slice[b + u * nt - v0] = q[u];
          float v[VE];
          unpack<T>(q[u], v);
          float top = v[0];
#pragma unroll
          for (int i = 1; i < VE; ++i) top = fmaxf(top, v[i]);
          if (top > m) {
            s *= ex2((m - top) * kLog2e);
            m = top;
          }
#pragma unroll
          for (int i = 0; i < VE; ++i) s += ex2((v[i] - m) * kLog2e);
        }
      }
    }
#pragma unroll
    for (int k = 16; k; k >>= 1)
      join(m, s, __shfl_xor_sync(0xffffffffu, m, k), __shfl_xor_sync(0xffffffffu, s, k));
    if ((tid & 31) == 0) warp_pair[tid >> 5] = make_float2(m, s);
    __syncthreads();
    m = -FLT_MAX, s = 0.f;
    for (int w = 0; w < nt / 32; ++w) join(m, s, warp_pair[w].x, warp_pair[w].y);
    if (size > 1) {
      if (tid == 0) mine = make_float2(m, s);
      cluster_barrier();
      m = -FLT_MAX, s = 0.f;
      for (uint32_t k = 0; k < size; ++k) {
        const float2 t = peer_pair(&mine, k);
        join(m, s, t.x, t.y);
      }
    }
    const float f = s != 0.f ? inv / s : 0.f, one = s != 0.f ? inv : 0.f;
    const int at = static_cast<int>(label) - head;  // label's place among the vectors' elements
    for (int b = v0 + tid; b < v1; b += nt) {
      float v[VE];
      unpack<T>(STAGED ? slice[b - v0] : xv[b], v);
#pragma unroll
      for (int i = 0; i < VE; ++i) {
        v[i] = ex2((v[i] - m) * kLog2e) * f;
        if (b * VE + i == at) v[i] -= one;
      }
      if (whole) {
        T e[VE];
#pragma unroll
        for (int i = 0; i < VE; ++i) e[i] = from_f32<T>(v[i]);
        reinterpret_cast<uint4*>(g + head)[b] = *reinterpret_cast<const uint4*>(e);
      } else {
#pragma unroll
        for (int i = 0; i < VE; ++i) g[head + b * VE + i] = from_f32<T>(v[i]);
      }
    }
    if (edge >= 0) g[edge] = from_f32<T>(ex2((xe - m) * kLog2e) * f - (edge == label ? one : 0.f));
    if (tid == 0) value = row_loss(m, s, to_f32(x[label]));
    if (size > 1) cluster_barrier();  // no CTA leaves while another reads its pair
  }
  if (rank == 0) finish(a, static_cast<int>(r), value, inv);
}

int launch_count(CeArgs& a, cudaStream_t st) {
  a.counts = std::min(kCountCtas, (a.R + 4095) / 4096);
  ce_count_kernel<<<a.counts, 1024, 0, st>>>(a.R, a.y, a.ignore, a.header);
  return check_launch("vcb_cross_entropy");
}

template <typename T, int G, int PER>
int launch_small(CeArgs a, cudaStream_t st) {
  const int rows = 256 / G;
  // up to four rows per group of lanes: one CTA and no count before it cost less
  // than a second launch
  if (a.R <= 4 * rows) {
    a.parts = 1, a.counts = 0;
  } else {
    a.parts = static_cast<int>(std::min<long long>((a.R + rows - 1LL) / rows, sm_count() * 16LL));
    const int rc = launch_count(a, st);
    if (rc) return rc;
  }
  ce_small_kernel<T, G, PER><<<a.parts, 256, 0, st>>>(a);
  return check_launch("vcb_cross_entropy");
}

constexpr int kSlice = 72 << 10;       // three CTAs per SM
constexpr int kSliceMost = 216 << 10;  // one

template <typename T>
int launch(CeArgs a, cudaStream_t st) {
  if (a.C <= 32) return launch_small<T, 8, 4>(a, st);
  if (a.C <= 128) return launch_small<T, 32, 4>(a, st);
  if (a.C <= 1024) return launch_small<T, 32, 32>(a, st);
  const long long bytes = static_cast<long long>(a.C) * sizeof(T);
  int size = 1;
  while (size < 8 && (bytes + size - 1) / size > kSlice) size *= 2;
  const long long part = ((bytes + 15) / 16 + size - 1) / size * 16;  // a slice, rounded up
  const bool staged = part <= kSliceMost;
  const int smem = staged ? static_cast<int>(part) : 0;
  if (static_cast<long long>(a.R) * size > 0x7fffffffLL)
    return fail(VCB_ERR_UNSUPPORTED, "vcb_cross_entropy: R=%d C=%d", a.R, a.C);
  a.parts = a.R;
  const int rc0 = launch_count(a, st);
  if (rc0) return rc0;
  const auto kernel = staged ? ce_row_kernel<T, true> : ce_row_kernel<T, false>;
  if (staged) {
    const int rc = ensure_smem(reinterpret_cast<const void*>(kernel), smem);
    if (rc) return rc;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(a.R * size));
  cfg.blockDim = dim3(part > (16 << 10) ? 512 : 256);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = size;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a);
  if (e != cudaSuccess) return cuda_fail(e, "vcb_cross_entropy");
  return check_launch("vcb_cross_entropy");
}

}  // namespace
}  // namespace vcb

using namespace vcb;

extern "C" size_t vcb_cross_entropy_workspace(int32_t R) {
  return kHeader * 4 + static_cast<size_t>(std::max(R, 0)) * sizeof(double);
}

extern "C" int vcb_cross_entropy(int32_t R, int32_t C, int32_t type, const void* logits, int64_t ld,
                                 const int64_t* labels, int64_t ignore_index, float* loss,
                                 void* grad, int64_t ldg, void* workspace, size_t workspace_bytes,
                                 void* stream) {
  if (R < 0 || C <= 0 || !valid_dtype(type) || ld < C || ldg < C || !loss)
    return fail(VCB_ERR_INVALID, "vcb_cross_entropy: R=%d C=%d type=%d ld=%lld ldg=%lld", R, C,
                type, (long long)ld, (long long)ldg);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (R == 0) return cuda_fail(cudaMemsetAsync(loss, 0, sizeof(float), st), "vcb_cross_entropy");
  const int eb = dtype_bytes(type);
  if (!logits || !labels || !grad || reinterpret_cast<uintptr_t>(logits) % eb ||
      reinterpret_cast<uintptr_t>(grad) % eb || reinterpret_cast<uintptr_t>(labels) % 8)
    return fail(VCB_ERR_INVALID, "vcb_cross_entropy: NULL or misaligned pointer");
  if (!workspace || workspace_bytes < vcb_cross_entropy_workspace(R) ||
      reinterpret_cast<uintptr_t>(workspace) % 16)
    return fail(VCB_ERR_INVALID, "vcb_cross_entropy: workspace of %zu bytes", workspace_bytes);
  CeArgs a{};
  a.R = R, a.C = C, a.ld = ld, a.ldg = ldg, a.ignore = ignore_index;
  a.x = logits, a.g = grad, a.loss = loss;
  a.y = reinterpret_cast<const long long*>(labels);
  a.header = static_cast<int*>(workspace);
  a.part = reinterpret_cast<double*>(a.header + kHeader);
  if (type == VCB_F32) return launch<float>(a, st);
  if (type == VCB_BF16) return launch<__nv_bfloat16>(a, st);
  return launch<__half>(a, st);
}
