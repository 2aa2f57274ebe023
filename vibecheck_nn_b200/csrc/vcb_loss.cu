// Softmax cross-entropy with its gradient, in one pass over the logits.
//
//   l_r = log sum_c exp(x_rc) - x_r,y(r),   loss = sum of l_r over the labelled
//   rows / their number n,   g_rc = (softmax(x_r)_c - [c = y(r)]) / n,
//   and 0 in rows whose label is ignore_index.
//
// Bound by HBM: a logit is read once and its gradient written once.  A row is
// cut over the CTAs of a cluster so that a slice (36 KB at most, while eight
// CTAs suffice) stays in shared memory between its two uses and six CTAs share an
// SM: one row is written while others are read.  The running maximum
// and sum of a softmax are kept in fp32 per thread, joined by shuffles and then
// over the cluster's shared memory, always in the same order.  Rows of up to
// 8 KB stay in the registers of a warp, of up to 128 classes in those of 8 or 32
// lanes without vectors.
//
// Measured: bf16 8192 x 131072 830 us with 3 rows of 10 ignored, 870 to 1,000 us with none
// (4.3 TB/s; the two passes of a row, 64 % of issue slots together, wait for the
// cluster in turn), 2048 x 50001 106 us (3.9 TB/s), fp32 100 x 10 one launch.  The loss
// alone: 556 us with 1 row of 5 ignored (870 with the gradient), 75 and 12.
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

constexpr int kCountCtas = 64;  // most partial counts of labelled rows
constexpr int kHeader = 128;    // words: partial counts, then the last ticket
constexpr int kTicket = kCountCtas;
// Finished CTAs take a ticket of their group of 64, whose last takes one of the
// launch: thousands of tickets of one address would follow each other at some
// 10 ns each.
constexpr int kGroup = 64;

struct CeArgs {
  int R, C, counts;
  long long ld, ldg, ignore;
  const void* x;
  void* g;
  const long long* y;
  int* header;        // kHeader words: partial counts, ticket
  int* tickets;       // one per group
  double* part;       // one partial loss per CTA (per cluster)
  int parts;
  float* loss;         // may be NULL, as g
  const float* scale;  // factor of the gradient, on the device, or NULL
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__global__ void __launch_bounds__(1024)
    ce_count_kernel(int R, const long long* __restrict__ y, long long ignore, int* header,
                    int* tickets, int groups) {
  __shared__ int sums[32];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  for (int i = blockIdx.x * 1024 + threadIdx.x; i < groups; i += gridDim.x * 1024) tickets[i] = 0;
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

// What a softmax entry of the gradient is multiplied with: the factor comes before the
// rounding to the logits' type, or loss scaling would multiply what float16 has
// already lost.
__device__ __forceinline__ float gradient_scale(const CeArgs& a, float inv) {
  return a.scale ? inv * *a.scale : inv;
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
    if (threadIdx.x == 0 && a.loss) *a.loss = static_cast<float>(value * inv);
    return;
  }
  if (threadIdx.x == 0) {
    a.part[part] = value;
    __threadfence();
    const int group = part / kGroup, groups = (a.parts + kGroup - 1) / kGroup;
    last = atomicAdd(a.tickets + group, 1) == min(kGroup, a.parts - group * kGroup) - 1;
    if (last) {
      __threadfence();
      last = atomicAdd(a.header + kTicket, 1) == groups - 1;
    }
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
    if (a.loss) *a.loss = static_cast<float>(t * inv);
  }
}

// ---- rows in registers: G lanes per row, PER logits per lane ----
template <typename T, int G, int PER>
__global__ void __launch_bounds__(256) ce_small_kernel(const CeArgs a) {
  constexpr int kRows = 256 / G;  // rows of a CTA per step
  const int lane = threadIdx.x % G, sub = threadIdx.x / G;
  const float inv = inv_count(a), scale = gradient_scale(a, inv);
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
    if (row && a.g) {
      const float f = bad ? NAN : live && s != 0.f ? scale / s : 0.f;
      const float one = live && s != 0.f ? scale : 0.f;
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

__device__ __forceinline__ void unpack(const uint4& q, float (&v)[4]) {
  v[0] = __uint_as_float(q.x), v[1] = __uint_as_float(q.y);
  v[2] = __uint_as_float(q.z), v[3] = __uint_as_float(q.w);
}

__device__ __forceinline__ float2 two(uint32_t w, __nv_bfloat16) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
__device__ __forceinline__ float2 two(uint32_t w, __half) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
__device__ __forceinline__ uint32_t from_two(float a, float b, __nv_bfloat16) {
  const __nv_bfloat162 t = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&t);
}
__device__ __forceinline__ uint32_t from_two(float a, float b, __half) {
  const __half2 t = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&t);
}

template <typename T>
__device__ __forceinline__ void unpack(const uint4& q, float (&v)[8]) {
  const float2 a = two(q.x, T()), b = two(q.y, T()), c = two(q.z, T()), d = two(q.w, T());
  v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
  v[4] = c.x, v[5] = c.y, v[6] = d.x, v[7] = d.y;
}
template <typename T>
__device__ __forceinline__ void unpack(const uint4& q, float (&v)[4]) {
  unpack(q, v);
}

template <typename T>
__device__ __forceinline__ uint4 pack(const float (&v)[8]) {
  return make_uint4(from_two(v[0], v[1], T()), from_two(v[2], v[3], T()),
                    from_two(v[4], v[5], T()), from_two(v[6], v[7], T()));
}
template <typename T>
__device__ __forceinline__ uint4 pack(const float (&v)[4]) {
  return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]),
                    __float_as_uint(v[3]));
}

// Pairs of floats in one instruction: issue slots bound the kernel next.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{\n\t.reg .b64 a, b, c, r;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "mov.b64 c, {%6, %7};\n\tfma.rn.f32x2 r, a, b, c;\n\tmov.b64 {%0, %1}, r;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  return fma2(a, make_float2(1.f, 1.f), b);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  return fma2(a, b, make_float2(-0.f, -0.f));
}

// exp(x - m) for the pair v[i], v[i + 1].  The difference comes first: x log2 e
// could overflow where a mask is the type's lowest value.
template <int N>
__device__ __forceinline__ float2 exp_pair(const float (&v)[N], int i, float m) {
  const float2 d = add2(make_float2(v[i], v[i + 1]), make_float2(-m, -m));
  const float2 t = mul2(d, make_float2(kLog2e, kLog2e));
  return make_float2(ex2(t.x), ex2(t.y));
}

// A thread's running maximum m and sum s of exp(x - m).
struct Running {
  float m = -FLT_MAX, s = 0.f;
  template <int N>
  __device__ __forceinline__ void add(const float (&v)[N]) {
    float top = v[0];
#pragma unroll
    for (int i = 1; i < N; ++i) top = fmaxf(top, v[i]);
    if (top > m) {
      s *= ex2((m - top) * kLog2e);
      m = top;
    }
    float2 part = exp_pair(v, 0, m);
#pragma unroll
    for (int i = 2; i < N; i += 2) part = add2(part, exp_pair(v, i, m));
    s += part.x + part.y;
  }
};

// Joins the sums of a warp's lanes; LANES: how many hold one (the others hold
// none).  One maximum over the warp, one rescaling per lane, then a plain sum in
// a fixed order.
template <int LANES>
__device__ __forceinline__ void join_lanes(float& m, float& s) {
  float top;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(top) : "f"(m));
  s *= ex2((m - top) * kLog2e);
  m = top;
#pragma unroll
  for (int k = LANES / 2; k; k >>= 1) s += __shfl_xor_sync(0xffffffffu, s, k);
  if (LANES < 32) s = __shfl_sync(0xffffffffu, s, 0);
}

// ---- rows of up to 32 NV vectors in the registers of a warp ----
template <typename T, int NV>
__global__ void __launch_bounds__(256) ce_warp_kernel(const CeArgs a) {
  constexpr int VE = 16 / sizeof(T);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int step = gridDim.x * 8;
  int r = blockIdx.x * 8 + warp;
  long long label = r < a.R ? a.y[r] : a.ignore;
  double total = 0.0;
  float inv = 0.f, scale = 0.f;
  while (r < a.R) {
    const bool more = r < a.R - step;
    const long long next = more ? a.y[r + step] : a.ignore;
    const T* x = static_cast<const T*>(a.x) + r * a.ld;
    T* g = static_cast<T*>(a.g) + r * a.ldg;
    // whole vectors, up to 7 elements before them (lanes 0..) and after (lanes 16..)
    const int head = min(static_cast<int>((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) /
                             static_cast<int>(sizeof(T)), a.C);
    const int vecs = (a.C - head) / VE;
    int edge = -1;
    if (lane < head) edge = lane;
    if (lane >= 16 && lane < 16 + a.C - head - vecs * VE) edge = head + vecs * VE + lane - 16;
    const bool whole = (reinterpret_cast<uintptr_t>(g + head) & 15) == 0;
    const bool live = label != a.ignore, bad = live && (label < 0 || label >= a.C);
    const bool read = live && !bad;
    const uint4* xv = reinterpret_cast<const uint4*>(x + head);
    uint4 q[NV];
    const float xe = read && edge >= 0 ? to_f32(x[edge]) : -INFINITY;
    const float xy = read && lane == 0 ? to_f32(x[label]) : 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (read && lane + 32 * i < vecs) q[i] = __ldcs(xv + lane + 32 * i);
    float m = fmaxf(-FLT_MAX, xe);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (read && lane + 32 * i < vecs) {
        float v[VE];
        unpack<T>(q[i], v);
#pragma unroll
        for (int j = 0; j < VE; ++j) m = fmaxf(m, v[j]);
      }
    }
    asm volatile("redux.sync.max.f32 %0, %0, 0xffffffff;" : "+f"(m));
    float s = ex2((xe - m) * kLog2e);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (read && lane + 32 * i < vecs) {
        float v[VE];
        unpack<T>(q[i], v);
        float2 part = exp_pair(v, 0, m);
#pragma unroll
        for (int j = 2; j < VE; j += 2) part = add2(part, exp_pair(v, j, m));
        s += part.x + part.y;
      }
    }
#pragma unroll
    for (int k = 16; k; k >>= 1) s += __shfl_xor_sync(0xffffffffu, s, k);
    if (inv == 0.f) {
      // the count of labelled rows (and zeroed tickets) come from the launch before
      asm volatile("griddepcontrol.wait;" ::: "memory");
      inv = inv_count(a);
      scale = gradient_scale(a, inv);
    }
    const float f = s != 0.f ? scale / s : 0.f, one = s != 0.f ? scale : 0.f;
    const int at = static_cast<int>(label) - head, label_vec = read && at >= 0 ? at / VE : -1;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int k = lane + 32 * i;
      if (k < vecs && a.g) {
        float v[VE];
        if (read) {
          unpack<T>(q[i], v);
#pragma unroll
          for (int j = 0; j < VE; j += 2) {
            const float2 e = mul2(exp_pair(v, j, m), make_float2(f, f));
            v[j] = e.x;
            v[j + 1] = e.y;
          }
          if (k == label_vec) {
#pragma unroll
            for (int j = 0; j < VE; ++j)
              if (j == at - k * VE) v[j] -= one;
          }
        } else {
#pragma unroll
          for (int j = 0; j < VE; ++j) v[j] = bad ? NAN : 0.f;
        }
        if (whole) {
          __stcs(reinterpret_cast<uint4*>(g + head) + k, pack<T>(v));
        } else {
#pragma unroll
          for (int j = 0; j < VE; ++j) g[head + k * VE + j] = from_f32<T>(v[j]);
        }
      }
    }
    if (edge >= 0 && a.g)
      g[edge] = from_f32<T>(read ? ex2((xe - m) * kLog2e) * f - (edge == label ? one : 0.f)
                                 : bad ? NAN : 0.f);
    if (live && lane == 0) total += bad ? NAN : row_loss(m, s, xy);
    if (!more) break;
    r += step;
    label = next;
  }
  if (inv == 0.f) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    inv = inv_count(a);
  }
  // rows of the CTA, in order
  __shared__ double rows[8];
  if (lane == 0) rows[warp] = total;
  __syncthreads();
  if (threadIdx.x == 0) {
    total = 0.0;
    for (int i = 0; i < 8; ++i) total += rows[i];
  }
  finish(a, blockIdx.x, total, inv);
}

// One cluster per row.  The row's 16-byte vectors are dealt over the CTAs;
// elements before the first and after the last vector (fewer than a vector each)
// belong to the first and the last CTA, one thread each.  STAGED: the slice stays
// in shared memory; otherwise it is read again.
template <typename T, bool STAGED>
__global__ void __launch_bounds__(512, 3) ce_row_kernel(const CeArgs a) {
  constexpr int VE = 16 / sizeof(T);
  extern __shared__ __align__(16) uint4 slice[];
  __shared__ float2 warp_pair[16], mine;
  const int tid = threadIdx.x, nt = blockDim.x, lane = tid & 31;
  const uint32_t rank = cluster_rank(), size = cluster_size(), lg = 31 - __clz(size);
  const long long r = blockIdx.x >> lg;
  const T* x = static_cast<const T*>(a.x) + r * a.ld;
  T* g = static_cast<T*>(a.g) + r * a.ldg;
  const long long label = a.y[r];
  const int head = min(static_cast<int>((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) /
                           static_cast<int>(sizeof(T)), a.C);
  const int vecs = (a.C - head) / VE, tail = a.C - head - vecs * VE;
  const int v0 = static_cast<int>((static_cast<long long>(vecs) * rank) >> lg);
  const int v1 = static_cast<int>((static_cast<long long>(vecs) * (rank + 1)) >> lg);
  int edge = -1;  // this thread's element outside the vectors
  if (rank == 0 && tid < head) edge = tid;
  if (rank == size - 1 && tid >= 32 && tid < 32 + tail) edge = head + vecs * VE + tid - 32;
  const bool whole = (reinterpret_cast<uintptr_t>(g + head) & 15) == 0;
  const uint4* xv = reinterpret_cast<const uint4*>(x + head);
  const auto put = [&](int b, const float (&v)[VE]) {
    if (whole) {
      __stcs(reinterpret_cast<uint4*>(g + head) + b, pack<T>(v));
    } else {
#pragma unroll
      for (int i = 0; i < VE; ++i) g[head + b * VE + i] = from_f32<T>(v[i]);
    }
  };
  // the count of labelled rows (and zeroed tickets) come from the launch before
  const auto count = [&] {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    return inv_count(a);
  };
  double value = 0.0;
  float inv;
  if (label == a.ignore || label < 0 || label >= a.C) {
    const float fill = label == a.ignore ? 0.f : NAN;
    float v[VE];
#pragma unroll
    for (int i = 0; i < VE; ++i) v[i] = fill;
    if (a.g) {
      for (int b = v0 + tid; b < v1; b += nt) put(b, v);
      if (edge >= 0) g[edge] = from_f32<T>(fill);
    }
    if (label != a.ignore) value = NAN;
    inv = count();
  } else {
    const float xe = edge >= 0 ? to_f32(x[edge]) : -INFINITY;
    Running run;
    if (edge >= 0) {
      run.m = fmaxf(run.m, xe);
      run.s = ex2((xe - run.m) * kLog2e);
    }
    constexpr int U = 4;  // loads in flight
    for (int b = v0 + tid; b < v1; b += U * nt) {
      uint4 q[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (b + u * nt < v1) q[u] = __ldcs(xv + b + u * nt);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (b + u * nt < v1) {
          if (STAGED) slice[b + u * nt - v0] = q[u];
          float v[VE];
          unpack<T>(q[u], v);
          run.add(v);
        }
      }
    }
    float m = run.m, s = run.s;
    join_lanes<32>(m, s);
    if (lane == 0) warp_pair[tid >> 5] = make_float2(m, s);
    __syncthreads();
    m = -FLT_MAX, s = 0.f;
    if (lane < nt / 32) m = warp_pair[lane].x, s = warp_pair[lane].y;
    join_lanes<16>(m, s);
    if (size > 1) {
      if (tid == 0) mine = make_float2(m, s);
      cluster_barrier();
      m = -FLT_MAX, s = 0.f;
      if (lane < static_cast<int>(size)) {
        const float2 t = peer_pair(&mine, lane);
        m = t.x, s = t.y;
      }
      join_lanes<8>(m, s);
    }
    inv = count();
    const float scale = gradient_scale(a, inv);
    const float f = s != 0.f ? scale / s : 0.f, one = s != 0.f ? scale : 0.f;
    const int at = static_cast<int>(label) - head;  // label's place among the vectors' elements
    const int label_vec = at >= 0 ? at / VE : -1;
    for (int b = a.g ? v0 + tid : v1; b < v1; b += nt) {
      float v[VE];
      unpack<T>(STAGED ? slice[b - v0] : xv[b], v);
#pragma unroll
      for (int i = 0; i < VE; i += 2) {
        const float2 e = mul2(exp_pair(v, i, m), make_float2(f, f));
        v[i] = e.x;
        v[i + 1] = e.y;
      }
      if (b == label_vec) {
#pragma unroll
        for (int i = 0; i < VE; ++i)
          if (i == at - b * VE) v[i] -= one;
      }
      put(b, v);
    }
    if (edge >= 0 && a.g)
      g[edge] = from_f32<T>(ex2((xe - m) * kLog2e) * f - (edge == label ? one : 0.f));
    if (tid == 0) value = row_loss(m, s, to_f32(x[label]));
    if (size > 1) cluster_barrier();  // no CTA leaves while another reads its pair
  }
  if (rank == 0) finish(a, static_cast<int>(r), value, inv);
}

int launch_count(CeArgs& a, cudaStream_t st) {
  a.counts = std::min(kCountCtas, (a.R + 4095) / 4096);
  ce_count_kernel<<<a.counts, 1024, 0, st>>>(a.R, a.y, a.ignore, a.header, a.tickets,
                                             (a.parts + kGroup - 1) / kGroup);
  return check_launch("vcb_cross_entropy");
}

// Up to four rows per group of lanes: one CTA and no count before it cost less than
// a second launch.
bool single(int R, int C) { return C <= 32 ? R <= 4 * 32 : C <= 128 && R <= 4 * 8; }

template <typename T, int G, int PER>
int launch_small(CeArgs a, cudaStream_t st) {
  const int rows = 256 / G;
  if (single(a.R, a.C)) {
    a.parts = 1, a.counts = 0;
  } else {
    a.parts = static_cast<int>(std::min<long long>((a.R + rows - 1LL) / rows, sm_count() * 16LL));
    const int rc = launch_count(a, st);
    if (rc) return rc;
  }
  ce_small_kernel<T, G, PER><<<a.parts, 256, 0, st>>>(a);
  return check_launch("vcb_cross_entropy");
}

// Launches a kernel of `ctas` CTAs in clusters of `size` that may start while the
// count before it ends.
template <typename K>
int launch_after_count(K kernel, const CeArgs& a, long long ctas, int threads, int smem, int size,
                       cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas));
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = size;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a);
  if (e != cudaSuccess) return cuda_fail(e, "vcb_cross_entropy");
  return check_launch("vcb_cross_entropy");
}

template <typename T, int NV>
int launch_warps(CeArgs a, cudaStream_t st) {
  const int per_sm = NV <= 4 ? 6 : NV <= 8 ? 4 : 2;
  a.parts = static_cast<int>(std::min<long long>((a.R + 7LL) / 8, 1LL * sm_count() * per_sm));
  const int rc = launch_count(a, st);
  return rc ? rc : launch_after_count(ce_warp_kernel<T, NV>, a, a.parts, 256, 0, 1, st);
}

// Bytes of a CTA's slice: six CTAs of the first share an SM, so that one row is
// written while others are read; the second is what one CTA can hold.
constexpr int kSlice = 36 << 10, kSliceMost = 216 << 10;

template <typename T>
int launch(CeArgs a, cudaStream_t st) {
  if (a.C <= 32) return launch_small<T, 8, 4>(a, st);
  if (a.C <= 128) return launch_small<T, 32, 4>(a, st);
  const long long bytes = static_cast<long long>(a.C) * sizeof(T);
  if (bytes <= 2048) return launch_warps<T, 4>(a, st);
  if (bytes <= 4096) return launch_warps<T, 8>(a, st);
  if (bytes <= 8192) return launch_warps<T, 16>(a, st);
  int size = 1;
  while (size < 8 && (bytes + size - 1) / size > kSlice) size *= 2;
  const long long part = ((bytes + 15) / 16 + size - 1) / size * 16;  // a slice, rounded up
  const bool staged = part <= kSliceMost;
  const int smem = staged ? static_cast<int>(part) : 0;
  // 256 threads for a slice of 36 KB: nine vectors each, against some 300
  // instructions per thread and row
  const int threads = part <= (12 << 10) ? 128 : part <= kSlice ? 256 : 512;
  if (static_cast<long long>(a.R) * size > 0x7fffffffLL)
    return fail(VCB_ERR_UNSUPPORTED, "vcb_cross_entropy: R=%d C=%d", a.R, a.C);
  a.parts = a.R;
  int rc = launch_count(a, st);
  if (rc) return rc;
  const auto kernel = staged ? ce_row_kernel<T, true> : ce_row_kernel<T, false>;
  if (staged) rc = ensure_smem(reinterpret_cast<const void*>(kernel), smem);
  if (rc) return rc;
  return launch_after_count(kernel, a, static_cast<long long>(a.R) * size, threads, smem, size, st);
}

}  // namespace

}  // namespace vcb

using namespace vcb;

extern "C" size_t vcb_cross_entropy_workspace(int32_t R, int32_t C) {
  if (R <= 0 || single(R, C)) return 0;
  const size_t rows = static_cast<size_t>(std::max(R, 0));
  return kHeader * 4 + (rows / kGroup + 2) / 2 * 8 + rows * sizeof(double);
}

extern "C" int vcb_cross_entropy_scaled(int32_t R, int32_t C, int32_t type, const void* logits,
                                        int64_t ld, const int64_t* labels, int64_t ignore_index,
                                        const float* scale, float* loss, void* grad, int64_t ldg,
                                        void* workspace, size_t workspace_bytes, void* stream) {
  if (R < 0 || C <= 0 || !valid_dtype(type) || ld < C || (grad && ldg < C))
    return fail(VCB_ERR_INVALID, "vcb_cross_entropy: R=%d C=%d type=%d ld=%lld ldg=%lld", R, C,
                type, (long long)ld, (long long)ldg);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (R == 0)
    return loss ? cuda_fail(cudaMemsetAsync(loss, 0, sizeof(float), st), "vcb_cross_entropy") : VCB_OK;
  const int eb = dtype_bytes(type);
  if (!logits || !labels || reinterpret_cast<uintptr_t>(logits) % eb ||
      reinterpret_cast<uintptr_t>(grad) % eb || reinterpret_cast<uintptr_t>(labels) % 8)
    return fail(VCB_ERR_INVALID, "vcb_cross_entropy: NULL or misaligned pointer");
  const size_t need = vcb_cross_entropy_workspace(R, C);
  if (need && (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 16))
    return fail(VCB_ERR_INVALID, "vcb_cross_entropy: workspace of %zu bytes", workspace_bytes);
  CeArgs a{};
  a.R = R, a.C = C, a.ld = ld, a.ldg = ldg, a.ignore = ignore_index;
  a.x = logits, a.g = grad, a.loss = loss, a.scale = scale;
  a.y = reinterpret_cast<const long long*>(labels);
  if (need) {
    a.header = static_cast<int*>(workspace);
    a.tickets = a.header + kHeader;
    a.part = reinterpret_cast<double*>(a.tickets + (R / kGroup + 2) / 2 * 2);
  }
  if (type == VCB_F32) return launch<float>(a, st);
  if (type == VCB_BF16) return launch<__nv_bfloat16>(a, st);
  return launch<__half>(a, st);
}

extern "C" int vcb_cross_entropy(int32_t R, int32_t C, int32_t type, const void* logits, int64_t ld,
                                 const int64_t* labels, int64_t ignore_index, float* loss,
                                 void* grad, int64_t ldg, void* workspace, size_t workspace_bytes,
                                 void* stream) {
  if (!loss || (R > 0 && !grad) || ldg < C)
    return fail(VCB_ERR_INVALID, "vcb_cross_entropy: loss=%p grad=%p ldg=%lld", loss, grad,
                (long long)ldg);
  return vcb_cross_entropy_scaled(R, C, type, logits, ld, labels, ignore_index, nullptr, loss, grad,
                                  ldg, workspace, workspace_bytes, stream);
}
