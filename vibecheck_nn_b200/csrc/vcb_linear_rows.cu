// Linear layer for few rows (up to 16 tokens), forward and both gradients.
//
// Bound by HBM: with few rows the weight is nearly all that is read (forward,
// dX = dZ W) or written (dW = dZ^T X), once each.
//
// Forward: a CTA takes four outputs n; its eight warps cut the contraction in
// vectors of 16 bytes per lane, so that thousands of warps read the weight at the
// same time; 32 sums per warp are reduced by exchanging halves (31 shuffles), then
// over the warps in order.
// Backward: a CTA takes a strip of columns k and a range of rows n.  A row of the
// weight is read, its share of dX added in registers, and the same row of dW written
// (x stays in registers), so W and dW pass once in one launch; db is the sum of the
// dz that are in shared memory anyway.  The ranges of a strip are a cluster, joined
// over distributed shared memory in order.  All sums are in fp32.
//
// Measured with cold inputs, on the device (calls in a captured graph): bf16 1 row 4096
// x 4096 forward 10.4 us (5 of HBM), backward 25 us (10 of HBM); fp32 8 rows 25 us (10)
// and 42 us (20).  Single calls between two events, as in the rules of vcb_linear.cu:
// 16, 31, 33 and 49 us.  Loads of several rows are in flight past conversions and
// stores: without that the backward took 47 and 66 us.
#include <algorithm>

#include "vcb_linear_tc.cuh"

namespace vcb {
namespace lin {
namespace {

constexpr int kRowThreads = 256, kRowWarps = 8, kOut = 4;

// V neighbouring elements as loaded.  They are unpacked where they are used: a use
// would wait for them, and more loads follow.
template <typename T, int V>
struct Raw {
  static constexpr int W = V * sizeof(T) / 4;
  uint32_t w[W + 1];
  bool odd;  // words of the elements from the second on, then the first and the last element

  // At p; 0 from `left` on.  vec: p is aligned to all V elements.
  __device__ __forceinline__ void load(const T* p, int left, bool vec) {
    odd = false;
    if (left < V) {
#pragma unroll
      for (int i = 0; i < W; ++i) {
        if constexpr (sizeof(T) == 4) {
          w[i] = i < left ? reinterpret_cast<const uint32_t*>(p)[i] : 0;
        } else {
          const uint16_t* h = reinterpret_cast<const uint16_t*>(p) + 2 * i;
          w[i] = (2 * i < left ? h[0] : 0u) | (2 * i + 1 < left ? h[1] : 0u) << 16;
        }
      }
    } else if (vec) {
      struct alignas(4 * W) Pack {
        uint32_t w[W];
      };
      const Pack q = *reinterpret_cast<const Pack*>(p);
#pragma unroll
      for (int i = 0; i < W; ++i) w[i] = q.w[i];
    } else {
      odd = sizeof(T) == 2 && reinterpret_cast<uintptr_t>(p) % 4 != 0;
      const uint32_t* q = reinterpret_cast<const uint32_t*>(p + odd);
#pragma unroll
      for (int i = 0; i < W - 1; ++i) w[i] = q[i];
      if (odd) {
        w[W - 1] = *reinterpret_cast<const uint16_t*>(p);
        w[W] = *reinterpret_cast<const uint16_t*>(p + V - 1);
      } else {
        w[W - 1] = q[W - 1];
      }
    }
  }
  __device__ __forceinline__ void values(float (&v)[V]) const {
    uint32_t o[W];
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const uint32_t low = i ? w[i - 1] >> 16 : w[W - 1], high = i < W - 1 ? w[i] : w[W];
      o[i] = odd ? low | high << 16 : w[i];
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      T e;
      if constexpr (sizeof(T) == 4) {
        e = __uint_as_float(o[i]);
      } else {
        const uint16_t h = static_cast<uint16_t>(i % 2 ? o[i / 2] >> 16 : o[i / 2]);
        e = *reinterpret_cast<const T*>(&h);
      }
      v[i] = to_f32(e);
    }
  }
};

// Sums of N values over the warp; lane l < N gets value l (N a power of two).
template <int N>
__device__ __forceinline__ float sums_of(float (&v)[N], int lane) {
#pragma unroll
  for (int o = 16; o >= N; o >>= 1) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  }
#pragma unroll
  for (int o = N / 2; o; o >>= 1) {
    const bool high = lane & o;
#pragma unroll
    for (int i = 0; i < o; ++i) {
      const float give = high ? v[i] : v[i + o], keep = high ? v[i + o] : v[i];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
    }
  }
  return v[0];
}

struct RowsFwd {
  Fwd f;
  int vec;  // rows of x and w are 16-byte aligned
};

template <typename T, int MR>
__global__ void __launch_bounds__(kRowThreads) rows_forward_kernel(const __grid_constant__ RowsFwd a) {
  constexpr int V = 16 / sizeof(T), NV = kOut * MR;
  const Fwd& f = a.f;
  __shared__ float part[kRowWarps][NV];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n0 = blockIdx.x * kOut, m0 = blockIdx.y * MR;
  const T *x = static_cast<const T*>(f.x), *w = static_cast<const T*>(f.w);
  float acc[NV] = {};
#pragma unroll 2
  for (int base = warp * 32 * V; base < f.K; base += kRowWarps * 32 * V) {
    const int c = base + lane * V, left = f.K - c;
    Raw<T, V> wr[kOut], xr[MR];
#pragma unroll
    for (int r = 0; r < kOut; ++r) wr[r].load(w + min(n0 + r, f.N - 1) * f.ldw + c, left, a.vec);
#pragma unroll
    for (int m = 0; m < MR; ++m) xr[m].load(x + min(m0 + m, f.M - 1) * f.ldx + c, left, a.vec);
    float wv[kOut][V];
#pragma unroll
    for (int r = 0; r < kOut; ++r) wr[r].values(wv[r]);
#pragma unroll
    for (int m = 0; m < MR; ++m) {
      float xv[V];
      xr[m].values(xv);
#pragma unroll
      for (int r = 0; r < kOut; ++r) {
#pragma unroll
        for (int i = 0; i < V; ++i) acc[m * kOut + r] = fmaf(xv[i], wv[r][i], acc[m * kOut + r]);
      }
    }
  }
  const float mine = sums_of<NV>(acc, lane);
  if (lane < NV) part[warp][lane] = mine;
  __syncthreads();
  const int t = threadIdx.x, n = n0 + t % kOut, m = m0 + t / kOut;
  if (t >= NV || n >= f.N || m >= f.M) return;
  float v[1] = {0.f};
#pragma unroll
  for (int k = 0; k < kRowWarps; ++k) v[0] += part[k][t];
  const Epilogue e{f.y, f.z, f.bias, f.res, f.ldy, f.ldz, f.ldr, f.act, 0};
  ColumnResidual<T, 1> res;
  res.fetch(e, f.M, f.N, m, n);
  emit_column<T, 1>(e, f.M, f.N, m, n, f.bias ? to_f32(static_cast<const T*>(f.bias)[n]) : 0.f, v,
                    res);
}

struct RowsBwd {
  Bwd b;
  int vec_x, vec_w, vec_dw;  // rows take vectors of V elements
  int split;                 // CTAs (a cluster) per strip
};

constexpr int kSpan = 512;  // rows n whose dz are in shared memory at a time

template <typename T, int V>
__device__ __forceinline__ void put_some(T* p, int left, bool vec, const float (&v)[V]) {
  struct alignas(sizeof(T) * V) Pack {
    T e[V];
  };
  if (vec && left >= V) {
    Pack q;
#pragma unroll
    for (int i = 0; i < V; ++i) q.e[i] = from_f32<T>(v[i]);
    *reinterpret_cast<Pack*>(p) = q;
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < left) p[i] = from_f32<T>(v[i]);
  }
}

template <typename T, int MR, int V>
__global__ void __launch_bounds__(kRowThreads) rows_backward_kernel(const __grid_constant__ RowsBwd a) {
  constexpr int kCols = 32 * V, kPart = kRowWarps * MR * kCols;
  const Bwd& b = a.b;
  // dz of kSpan rows ([n][m]); at the end the warps' sums of dX, then the CTA's
  __shared__ __align__(16) float buf[kSpan * MR > kPart ? kSpan * MR : kPart];
  __shared__ float mine[MR * kCols];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int size = a.split, rank = blockIdx.x % size, strip = blockIdx.x / size;
  const int c = strip * kCols + lane * V, left = b.K - c;
  const int n_begin = static_cast<int>(static_cast<long long>(b.N) * rank / size);
  const int n_end = static_cast<int>(static_cast<long long>(b.N) * (rank + 1) / size);
  const T *dy = static_cast<const T*>(b.dy), *z = static_cast<const T*>(b.z);
  const T* w = static_cast<const T*>(b.w) + c;
  T* dw = static_cast<T*>(b.dw) + c;
  float x[MR][V], acc[MR][V] = {};
  if (b.dw) {
#pragma unroll
    for (int m = 0; m < MR; ++m) {
      Raw<T, V> r;
      r.load(static_cast<const T*>(b.x) + min(m, b.M - 1) * b.ldx + c, m < b.M ? left : 0, a.vec_x);
      r.values(x[m]);
    }
  }
  for (int n0 = n_begin; n0 < n_end; n0 += kSpan) {
    const int rows = min(kSpan, n_end - n0);
    __syncthreads();
    for (int t = threadIdx.x; t < rows; t += kRowThreads) {
      const int n = n0 + t;
      float sum = 0.f;
#pragma unroll
      for (int m = 0; m < MR; ++m) {
        float v = 0.f;
        if (m < b.M)
          v = act_grad(to_f32(dy[m * b.lddy + n]),
                       b.act == VCB_ACT_NONE ? 0.f : to_f32(z[m * b.ldz + n]), b.act);
        buf[t * MR + m] = v;
        sum += v;
      }
      if (b.db && strip == 0) static_cast<T*>(b.db)[n] = from_f32<T>(sum);
    }
    __syncthreads();
    constexpr int U = 4;  // rows of W in flight; the stores of dW between them would end that
    for (int t0 = warp; t0 < rows; t0 += U * kRowWarps) {
      Raw<T, V> wr[U];
      if (b.dx) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int t = t0 + u * kRowWarps;
          if (t < rows) wr[u].load(w + (long long)(n0 + t) * b.ldw, left, a.vec_w);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int t = t0 + u * kRowWarps;
        if (t >= rows) break;
        const long long n = n0 + t;
        float dz[MR];
#pragma unroll
        for (int m = 0; m < MR; ++m) dz[m] = buf[t * MR + m];
        if (b.dx) {
          float v[V];
          wr[u].values(v);
#pragma unroll
          for (int m = 0; m < MR; ++m) {
#pragma unroll
            for (int i = 0; i < V; ++i) acc[m][i] = fmaf(dz[m], v[i], acc[m][i]);
          }
        }
        if (b.dw) {
          float v[V] = {};
#pragma unroll
          for (int m = 0; m < MR; ++m) {
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] = fmaf(dz[m], x[m][i], v[i]);
          }
          put_some<T, V>(dw + n * b.lddw, left, a.vec_dw, v);
        }
      }
    }
  }
  if (!b.dx) return;  // the same for all CTAs
  __syncthreads();
#pragma unroll
  for (int m = 0; m < MR; ++m) {
#pragma unroll
    for (int i = 0; i < V; ++i) buf[(warp * MR + m) * kCols + lane * V + i] = acc[m][i];
  }
  __syncthreads();
  for (int e = threadIdx.x; e < MR * kCols; e += kRowThreads) {
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < kRowWarps; ++k) v += buf[k * MR * kCols + e];
    mine[e] = v;
  }
  cluster_sync();
  for (int e = rank * kRowThreads + threadIdx.x; e < MR * kCols; e += size * kRowThreads) {
    const int m = e / kCols, k = strip * kCols + e % kCols;
    float v = 0.f;
    for (int g = 0; g < size; ++g) v += peer_f32(map_rank(smem_u32(mine + e), g));
    if (m < b.M && k < b.K) static_cast<T*>(b.dx)[m * b.lddx + k] = from_f32<T>(v);
  }
  cluster_sync();  // no CTA leaves while its sums are read
}

bool aligned(const void* p, long long ld, int elem, int bytes) {
  return reinterpret_cast<uintptr_t>(p) % bytes == 0 && ld * elem % bytes == 0;
}

template <typename T>
int forward(const Fwd& f, cudaStream_t st) {
  RowsFwd a{f, aligned(f.x, f.ldx, sizeof(T), 16) && aligned(f.w, f.ldw, sizeof(T), 16)};
  const dim3 grid((f.N + kOut - 1) / kOut, f.M > 8 ? 2 : 1);
  if (f.M == 1)
    rows_forward_kernel<T, 1><<<grid, kRowThreads, 0, st>>>(a);
  else if (f.M == 2)
    rows_forward_kernel<T, 2><<<grid, kRowThreads, 0, st>>>(a);
  else if (f.M <= 4)
    rows_forward_kernel<T, 4><<<grid, kRowThreads, 0, st>>>(a);
  else
    rows_forward_kernel<T, 8><<<grid, kRowThreads, 0, st>>>(a);
  return check_launch("vcb_linear_forward");
}

template <typename T, int MR, int V>
int backward(const Bwd& b, cudaStream_t st) {
  const char* who = "vcb_linear_backward";
  const int e = sizeof(T), strips = (b.K + 32 * V - 1) / (32 * V);
  RowsBwd a{b, aligned(b.x, b.ldx, e, V * e), aligned(b.w, b.ldw, e, V * e),
            aligned(b.dw, b.lddw, e, V * e), 1};
  // a strip's rows over a cluster while that leaves every CTA some 32 rows
  while (a.split < 8 && strips * a.split < 4 * sm_count() && b.N / (2 * a.split) >= 32) a.split *= 2;
  if (static_cast<long long>(strips) * a.split > 0x7fffffffLL)
    return fail(VCB_ERR_UNSUPPORTED, "%s: K=%d", who, b.K);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(strips * a.split));
  cfg.blockDim = dim3(kRowThreads);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = a.split;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  const cudaError_t err = cudaLaunchKernelEx(&cfg, rows_backward_kernel<T, MR, V>, a);
  if (err != cudaSuccess) return cuda_fail(err, who);
  return check_launch(who);
}

template <typename T>
int backward(const Bwd& b, cudaStream_t st) {
  if (b.M == 1) return backward<T, 1, 4>(b, st);
  if (b.M == 2) return backward<T, 2, 4>(b, st);
  if (b.M <= 4) return backward<T, 4, 4>(b, st);
  if constexpr (sizeof(T) == 4) {  // 16-bit types take the tensor cores from 9 rows on
    if (b.M > 8) return backward<T, 16, 2>(b, st);
  }
  return backward<T, 8, 4>(b, st);
}

}  // namespace

int rows_forward(const Fwd& f, cudaStream_t st) {
  return f.type == VCB_F32    ? forward<float>(f, st)
         : f.type == VCB_BF16 ? forward<__nv_bfloat16>(f, st)
                              : forward<__half>(f, st);
}

int rows_backward(const Bwd& b, cudaStream_t st) {
  return b.type == VCB_F32    ? backward<float>(b, st)
         : b.type == VCB_BF16 ? backward<__nv_bfloat16>(b, st)
                              : backward<__half>(b, st);
}

}  // namespace lin
}  // namespace vcb
