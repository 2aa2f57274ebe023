// The linear layer's float32 products on the tensor cores.
//
// A float32 operand row is scaled by a power of two, so that its largest entry
// lies in [2^14, 2^15), and split in two half-precision numbers,
//   x 2^-e = h + l + d,  h = fp16(x 2^-e),  l = fp16(x 2^-e - h),
// |d| <= 2^-22 |x| 2^-e (and 2^-40 of the row's largest where l is subnormal).
// The tensor cores form  h h' + h l' + l h'  with exact products and fp32
// accumulators; l l' is below 2^-22 of the product and left out.  That is the
// precision of three TF32 products at twice their rate: fp16 multiplies twice as
// fast as TF32 and has as many significant bits, and the row scales supply the
// exponents that it lacks.  A scale belongs to a row along which nothing is
// summed (a row of the output, or a column of it), so it leaves the product as a
// factor 2^(e + e').  An infinite or NaN entry makes the outputs of its row
// infinite or NaN.
//
// The tensor cores drop low-order bits in every accumulation.  So an accumulator
// in tensor memory takes one 64-deep stage (12 MMAs) only, and the epilogue warps
// add the stages' sums in registers, rounding to nearest, while the next stage
// fills the other accumulator.
//
// Measured: 4096^3 forward 355 us in short bursts (387 TFLOP/s of fp32 products, 1,160
// of fp16), 424 us back to back under the power cap, both gradients 750 us; largest
// error 3e-7 of the largest output, against 1.1e-6 of an fp32 sum.
//
// Preparation is bound by HBM: forward, one launch reads each row once, finds its
// scale and writes both halves.  Backward, dz needs row scales for dX and column
// scales for dW, so a first launch finds all scales (and db, and never stores
// dz), a second writes the halves.  Then products as in vcb_linear_tc.cu:
// f32_kernel<256, true> in CTA pairs for large ones, f32_kernel<64 / 128, false>
// with the contraction cut over a cluster for the rest.
#include <algorithm>
#include <array>
#include <atomic>
#include <initializer_list>

#include "vcb_linear_tc.cuh"

namespace vcb {
namespace lin {
namespace {

__device__ int g_f32_fault;
std::atomic<bool> g_launched{false};

// Exponent e of the scale 2^-e for a row whose largest |entry| has these bits.
__device__ __forceinline__ int scale_exp(uint32_t bits) {
  const int b = static_cast<int>(bits >> 23);
  if (bits == 0 || b >= 255) return 0;  // all zero, or not finite
  return max(b - 127 - 14, -126);
}

__device__ __forceinline__ float exp2i(int k) { return __int_as_float((k + 127) << 23); }

// v 2^e for the sum e of two scale_exp(): in two steps, each in range.
__device__ __forceinline__ float scaled(float v, int e) {
  const int h = e >> 1;
  return v * exp2i(h) * exp2i(e - h);
}

// Larger |entry|, NaN left aside: it needs no scale.
__device__ __forceinline__ float more(float m, float x) { return fmaxf(m, fabsf(x)); }

__device__ __forceinline__ void halves4(const float (&x)[4], const float (&scale)[4], uint2& high,
                                        uint2& low) {
  __half2 h[2], l[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const float a = x[2 * k] * scale[2 * k], b = x[2 * k + 1] * scale[2 * k + 1];
    h[k] = __floats2half2_rn(a, b);
    const float2 back = __half22float2(h[k]);
    // an infinite h has no remainder
    l[k] = __floats2half2_rn(isinf(back.x) ? 0.f : a - back.x, isinf(back.y) ? 0.f : b - back.y);
  }
  high = *reinterpret_cast<const uint2*>(h);
  low = *reinterpret_cast<const uint2*>(l);
}

__device__ __forceinline__ void put_halves(__half* h, long long plane, const float (&v)[4],
                                           float scale) {
  const float all[4] = {scale, scale, scale, scale};
  uint2 high, low;
  halves4(v, all, high, low);
  *reinterpret_cast<uint2*>(h) = high;
  *reinterpret_cast<uint2*>(h + plane) = low;
}

// Four entries of a row from column c; 0 beyond the last.
__device__ __forceinline__ void row4(const float* row, int c, int cols, bool vec, float (&v)[4]) {
  if (vec && c + 4 <= cols) {
    load4(row + c, v);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = c + k < cols ? row[c + k] : 0.f;
  }
}

// ---- preparation, forward: halves of the rows of two matrices ----
struct RowJob {
  const float* src;
  long long ld, rows;
  int cols, vec;
  __half* h;        // rows x ldh, the second halves `plane` elements further
  long long ldh, plane;
  uint32_t* most;   // bits of the largest |entry| of each row
};

struct RowJobs {
  RowJob j[2];
};

// TPR threads per row, of which KEEP vectors per thread stay in registers.
template <int TPR, int KEEP>
__global__ void __launch_bounds__(256) rows_kernel(const __grid_constant__ RowJobs a) {
  __shared__ uint32_t warp_most[8];
  let_next_start();
  long long r = static_cast<long long>(blockIdx.x) * (256 / TPR) + threadIdx.x / TPR;
  const int t = threadIdx.x % TPR;
  const bool second = r >= a.j[0].rows;
  const RowJob& q = a.j[second];
  if (second) r -= a.j[0].rows;
  const bool row = r < q.rows;  // uniform over the threads of a row
  const float* src = q.src + r * q.ld;
  float v[KEEP][4];
  float most = 0.f;
  if (row) {
#pragma unroll
    for (int k = 0; k < KEEP; ++k) row4(src, (k * TPR + t) * 4, q.cols, q.vec, v[k]);
#pragma unroll
    for (int k = 0; k < KEEP; ++k) {
#pragma unroll
      for (int i = 0; i < 4; ++i) most = more(most, v[k][i]);
    }
    for (int c = (KEEP * TPR + t) * 4; c < q.cols; c += TPR * 4) {
      float w[4];
      row4(src, c, q.cols, q.vec, w);
#pragma unroll
      for (int i = 0; i < 4; ++i) most = more(most, w[i]);
    }
  }
  uint32_t m = __reduce_max_sync(0xffffffffu, __float_as_uint(most));
  if (TPR > 32) {
    if ((threadIdx.x & 31) == 0) warp_most[threadIdx.x >> 5] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < TPR / 32; ++w) m = max(m, warp_most[threadIdx.x / TPR * (TPR / 32) + w]);
  }
  if (!row) return;
  if (t == 0) q.most[r] = m;
  const float scale = exp2i(-scale_exp(m));
  __half* h = q.h + r * q.ldh;
#pragma unroll
  for (int k = 0; k < KEEP; ++k) {
    const int c = (k * TPR + t) * 4;
    if (c < q.cols) put_halves(h + c, q.plane, v[k], scale);
  }
  for (int c = (KEEP * TPR + t) * 4; c < q.cols; c += TPR * 4) {
    float w[4];
    row4(src, c, q.cols, q.vec, w);
    put_halves(h + c, q.plane, w, scale);
  }
}

// ---- preparation, backward ----
// A matrix in strips of columns, 4 columns per lane; with z the entries are dz = dy
// act'(z).
struct ColJob {
  const float *src, *z;
  long long ld, ldz, rows;
  int cols, vec, act;
  uint32_t *col_most, *row_most;  // row_most may be NULL; zero on entry
  float* sum;                     // column sums, or NULL
  __half *by_col, *by_row;        // halves with column scales; with row scales, or NULL
  long long ldh, plane;
};

struct ColJobs {
  ColJob j[3];
  int count;
  int cluster;  // CTAs per strip of scales_kernel
  int wide;     // strips of halves_kernel, for each block of rows
};

constexpr int kStripThreads = 256, kStripWarps = kStripThreads / 32;

// Entries of N rows from r, `step` rows apart; 0 from row `end` on.  All loads come
// before the first use.
template <int N>
__device__ __forceinline__ void job_rows(const ColJob& q, long long r, long long step,
                                         long long end, int c, float (&v)[N][4]) {
  float t[N][4];
#pragma unroll
  for (int u = 0; u < N; ++u) {
#pragma unroll
    for (int k = 0; k < 4; ++k) v[u][k] = t[u][k] = 0.f;
    if (r + u * step >= end) continue;
    row4(q.src + (r + u * step) * q.ld, c, q.cols, q.vec, v[u]);
    if (q.act != VCB_ACT_NONE) row4(q.z + (r + u * step) * q.ldz, c, q.cols, q.vec, t[u]);
  }
  if (q.act != VCB_ACT_NONE) {
#pragma unroll
    for (int u = 0; u < N; ++u) act_grads(v[u], t[u], q.act);
  }
}

// The job and strip (of `width` columns) of strip s of a launch.
__device__ __forceinline__ const ColJob& strip_of(const ColJobs& a, int& s, int width = 32) {
  int k = 0;
  while (k + 1 < a.count) {
    const int strips = (a.j[k].cols + width - 1) / width;
    if (s < strips) break;
    s -= strips;
    ++k;
  }
  return a.j[k];
}

// Largest entries of every column (a cluster of up to 8 CTAs per strip of 32 columns,
// a part of the rows each, 8 lanes per row) and of every row (atomic maxima: any
// order gives the same), column sums in the order of the ranks.
__global__ void __launch_bounds__(kStripThreads, 4)
    scales_kernel(const __grid_constant__ ColJobs a) {
  __shared__ float part[kStripWarps][32], sum_mine[32];
  __shared__ uint32_t most_part[kStripWarps][32], most_mine[32];
  let_next_start();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int size = a.cluster, rank = blockIdx.x % size;
  int strip = blockIdx.x / size;
  const ColJob& q = strip_of(a, strip);
  const int c = strip * 32 + (lane & 7) * 4;
  const long long r0 = q.rows * rank / size, r1 = q.rows * (rank + 1) / size;
  float sum[4] = {};
  float most[4] = {};
  constexpr int U = 4, W = kStripWarps * 4;  // rows in flight per lane, rows of a CTA's step
  for (long long base = r0 + warp * 4; base < r1; base += U * W) {
    float v[U][4];
    job_rows<U>(q, base + (lane >> 3), W, r1, c, v);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long r = base + u * W + (lane >> 3);
      float top = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        most[i] = more(most[i], v[u][i]);
        sum[i] += v[u][i];
        top = more(top, v[u][i]);
      }
      if (q.row_most) {
        uint32_t m = __float_as_uint(top);
#pragma unroll
        for (int k = 4; k; k >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, k));
        if ((lane & 7) == 0 && r < r1) atomicMax(q.row_most + r, m);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int k = 8; k < 32; k *= 2) {
      sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], k);
      most[i] = fmaxf(most[i], __shfl_xor_sync(0xffffffffu, most[i], k));
    }
    if (lane < 8) {
      part[warp][lane * 4 + i] = sum[i];
      most_part[warp][lane * 4 + i] = __float_as_uint(most[i]);
    }
  }
  __syncthreads();
  if (threadIdx.x < 32) {
    float s = 0.f;
    uint32_t m = 0;
    for (int w = 0; w < kStripWarps; ++w) {
      s += part[w][threadIdx.x];
      m = max(m, most_part[w][threadIdx.x]);
    }
    sum_mine[threadIdx.x] = s;
    most_mine[threadIdx.x] = m;
  }
  cluster_sync();
  const int col = strip * 32 + threadIdx.x;
  if (rank == 0 && threadIdx.x < 32 && col < q.cols) {
    float s = 0.f;
    uint32_t m = 0;
    for (int k = 0; k < size; ++k) {
      s += peer_f32(map_rank(smem_u32(sum_mine + threadIdx.x), k));
      m = max(m, __float_as_uint(peer_f32(map_rank(smem_u32(most_mine + threadIdx.x), k))));
    }
    if (q.sum) q.sum[col] = s;
    q.col_most[col] = m;
  }
  cluster_sync();  // no CTA leaves while its figures are read
}

constexpr int kHalvesRows = 32;  // rows of a CTA

__global__ void __launch_bounds__(kStripThreads) halves_kernel(const __grid_constant__ ColJobs a) {
  after_previous();
  let_next_start();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int block = blockIdx.x / a.wide;
  int strip = blockIdx.x % a.wide;
  const ColJob& q = strip_of(a, strip, 128);
  const int c = strip * 128 + lane * 4;
  if (c >= q.cols) return;
  float scale[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) scale[i] = c + i < q.cols ? exp2i(-scale_exp(q.col_most[c + i])) : 0.f;
  const long long end = min(q.rows, (block + 1LL) * kHalvesRows);
  constexpr int U = kHalvesRows / kStripWarps;  // rows of a warp
  const long long r0 = static_cast<long long>(block) * kHalvesRows + warp;
  float v[U][4];
  job_rows<U>(q, r0, kStripWarps, end, c, v);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const long long r = r0 + u * kStripWarps;
    if (r >= end) break;
    if (q.by_row)
      put_halves(q.by_row + r * q.ldh + c, q.plane, v[u], exp2i(-scale_exp(q.row_most[r])));
    if (q.by_col) {
      uint2 high, low;
      halves4(v[u], scale, high, low);
      __half* at = q.by_col + r * q.ldh + c;
      *reinterpret_cast<uint2*>(at) = high;
      *reinterpret_cast<uint2*>(at + q.plane) = low;
    }
  }
}

// ---- products ----
struct alignas(64) Prod32 {
  CUtensorMap a, b;  // (64, rows, 2 halves) boxes
  int J, I, a_mn, b_mn, tiles_j, tiles_i, nk;
  uint32_t idesc;
  const uint32_t *most_a, *most_b;  // scales of the rows of A (j) and of B (i)
  Epilogue epi;
};

struct Launch32 {
  Prod32 p[2];
  int units0, units, split;
};

// Sixteen epilogue warps: what they do at a tile's end (scales, activation, stores)
// runs beside two stages of the next tile's MMAs only, so it is spread as wide as
// registers allow.
constexpr int kEpi = 16, kF32Threads = (kEpi + 2) * 32;

template <int BN, bool PAIR>
struct Cfg {
  static constexpr int kRowsB = PAIR ? BN / 2 : BN;
  static constexpr int kBytesB = 2 * kRowsB * 128;
  static constexpr int kStage = 2 * kBytesA + kBytesB;
  static constexpr int kStages = 196608 / kStage;
  static constexpr int kSmem = kStages * kStage + 1024;
  static constexpr int kBufs = BN == 256 ? 2 : 4;
  static constexpr int kColumns = kBufs * BN;  // of tensor memory
  static constexpr int kCols = BN / (kEpi / 4);  // of an epilogue thread
  static constexpr int kArrivals = kEpi * (PAIR ? 2 : 1);
};

__device__ __forceinline__ void tma_3d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x,
                                       int y) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(0), "r"(bar)
      : "memory");
}

__device__ __forceinline__ void tma_3d_pair(uint32_t dst, const CUtensorMap* map, uint32_t bar,
                                            int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::"
      "bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(0), "r"(bar)
      : "memory");
}

// Both halves of an operand's rows.  K-major: all h rows, then all l rows.
// MN-major: per 64 rows, 8 KB of h and 8 KB of l.
template <bool PAIR>
__device__ __forceinline__ void load_halves(uint32_t dst, const CUtensorMap* map, uint32_t bar,
                                            int mn, int row, int rows, int t) {
  if (!mn) {
    if (PAIR) tma_3d_pair(dst, map, bar, t, row); else tma_3d(dst, map, bar, t, row);
  } else {
    for (int q = 0; q < rows; q += 64) {
      if (PAIR) tma_3d_pair(dst + q * 256, map, bar, row + q, t);
      else tma_3d(dst + q * 256, map, bar, row + q, t);
    }
  }
}

// One tile of `out` per unit of work.  PAIR: persistent CTA pairs, 256 x 256.
// Otherwise a 128 x BN tile per cluster of L.split CTAs, each with a part of the
// contraction (none, where it has fewer stages than CTAs); the parts are joined in the order of the ranks.
template <int BN, bool PAIR>
__global__ void __launch_bounds__(kF32Threads, 1) f32_kernel(const __grid_constant__ Launch32 L) {
  using C = Cfg<BN, PAIR>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem = (smem_u32(smem_raw) + 1023) & ~1023u;
  __shared__ __align__(8) uint64_t full[C::kStages], empty[C::kStages];
  __shared__ __align__(8) uint64_t acc_full[C::kBufs], acc_free[C::kBufs], done;
  __shared__ uint32_t tmem_slot;
  __shared__ int failed;
  const volatile int* vfailed = &failed;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t rank = ctarank();
  const int size = PAIR ? 2 : L.split;
  const int first = blockIdx.x / size, step = PAIR ? gridDim.x / 2 : L.units;
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int q = 0; q < C::kBufs; ++q) {
      mbar_init(&acc_full[q], 1);
      mbar_init(&acc_free[q], C::kArrivals);
    }
    mbar_init(&done, 1);
    failed = 0;
    mbar_fence_init();
  }
  if (warp == 0) {
    if (PAIR) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                       smem_u32(&tmem_slot)),
                   "r"(C::kColumns));
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                       smem_u32(&tmem_slot)),
                   "r"(C::kColumns));
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
  }
  fence_before_sync();
  __syncthreads();
  if (PAIR) cluster_sync();  // barriers of both CTAs are ready
  fence_after_sync();
  after_previous();
  const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_slot, 0);
  // the part of a contraction of nk stages
  const auto begin = [&](int nk) { return PAIR ? 0 : static_cast<int>((long long)nk * rank / size); };
  const auto end = [&](int nk) {
    return PAIR ? nk : static_cast<int>((long long)nk * (rank + 1) / size);
  };

  if (warp == kEpi) {  // TMA producer
    const bool one = elect_one();
    unsigned g = 0;
    Ring ring;
    bool ok = true;
    const uint32_t full0 = PAIR ? map_rank(smem_u32(full), 0) : smem_u32(full);
    for (int u = first; ok && u < L.units; u += step) {
      const Prod32& p = L.p[u >= L.units0];
      int ti, tj;
      tile_at(p.tiles_i, p.tiles_j, u >= L.units0 ? u - L.units0 : u, ti, tj);
      const int ja = PAIR ? (tj * 2 + rank) * kTileJ : tj * kTileJ;
      const int ib = PAIR ? (ti * 2 + rank) * C::kRowsB : ti * BN;
      const int a_mn = p.a_mn, b_mn = p.b_mn, k1 = end(p.nk);
      for (int kb = begin(p.nk); kb < k1; ++kb, ++g, ring.next(C::kStages)) {
        const int s = ring.s;
        if (g >= C::kStages && !mbar_wait(&empty[s], ring.parity ^ 1, kSpinLimit, vfailed)) {
          ok = false;
          break;
        }
        if (one) {
          if (!PAIR || rank == 0) mbar_expect_tx(&full[s], (PAIR ? 2 : 1) * C::kStage);
          const uint32_t bar = full0 + s * 8, st = smem + s * C::kStage;
          load_halves<PAIR>(st, &p.a, bar, a_mn, ja, kTileJ, kb * kBK);
          load_halves<PAIR>(st + 2 * kBytesA, &p.b, bar, b_mn, ib, C::kRowsB, kb * kBK);
        }
      }
    }
    if (!ok) failed = 1;
    if (!PAIR || rank == 0)  // the copies in flight land before the CTAs leave
      for (unsigned k = g > C::kStages ? g - C::kStages : 0; k < g; ++k)
        if (!mbar_wait(&full[k % C::kStages], (k / C::kStages) & 1, kSpinLimit)) failed = 1;
  } else if (warp == kEpi + 1) {  // MMA issuer
    if (!PAIR || rank == 0) {
      const bool one = elect_one();
      Ring ring, buf;
      unsigned chunks = 0;
      bool ok = true;
      for (int u = first; ok && u < L.units; u += step) {
        const Prod32& p = L.p[u >= L.units0];
        const int a_mn = p.a_mn, b_mn = p.b_mn, k1 = end(p.nk);
        const Desc da = operand(smem, a_mn, C::kStage, 16384);
        const Desc db = operand(smem + 2 * kBytesA, b_mn, C::kStage, 16384);
        const uint32_t la = (a_mn ? 8192 : kBytesA) >> 4, lb = (b_mn ? 8192 : C::kBytesB / 2) >> 4;
        const uint32_t idesc = p.idesc;
        for (int kb = begin(p.nk); kb < k1;
             ++kb, ++chunks, ring.next(C::kStages), buf.next(C::kBufs)) {
          if (!mbar_wait(&full[ring.s], ring.parity, kSpinLimit, vfailed) ||
              (chunks >= C::kBufs &&
               !mbar_wait(&acc_free[buf.s], buf.parity ^ 1, kDoneLimit, vfailed))) {
            ok = false;
            break;
          }
          fence_after_sync();
          if (one) {
            const uint32_t d = tmem + buf.s * BN;
            const uint64_t a0 = da.base + ring.s * da.stage, b0 = db.base + ring.s * db.stage;
#pragma unroll
            for (int k = 0; k < kBK / 16; ++k) {
              const uint64_t ah = a0 + k * da.k, bh = b0 + k * db.k;
              mma_f16<PAIR>(d, ah + la, bh, idesc, k == 0 ? 0u : 1u);
              mma_f16<PAIR>(d, ah, bh + lb, idesc, 1u);
              mma_f16<PAIR>(d, ah, bh, idesc, 1u);
            }
            if (PAIR) {
              commit_pair(&empty[ring.s]);
              commit_pair(&acc_full[buf.s]);
            } else {
              mma_commit(&empty[ring.s]);
              mma_commit(&acc_full[buf.s]);
            }
          }
        }
      }
      if (!ok) failed = 1;
      if (one) {  // every MMA has finished before tensor memory is freed
        if (PAIR) commit_pair(&done); else mma_commit(&done);
      }
    }
    if (!mbar_wait(&done, 0, kDoneLimit)) failed = 1;
  } else {
    constexpr int kCols = C::kCols;
    const int quad = warp & 3, col0 = (warp >> 2) * kCols;
    const uint32_t base = tmem + ((uint32_t)(quad * 32) << 16) + col0;
    Ring buf;
    bool ok = true;
    for (int u = first; u < L.units; u += step) {
      const Prod32& p = L.p[u >= L.units0];
      int ti, tj;
      tile_at(p.tiles_i, p.tiles_j, u >= L.units0 ? u - L.units0 : u, ti, tj);
      const int j0 = (PAIR ? (tj * 2 + rank) * kTileJ : tj * kTileJ) + quad * 32;
      const int i0 = ti * BN + col0;
      const int chunks = end(p.nk) - begin(p.nk);
      float acc[kCols];
#pragma unroll
      for (int k = 0; k < kCols; ++k) acc[k] = 0.f;
      for (int kb = 0; ok && kb < chunks; ++kb, buf.next(C::kBufs)) {
        ok = __all_sync(0xffffffffu, mbar_wait(&acc_full[buf.s], buf.parity, kDoneLimit, vfailed));
        if (!ok) break;
        fence_after_sync();
#pragma unroll
        for (int c = 0; c < kCols; c += 16) {
          uint32_t r[16];
          tmem_ld16(base + buf.s * BN + c, r);
          tmem_wait_ld(r);
#pragma unroll
          for (int k = 0; k < 16; ++k)
            acc[c + k] = __fadd_rn(acc[c + k], __uint_as_float(r[k]));
        }
        fence_before_sync();
        __syncwarp();
        if (lane == 0) {
          if (PAIR)
            arrive_leader(&acc_free[buf.s]);
          else
            mbar_arrive(&acc_free[buf.s]);
        }
      }
      if (!ok) {
#pragma unroll
        for (int k = 0; k < kCols; ++k) acc[k] = NAN;
      }
      if (!PAIR && size > 1) {  // partial sums where the stages were
#pragma unroll
        for (int k = 0; k < kCols; ++k)
          asm volatile("st.shared.f32 [%0], %1;" ::"r"(
                           smem + ((col0 + k) * kTileJ + quad * 32 + lane) * 4),
                       "f"(acc[k])
                       : "memory");
        break;
      }
      const int I = p.I, J = p.J, j = j0 + (lane & ~3);
      const int ea = j0 + lane < J ? scale_exp(__ldg(p.most_a + j0 + lane)) : 0;
      float bias[4];
      bias_at<float>(p.epi, J, j, bias);
#pragma unroll
      for (int c = 0; c < kCols; c += 16) {
        if (i0 + c < I) {  // warp-uniform
          const int eb = i0 + c + (lane & 15) < I
                             ? scale_exp(__ldg(p.most_b + i0 + c + (lane & 15))) : 0;
          Residual<float, 4> res;
          res.fetch(p.epi, I, J, i0 + c + (lane & 3), j);
          float v[16];
#pragma unroll
          for (int k = 0; k < 16; ++k)
            v[k] = scaled(acc[c + k], ea + __shfl_sync(0xffffffffu, eb, k));
          transpose4(v, lane);
          emit<float, 4>(p.epi, I, J, i0 + c + (lane & 3), j, bias, v, res);
        }
      }
    }
    if (!ok) failed = 1;
  }
  fence_before_sync();
  __syncthreads();
  if (PAIR || size > 1) cluster_sync();
  if (!PAIR && size > 1) {
    if (warp < kEpi) {
      const Prod32& p = L.p[first >= L.units0];
      int ti, tj;
      tile_at(p.tiles_i, p.tiles_j, first >= L.units0 ? first - L.units0 : first, ti, tj);
      const Epilogue e = p.epi;
      const int i0 = ti * BN, j = tj * kTileJ + lane * 4;
      const int columns = min(BN, p.I - i0);
      float bias[4];
      int ea[4];
      bias_at<float>(e, p.J, j, bias);
#pragma unroll
      for (int k = 0; k < 4; ++k) ea[k] = j + k < p.J ? scale_exp(__ldg(p.most_a + j + k)) : 0;
      for (int c = rank * kEpi + warp; c < columns; c += size * kEpi) {
        const uint32_t at = smem + (c * kTileJ + lane * 4) * 4;
        float v[4] = {};
        for (int k = 0; k < size; ++k) {
          const float4 t = peer_f32x4(map_rank(at, k));
          v[0] += t.x, v[1] += t.y, v[2] += t.z, v[3] += t.w;
        }
        const int eb = scale_exp(__ldg(p.most_b + i0 + c));
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = scaled(v[k], ea[k] + eb);
        Residual<float, 1> res;
        res.fetch(e, p.I, p.J, i0 + c, j);
        emit<float, 1>(e, p.I, p.J, i0 + c, j, bias, v, res);
      }
    }
    cluster_sync();  // no CTA leaves while its partial sums are read
  }
  if (warp == 0) {
    if (PAIR)
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                   "r"(C::kColumns));
    else
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                   "r"(C::kColumns));
  }
  if (threadIdx.x == 0 && failed) atomicExch(&g_f32_fault, 1);
}

// ---- host ----
// M N K from which the tensor cores are used.  Forward: 64 x 1024 x 1024 (2^26) 12.6
// us against 15.4 on the FP32 units, 64 x 512 x 512 9.9 against 5.8.  Backward, with
// two more launches: 146 x 800 x 810 (2^26.5) 40 against 48, 300 x 300 x 1000 28
// against 36, 512 x 512 x 256 (2^26) 28 against 26, 128 x 512 x 512 30 against 20.
constexpr long long kTcLeast = 1LL << 26;

long long pad8(long long n) { return (n + 7) / 8 * 8; }
size_t up256(size_t n) { return (n + 255) / 256 * 256; }
size_t halves_bytes(long long rows, long long cols) { return up256(rows * pad8(cols) * 4); }

// Both halves of a row-major (rows x cols) operand: planes of rows x ld.
struct Halves {
  __half* p;
  int rows, cols;
  long long ld, plane;
  uint32_t* most;  // of the rows (or columns) that the product does not sum over
  bool mn;
};

struct Arena {
  uint8_t* at;
  template <typename T>
  T* take(size_t bytes) {
    T* p = reinterpret_cast<T*>(at);
    at += up256(bytes);
    return p;
  }
};

Halves make_halves(Arena& ws, int rows, int cols, bool mn, uint32_t* most) {
  Halves h{ws.take<__half>(halves_bytes(rows, cols)), rows, cols, pad8(cols), 0, most, mn};
  h.plane = h.rows * h.ld;
  return h;
}

int make_map(CUtensorMap* map, const Halves& h, int box_rows, const char* who) {
  const auto fn = encode_fn();
  if (!fn) return fail(VCB_ERR_CUDA, "%s: cuTensorMapEncodeTiled unavailable", who);
  const cuuint64_t dims[3] = {(cuuint64_t)h.cols, (cuuint64_t)h.rows, 2};
  const cuuint64_t strides[2] = {(cuuint64_t)h.ld * 2, (cuuint64_t)h.plane * 2};
  const cuuint32_t box[3] = {kBK, (cuuint32_t)box_rows, 2}, estr[3] = {1, 1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, h.p, dims, strides, box, estr,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(VCB_ERR_CUDA, "%s: tensor map encode failed (%d)", who, (int)r);
  return VCB_OK;
}

struct Plan32 {
  bool pair;
  int bn, split;
  double cycles;
};

// As the 16-bit products' plan: rounds of tiles over the SMs times the stages'
// cycles (12 MMAs: 1,536 for a pair's tile, 768 for 64 or 128 columns), plus start
// and epilogue.
struct Shape {
  int I, J, T;
};

// CTAs at a time in clusters of 1, 2, 4 and 8.
int slots_of(int size) {
  static const std::array<int, 4> slots = [] {
    using C = Cfg<128, false>;
    std::array<int, 4> n;
    for (int k = 0; k < 4; ++k)
      n[k] = cluster_slots(f32_kernel<128, false>, kF32Threads, C::kSmem, 1 << k);
    return n;
  }();
  return slots[size == 1 ? 0 : size == 2 ? 1 : size == 4 ? 2 : 3];
}

Plan32 plan_of(std::initializer_list<Shape> products) {
  const int sms = sm_count();
  const auto ceil = [](long long a, long long b) { return (a + b - 1) / b; };
  long long nk = 1, pairs = 0;
  for (const Shape& s : products) {
    nk = std::max(nk, ceil(s.T, kBK));
    pairs += ceil(s.I, 256) * ceil(s.J, 256);
  }
  Plan32 best{true, 256, 1, static_cast<double>(ceil(pairs, sms / 2)) * (nk * 1540 + 4000) + 4000};
  for (int bn : {64, 128}) {
    long long tiles = 0;
    for (const Shape& s : products) tiles += ceil(s.I, bn) * ceil(s.J, kTileJ);
    for (int split : {1, 2, 4, 8}) {
      if (split > nk) break;
      const double t = static_cast<double>(ceil(tiles * split, slots_of(split))) *
                           (ceil(nk, split) * (bn == 64 ? 800 : 1000) + 4000 + 20.0 * bn) +
                       (split > 1 ? 1500 + 8.0 * bn : 0);
      if (t < best.cycles) best = {false, bn, split, t};
    }
  }
  return best;
}

int set_prod(Prod32& r, int I, int J, int T, const Halves& a, const Halves& b, const Plan32& plan,
             const Epilogue& epi, const char* who) {
  r.I = I, r.J = J;
  r.a_mn = a.mn, r.b_mn = b.mn;
  const int tj = plan.pair ? 256 : kTileJ;
  r.tiles_j = (J + tj - 1) / tj;
  r.tiles_i = (I + plan.bn - 1) / plan.bn;
  r.nk = std::max(1, (T + kBK - 1) / kBK);
  r.idesc = idesc_16(VCB_F16, tj, plan.bn, a.mn, b.mn);
  r.most_a = a.most, r.most_b = b.most;
  r.epi = epi;
  r.epi.vec = vector_rows(epi, 4);
  int rc = make_map(&r.a, a, a.mn ? kBK : kTileJ, who);
  if (!rc) rc = make_map(&r.b, b, b.mn ? kBK : plan.pair ? kTileJ : plan.bn, who);
  return rc;
}

template <int BN, bool PAIR>
int launch(const Launch32& L, bool chained, cudaStream_t st, const char* who) {
  using C = Cfg<BN, PAIR>;
  g_launched = true;
  const auto kernel = f32_kernel<BN, PAIR>;
  const int rc = ensure_smem(reinterpret_cast<const void*>(kernel), C::kSmem);
  if (rc) return rc;
  const int size = PAIR ? 2 : L.split;
  return launch_clusters(kernel, L, size * (PAIR ? std::min(L.units, sm_count() / 2) : L.units),
                         kF32Threads, C::kSmem, size, chained, st, who);
}

int launch_plan(const Launch32& L, const Plan32& plan, bool chained, cudaStream_t st,
                const char* who) {
  if (plan.pair) return launch<256, true>(L, chained, st, who);
  return plan.bn == 64 ? launch<64, false>(L, chained, st, who)
                       : launch<128, false>(L, chained, st, who);
}

bool vec16(const void* p, long long ld) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 4 == 0;
}

bool fits(long long M, long long N, long long K, long long least) {
  const long long most = 1LL << 28;
  return M * N * K >= least && M < most && N < most && K < most && (M + 63) / 64 * ((N + 127) / 128) < most &&
         (M + 63) / 64 * ((K + 127) / 128) < most && (N + 63) / 64 * ((K + 127) / 128) < most;
}

}  // namespace

bool f32_forward_fits(const Fwd& f) { return f.type == VCB_F32 && fits(f.M, f.N, f.K, kTcLeast); }

size_t f32_forward_bytes(int M, int N, int K) {
  if (!fits(M, N, K, kTcLeast)) return 0;
  return halves_bytes(M, K) + halves_bytes(N, K) + up256(M * 4LL) + up256(N * 4LL) + 256;
}

int f32_forward(const Fwd& f, void* ws, cudaStream_t st) {
  const char* who = "vcb_linear_forward";
  Arena arena{reinterpret_cast<uint8_t*>(up256(reinterpret_cast<size_t>(ws)))};
  const Halves w = make_halves(arena, f.N, f.K, false, arena.take<uint32_t>(f.N * 4LL));
  const Halves x = make_halves(arena, f.M, f.K, false, arena.take<uint32_t>(f.M * 4LL));
  RowJobs jobs{};
  const auto job = [](const void* p, long long ld, const Halves& h) {
    return RowJob{static_cast<const float*>(p), ld, h.rows, h.cols, vec16(p, ld), h.p, h.ld,
                  h.plane, h.most};
  };
  jobs.j[0] = job(f.w, f.ldw, w);
  jobs.j[1] = job(f.x, f.ldx, x);
  const long long rows = static_cast<long long>(f.N) + f.M;
  // a warp per row while that keeps a row in registers: what a thread does once is spread
  // over more entries (1000^3 27.6 -> 25.6 us against a CTA per row)
  const auto launch_rows = [&](void (*kernel)(RowJobs), int per) {
    kernel<<<static_cast<unsigned>((rows + per - 1) / per), 256, 0, st>>>(jobs);
  };
  if (f.K <= 512)
    launch_rows(rows_kernel<32, 4>, 8);
  else if (f.K <= 2048)
    launch_rows(rows_kernel<32, 16>, 8);
  else
    launch_rows(rows_kernel<256, 4>, 1);
  int rc = check_launch(who);
  if (rc) return rc;
  const Plan32 plan = plan_of({{f.M, f.N, f.K}});
  Launch32 L{};
  rc = set_prod(L.p[0], f.M, f.N, f.K, w, x, plan,
                {f.y, f.z, f.bias, f.res, f.ldy, f.ldz, f.ldr, f.act, 0}, who);
  if (rc) return rc;
  L.units0 = L.units = L.p[0].tiles_i * L.p[0].tiles_j;
  L.split = plan.split;
  return launch_plan(L, plan, true, st, who);
}

bool f32_backward_fits(const Bwd& b) {
  return b.type == VCB_F32 && (b.dx || b.dw) && fits(b.M, b.N, b.K, kTcLeast);
}

size_t f32_backward_bytes(int M, int N, int K) {
  if (!fits(M, N, K, kTcLeast)) return 0;
  return 2 * halves_bytes(M, N) + halves_bytes(N, K) + halves_bytes(M, K) + up256(M * 4LL) +
         up256(N * 4LL) + 2 * up256(K * 4LL) + 256;
}

int f32_backward(const Bwd& b, void* ws, cudaStream_t st) {
  const char* who = "vcb_linear_backward";
  Arena arena{reinterpret_cast<uint8_t*>(up256(reinterpret_cast<size_t>(ws)))};
  uint32_t* row_most = arena.take<uint32_t>(b.M * 4LL);
  const Halves dzr = make_halves(arena, b.M, b.N, false, row_most);
  const Halves dzc = make_halves(arena, b.M, b.N, true, arena.take<uint32_t>(b.N * 4LL));
  const Halves w = make_halves(arena, b.N, b.K, true, arena.take<uint32_t>(b.K * 4LL));
  const Halves x = make_halves(arena, b.M, b.K, true, arena.take<uint32_t>(b.K * 4LL));
  ColJobs jobs{};
  long long strips = 0, wide = 0, tall = 0;
  const auto add = [&](const void* p, long long ld, const Halves& h) -> ColJob& {
    ColJob& q = jobs.j[jobs.count++];
    q.src = static_cast<const float*>(p);
    q.ld = ld, q.rows = h.rows, q.cols = h.cols, q.vec = vec16(p, ld);
    q.col_most = h.most, q.by_col = h.p, q.ldh = h.ld, q.plane = h.plane;
    strips += (h.cols + 31) / 32;
    wide += (h.cols + 127) / 128;
    tall = std::max(tall, q.rows);
    return q;
  };
  ColJob& dz = add(b.dy, b.lddy, dzc);
  dz.act = b.act, dz.z = static_cast<const float*>(b.z), dz.ldz = b.ldz;
  if (b.act != VCB_ACT_NONE) dz.vec = dz.vec && vec16(b.z, b.ldz);
  dz.sum = static_cast<float*>(b.db);
  if (b.dx) dz.by_row = dzr.p, dz.row_most = row_most;
  if (!b.dw) dz.by_col = nullptr;
  if (b.dx) add(b.w, b.ldw, w);
  if (b.dw) add(b.x, b.ldx, x);
  const long long blocks = (tall + kHalvesRows - 1) / kHalvesRows;
  if (strips * 8 > 0x7fffffffLL || wide * blocks > 0x7fffffffLL)
    return fail(VCB_ERR_UNSUPPORTED, "%s: M=%d N=%d K=%d", who, b.M, b.N, b.K);
  cudaError_t e = cudaSuccess;
  if (b.dx) e = cudaMemsetAsync(row_most, 0, b.M * 4LL, st);
  if (e != cudaSuccess) return cuda_fail(e, who);
  jobs.cluster = 1;  // a CTA's step is 128 rows
  while (jobs.cluster < 8 && tall > 128 * jobs.cluster) jobs.cluster *= 2;
  int rc = launch_clusters(scales_kernel, jobs, static_cast<unsigned>(strips * jobs.cluster),
                           kStripThreads, 0, jobs.cluster, false, st, who);
  if (rc) return rc;
  jobs.wide = static_cast<int>(wide);
  rc = launch_clusters(halves_kernel, jobs, static_cast<unsigned>(wide * blocks), kStripThreads, 0,
                       1, true, st, who);
  if (rc) return rc;
  const Epilogue ex{b.dx, nullptr, nullptr, nullptr, b.lddx, 0, 0, VCB_ACT_NONE, 0};
  const Epilogue ew{b.dw, nullptr, nullptr, nullptr, b.lddw, 0, 0, VCB_ACT_NONE, 0};
  const Shape shape_x{b.M, b.K, b.N}, shape_w{b.N, b.K, b.M};
  Plan32 px = plan_of({shape_x}), pw = plan_of({shape_w});
  const Plan32 both = plan_of({shape_x, shape_w});
  // One launch for both products unless their shapes want different cuts by more than
  // a launch costs.
  const bool together = b.dx && b.dw && both.cycles < px.cycles + pw.cycles + 4000;
  if (together) px = pw = both;
  Launch32 L{};
  if (b.dx) {
    rc = set_prod(L.p[0], b.M, b.K, b.N, w, dzr, px, ex, who);
    if (rc) return rc;
    L.units0 = L.units = L.p[0].tiles_i * L.p[0].tiles_j;
    L.split = px.split;
    if (!together) {
      rc = launch_plan(L, px, true, st, who);
      if (rc || !b.dw) return rc;
      L.units0 = L.units = 0;
    }
  }
  Prod32& p = L.p[together ? 1 : 0];
  rc = set_prod(p, b.N, b.K, b.M, x, dzc, pw, ew, who);
  if (rc) return rc;
  L.units += p.tiles_i * p.tiles_j;
  if (!together) L.units0 = L.units;
  L.split = pw.split;
  return launch_plan(L, pw, together || !b.dx, st, who);
}

int f32_fault_take(cudaStream_t st, int* was_set) {
  *was_set = 0;
  if (!g_launched) return VCB_OK;
  int h = 0;
  cudaError_t e =
      cudaMemcpyFromSymbolAsync(&h, g_f32_fault, sizeof(int), 0, cudaMemcpyDeviceToHost, st);
  if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  if (e == cudaSuccess && h) {
    const int zero = 0;
    e = cudaMemcpyToSymbolAsync(g_f32_fault, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, st);
    if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  }
  *was_set = h;
  return cuda_fail(e, "vcb_fault_check");
}

}  // namespace lin
}  // namespace vcb
