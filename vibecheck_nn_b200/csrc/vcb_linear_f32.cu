// The linear layer's float32 products on the tensor cores.
//
// A float32 number is the sum of three bfloat16 numbers,
//   b1 = bf16(x),  b2 = bf16(x - b1),  b3 = x - b1 - b2,
// exactly (24 bits in three times 8) while |x| >= 2^-110; below that b3, then b2,
// end at bfloat16's smallest step, 2^-133.  Each has float32's exponents, so
// entries of any size share a row.  The tensor cores form
//   b1 b1' + (b1 b2' + b2 b1') + (b2 b2' + b1 b3' + b3 b1')
// with exact products and fp32 accumulators.  b2 b3' + b3 b2' + b3 b3' are left out:
// below 2^-24 |x x'|, what rounding one product to float32 may lose.  So an output's
// error is bounded by its own sum of |x x'|, as that of a float32 sum is, whatever
// else lies in the rows.  (Two fp16 halves under one scale per row took three products
// instead of six, but their error went by the row's largest entry: a column at 2^30
// that met zero weights cost the other columns three digits.)  An infinite or NaN
// entry makes the outputs that it meets infinite or NaN: its products with b2' and
// b3', which may be 0, are formed too.
//
// The tensor cores drop low-order bits in every accumulation.  So an accumulator
// in tensor memory takes one 64-deep stage (24 MMAs) only, the smaller products
// first, and the epilogue warps add the stages' sums in registers, rounding to
// nearest, while the next stage fills the other accumulator.
//
// Measured: 4096^3 forward 605 us in short bursts (227 TFLOP/s of fp32 products, 1,360
// of bfloat16), 680 us back to back under the power cap, both gradients 1,065 us;
// largest error 1.7e-7 of the largest output, against 1.1e-6 of an fp32 sum.
//
// Preparation is bound by HBM: one launch reads each operand once and writes its
// three parts (backward: dz = dy act'(z) and db in strips of columns, W and X flat
// beside them).  The parts of dz serve both products, read along either index.
// Then products as in vcb_linear_tc.cu: f32_kernel<256, true> in CTA pairs for
// large ones, f32_kernel<64 / 128, false> with the contraction cut over a cluster
// for the rest.
#include <algorithm>
#include <array>
#include <initializer_list>

#include "vcb_linear_tc.cuh"

namespace vcb {
namespace lin {
namespace {

constexpr int kParts = 3;
constexpr uint32_t kLargest16 = 0x7F7F0000u;  // of bfloat16, as a float's bits

// The parts of four entries.  What would round up to infinity is cut instead; an
// infinite entry has no remainder.
__device__ __forceinline__ void split4(const float (&x)[4], uint2 (&part)[kParts]) {
  uint32_t w[kParts][2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    float r[2] = {x[2 * k], x[2 * k + 1]}, top[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t bits = __float_as_uint(r[i]), size = bits & 0x7FFFFFFFu;
      top[i] = size > kLargest16 && size < 0x7F800000u
                   ? __uint_as_float(kLargest16 | (bits & 0x80000000u)) : r[i];
    }
#pragma unroll
    for (int p = 0; p < kParts; ++p) {
      const __nv_bfloat162 h =
          p ? __floats2bfloat162_rn(r[0], r[1]) : __floats2bfloat162_rn(top[0], top[1]);
      const uint32_t u = w[p][k] = *reinterpret_cast<const uint32_t*>(&h);
      const float back[2] = {__uint_as_float(u << 16), __uint_as_float(u & 0xFFFF0000u)};
#pragma unroll
      for (int i = 0; i < 2; ++i) r[i] = isinf(back[i]) ? 0.f : r[i] - back[i];
    }
  }
#pragma unroll
  for (int p = 0; p < kParts; ++p) part[p] = make_uint2(w[p][0], w[p][1]);
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

// ---- preparation ----
// A row-major matrix and its parts: `plane` elements apart, rows of ldp (a multiple of
// 8) elements.
struct Matrix {
  const float* src;
  long long ld, rows;
  int cols, vec;
  __nv_bfloat16* parts;
  long long ldp, plane;
};

struct Prep32 {
  Matrix dz;              // in strips of columns (backward); its src is dy
  const float* z;
  float* sum;             // column sums of dz (db), or NULL
  long long ldz;
  int act, strips;        // strips of 32 columns, 0 for none
  int cluster;            // CTAs per strip
  Matrix flat[2];
  int flats;
};

constexpr int kPrepThreads = 256, kPrepWarps = kPrepThreads / 32, kStrip = 32;

// Strips: a cluster of up to 8 CTAs each, a part of the rows per CTA, 8 lanes per
// row; column sums in the order of the ranks.  The remaining CTAs: 8 entries per
// thread, neighbouring threads on neighbouring entries of all rows.
__global__ void __launch_bounds__(kPrepThreads, 4) parts_kernel(const __grid_constant__ Prep32 a) {
  __shared__ float part[kPrepWarps][kStrip], mine[kStrip];
  let_next_start();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int size = a.cluster, strip = blockIdx.x / size;
  if (strip < a.strips) {
    const Matrix& q = a.dz;
    const int rank = blockIdx.x % size, c = strip * kStrip + (lane & 7) * 4;
    const long long r0 = q.rows * rank / size, r1 = q.rows * (rank + 1) / size;
    float sum[4] = {};
    constexpr int U = 4, W = kPrepWarps * 4;  // rows in flight per lane, rows of a CTA's step
    for (long long base = r0 + warp * 4 + (lane >> 3); base < r1; base += U * W) {
      float v[U][4], t[U][4];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const long long r = base + u * W;
        if (r >= r1) continue;
        row4(q.src + r * q.ld, c, q.cols, q.vec, v[u]);
        if (a.act != VCB_ACT_NONE) row4(a.z + r * a.ldz, c, q.cols, q.vec, t[u]);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const long long r = base + u * W;
        if (r >= r1) continue;
        if (a.act != VCB_ACT_NONE) act_grads(v[u], t[u], a.act);
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[i] += v[u][i];
        if (c < q.cols) {
          uint2 p[kParts];
          split4(v[u], p);
          __nv_bfloat16* at = q.parts + r * q.ldp + c;
#pragma unroll
          for (int k = 0; k < kParts; ++k) *reinterpret_cast<uint2*>(at + k * q.plane) = p[k];
        }
      }
    }
    if (!a.sum) return;  // the same for all CTAs
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int k = 8; k < 32; k *= 2) sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], k);
      if (lane < 8) part[warp][lane * 4 + i] = sum[i];
    }
    __syncthreads();
    if (threadIdx.x < kStrip) {
      float s = 0.f;
      for (int w = 0; w < kPrepWarps; ++w) s += part[w][threadIdx.x];
      mine[threadIdx.x] = s;
    }
    cluster_sync();
    const int col = strip * kStrip + threadIdx.x;
    if (rank == 0 && threadIdx.x < kStrip && col < q.cols) {
      float s = 0.f;
      for (int k = 0; k < size; ++k) s += peer_f32(map_rank(smem_u32(mine + threadIdx.x), k));
      a.sum[col] = s;
    }
    cluster_sync();  // no CTA leaves while its sums are read
    return;
  }
  const long long first = (long long)(blockIdx.x - a.strips * size) * kPrepThreads + threadIdx.x;
  const long long step = (long long)(gridDim.x - a.strips * size) * kPrepThreads;
  for (int m = 0; m < a.flats; ++m) {
    const Matrix& q = a.flat[m];
    const int nv = (q.cols + 7) / 8;
    long long row = first / nv;
    int v = static_cast<int>(first - row * nv);
    const long long down = step / nv;
    const int right = static_cast<int>(step - down * nv);
    constexpr int U = 2;  // vectors of 8 in flight
    while (row < q.rows) {
      float x[U][2][4];
      __nv_bfloat16* out[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        out[u] = row < q.rows ? q.parts + row * q.ldp + v * 8 : nullptr;
        if (out[u]) {
          row4(q.src + row * q.ld, v * 8, q.cols, q.vec, x[u][0]);
          row4(q.src + row * q.ld, v * 8 + 4, q.cols, q.vec, x[u][1]);
        }
        row += down, v += right;
        if (v >= nv) v -= nv, ++row;
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (!out[u]) continue;
        uint2 lo[kParts], hi[kParts];
        split4(x[u][0], lo);
        split4(x[u][1], hi);
#pragma unroll
        for (int k = 0; k < kParts; ++k)
          *reinterpret_cast<uint4*>(out[u] + k * q.plane) =
              make_uint4(lo[k].x, lo[k].y, hi[k].x, hi[k].y);
      }
    }
  }
}

// ---- products ----
struct alignas(64) Prod32 {
  CUtensorMap a, b;  // (64, rows, parts) boxes
  int J, I, a_mn, b_mn, tiles_j, tiles_i, nk;
  uint32_t idesc;
  Epilogue epi;
};

struct Launch32 {
  Prod32 p[2];
  int units0, units, split;
  int* fault;
};

// Sixteen epilogue warps: what they do at a tile's end (activation, stores)
// runs beside two stages of the next tile's MMAs only, so it is spread as wide as
// registers allow.
constexpr int kEpi = 16, kF32Threads = (kEpi + 2) * 32;

template <int BN, bool PAIR>
struct Cfg {
  static constexpr int kRowsB = PAIR ? BN / 2 : BN;
  static constexpr int kBytesB = kParts * kRowsB * 128;
  static constexpr int kStage = kParts * kBytesA + kBytesB;
  static constexpr int kStages = 221184 / kStage;
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

// The parts of an operand's rows.  K-major: all rows of b1, then of b2 and b3.
// MN-major: per 64 rows, 8 KB of each.
constexpr uint32_t kBoxMn = kParts * 8192;
template <bool PAIR>
__device__ __forceinline__ void load_parts(uint32_t dst, const CUtensorMap* map, uint32_t bar,
                                            int mn, int row, int rows, int t) {
  if (!mn) {
    if (PAIR) tma_3d_pair(dst, map, bar, t, row); else tma_3d(dst, map, bar, t, row);
  } else {
    for (int q = 0; q < rows; q += 64) {
      if (PAIR) tma_3d_pair(dst + q / 64 * kBoxMn, map, bar, row + q, t);
      else tma_3d(dst + q / 64 * kBoxMn, map, bar, row + q, t);
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
          load_parts<PAIR>(st, &p.a, bar, a_mn, ja, kTileJ, kb * kBK);
          load_parts<PAIR>(st + kParts * kBytesA, &p.b, bar, b_mn, ib, C::kRowsB, kb * kBK);
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
        const Desc da = operand(smem, a_mn, C::kStage, kBoxMn);
        const Desc db = operand(smem + kParts * kBytesA, b_mn, C::kStage, kBoxMn);
        // from a part to the next
        const uint32_t pa = (a_mn ? 8192 : kBytesA) >> 4;
        const uint32_t pb = (b_mn ? 8192 : C::kBytesB / kParts) >> 4;
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
            // the smallest products first: what their sums lose is of their size
#pragma unroll
            for (int sum = kParts - 1; sum >= 0; --sum) {
#pragma unroll
              for (int p = 0; p <= sum; ++p) {
#pragma unroll
                for (int k = 0; k < kBK / 16; ++k)
                  mma_f16<PAIR>(d, a0 + p * pa + k * da.k, b0 + (sum - p) * pb + k * db.k, idesc,
                                sum == kParts - 1 && p == 0 && k == 0 ? 0u : 1u);
              }
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
      float bias[4];
      bias_at<float>(p.epi, J, j, bias);
#pragma unroll
      for (int c = 0; c < kCols; c += 16) {
        if (i0 + c < I) {  // warp-uniform
          Residual<float, 4> res;
          res.fetch(p.epi, I, J, i0 + c + (lane & 3), j);
          float v[16];
#pragma unroll
          for (int k = 0; k < 16; ++k) v[k] = acc[c + k];
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
      bias_at<float>(e, p.J, j, bias);
      for (int c = rank * kEpi + warp; c < columns; c += size * kEpi) {
        const uint32_t at = smem + (c * kTileJ + lane * 4) * 4;
        float v[4] = {};
        for (int k = 0; k < size; ++k) {
          const float4 t = peer_f32x4(map_rank(at, k));
          v[0] += t.x, v[1] += t.y, v[2] += t.z, v[3] += t.w;
        }
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
  if (threadIdx.x == 0 && failed) atomicOr(L.fault, kFaultLinear);
}

// ---- host ----
// M N K from which the tensor cores are used.  Forward: 64 x 1024 x 1024 (2^26) 17 us
// against 21 on the FP32 units, 512 x 512 x 256 (2^26) 15 against 22, but 64 x 512 x 512
// 15 against 12 and 128 x 512 x 512 (2^25) 17 against 16.  Both gradients: 146 x 800 x
// 810 (2^26.5) 26 against 41, 512 x 512 x 256 20 against 32, 128 x 512 x 512 19 against
// 21, 20000 x 50 x 50 (2^25.6) 106 against 90.
constexpr long long kTcLeast = 1LL << 26;

long long pad8(long long n) { return (n + 7) / 8 * 8; }
size_t up256(size_t n) { return (n + 255) / 256 * 256; }
size_t parts_bytes(long long rows, long long cols) {
  return up256(rows * pad8(cols) * 2 * kParts);
}

struct Arena {
  uint8_t* at;
  template <typename T>
  T* take(size_t bytes) {
    T* p = reinterpret_cast<T*>(at);
    at += up256(bytes);
    return p;
  }
};

Matrix matrix(Arena& ws, const void* p, long long ld, int rows, int cols) {
  const bool vec = reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 4 == 0;
  return {static_cast<const float*>(p), ld, rows, cols, vec,
          ws.take<__nv_bfloat16>(parts_bytes(rows, cols)), pad8(cols), rows * pad8(cols)};
}

int make_map(CUtensorMap* map, const Matrix& h, int box_rows, const char* who) {
  const auto fn = encode_fn();
  if (!fn) return fail(VCB_ERR_CUDA, "%s: cuTensorMapEncodeTiled unavailable", who);
  const cuuint64_t dims[3] = {(cuuint64_t)h.cols, (cuuint64_t)h.rows, kParts};
  const cuuint64_t strides[2] = {(cuuint64_t)h.ldp * 2, (cuuint64_t)h.plane * 2};
  const cuuint32_t box[3] = {kBK, (cuuint32_t)box_rows, kParts}, estr[3] = {1, 1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, h.parts, dims, strides, box, estr,
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
// cycles, plus start and epilogue.  The cycles are measured (24 MMAs alone: 3,072 for a
// pair's tile, 1,536 for 64 or 128 columns; the operands' way from L2 and the clock
// under load add the rest).
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
  Plan32 best{true, 256, 1, static_cast<double>(ceil(pairs, sms / 2)) * (nk * 4200 + 4000) + 4000};
  for (int bn : {64, 128}) {
    long long tiles = 0;
    for (const Shape& s : products) tiles += ceil(s.I, bn) * ceil(s.J, kTileJ);
    for (int split : {1, 2, 4, 8}) {
      if (split > nk) break;
      const double t = static_cast<double>(ceil(tiles * split, slots_of(split))) *
                           (ceil(nk, split) * (bn == 64 ? 1950 : 2700) + 4000 + 20.0 * bn) +
                       (split > 1 ? 1500 + 8.0 * bn : 0);
      if (t < best.cycles) best = {false, bn, split, t};
    }
  }
  return best;
}

// mn: the operand is contiguous along its row index, not along the contraction.
int set_prod(Prod32& r, int I, int J, int T, const Matrix& a, bool a_mn, const Matrix& b, bool b_mn,
             const Plan32& plan, const Epilogue& epi, const char* who) {
  r.I = I, r.J = J;
  r.a_mn = a_mn, r.b_mn = b_mn;
  const int tj = plan.pair ? 256 : kTileJ;
  r.tiles_j = (J + tj - 1) / tj;
  r.tiles_i = (I + plan.bn - 1) / plan.bn;
  r.nk = std::max(1, (T + kBK - 1) / kBK);
  r.idesc = idesc_16(VCB_BF16, tj, plan.bn, a_mn, b_mn);
  r.epi = epi;
  r.epi.vec = vector_rows(epi, 4);
  int rc = make_map(&r.a, a, a_mn ? kBK : kTileJ, who);
  if (!rc) rc = make_map(&r.b, b, b_mn ? kBK : plan.pair ? kTileJ : plan.bn, who);
  return rc;
}

template <int BN, bool PAIR>
int launch(Launch32& L, bool chained, cudaStream_t st, const char* who) {
  using C = Cfg<BN, PAIR>;
  const auto kernel = f32_kernel<BN, PAIR>;
  int rc = fault_word(&L.fault);
  if (!rc) rc = ensure_smem(reinterpret_cast<const void*>(kernel), C::kSmem);
  if (rc) return rc;
  const int size = PAIR ? 2 : L.split;
  return launch_clusters(kernel, L, size * (PAIR ? std::min(L.units, sm_count() / 2) : L.units),
                         kF32Threads, C::kSmem, size, chained, st, who);
}

int launch_plan(Launch32& L, const Plan32& plan, bool chained, cudaStream_t st,
                const char* who) {
  if (plan.pair) return launch<256, true>(L, chained, st, who);
  return plan.bn == 64 ? launch<64, false>(L, chained, st, who)
                       : launch<128, false>(L, chained, st, who);
}

int launch_prep(Prep32& a, cudaStream_t st, const char* who) {
  long long vectors = 0;
  for (int k = 0; k < a.flats; ++k)
    vectors = std::max(vectors, a.flat[k].rows * ((a.flat[k].cols + 7LL) / 8));
  const long long ctas =
      std::min<long long>((vectors + kPrepThreads - 1) / kPrepThreads, 4LL * sm_count());
  a.cluster = 1;  // a CTA's step is 128 rows
  while (a.strips && a.cluster < 8 && a.dz.rows > 128 * a.cluster) a.cluster *= 2;
  const long long grid = (a.strips + (ctas + a.cluster - 1) / a.cluster) * a.cluster;
  return launch_clusters(parts_kernel, a, static_cast<unsigned>(grid), kPrepThreads, 0, a.cluster,
                         false, st, who);
}

bool fits(long long M, long long N, long long K, long long least) {
  const long long most = 1LL << 28;
  return M * N * K >= least && M < most && N < most && K < most && (M + 63) / 64 * ((N + 127) / 128) < most &&
         (M + 63) / 64 * ((K + 127) / 128) < most && (N + 63) / 64 * ((K + 127) / 128) < most;
}

}  // namespace

bool f32_forward_fits(const Fwd& f) { return f.type == VCB_F32 && fits(f.M, f.N, f.K, kTcLeast); }

size_t f32_forward_bytes(int M, int N, int K) {
  return fits(M, N, K, kTcLeast) ? parts_bytes(M, K) + parts_bytes(N, K) + 256 : 0;
}

int f32_forward(const Fwd& f, void* ws, cudaStream_t st) {
  const char* who = "vcb_linear_forward";
  Arena arena{reinterpret_cast<uint8_t*>(up256(reinterpret_cast<size_t>(ws)))};
  Prep32 prep{};
  const Matrix w = matrix(arena, f.w, f.ldw, f.N, f.K), x = matrix(arena, f.x, f.ldx, f.M, f.K);
  prep.flat[0] = w, prep.flat[1] = x, prep.flats = 2;
  int rc = launch_prep(prep, st, who);
  if (rc) return rc;
  const Plan32 plan = plan_of({{f.M, f.N, f.K}});
  Launch32 L{};
  rc = set_prod(L.p[0], f.M, f.N, f.K, w, false, x, false, plan,
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
  return parts_bytes(M, N) + parts_bytes(N, K) + parts_bytes(M, K) + 256;
}

int f32_backward(const Bwd& b, void* ws, cudaStream_t st) {
  const char* who = "vcb_linear_backward";
  Arena arena{reinterpret_cast<uint8_t*>(up256(reinterpret_cast<size_t>(ws)))};
  Prep32 prep{};
  const Matrix dz = prep.dz = matrix(arena, b.dy, b.lddy, b.M, b.N);
  const Matrix w = matrix(arena, b.w, b.ldw, b.N, b.K), x = matrix(arena, b.x, b.ldx, b.M, b.K);
  prep.z = static_cast<const float*>(b.z), prep.ldz = b.ldz, prep.act = b.act;
  if (b.act != VCB_ACT_NONE)
    prep.dz.vec = dz.vec && reinterpret_cast<uintptr_t>(b.z) % 16 == 0 && b.ldz % 4 == 0;
  prep.sum = static_cast<float*>(b.db);
  prep.strips = (b.N + kStrip - 1) / kStrip;
  if (b.dx) prep.flat[prep.flats++] = w;
  if (b.dw) prep.flat[prep.flats++] = x;
  int rc = launch_prep(prep, st, who);
  if (rc) return rc;
  const Epilogue ex{b.dx, nullptr, nullptr, nullptr, b.lddx, 0, 0, VCB_ACT_NONE, 0};
  const Epilogue ew{b.dw, nullptr, nullptr, nullptr, b.lddw, 0, 0, VCB_ACT_NONE, 0};
  const Shape shape_x{b.M, b.K, b.N}, shape_w{b.N, b.K, b.M};
  Plan32 px = plan_of({shape_x}), pw = plan_of({shape_w});
  const Plan32 both = plan_of({shape_x, shape_w});
  // One launch for both products unless their shapes want different cuts by more than
  // a launch costs.
  const bool together = b.dx && b.dw && both.cycles < px.cycles + pw.cycles + 9000;
  if (together) px = pw = both;
  Launch32 L{};
  if (b.dx) {
    rc = set_prod(L.p[0], b.M, b.K, b.N, w, true, dz, false, px, ex, who);
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
  rc = set_prod(p, b.N, b.K, b.M, x, true, dz, true, pw, ew, who);
  if (rc) return rc;
  L.units += p.tiles_i * p.tiles_j;
  if (!together) L.units0 = L.units;
  L.split = pw.split;
  return launch_plan(L, pw, together || !b.dx, st, who);
}

}  // namespace lin
}  // namespace vcb
