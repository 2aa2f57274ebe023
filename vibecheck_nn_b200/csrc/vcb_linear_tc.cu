// The linear layer's products in 16-bit types on the tensor cores
// (tcgen05.mma kind::f16, fp32 accumulators in tensor memory).
//
// Every product of the layer is  out(i, j) = sum_t B(i, t) A(j, t)  with j the
// contiguous index of the output:
//   forward  Y  (i = m, j = n, t = k):  A = W    B = X
//   dX          (i = m, j = k, t = n):  A = W^T  B = dZ
//   dW          (i = n, j = k, t = m):  A = X^T  B = dZ^T
// The MMA's M rows (tensor memory lanes) are the j's: neighbouring lanes then
// store neighbouring elements of a row of the output, so the epilogue needs no
// staging, a bias is one register per lane, and few rows i cost only a narrow
// MMA (N = 16 for up to 16 tokens).  Transposed operands are read as they lie:
// a 16-bit operand of tcgen05.mma may be contiguous along its row index
// ("MN-major") as well as along t ("K-major"); TMA brings 64 x 64 boxes with
// 128-byte swizzle for the former.
//
// Two kernels:
//  * pair_kernel, large products: two CTAs per 256 x 256 tile
//    (cta_group::2), persistent, six 32 KB stages per CTA, two accumulators in
//    tensor memory so that a tile's epilogue overlaps the next tile's MMAs.  A
//    single CTA's 128 x 256 tile would need 96 B per cycle and SM from L2 at
//    full MMA rate, the pair needs 64.
//  * split_kernel, everything else: a 128 x bn tile, its contraction cut over
//    the up to 8 CTAs of a cluster when there are few tiles (few tokens: the
//    weight is what is read, and every SM takes part in reading it).  The
//    partial sums are joined over distributed shared memory in the order of
//    the ranks: no atomics, no second launch, the same bits every time.
// A contraction that would give one accumulator more than kLongest stages goes to
// sum_kernel (vcb_linear_sum.cuh), which empties accumulators on the way.
// Measured: bf16 8192 x 8192 x 4096 with GELU, residual and pre-activation 350 us in
// short bursts (1,570 TFLOP/s, 93 % of the library's measured rate), 465 us back to back
// under the power cap (1,180); 4096^3 105 us; 2048 x 8192 x 1024 with the same epilogue
// 64 us (epilogue-bound: 20 us of MMAs); both gradients at 2047 x 2050 x 1999 57 us, 20
// of them the preparation.
// Every mbarrier wait is bounded: when one runs out the CTA raises the fault
// word (vcb_fault_check), writes NaN to the tiles it has not finished, waits
// for its copies and MMAs in flight, frees its tensor memory and returns.
#include <algorithm>
#include <array>

#include "vcb_linear_sum.cuh"

namespace vcb {
namespace lin {
namespace {

struct alignas(64) Prod {
  CUtensorMap a, b;
  int J, I, T;
  int a_mn, b_mn;
  int bn;                // columns of the tile (rows i), a multiple of 16
  int tiles_j, tiles_i;
  int nk;                // stages of a full contraction
  uint32_t idesc;
  Epilogue epi;
};

struct Launch {
  Prod p[2];
  int units0, units;  // tiles of the first product, of both
  int split;          // split_kernel: CTAs per tile of the first product (cluster size)
  int stages;
  int* fault;
};

// W columns of the accumulator, NaN if !ok.
template <int W>
__device__ __forceinline__ void accumulator(uint32_t at, bool ok, float (&v)[W]) {
  uint32_t raw[W];
  if (ok) {
    if constexpr (W == 16) tmem_ld16(at, raw); else tmem_ld8(at, raw);
    tmem_wait_ld(raw);
  }
#pragma unroll
  for (int k = 0; k < W; ++k) v[k] = ok ? __uint_as_float(raw[k]) : NAN;
}

// Epilogue of one of WARPS warps: lanes 32 (warp % 4).. of the accumulator at `acc`,
// chunk warp / 4 of W columns and every (WARPS / 4)th from there.  Residuals are
// fetched two chunks ahead.  `ok` false: NaN instead.
template <typename T, int W, int WARPS>
struct TileEpilogue {
  static constexpr int kStep = WARPS / 4 * W;
  const Epilogue& e;
  int I, J, bn, i0, lane, j, first;
  Residual<T, W / 4> res[2];

  __device__ __forceinline__ TileEpilogue(const Prod& p, int warp, int lane_, int j0, int i0_)
      : e(p.epi), I(p.I), J(p.J), bn(p.bn), i0(i0_), lane(lane_),
        j(j0 + (warp & 3) * 32 + (lane_ & ~3)), first((warp >> 2) * W) {
    // before the accumulator is ready
    fetch(res[0], first);
    fetch(res[1], first + kStep);
  }
  __device__ __forceinline__ void fetch(Residual<T, W / 4>& r, int c) {
    if (c < bn) r.fetch(e, I, J, i0 + c + (lane & 3), j);
  }
  __device__ __forceinline__ void chunk(uint32_t at, int c, const float (&bias)[4],
                                        Residual<T, W / 4>& r, bool ok) {
    if (c >= bn || i0 + c >= I) return;  // warp-uniform
    float v[W];
    accumulator(at + c, ok, v);
    transpose4(v, lane);
    emit<T, W / 4>(e, I, J, i0 + c + (lane & 3), j, bias, v, r);
    fetch(r, c + 2 * kStep);
  }
  __device__ __forceinline__ void run(uint32_t acc, int warp, bool ok) {
    float bias[4];
    bias_at<T>(e, J, j, bias);
    const uint32_t at = acc + ((uint32_t)((warp & 3) * 32) << 16);
    for (int c = first; c < bn; c += 2 * kStep) {
      chunk(at, c, bias, res[0], ok);
      chunk(at, c + kStep, bias, res[1], ok);
    }
  }
};

// The same where rows take no vectors: a lane keeps its column, so a warp's stores
// and loads are 32 neighbouring elements.  Residuals one chunk ahead: registers for
// two would be spilled.
template <typename T, int W, int WARPS>
struct ColumnEpilogue {
  static constexpr int kStep = WARPS / 4 * W;
  const Epilogue& e;
  int I, J, bn, i0, j, first;
  float bias;
  ColumnResidual<T, W> res;

  __device__ __forceinline__ ColumnEpilogue(const Prod& p, int warp, int lane, int j0, int i0_)
      : e(p.epi), I(p.I), J(p.J), bn(p.bn), i0(i0_), j(j0 + (warp & 3) * 32 + lane),
        first((warp >> 2) * W) {
    bias = e.bias && j < J ? to_f32(static_cast<const T*>(e.bias)[j]) : 0.f;
    fetch(first);
  }
  __device__ __forceinline__ void fetch(int c) {
    if (c < bn) res.fetch(e, I, J, i0 + c, j);
  }
  __device__ __forceinline__ void run(uint32_t acc, int warp, bool ok) {
    const uint32_t at = acc + ((uint32_t)((warp & 3) * 32) << 16);
    for (int c = first; c < bn && i0 + c < I; c += kStep) {
      float v[W];
      accumulator(at + c, ok, v);
      emit_column<T, W>(e, I, J, i0 + c, j, bias, v, res);
      fetch(c + kStep);
    }
  }
};

// Sixteen epilogue warps with 8 columns at a time: an epilogue warp waits for tensor
// memory, shuffles and conversions in turn, so a short contraction leaves the
// epilogue as the bound.
constexpr int kPairEpi = 16, kPairThreads = (kPairEpi + 2) * 32;
constexpr int kPairStages = 6;
constexpr int kPairStage = 2 * kBytesA;  // per CTA: 128 rows of A and 128 of B
constexpr int kPairSmem = kPairStages * kPairStage + 1024;

template <typename T>
__global__ void __launch_bounds__(kPairThreads, 1)
    pair_kernel(const __grid_constant__ Launch L) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem = (smem_u32(smem_raw) + 1023) & ~1023u;
  __shared__ __align__(8) uint64_t full[kPairStages], empty[kPairStages];
  __shared__ __align__(8) uint64_t acc_full[2], acc_free[2], done;
  __shared__ uint32_t tmem_slot;
  __shared__ int failed;
  const volatile int* vfailed = &failed;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t rank = ctarank();
  const int first = blockIdx.x >> 1, step = gridDim.x >> 1;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kPairStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int q = 0; q < 2; ++q) {
      mbar_init(&acc_full[q], 1);
      mbar_init(&acc_free[q], 2 * kPairEpi);
    }
    mbar_init(&done, 1);
    failed = 0;
    mbar_fence_init();
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(&tmem_slot)),
                 "r"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
  fence_before_sync();
  __syncthreads();
  cluster_sync();  // barriers of both CTAs are ready
  fence_after_sync();
  after_previous();
  const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_slot, 0);

  if (warp == kPairEpi) {
    {  // TMA producer: this CTA's halves of A and B, counted by the leader
      const bool one = elect_one();
      unsigned g = 0;
      Ring ring;
      bool ok = true;
      const uint32_t full0 = map_rank(smem_u32(full), 0);
      for (int u = first; ok && u < L.units; u += step) {
        const Prod& p = L.p[u >= L.units0];
        int ti, tj;
        tile_at(p.tiles_i, p.tiles_j, u >= L.units0 ? u - L.units0 : u, ti, tj);
        const int ja = (tj * 2 + rank) * kTileJ, ib = (ti * 2 + rank) * kTileJ;
        const int nk = p.nk, a_mn = p.a_mn, b_mn = p.b_mn;
        for (int kb = 0; kb < nk; ++kb, ++g, ring.next(kPairStages)) {
          const int s = ring.s;
          if (g >= kPairStages && !mbar_wait(&empty[s], ring.parity ^ 1, kSpinLimit, vfailed)) {
            ok = false;
            break;
          }
          if (one) {
            if (rank == 0) mbar_expect_tx(&full[s], 2 * kPairStage);
            const uint32_t bar = full0 + s * 8, st = smem + s * kPairStage;
            load_operand<true>(st, &p.a, bar, a_mn, ja, kTileJ, kb * kBK);
            load_operand<true>(st + kBytesA, &p.b, bar, b_mn, ib, kTileJ, kb * kBK);
          }
        }
      }
      if (!ok) failed = 1;
      if (rank == 0)  // the copies in flight land before the pair leaves
        for (unsigned k = g > kPairStages ? g - kPairStages : 0; k < g; ++k)
          if (!mbar_wait(&full[k % kPairStages], (k / kPairStages) & 1, kSpinLimit)) failed = 1;
    }
  } else if (warp == kPairEpi + 1) {
    if (rank == 0) {  // MMA issuer of the pair
      const bool one = elect_one();
      unsigned t = 0;
      Ring ring;
      bool ok = true;
      for (int u = first; ok && u < L.units; u += step, ++t) {
        const Prod& p = L.p[u >= L.units0];
        const int q = t & 1, nk = p.nk;
        const Desc da = operand(smem, p.a_mn, kPairStage);
        const Desc db = operand(smem + kBytesA, p.b_mn, kPairStage);
        const uint32_t idesc = p.idesc;
        if (t >= 2 && !mbar_wait(&acc_free[q], ((t >> 1) - 1) & 1, kDoneLimit, vfailed)) {
          ok = false;
          break;
        }
        for (int kb = 0; kb < nk; ++kb, ring.next(kPairStages)) {
          const int s = ring.s;
          if (!mbar_wait(&full[s], ring.parity, kSpinLimit, vfailed)) {
            ok = false;
            break;
          }
          fence_after_sync();
          if (one) {
            mma_stage<true>(tmem + q * 256, da, db, s, idesc, kb == 0);
            commit_pair(&empty[s]);
          }
        }
        if (ok && one) commit_pair(&acc_full[q]);
      }
      if (!ok) failed = 1;
      if (one) commit_pair(&done);  // every MMA has finished before tensor memory is freed
    }
    if (!mbar_wait(&done, 0, kDoneLimit)) failed = 1;
  } else {
    unsigned t = 0;
    bool ok = true;
    for (int u = first; u < L.units; u += step, ++t) {
      const Prod& p = L.p[u >= L.units0];
      int ti, tj;
      tile_at(p.tiles_i, p.tiles_j, u >= L.units0 ? u - L.units0 : u, ti, tj);
      const int q = t & 1, j0 = (tj * 2 + rank) * kTileJ, i0 = ti * 2 * kTileJ;
      const auto ready = [&] {
        ok = ok && mbar_wait(&acc_full[q], (t >> 1) & 1, kDoneLimit, vfailed);
        ok = __all_sync(0xffffffffu, ok);
        fence_after_sync();
      };
      if (p.epi.vec) {
        TileEpilogue<T, 8, kPairEpi> epilogue(p, warp, lane, j0, i0);
        ready();
        epilogue.run(tmem + q * 256, warp, ok);
      } else {
        ColumnEpilogue<T, 8, kPairEpi> epilogue(p, warp, lane, j0, i0);
        ready();
        epilogue.run(tmem + q * 256, warp, ok);
      }
      fence_before_sync();
      __syncwarp();
      if (lane == 0)
        arrive_leader(&acc_free[q]);
    }
    if (!ok) failed = 1;
  }
  fence_before_sync();
  __syncthreads();
  cluster_sync();
  if (warp == 0)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
  if (threadIdx.x == 0 && failed) atomicOr(L.fault, kFaultLinear);
}

// One tile per CTA; the tiles of the first product are shared by the
// L.split CTAs of a cluster, each taking a part of the contraction.
template <typename T>
__global__ void __launch_bounds__(kThreads)
    split_kernel(const __grid_constant__ Launch L) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem = (smem_u32(smem_raw) + 1023) & ~1023u;
  __shared__ __align__(8) uint64_t full[kMostStages], empty[kMostStages], acc_full;
  __shared__ uint32_t tmem_slot;
  __shared__ int failed;
  const volatile int* vfailed = &failed;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int size = L.split, rank = blockIdx.x % size, cluster = blockIdx.x / size;
  // this CTA's tile and part of the contraction
  const bool second = cluster >= L.units0;
  const Prod& p = L.p[second];
  const int u = second ? (cluster - L.units0) * size + rank : cluster;
  const bool idle = second && u >= p.tiles_i * p.tiles_j;
  int ti = 0, tj = 0;
  if (!idle) tile_at(p.tiles_i, p.tiles_j, u, ti, tj);
  const int parts = second ? 1 : size, part = second ? 0 : rank;
  const int k0 = idle ? 0 : static_cast<int>((long long)p.nk * part / parts);
  const int k1 = idle ? 0 : static_cast<int>((long long)p.nk * (part + 1) / parts);
  const int stages = L.stages, stage_bytes = kBytesA + p.bn * kBK * 2;
  const uint32_t columns = max(32, p.bn <= 32 ? 32 : p.bn <= 64 ? 64 : p.bn <= 128 ? 128 : 256);
  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(&acc_full, 1);
    failed = 0;
    mbar_fence_init();
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(&tmem_slot)),
                 "r"(columns));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  after_previous();
  const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_slot, 0);
  const int j0 = tj * kTileJ, i0 = ti * p.bn;
  bool ok = true;

  if (warp == kEpiWarps) {
    {  // TMA producer
      const bool one = elect_one();
      int g = 0;
      Ring ring;
      const int a_mn = p.a_mn, b_mn = p.b_mn, bn = p.bn;
      for (int kb = k0; kb < k1; ++kb, ++g, ring.next(stages)) {
        const int s = ring.s;
        if (g >= stages && !mbar_wait(&empty[s], ring.parity ^ 1, kSpinLimit, vfailed)) {
          ok = false;
          break;
        }
        if (one) {
          mbar_expect_tx(&full[s], stage_bytes);
          const uint32_t st = smem + s * stage_bytes, bar = smem_u32(&full[s]);
          load_operand<false>(st, &p.a, bar, a_mn, j0, kTileJ, kb * kBK);
          load_operand<false>(st + kBytesA, &p.b, bar, b_mn, i0, bn, kb * kBK);
        }
      }
      if (!ok) failed = 1;
      for (int k = g > stages ? g - stages : 0; k < g; ++k)
        if (!mbar_wait(&full[k % stages], (k / stages) & 1, kSpinLimit)) failed = 1;
    }
  } else if (warp == kEpiWarps + 1) {
    {  // MMA issuer
      const bool one = elect_one();
      Ring ring;
      const Desc da = operand(smem, p.a_mn, stage_bytes);
      const Desc db = operand(smem + kBytesA, p.b_mn, stage_bytes);
      const uint32_t idesc = p.idesc;
      for (int kb = k0; kb < k1; ++kb, ring.next(stages)) {
        const int s = ring.s;
        if (!mbar_wait(&full[s], ring.parity, kSpinLimit, vfailed)) {
          ok = false;
          break;
        }
        fence_after_sync();
        if (one) {
          mma_stage<false>(tmem, da, db, s, idesc, kb == k0);
          mma_commit(&empty[s]);
        }
      }
      if (!ok) failed = 1;
      if (one) mma_commit(&acc_full);
      if (!mbar_wait(&acc_full, 0, kDoneLimit)) failed = 1;
    }
  } else {
    const auto ready = [&] {
      ok = mbar_wait(&acc_full, 0, kDoneLimit) && !*vfailed;
      ok = __all_sync(0xffffffffu, ok);
      fence_after_sync();
    };
    if (parts == 1 && !p.epi.vec) {
      ColumnEpilogue<T, 16, kEpiWarps> epilogue(p, warp, lane, j0, idle ? p.I : i0);
      ready();
      epilogue.run(tmem, warp, ok);
    } else if (parts == 1) {
      TileEpilogue<T, 16, kEpiWarps> epilogue(p, warp, lane, j0, idle ? p.I : i0);
      ready();
      epilogue.run(tmem, warp, ok);
    } else {
      ready();
      // partial sums where the stages were, a column's 128 rows together
      const uint32_t base = tmem + ((uint32_t)((warp & 3) * 32) << 16);
      for (int c = (warp >> 2) * 16; c < p.bn && i0 + c < p.I; c += 32) {
        uint32_t r[16];
        tmem_ld16(base + c, r);
        tmem_wait_ld(r);
#pragma unroll
        for (int k = 0; k < 16; ++k)
          asm volatile("st.shared.f32 [%0], %1;" ::"r"(
                           smem + ((c + k) * kTileJ + (warp & 3) * 32 + lane) * 4),
                       "f"(ok ? __uint_as_float(r[k]) : NAN)
                       : "memory");
      }
    }
  }
  fence_before_sync();
  __syncthreads();
  if (warp == 0)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                 "r"(columns));
  if (threadIdx.x == 0 && failed) atomicOr(L.fault, kFaultLinear);
  if (size == 1) return;
  cluster_sync();
  if (parts > 1 && warp < kEpiWarps) {
    // columns are dealt over the ranks and their warps; 4 rows per lane
    const Epilogue e = p.epi;
    const int columns = min(p.bn, p.I - i0), j = j0 + lane * 4;
    float bias[4];
    bias_at<T>(e, p.J, j, bias);
    for (int c = rank * kEpiWarps + warp; c < columns; c += size * kEpiWarps) {
      const uint32_t at = smem + (c * kTileJ + lane * 4) * 4;
      float v[4] = {};
      for (int k = 0; k < size; ++k) {
        const float4 t = peer_f32x4(map_rank(at, k));
        v[0] += t.x, v[1] += t.y, v[2] += t.z, v[3] += t.w;
      }
      Residual<T, 1> res;
      res.fetch(e, p.I, p.J, i0 + c, j);
      emit<T, 1>(e, p.I, p.J, i0 + c, j, bias, v, res);
    }
  }
  cluster_sync();  // no CTA leaves while its partial sums are read
}

// What a backward pass needs first: dz = dy act'(z) in rows that TMA can read,
// db, and copies of operands whose rows TMA cannot read (not 16-byte aligned).  dz is
// rounded to the operands' type, which a tensor-core operand has to have; db sums the
// values before that.
struct Copy {
  const void* src;
  void* dst;
  long long lds, ldd, rows;
  int cols;
};

struct Prep {
  int M, N, act, strips;  // strips of 4 lanes columns of dy, 0 for none
  int lanes;              // of a row in a strip: 8 or 4
  const void *dy, *z;
  void *dz, *db;          // either may be NULL
  long long lddy, ldz, lddz;
  Copy copy[2];
  int copies;
  int cluster;  // CTAs per strip
};

constexpr int kPrepThreads = 256, kPrepWarps = kPrepThreads / 32;
constexpr int kStrip = 32;  // columns at most

// Four elements of a row as loaded: two words, or an element in each.  They are
// unpacked where they are used: more loads follow these.
struct Loaded {
  uint32_t w[4];
};

// From p, `align` bytes aligned (8, 4 or 2); 0 from `left` on.
template <typename T>
__device__ __forceinline__ void four_at(const T* p, int align, int left, Loaded& e) {
  if (align == 8 && left >= 4) {
    const uint2 t = __ldcs(reinterpret_cast<const uint2*>(p));
    e.w[0] = t.x, e.w[1] = t.y;
  } else if (align >= 4 && left >= 4) {
    e.w[0] = __ldcs(reinterpret_cast<const uint32_t*>(p));
    e.w[1] = __ldcs(reinterpret_cast<const uint32_t*>(p) + 1);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      e.w[i] = i < left ? __ldcs(reinterpret_cast<const uint16_t*>(p) + i) : 0;
  }
}

template <typename T>
__device__ __forceinline__ void values(const Loaded& e, bool packed, float (&v)[4]) {
  const uint32_t w[2] = {packed ? e.w[0] : e.w[0] | e.w[1] << 16,
                         packed ? e.w[1] : e.w[2] | e.w[3] << 16};
  T t[4];
  *reinterpret_cast<uint2*>(t) = make_uint2(w[0], w[1]);
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = to_f32(t[i]);
}

// Alignment of all rows of a 16-bit matrix at columns that are multiples of 4.
__device__ __forceinline__ int rows_align(const void* p, long long ld) {
  const unsigned bits = static_cast<unsigned>(reinterpret_cast<uintptr_t>(p)) |
                        static_cast<unsigned>(ld * 2);
  return bits % 8 == 0 ? 8 : bits % 4 == 0 ? 4 : 2;
}

// Eight elements at p, 2-byte aligned; 0 from `left` on.
__device__ __forceinline__ uint4 eight_at(const uint16_t* p, int left) {
  if (left < 8) {
    uint32_t w[4] = {};
#pragma unroll
    for (int i = 0; i < 7; ++i)
      if (i < left) w[i / 2] |= static_cast<uint32_t>(p[i]) << 16 * (i % 2);
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  const bool odd = reinterpret_cast<uintptr_t>(p) % 4 != 0;
  const uint32_t* w = reinterpret_cast<const uint32_t*>(p + odd);
  const uint32_t w0 = __ldcs(w), w1 = __ldcs(w + 1), w2 = __ldcs(w + 2);
  if (!odd) return make_uint4(w0, w1, w2, __ldcs(w + 3));
  // the six elements between the first and the last as aligned words
  const uint32_t a0 = p[0], a7 = p[7];
  return make_uint4(a0 | w0 << 16, w0 >> 16 | w1 << 16, w1 >> 16 | w2 << 16, w2 >> 16 | a7 << 16);
}

// A cluster of up to 8 CTAs per strip of 32 or 16 columns: each sums its part of the
// rows (4 columns per lane), rank 0 adds the sums in order.  Bound by
// HBM: dy and z are read and dz is written once; strips are narrow so that a matrix
// of 2,000 columns keeps every SM reading.  The remaining CTAs copy.
template <typename T, int LANES>  // of a row in a strip
__global__ void __launch_bounds__(kPrepThreads, 5)
    prep_kernel(const __grid_constant__ Prep a) {
  __shared__ float part[kPrepWarps][kStrip], mine[kStrip];
  let_next_start();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int size = a.cluster, strip = blockIdx.x / size;
  if (strip < a.strips) {
    constexpr int lanes = LANES, rows = 32 / lanes;  // rows of a warp
    const int rank = blockIdx.x % size, c = (strip * lanes + lane % lanes) * 4;
    const long long r0 = static_cast<long long>(a.M) * rank / size;
    const long long r1 = static_cast<long long>(a.M) * (rank + 1) / size;
    const T *dy = static_cast<const T*>(a.dy) + c, *z = static_cast<const T*>(a.z) + c;
    const int ay = rows_align(a.dy, a.lddy), az = rows_align(a.z, a.ldz), left = a.N - c;
    float sum[4] = {};
    constexpr int U = 2, W = kPrepWarps * rows;  // rows in flight, rows of a CTA's step
    for (long long r = r0 + warp * rows + lane / lanes; r < r1; r += U * W) {
      Loaded g[U], t[U];
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const long long row = r + k * W;
        if (row >= r1) continue;
        four_at(dy + row * a.lddy, ay, left, g[k]);
        if (a.act != VCB_ACT_NONE) four_at(z + row * a.ldz, az, left, t[k]);
      }
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const long long row = r + k * W;
        if (row >= r1) continue;
        float v[4], w[4];
        values<T>(g[k], ay >= 4 && left >= 4, v);
        if (a.act != VCB_ACT_NONE) {
          values<T>(t[k], az >= 4 && left >= 4, w);
          act_grads(v, w, a.act);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[i] += v[i];
        // lddz is a multiple of 8, so a vector that crosses N stays in its row
        if (a.dz && left > 0) store4(static_cast<T*>(a.dz) + row * a.lddz + c, v);
      }
    }
    if (a.db) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int k = lanes; k < 32; k *= 2) sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], k);
        if (lane < lanes) part[warp][lane * 4 + i] = sum[i];
      }
      __syncthreads();
      if (threadIdx.x < lanes * 4) {
        float v = 0.f;
        for (int w = 0; w < kPrepWarps; ++w) v += part[w][threadIdx.x];
        mine[threadIdx.x] = v;
      }
    }
    cluster_sync();
    if (a.db && rank == 0 && threadIdx.x < lanes * 4) {
      const int col = strip * lanes * 4 + threadIdx.x;
      float v = 0.f;
      for (int k = 0; k < size; ++k) v += peer_f32(map_rank(smem_u32(mine + threadIdx.x), k));
      if (col < a.N) static_cast<T*>(a.db)[col] = from_f32<T>(v);
    }
    cluster_sync();  // no CTA leaves while its sums are read
    return;
  }
  // copies: eight elements per thread, written as one 16-byte vector; neighbouring
  // threads take neighbouring vectors of all rows, four of them in flight
  const long long first = (long long)(blockIdx.x - a.strips * size) * kPrepThreads + threadIdx.x;
  const long long step = (long long)(gridDim.x - a.strips * size) * kPrepThreads;
  for (int k = 0; k < a.copies; ++k) {
    const Copy& q = a.copy[k];
    const int nv = (q.cols + 7) / 8;
    long long row = first / nv;
    int v = static_cast<int>(first - row * nv);
    const long long down = step / nv;
    const int right = static_cast<int>(step - down * nv);
    constexpr int U = 4;
    while (row < q.rows) {
      uint4 o[U];
      uint16_t* out[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        out[u] = row < q.rows ? static_cast<uint16_t*>(q.dst) + row * q.ldd + v * 8 : nullptr;
        if (out[u]) o[u] = eight_at(static_cast<const uint16_t*>(q.src) + row * q.lds + v * 8, q.cols - v * 8);
        row += down, v += right;
        if (v >= nv) v -= nv, ++row;
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (out[u]) *reinterpret_cast<uint4*>(out[u]) = o[u];
    }
  }
}

// ---- host ----

// Row-major (rows x cols) 16-bit matrix in boxes of box_rows x 64 columns.
int make_map(CUtensorMap* map, const void* p, int rows, int cols, long long ld, int box_rows,
             const char* who) {
  const auto fn = encode_fn();
  if (!fn) return fail(VCB_ERR_CUDA, "%s: cuTensorMapEncodeTiled unavailable", who);
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)ld * 2};
  const cuuint32_t box[2] = {kBK, (cuuint32_t)box_rows}, estr[2] = {1, 1};
  const CUresult r =
      fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, const_cast<void*>(p), dims, strides, box, estr,
         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(VCB_ERR_CUDA, "%s: tensor map encode failed (%d)", who, (int)r);
  return VCB_OK;
}

}  // namespace

// How a launch cuts its work: pairs, or bn columns and `split` CTAs per tile.
struct Plan {
  bool pair;
  int bn, split;
};

// CTAs at a time in clusters of 1, 2, 4 and 8 (most of an SM's shared memory each).
int slots_of(int size) {
  static const std::array<int, 4> slots = [] {
    std::array<int, 4> n;
    for (int k = 0; k < 4; ++k)
      n[k] = cluster_slots(split_kernel<__half>, kThreads, 200 << 10, 1 << k);
    return n;
  }();
  return slots[size == 1 ? 0 : size == 2 ? 1 : size == 4 ? 2 : 3];
}

// Cycles of a launch: rounds of tiles over those places times the longer of the MMAs
// (128 rows take 64 cycles per 16 of the contraction up to 128 columns, then
// half a cycle a column; a pair's 256 x 256 takes 128) and the operands'
// way from L2 (about 60 B per cycle and SM), plus a start and an epilogue.
Plan plan_of(int I, int J, int T, bool pair_possible, bool by64) {
  const int sms = sm_count();
  const int nk = std::max(1, (T + kBK - 1) / kBK);
  const auto ceil = [](long long a, long long b) { return (a + b - 1) / b; };
  Plan best{false, 16, 1};
  double least = 1e300;
  for (int bn : {16, 32, 48, 64, 96, 128, 192, 256}) {
    if (by64 && bn % 64) continue;  // an MN-major operand comes in boxes of 64
    const long long tiles = ceil(I, bn) * ceil(J, kTileJ);
    for (int split : {1, 2, 4, 8}) {
      if (split > nk) break;
      const double stage = std::max(4.0 * std::max(64, bn / 2), (kTileJ + bn) * 128 / 60.0);
      const double rounds = static_cast<double>(ceil(tiles * split, slots_of(split)));
      const double t = rounds * (ceil(nk, split) * stage + 2500 + 12.0 * bn) +
                       (split > 1 ? 1500 + 6.0 * bn : 0);
      if (t < least) least = t, best = {false, bn, split};
    }
  }
  if (pair_possible) {
    const long long tiles = ceil(I, 256) * ceil(J, 256);
    const double t = static_cast<double>(ceil(tiles, sms / 2)) * nk * 540 + 8000;
    if (t < least) best = {true, 256, 1};
  }
  return best;
}

struct Operand {
  const void* p;
  long long ld;
  bool mn;  // contiguous along its row index, not along the contraction
};

int set_prod(Prod& r, int type, int I, int J, int T, const Operand& a, const Operand& b, int bn,
             bool pair, const char* who) {
  r.I = I, r.J = J, r.T = T;
  r.a_mn = a.mn, r.b_mn = b.mn;
  r.bn = bn;
  const int tj = pair ? 256 : kTileJ;
  r.tiles_j = (J + tj - 1) / tj;
  r.tiles_i = (I + bn - 1) / bn;
  r.nk = std::max(1, (T + kBK - 1) / kBK);
  r.idesc = idesc_16(type, tj, bn, a.mn, b.mn);
  const int rows_a = kTileJ, rows_b = pair ? kTileJ : bn;
  int rc = a.mn ? make_map(&r.a, a.p, T, J, a.ld, kBK, who) : make_map(&r.a, a.p, J, T, a.ld, rows_a, who);
  if (!rc)
    rc = b.mn ? make_map(&r.b, b.p, T, I, b.ld, kBK, who) : make_map(&r.b, b.p, I, T, b.ld, rows_b, who);
  return rc;
}

template <typename T>
int launch_tc(Launch& L, const Plan& plan, bool chained, cudaStream_t st, const char* who) {
  int rc = fault_word(&L.fault);
  if (rc) return rc;
  if (plan.pair) {
    const auto kernel = pair_kernel<T>;
    rc = ensure_smem(reinterpret_cast<const void*>(kernel), kPairSmem);
    if (rc) return rc;
    const int grid = 2 * std::min(L.units, sm_count() / 2);
    return launch_clusters(kernel, L, grid, kPairThreads, kPairSmem, 2, chained, st, who);
  }
  const auto kernel = split_kernel<T>;
  const int bn = std::max(L.units0 ? L.p[0].bn : 0, L.units > L.units0 ? L.p[1].bn : 0);
  const int nk = std::max(L.units0 ? (L.p[0].nk + plan.split - 1) / plan.split : 0,
                          L.units > L.units0 ? L.p[1].nk : 0);
  const int stage = kBytesA + bn * kBK * 2;
  const long long clusters =
      L.units0 + (L.units - L.units0 + plan.split - 1LL) / plan.split;
  // two CTAs per SM overlap one's epilogue with the other's loads
  const int room = clusters * plan.split > slots_of(plan.split) ? 100 << 10 : 200 << 10;
  L.stages = std::max(2, std::min({kMostStages, nk, room / stage}));
  L.split = plan.split;
  const int smem = std::max(L.stages * stage, plan.split > 1 ? bn * kTileJ * 4 : 0) + 1024;
  rc = ensure_smem(reinterpret_cast<const void*>(kernel), 227 * 1024 - 1024);
  if (rc) return rc;
  return launch_clusters(kernel, L, static_cast<unsigned>(clusters * plan.split), kThreads, smem,
                         plan.split, chained, st, who);
}

int launch_type(Launch& L, const Plan& plan, int type, bool chained, cudaStream_t st,
                const char* who) {
  return type == VCB_BF16 ? launch_tc<__nv_bfloat16>(L, plan, chained, st, who)
                          : launch_tc<__half>(L, plan, chained, st, who);
}

namespace {

// One accumulator would take more than kLongest stages of a contraction of T entries.
bool too_long(const Plan& plan, int T) {
  const int nk = (T + kBK - 1) / kBK;
  return (nk + plan.split - 1) / plan.split > kLongest;
}

// CTAs of a cluster per tile of a long product, 0 for pairs: cycles as in plan_of.
int long_plan(int I, int J, int T) {
  const auto ceil = [](long long x, long long y) { return (x + y - 1) / y; };
  const long long nk = ceil(T, kBK), tiles = ceil(I, 128) * ceil(J, kTileJ);
  double least = static_cast<double>(ceil(ceil(I, 256) * ceil(J, 256), sm_count() / 2)) *
                     (nk * 540 + 4000) + 4000;
  int best = 0;
  for (int split : {1, 2, 4, 8}) {
    const double t = static_cast<double>(ceil(tiles * split, slots_of(split))) *
                         (ceil(nk, split) * 560 + 6500) + (split > 1 ? 2500 : 0);
    if (t < least) least = t, best = split;
  }
  return best;
}

// out(i, j) = sum_t b(i, t) a(j, t) for long T.
template <typename E>
int launch_long(int type, int I, int J, int T, const Operand& a, const Operand& b,
                const Epilogue& epi, bool chained, cudaStream_t st, const char* who) {
  SumLaunch L{};
  L.split = long_plan(I, J, T);
  const bool pair = L.split == 0;
  const auto of = [&](const Operand& o, int rows) {
    const int r = o.mn ? T : rows;
    return SumOperand{o.p, r, o.mn ? rows : T, o.ld, r * o.ld, o.mn};
  };
  const int rc = set_sum<1>(L.p[0], type, I, J, T, of(a, J), of(b, I), pair ? 256 : 128, pair, epi,
                            2, who);
  if (rc) return rc;
  L.units0 = L.units = L.p[0].tiles_i * L.p[0].tiles_j;
  return pair ? launch_sum<E, 1, 256, true>(L, chained, st, who)
              : launch_sum<E, 1, 128, false>(L, chained, st, who);
}

int long_product(int type, int I, int J, int T, const Operand& a, const Operand& b,
                 const Epilogue& epi, bool chained, cudaStream_t st, const char* who) {
  return type == VCB_BF16
             ? launch_long<__nv_bfloat16>(type, I, J, T, a, b, epi, chained, st, who)
             : launch_long<__half>(type, I, J, T, a, b, epi, chained, st, who);
}

// M N K from which the tensor cores are used.  As the operands lie: bf16 64 x 256 x
// 256 (2^22) 4.9 us against 5.4 on the FP32 units, 100 x 200 x 200 9.2 against 11.3,
// 8 x 1024 x 1024 backward 10 against 45.  With a launch that prepares them: 128 x
// 128 x 128 backward (2^21, GELU) 17 against 13, 2000 x 63 x 63 (2^23) 15 against
// 11, 64 x 300 x 301 backward (2^22.5) 17 and 17.
constexpr long long kTcLeast = 1LL << 20, kTcLeastPrepared = 1LL << 23;

long long pad8(long long n) { return (n + 7) / 8 * 8; }
size_t matrix_bytes(long long rows, long long cols) {
  return static_cast<size_t>(rows) * pad8(cols) * 2 + 256;
}

bool tma_rows(const void* p, long long ld) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 8 == 0;
}

// Sizes that 32-bit tile and TMA coordinates describe.
bool fits(long long M, long long N, long long K, bool prepared) {
  const long long most = 1LL << 30;
  return M * N * K >= (prepared ? kTcLeastPrepared : kTcLeast) && M < most && N < most && K < most &&
         ((M + 15) / 16) * ((N + 127) / 128) < most && ((N + 15) / 16) * ((K + 127) / 128) < most &&
         ((M + 15) / 16) * ((K + 127) / 128) < most;
}

// Workspace in 256-byte pieces.
struct Arena {
  uint8_t* at;
  void* take(size_t n) {
    at = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(at) + 255) & ~uintptr_t{255});
    void* p = at;
    at += n;
    return p;
  }
};

// An operand as TMA can read it: itself, or a copy that `prep` makes.
Operand readable(const void* p, long long ld, int rows, int cols, bool mn, Prep& prep, Arena& ws) {
  if (tma_rows(p, ld)) return {p, ld, mn};
  Copy& c = prep.copy[prep.copies++];
  c = {p, ws.take(matrix_bytes(rows, cols)), ld, pad8(cols), rows, cols};
  return {c.dst, c.ldd, mn};
}

int launch_prep(Prep& a, int type, cudaStream_t st, const char* who) {
  long long vectors = 0;
  for (int k = 0; k < a.copies; ++k)
    vectors = std::max(vectors, a.copy[k].rows * ((a.copy[k].cols + 7LL) / 8));
  const long long ctas =
      std::min<long long>((vectors + kPrepThreads - 1) / kPrepThreads, 4LL * sm_count());
  a.cluster = 1;  // a CTA's step is 64 rows or more
  while (a.strips && a.cluster < 8 && a.M > 64 * a.cluster) a.cluster *= 2;
  const long long grid = (a.strips + (ctas + a.cluster - 1) / a.cluster) * (long long)a.cluster;
  if (grid == 0) return VCB_OK;
  const auto kernel = type == VCB_BF16
                          ? a.lanes == 4 ? prep_kernel<__nv_bfloat16, 4> : prep_kernel<__nv_bfloat16, 8>
                          : a.lanes == 4 ? prep_kernel<__half, 4> : prep_kernel<__half, 8>;
  return launch_clusters(kernel, a, static_cast<unsigned>(grid), kPrepThreads, 0, a.cluster, false,
                         st, who);
}

}  // namespace

bool tc_forward_fits(const Fwd& f) {
  return f.type != VCB_F32 &&
         fits(f.M, f.N, f.K, !tma_rows(f.x, f.ldx) || !tma_rows(f.w, f.ldw));
}

size_t tc_forward_bytes(int M, int N, int K) {
  return fits(M, N, K, true) ? matrix_bytes(M, K) + matrix_bytes(N, K) + 256 : 0;
}

int tc_forward(const Fwd& f, void* ws, cudaStream_t st) {
  const char* who = "vcb_linear_forward";
  Prep prep{};
  Arena arena{static_cast<uint8_t*>(ws)};
  const Operand a = readable(f.w, f.ldw, f.N, f.K, false, prep, arena);
  const Operand b = readable(f.x, f.ldx, f.M, f.K, false, prep, arena);
  int rc = launch_prep(prep, f.type, st, who);
  if (rc) return rc;
  const Plan plan = plan_of(f.M, f.N, f.K, true, false);
  const Epilogue epi{f.y, f.z, f.bias, f.res, f.ldy, f.ldz, f.ldr, f.act, 0};
  if (too_long(plan, f.K))
    return long_product(f.type, f.M, f.N, f.K, a, b, epi, prep.copies > 0, st, who);
  Launch L{};
  Prod& p = L.p[0];
  rc = set_prod(p, f.type, f.M, f.N, f.K, a, b, plan.bn, plan.pair, who);
  if (rc) return rc;
  p.epi = epi;
  p.epi.vec = vector_rows(p.epi, 2);
  L.units0 = L.units = p.tiles_i * p.tiles_j;
  return launch_type(L, plan, f.type, prep.copies > 0, st, who);
}

int tc_path(int M, int N, int K, int product) {
  const int I = product == 2 ? N : M, J = product == 0 ? N : K;
  const int T = product == 0 ? K : product == 1 ? N : M;
  const Plan plan = plan_of(I, J, T, true, product == 2);
  if (!too_long(plan, T)) return plan.pair ? 3 : 2;
  return long_plan(I, J, T) ? 4 : 5;
}

bool tc_backward_fits(const Bwd& b) {
  const bool prepared = b.act != VCB_ACT_NONE || b.db || !tma_rows(b.dy, b.lddy) ||
                        !tma_rows(b.x, b.ldx) || !tma_rows(b.w, b.ldw);
  return b.type != VCB_F32 && (b.dx || b.dw) && fits(b.M, b.N, b.K, prepared);
}

size_t tc_backward_bytes(int M, int N, int K, int act, bool rows16) {
  if ((rows16 && act == VCB_ACT_NONE) || !fits(M, N, K, true)) return 0;
  return matrix_bytes(M, N) + (rows16 ? 0 : matrix_bytes(N, K) + matrix_bytes(M, K)) + 256;
}

int tc_backward(const Bwd& b, void* ws, cudaStream_t st) {
  const char* who = "vcb_linear_backward";
  Prep prep{};
  Arena arena{static_cast<uint8_t*>(ws)};
  prep.M = b.M, prep.N = b.N, prep.act = b.act;
  prep.dy = b.dy, prep.lddy = b.lddy, prep.z = b.z, prep.ldz = b.ldz, prep.db = b.db;
  Operand dz{b.dy, b.lddy, false};
  if (b.act != VCB_ACT_NONE || !tma_rows(b.dy, b.lddy)) {
    prep.lddz = pad8(b.N);
    prep.dz = arena.take(matrix_bytes(b.M, b.N));
    dz = {prep.dz, prep.lddz, false};
  }
  if (prep.dz || prep.db) {
    // narrower strips where those of 32 columns would leave a third of the SMs' places
    // empty: bf16 4096 x 1024 x 1024 (GELU) 58 -> 54 us, 5273 x 444 x 131 50 -> 44 us
    prep.lanes = ((b.N + 31) / 32) * 8 < 3 * sm_count() ? 4 : 8;
    prep.strips = (b.N + 4 * prep.lanes - 1) / (4 * prep.lanes);
  }
  Operand w{}, x{};
  if (b.dx) w = readable(b.w, b.ldw, b.N, b.K, true, prep, arena);
  if (b.dw) x = readable(b.x, b.ldx, b.M, b.K, true, prep, arena);
  int rc = launch_prep(prep, b.type, st, who);
  if (rc) return rc;
  const bool prepared = prep.strips || prep.copies;
  // dX and dW share a launch when both are pairs or both are not, and both are short
  // enough for one accumulator; the contraction of dW, the rows, is then not cut
  const Plan px = plan_of(b.M, b.K, b.N, true, false), pw = plan_of(b.N, b.K, b.M, true, true);
  Launch L{};
  Operand dzt = dz;
  dzt.mn = true;
  const Epilogue ex{b.dx, nullptr, nullptr, nullptr, b.lddx, 0, 0, VCB_ACT_NONE, 0};
  const Epilogue ew{b.dw, nullptr, nullptr, nullptr, b.lddw, 0, 0, VCB_ACT_NONE, 0};
  const bool long_x = b.dx && too_long(px, b.N), long_w = b.dw && too_long(pw, b.M);
  const bool together = b.dx && b.dw && px.pair == pw.pair && !long_x &&
                        !too_long({pw.pair, pw.bn, 1}, b.M);
  if (long_x) {
    rc = long_product(b.type, b.M, b.K, b.N, w, dz, ex, prepared, st, who);
    if (rc) return rc;
  } else if (b.dx) {
    rc = set_prod(L.p[0], b.type, b.M, b.K, b.N, w, dz, px.bn, px.pair, who);
    if (rc) return rc;
    L.p[0].epi = ex;
    L.p[0].epi.vec = vector_rows(L.p[0].epi, 2);
    L.units0 = L.units = L.p[0].tiles_i * L.p[0].tiles_j;
  }
  if (b.dx && !long_x && !together) {
    rc = launch_type(L, px, b.type, prepared, st, who);
    if (rc) return rc;
    L.units0 = L.units = 0;
  }
  if (long_w)
    return long_product(b.type, b.N, b.K, b.M, x, dzt, ew, prepared && !b.dx, st, who);
  if (b.dw) {
    Prod& p = L.p[1];
    rc = set_prod(p, b.type, b.N, b.K, b.M, x, dzt, pw.bn, pw.pair, who);
    if (rc) return rc;
    p.epi = ew;
    p.epi.vec = vector_rows(p.epi, 2);
    L.units += p.tiles_i * p.tiles_j;
    Plan plan = pw;
    if (together) plan.split = px.split;
    if (!together) {  // the only product of its launch
      L.p[0] = L.p[1];
      L.units0 = L.units;
    }
    rc = launch_type(L, plan, b.type, prepared && (together || !b.dx), st, who);
  }
  return rc;
}

}  // namespace lin
}  // namespace vcb
