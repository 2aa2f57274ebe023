// The linear layer's products whose accumulators in tensor memory are emptied on the
// way: the tensor cores drop low-order bits in every accumulation, a loss that grows
// with the number of accumulations, always towards zero.  An accumulator takes kPer
// stages of 64 entries; the epilogue warps add those sums in registers, rounding to
// nearest, while the next stages fill the other accumulator.
//
// PARTS = 3: float32 operands as three bfloat16 parts each (vcb_linear_f32.cu), one
// stage per accumulator.  PARTS = 1: 16-bit operands whose contraction is longer than
// an accumulator may take (vcb_linear_tc.cu).
#pragma once

#include <algorithm>

#include "vcb_linear_tc.cuh"

namespace vcb {
namespace lin {
namespace {

// Most stages (8,192 entries) of a 16-bit product's accumulator.  Same-signed entries, the
// worst case, lose 5e-5 in 8,192 (a tenth of half a unit of float16), but 2e-4 in
// 32,768, 8e-4 in 131,072 and 6e-3 in 2^20.
// Beside one accumulator per tile, measured: bf16 dW and dX at 131072 x 2048 x 2048 2,254
// us against 2,166, 40000 x 1100 x 1030 508 against 467, 9000 x 512 x 512 54 against 106.
constexpr int kLongest = 128;

struct alignas(64) SumProd {
  CUtensorMap a, b;  // (64, rows, parts) boxes
  int J, I, a_mn, b_mn, tiles_j, tiles_i, nk;
  uint32_t idesc;
  Epilogue epi;
};

struct SumLaunch {
  SumProd p[2];
  int units0, units, split;
  int* fault;
};

// Sixteen epilogue warps: what they do at a tile's end (activation, stores)
// runs beside two stages of the next tile's MMAs only, so it is spread as wide as
// registers allow.
constexpr int kEpi = 16, kSumThreads = (kEpi + 2) * 32;

template <int PARTS, int BN, bool PAIR>
struct Cfg {
  static constexpr int kRowsB = PAIR ? BN / 2 : BN;
  static constexpr int kBytesB = PARTS * kRowsB * 128;
  static constexpr int kStage = PARTS * kBytesA + kBytesB;
  static constexpr int kStages = 221184 / kStage;
  // stages of an accumulator
  static constexpr int kPer = PARTS == 1 ? kLongest : 1;
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

// The parts of an operand's rows.  K-major: all rows of the first part, then of the
// others.  MN-major: per 64 rows, 8 KB of each.
template <int PARTS, bool PAIR>
__device__ __forceinline__ void load_parts(uint32_t dst, const CUtensorMap* map, uint32_t bar,
                                            int mn, int row, int rows, int t) {
  if (!mn) {
    if (PAIR) tma_3d_pair(dst, map, bar, t, row); else tma_3d(dst, map, bar, t, row);
  } else {
    for (int q = 0; q < rows; q += 64) {
      if (PAIR) tma_3d_pair(dst + q / 64 * (PARTS * 8192), map, bar, row + q, t);
      else tma_3d(dst + q / 64 * (PARTS * 8192), map, bar, row + q, t);
    }
  }
}

// One tile of `out` per unit of work.  PAIR: persistent CTA pairs, 256 x 256.
// Otherwise a 128 x BN tile per cluster of L.split CTAs, each with a part of the
// contraction (none, where it has fewer stages than CTAs); the parts are joined in the
// order of the ranks.
template <typename T, int PARTS, int BN, bool PAIR>
__global__ void __launch_bounds__(kSumThreads, 1) sum_kernel(const __grid_constant__ SumLaunch L) {
  using C = Cfg<PARTS, BN, PAIR>;
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
      const SumProd& p = L.p[u >= L.units0];
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
          load_parts<PARTS, PAIR>(st, &p.a, bar, a_mn, ja, kTileJ, kb * kBK);
          load_parts<PARTS, PAIR>(st + PARTS * kBytesA, &p.b, bar, b_mn, ib, C::kRowsB, kb * kBK);
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
        const SumProd& p = L.p[u >= L.units0];
        const int a_mn = p.a_mn, b_mn = p.b_mn, k1 = end(p.nk);
        const Desc da = operand(smem, a_mn, C::kStage, PARTS * 8192);
        const Desc db = operand(smem + PARTS * kBytesA, b_mn, C::kStage, PARTS * 8192);
        // from a part to the next
        const uint32_t pa = (a_mn ? 8192 : kBytesA) >> 4;
        const uint32_t pb = (b_mn ? 8192 : C::kBytesB / PARTS) >> 4;
        const uint32_t idesc = p.idesc;
        const int k0 = begin(p.nk);
        for (int kb = k0; kb < k1; ++kb, ring.next(C::kStages)) {
          const int at = (kb - k0) % C::kPer;  // in its accumulator
          const bool last = at == C::kPer - 1 || kb == k1 - 1;
          if (!mbar_wait(&full[ring.s], ring.parity, kSpinLimit, vfailed) ||
              (at == 0 && chunks >= C::kBufs &&
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
            for (int sum = PARTS - 1; sum >= 0; --sum) {
#pragma unroll
              for (int q = 0; q <= sum; ++q) {
#pragma unroll
                for (int k = 0; k < kBK / 16; ++k)
                  mma_f16<PAIR>(d, a0 + q * pa + k * da.k, b0 + (sum - q) * pb + k * db.k, idesc,
                                sum == PARTS - 1 && q == 0 && k == 0 && at == 0 ? 0u : 1u);
              }
            }
            if (PAIR) commit_pair(&empty[ring.s]); else mma_commit(&empty[ring.s]);
            if (last) {
              if (PAIR) commit_pair(&acc_full[buf.s]); else mma_commit(&acc_full[buf.s]);
            }
          }
          if (last) ++chunks, buf.next(C::kBufs);
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
      const SumProd& p = L.p[u >= L.units0];
      int ti, tj;
      tile_at(p.tiles_i, p.tiles_j, u >= L.units0 ? u - L.units0 : u, ti, tj);
      const int j0 = (PAIR ? (tj * 2 + rank) * kTileJ : tj * kTileJ) + quad * 32;
      const int i0 = ti * BN + col0;
      const int chunks = (end(p.nk) - begin(p.nk) + C::kPer - 1) / C::kPer;
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
      bias_at<T>(p.epi, J, j, bias);
#pragma unroll
      for (int c = 0; c < kCols; c += 16) {
        if (i0 + c < I) {  // warp-uniform
          Residual<T, 4> res;
          res.fetch(p.epi, I, J, i0 + c + (lane & 3), j);
          float v[16];
#pragma unroll
          for (int k = 0; k < 16; ++k) v[k] = acc[c + k];
          transpose4(v, lane);
          emit<T, 4>(p.epi, I, J, i0 + c + (lane & 3), j, bias, v, res);
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
      const SumProd& p = L.p[first >= L.units0];
      int ti, tj;
      tile_at(p.tiles_i, p.tiles_j, first >= L.units0 ? first - L.units0 : first, ti, tj);
      const Epilogue e = p.epi;
      const int i0 = ti * BN, j = tj * kTileJ + lane * 4;
      const int columns = min(BN, p.I - i0);
      float bias[4];
      bias_at<T>(e, p.J, j, bias);
      for (int c = rank * kEpi + warp; c < columns; c += size * kEpi) {
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
// A row-major 16-bit matrix in PARTS planes; mn: it is contiguous along its row index,
// not along the contraction.
struct SumOperand {
  const void* p;
  int rows, cols;
  long long ld, plane;
  bool mn;
};

template <int PARTS>
int sum_map(CUtensorMap* map, const SumOperand& h, int box_rows, const char* who) {
  const auto fn = encode_fn();
  if (!fn) return fail(VCB_ERR_CUDA, "%s: cuTensorMapEncodeTiled unavailable", who);
  const cuuint64_t dims[3] = {(cuuint64_t)h.cols, (cuuint64_t)h.rows, PARTS};
  const cuuint64_t strides[2] = {(cuuint64_t)h.ld * 2, (cuuint64_t)h.plane * 2};
  const cuuint32_t box[3] = {kBK, (cuuint32_t)box_rows, PARTS}, estr[3] = {1, 1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, const_cast<void*>(h.p), dims,
                        strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(VCB_ERR_CUDA, "%s: tensor map encode failed (%d)", who, (int)r);
  return VCB_OK;
}

// out(i, j) = sum_t b(i, t) a(j, t); type: of the operands, elem: bytes of an output.
template <int PARTS>
int set_sum(SumProd& r, int type, int I, int J, int T, const SumOperand& a, const SumOperand& b,
            int bn, bool pair, const Epilogue& epi, int elem, const char* who) {
  r.I = I, r.J = J;
  r.a_mn = a.mn, r.b_mn = b.mn;
  const int tj = pair ? 256 : kTileJ;
  r.tiles_j = (J + tj - 1) / tj;
  r.tiles_i = (I + bn - 1) / bn;
  r.nk = std::max(1, (T + kBK - 1) / kBK);
  r.idesc = idesc_16(type, tj, bn, a.mn, b.mn);
  r.epi = epi;
  r.epi.vec = vector_rows(epi, elem);
  int rc = sum_map<PARTS>(&r.a, a, a.mn ? kBK : kTileJ, who);
  if (!rc) rc = sum_map<PARTS>(&r.b, b, b.mn ? kBK : pair ? kTileJ : bn, who);
  return rc;
}

template <typename T, int PARTS, int BN, bool PAIR>
int launch_sum(SumLaunch& L, bool chained, cudaStream_t st, const char* who) {
  using C = Cfg<PARTS, BN, PAIR>;
  int rc = fault_word(&L.fault);
  const auto kernel = sum_kernel<T, PARTS, BN, PAIR>;
  if (!rc) rc = ensure_smem(reinterpret_cast<const void*>(kernel), C::kSmem);
  if (rc) return rc;
  const int size = PAIR ? 2 : L.split;
  return launch_clusters(kernel, L, size * (PAIR ? std::min(L.units, sm_count() / 2) : L.units),
                         kSumThreads, C::kSmem, size, chained, st, who);
}

}  // namespace
}  // namespace lin
}  // namespace vcb
