// Primitives that the linear layer's tensor-core kernels share: TMA loads and
// tcgen05.mma kind::f16 for one CTA or a pair, shared-memory operands that are
// contiguous along either index, clusters, and the order of the tiles.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>

#include "vcb_linear.cuh"
#include "vcb_tcgen05.cuh"

namespace vcb {
namespace lin {
namespace {

using namespace tc5;

constexpr int kBK = 64;                      // contraction per stage: 128 bytes
constexpr int kTileJ = 128;                  // MMA rows of one CTA
constexpr int kBytesA = kTileJ * kBK * 2;    // 16 KB
constexpr int kEpiWarps = 8;
constexpr int kThreads = (kEpiWarps + 2) * 32;
constexpr int kMostStages = 12;
constexpr unsigned kSpinLimit = 1u << 20;    // pipeline waits (a stage is microseconds)
constexpr unsigned kDoneLimit = 1u << 24;    // waits for a whole mainloop

// One lane of a converged warp.  The producer's and the issuer's loops are run
// by all 32 lanes and only the instruction itself by the elected one: what it
// takes (descriptors, addresses, the instruction word) is then uniform over the
// warp and stays in uniform registers.  Run by lane 0 alone, every operand went
// through a vector register first: 620 cycles per stage instead of the MMAs'.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(p));
  return p != 0;
}

__device__ __forceinline__ uint32_t ctarank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}

// A kernel that prepares operands lets the product's CTAs take their places, barriers
// and tensor memory as its own run out; each thread of the product waits for all that
// was prepared before it touches anything else.
__device__ __forceinline__ void let_next_start() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

__device__ __forceinline__ void after_previous() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile(
      "barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::
          : "memory");
}

__device__ __forceinline__ uint32_t map_rank(uint32_t saddr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(saddr), "r"(rank));
  return r;
}

// Arrive on `bar` of the pair's first CTA.  Relaxed: what it hands over are reads of
// tensor memory that have completed (a release would fence all memory, some 500
// cycles each time).
__device__ __forceinline__ void arrive_leader(uint64_t* bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(
                   map_rank(smem_u32(bar), 0))
               : "memory");
}

__device__ __forceinline__ void tma_2d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x,
                                       int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(bar)
      : "memory");
}

// As tma_2d for a CTA pair: `bar` may lie in the other CTA of the pair.
__device__ __forceinline__ void tma_2d_pair(uint32_t dst, const CUtensorMap* map, uint32_t bar,
                                            int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::"
      "bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(bar)
      : "memory");
}

// One operand's rows [row, row + rows) x contraction [t, t + 64).  K-major: one
// box of `rows` rows; MN-major: boxes of 64 (rows) x 64 (t), 8 KB each.
template <bool PAIR>
__device__ __forceinline__ void load_operand(uint32_t dst, const CUtensorMap* map, uint32_t bar,
                                             int mn, int row, int rows, int t) {
  if (!mn) {
    if (PAIR) tma_2d_pair(dst, map, bar, t, row); else tma_2d(dst, map, bar, t, row);
  } else {
    for (int q = 0; q < rows; q += 64) {
      if (PAIR) tma_2d_pair(dst + q * 128, map, bar, row + q, t);
      else tma_2d(dst + q * 128, map, bar, row + q, t);
    }
  }
}

// Shared-memory operand, 128-byte swizzle.  K-major: 8-row groups 1,024 B
// apart.  MN-major: 64 rows contiguous per t, 8-t groups 1,024 B apart (stride
// offset), 64-row boxes `box` B apart (leading offset).
__device__ __forceinline__ uint64_t operand_desc(uint32_t saddr, int mn, uint32_t box) {
  uint64_t d = (uint64_t)((saddr >> 4) & 0x3FFF);
  d |= (uint64_t)(mn ? box >> 4 : 1) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}

// Instruction descriptor: D f32, A and B both f16 (0) or bf16 (1).
inline uint32_t idesc_16(int type, int M, int N, int a_mn, int b_mn) {
  const uint32_t f = type == VCB_BF16 ? 1 : 0;
  return (1u << 4) | (f << 7) | (f << 10) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) |
         ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

template <bool PAIR>
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                        uint32_t accumulate) {
  if (PAIR)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate));
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate));
}

// One operand's descriptors: of the first stage, and their steps (in the
// descriptor's 16-byte units) per 16 of the contraction and per stage.  The
// address field of a descriptor has room for every stage, so adding to the low
// word suffices.
struct Desc {
  uint64_t base;
  uint32_t k, stage;
};

__device__ __forceinline__ Desc operand(uint32_t saddr, int mn, uint32_t stage_bytes,
                                        uint32_t box = 8192) {
  return {operand_desc(saddr, mn, box), (mn ? 2048u : 32u) >> 4, stage_bytes >> 4};
}

// The four MMAs of stage s.
template <bool PAIR>
__device__ __forceinline__ void mma_stage(uint32_t d, const Desc& a, const Desc& b, uint32_t s,
                                          uint32_t idesc, bool first) {
  const uint64_t da = a.base + s * a.stage, db = b.base + s * b.stage;
#pragma unroll
  for (int k = 0; k < kBK / 16; ++k)
    mma_f16<PAIR>(d, da + k * a.k, db + k * b.k, idesc, first && k == 0 ? 0u : 1u);
}

// A position in a ring of stages and the parity of its use.
struct Ring {
  int s = 0;
  unsigned parity = 0;
  __device__ __forceinline__ void next(int stages) {
    if (++s == stages) s = 0, parity ^= 1;
  }
};

// Arrive on `bar` of both CTAs of the pair when the MMAs issued so far are done.
__device__ __forceinline__ void commit_pair(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 "
      "[%0], %1;" ::"r"(smem_u32(bar)),
      "h"((uint16_t)3)
      : "memory");
}

__device__ __forceinline__ float peer_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

__device__ __forceinline__ float4 peer_f32x4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

// Tile u of a product: eight tile rows i share the tiles j that run beside
// them, so that concurrent CTAs read few distinct operand rows.
__device__ __forceinline__ void tile_at(int tiles_i, int tiles_j, int u, int& ti, int& tj) {
  constexpr int G = 8;
  const int per = G * tiles_j, g = u / per, in = u - g * per;
  const int rows = min(G, tiles_i - g * G);
  ti = g * G + in % rows;
  tj = in / rows;
}

// Launches in clusters of `size`; with `chained` as the kernel before it runs out.
template <typename Args>
int launch_clusters(void (*kernel)(Args), const Args& args, dim3 grid, int threads, int smem,
                    int size, bool chained, cudaStream_t st, const char* who) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = size;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = chained ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args);
  if (e != cudaSuccess) return cuda_fail(e, who);
  return check_launch(who);
}

// CTAs of a kernel with one CTA per SM that run at the same time in clusters of `size`:
// a cluster lies in one group of SMs, and the groups of a B200 hold 15 clusters of 8
// rather than 148 / 8.  A sixteenth would run alone after them.
template <typename Args>
int cluster_slots(void (*kernel)(Args), int threads, int smem, int size) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(size);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = size;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  int clusters = 0;
  if (ensure_smem(reinterpret_cast<const void*>(kernel), smem) != VCB_OK ||
      cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg) != cudaSuccess || clusters < 1) {
    cudaGetLastError();
    clusters = sm_count() / size;
  }
  return clusters * size;
}

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static const PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) !=
            cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  }();
  return fn;
}

}  // namespace
}  // namespace lin
}  // namespace vcb
