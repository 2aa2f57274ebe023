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
// Preparation (two 2048^2 operands: 16 us, 27 % of DRAM, 56 % of issue slots): one
// launch reads each operand once and writes its three parts (backward: dz = dy act'(z) and db in strips of columns, W and X flat
// beside them).  The parts of dz serve both products, read along either index.
// Then products as in vcb_linear_tc.cu: sum_kernel<float, 3, 256, true> in CTA pairs for
// large ones, sum_kernel<float, 3, 64 / 128, false> with the contraction cut over a cluster
// for the rest.
#include <algorithm>
#include <array>
#include <initializer_list>

#include "vcb_linear_sum.cuh"

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
    using C = Cfg<kParts, 128, false>;
    std::array<int, 4> n;
    for (int k = 0; k < 4; ++k)
      n[k] = cluster_slots(sum_kernel<float, kParts, 128, false>, kSumThreads, C::kSmem, 1 << k);
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

int set_prod(SumProd& r, int I, int J, int T, const Matrix& a, bool a_mn, const Matrix& b, bool b_mn,
             const Plan32& plan, const Epilogue& epi, const char* who) {
  const auto of = [](const Matrix& m, bool mn) {
    return SumOperand{m.parts, static_cast<int>(m.rows), m.cols, m.ldp, m.plane, mn};
  };
  return set_sum<kParts>(r, VCB_BF16, I, J, T, of(a, a_mn), of(b, b_mn), plan.bn, plan.pair, epi, 4,
                         who);
}

int launch_plan(SumLaunch& L, const Plan32& plan, bool chained, cudaStream_t st,
                const char* who) {
  if (plan.pair) return launch_sum<float, kParts, 256, true>(L, chained, st, who);
  return plan.bn == 64 ? launch_sum<float, kParts, 64, false>(L, chained, st, who)
                       : launch_sum<float, kParts, 128, false>(L, chained, st, who);
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
  SumLaunch L{};
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

namespace {
// One launch for both products unless their shapes want different cuts by more than
// a launch costs.
struct BackwardPlan {
  Plan32 x, w;
  bool together;
};

BackwardPlan backward_plan(int M, int N, int K, bool dx, bool dw) {
  const Shape x{M, K, N}, w{N, K, M};
  BackwardPlan p{plan_of({x}), plan_of({w}), false};
  const Plan32 both = plan_of({x, w});
  p.together = dx && dw && both.cycles < p.x.cycles + p.w.cycles + 9000;
  if (p.together) p.x = p.w = both;
  return p;
}
}  // namespace

int f32_path(int M, int N, int K, int product) {
  if (product == 0) return plan_of({{M, N, K}}).pair ? 3 : 2;
  const BackwardPlan p = backward_plan(M, N, K, true, true);
  return (product == 1 ? p.x : p.w).pair ? 3 : 2;
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
  const BackwardPlan plan = backward_plan(b.M, b.N, b.K, b.dx, b.dw);
  const Plan32 px = plan.x, pw = plan.w;
  const bool together = plan.together;
  SumLaunch L{};
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
  SumProd& p = L.p[together ? 1 : 0];
  rc = set_prod(p, b.N, b.K, b.M, x, true, dz, true, pw, ew, who);
  if (rc) return rc;
  L.units += p.tiles_i * p.tiles_j;
  if (!together) L.units0 = L.units;
  L.split = pw.split;
  return launch_plan(L, pw, together || !b.dx, st, who);
}

}  // namespace lin
}  // namespace vcb
