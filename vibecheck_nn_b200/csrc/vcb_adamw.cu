// AdamW over many tensors in one launch, moments in 32 or in 8 bits.
//
//   m = b1 m + (1 - b1) g,   v = b2 v + (1 - b2) g^2,
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v / (1 - b2^t)) + eps)
//
// 8-bit moments are kept per block of 256 elements with the block's largest
// |m| = M and v = V in fp32:  m = M sgn(c) (c / 127)^2,  v = V (c / 255)^4.
// The powers spend the codes near zero, where most moments of a block lie:
// v spans 4e9 : 1 inside a block.  A new value between two codes goes up with
// the probability that keeps its mean, or an average that moves by (1 - b2) =
// 0.1 % a step would be rounded back for ever.  A v that is not zero never
// gets code 0: m / (sqrt(0) + eps) would be a jump.  The random bits are a
// hash of the element's place in the state, the step and the seed, so a run
// is repeatable.  The weight moves by the moments before they are coded.
//
// Bound by HBM: each weight, gradient and moment is read once and written
// once.  One warp takes one block of 256 elements (8 per lane, as two groups
// of 4 so that every access of a warp is contiguous), holds it in registers,
// and finds M and V by shuffles; no shared memory, no second pass.  The tensor
// table travels as a kernel parameter, so nothing is uploaded per step.
//
// Measured on 134 M weights: fp32 with 32-bit moments 546 us (6.9 TB/s, at HBM's
// rate); fp32 with 8-bit moments 380 us (the square roots, the search for codes and
// the noise of two moments per weight are as long as its 12 bytes), bf16 with 8-bit
// moments 400 us (arithmetic alone).
#include <cfloat>

#include "vcb_common.cuh"
#include "vcb_types.cuh"

namespace vcb {
namespace {

constexpr int kBlock = 256;       // elements per 8-bit scale, one warp's share
constexpr int kWarps = 8;
constexpr int kChunk = kBlock * kWarps;  // elements per CTA

struct Entry {
  void* p;
  const void* g;
  long long n, off;
  int first;  // first CTA of this tensor
  int vec;    // p and g aligned to 4 elements
};

// Kernel parameters may take 32,764 bytes; a small table keeps the launch of
// a small network cheap.
constexpr int kSmallTable = 32, kLargeTable = 640;

template <int CAP>
struct Table {
  int count;
  Entry e[CAP];
};

struct State {
  void *m, *v;
  float *ms, *vs;
  vcb_adamw_opts o;
};

// Approximate square root and reciprocal; what lies below the normal range
// counts as 0.
__device__ __forceinline__ float sqrt_flush(float x) {
  float y;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float rcp_flush(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Largest of the three magnitudes, NaN when one is.
__device__ __forceinline__ float max_nan(float a, float b, float c) {
  float y;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}

// Two floats in one instruction: the kernel is bound by issue slots.  Each
// result is rounded by itself, as by the scalar instructions.
struct F2 {
  float x, y;
};

#define VCB_F2_OP2(name, op)                                                           \
  __device__ __forceinline__ F2 name(F2 a, F2 b) {                                     \
    F2 r;                                                                              \
    asm("{\n\t.reg .b64 a, b, r;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t" op \
        " r, a, b;\n\tmov.b64 {%0, %1}, r;\n\t}"                                      \
        : "=f"(r.x), "=f"(r.y)                                                         \
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));                                     \
    return r;                                                                          \
  }
VCB_F2_OP2(mul2, "mul.rn.f32x2")
VCB_F2_OP2(add2, "add.rn.f32x2")
VCB_F2_OP2(add2_rz, "add.rz.f32x2")
#undef VCB_F2_OP2

__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("{\n\t.reg .b64 a, b, c, r;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "mov.b64 c, {%6, %7};\n\tfma.rn.f32x2 r, a, b, c;\n\tmov.b64 {%0, %1}, r;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}

__device__ __forceinline__ F2 both(float x) { return {x, x}; }

// Sums of products are added one by one: an add.f32x2 of a mul.f32x2 becomes one
// fma, whose single rounding gives other codes.
__device__ __forceinline__ F2 sum_of(F2 a, F2 b) {
  return {__fadd_rn(a.x, b.x), __fadd_rn(a.y, b.y)};
}

// 32 noise bits of an element: three multiply-xorshift rounds (multiplicative
// hashing) with the fractional bits of the golden ratio, sqrt 2 and sqrt 3.
// x: (index + key) kGolden.
constexpr uint32_t kGolden = 0x9E3779B9u;
__device__ __forceinline__ uint32_t noise(uint32_t x) {
  x = (x ^ (x >> 16)) * 0x6A09E667u;
  x = (x ^ (x >> 15)) * 0xBB67AE85u;
  return x ^ (x >> 16);
}

// Conversions between small integers and floats go by the mantissa of 2^23 + n,
// not by the conversion instructions: those share a pipe of an eighth of the
// rate with the square roots, and the twelve of them per element were what bound
// the kernel.
constexpr float kBig = 8388608.f;  // 2^23

// 2^23 + byte / half word k of w.
__device__ __forceinline__ float big_byte(uint32_t w, int k) {
  return __uint_as_float(__byte_perm(w, 0x4B000000u, 0x7440 | k));
}
__device__ __forceinline__ float big_half(uint32_t w, int k) {
  return __uint_as_float(__byte_perm(w, 0x4B000000u, k ? 0x7432 : 0x7410));
}

// floor(x) for 0 <= x < 2^22.
__device__ __forceinline__ F2 floor2(F2 x) { return add2(add2_rz(x, both(kBig)), both(-kBig)); }

// The low bytes of four integers held as floats, each 2^23 + n.
__device__ __forceinline__ uint32_t pack4(F2 n, F2 k) {
  const uint32_t a = __byte_perm(__float_as_uint(n.x), __float_as_uint(n.y), 0x0040);
  const uint32_t b = __byte_perm(__float_as_uint(k.x), __float_as_uint(k.y), 0x0040);
  return __byte_perm(a, b, 0x5410);
}

__device__ __forceinline__ F2 four(F2 c) {
  const F2 q = mul2(c, c);
  return mul2(q, q);
}

// Moments of the codes k and k + 1 of a word; signed codes come as c + 128 (the
// sign bit flipped in all four bytes).
__device__ __forceinline__ F2 m_value(uint32_t flipped, int k, float scale) {
  const F2 c = add2({big_byte(flipped, k), big_byte(flipped, k + 1)}, both(-kBig - 128.f));
  return mul2(both(scale), mul2(mul2(c, {fabsf(c.x), fabsf(c.y)}), both(1.f / 16129.f)));
}

__device__ __forceinline__ F2 v_value(uint32_t codes, int k, float scale) {
  const F2 c = add2({big_byte(codes, k), big_byte(codes, k + 1)}, both(-kBig));
  return mul2(both(scale), mul2(four(c), both(static_cast<float>(1.0 / 4228250625.0))));
}

// Square roots here are approximate; a factor just above 1 keeps a root from
// falling below its integer, and one comparison takes back what that adds.
constexpr float kAbove = 1.f + 0x1p-20f;

// The codes of |m| / M = y / 127^2: the largest c with c^2 <= y, or the next one
// with the probability (y - c^2) / (2c + 1).  r: 16 random bits.  Returns 2^23 +
// 128 + the signed code.
__device__ __forceinline__ F2 m_code(F2 m, float inv, F2 r) {
  const F2 y = mul2(mul2({fabsf(m.x), fabsf(m.y)}, both(inv)), both(16129.f));
  F2 c = floor2(mul2({sqrt_flush(y.x), sqrt_flush(y.y)}, both(kAbove)));
  const F2 q = mul2(c, c);
  if (q.x > y.x) c.x -= 1.f;
  if (q.y > y.y) c.y -= 1.f;
  const F2 odds = mul2(r, fma2(both(2.f), c, both(1.f)));
  const F2 rest = mul2(fma2({-c.x, -c.y}, c, y), both(65536.f));
  if (odds.x < rest.x) c.x += 1.f;
  if (odds.y < rest.y) c.y += 1.f;
  c = {copysignf(fminf(c.x, 127.f), m.x), copysignf(fminf(c.y, 127.f), m.y)};
  return add2(c, both(kBig + 128.f));
}

// The codes of v / V = y / 255^4; root: about y^(1/4), kAbove included.  Returns
// 2^23 + code.
__device__ __forceinline__ F2 v_code(F2 v, float inv, F2 root, F2 r) {
  const F2 y = mul2(mul2(v, both(inv)), both(4228250625.f));
  F2 c = floor2(root);
  const F2 q = four(c);
  if (q.x > y.x) c.x -= 1.f;
  if (q.y > y.y) c.y -= 1.f;
  const F2 lo = four(c), minus = {-lo.x, -lo.y};
  const F2 odds = mul2(r, sum_of(four(add2(c, both(1.f))), minus));
  const F2 rest = mul2(sum_of(y, minus), both(65536.f));
  if (odds.x < rest.x) c.x += 1.f;
  if (odds.y < rest.y) c.y += 1.f;
  c = {fminf(c.x, 255.f), fminf(c.y, 255.f)};
  if (y.x > 0.f) c.x = fmaxf(c.x, 1.f);
  if (y.y > 0.f) c.y = fmaxf(c.y, 1.f);
  return add2(c, both(kBig));
}

// Four elements of a tensor, of which `live` exist; `whole`: all do, and their
// address is that of a vector.
template <typename T>
__device__ __forceinline__ void get4(const T* p, int live, bool whole, F2 (&v)[2]) {
  float t[4];
  if (whole) {
    load4(p, t);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) t[i] = i < live ? to_f32(p[i]) : 0.f;
  }
  v[0] = {t[0], t[1]}, v[1] = {t[2], t[3]};
}

template <typename T>
__device__ __forceinline__ void put4(T* p, int live, bool whole, const F2 (&v)[2]) {
  const float t[4] = {v[0].x, v[0].y, v[1].x, v[1].y};
  if (whole) {
    store4(p, t);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < live) p[i] = from_f32<T>(t[i]);
  }
}

template <typename PT, typename GT, int BITS, int CAP>
__global__ void __launch_bounds__(kWarps * 32, 5)
    adamw_kernel(const __grid_constant__ Table<CAP> tab, const __grid_constant__ State s) {
  // the tensor of this CTA: the last whose first CTA is not behind it
  int lo = 0, hi = tab.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (tab.e[mid].first <= static_cast<int>(blockIdx.x)) lo = mid; else hi = mid - 1;
  }
  const Entry& e = tab.e[lo];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long at = static_cast<long long>(blockIdx.x - e.first) * kChunk + warp * kBlock;
  if (at >= e.n) return;
  PT* p = static_cast<PT*>(e.p) + at;
  const GT* g = static_cast<const GT*>(e.g) + at;
  const long long off = e.off + at;  // of this block in the state
  const int left = static_cast<int>(min(e.n - at, static_cast<long long>(kBlock)));
  const bool whole = e.vec && left == kBlock;  // of the warp
  // per lane two groups of four, each in two pairs
  F2 pv[2][2], gv[2][2], m[2][2], v[2][2], root[2][2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int i = h * 128 + lane * 4;
    get4(p + i, left - i, whole, pv[h]);
    get4(g + i, left - i, whole, gv[h]);
  }
  float ms = 0.f, vs = 0.f;
  if (BITS == 8) {
    ms = s.ms[off / kBlock];
    vs = s.vs[off / kBlock];
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const long long i = off + h * 128 + lane * 4;
    if (BITS == 8) {
      const uint32_t mc =
          *reinterpret_cast<const uint32_t*>(static_cast<const int8_t*>(s.m) + i) ^ 0x80808080u;
      const uint32_t vc = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(s.v) + i);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        m[h][j] = m_value(mc, 2 * j, ms);
        v[h][j] = v_value(vc, 2 * j, vs);
      }
    } else {
      get4(static_cast<const float*>(s.m) + i, 4, true, m[h]);
      get4(static_cast<const float*>(s.v) + i, 4, true, v[h]);
    }
  }
  const vcb_adamw_opts& o = s.o;
  float big = 0.f, most = 0.f;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const F2 gj = gv[h][j];
      m[h][j] = sum_of(mul2(m[h][j], both(o.b1)), mul2(gj, both(o.c1)));
      v[h][j] = sum_of(mul2(v[h][j], both(o.b2)), mul2(mul2(gj, both(o.c2)), gj));
      root[h][j] = {sqrt_flush(v[h][j].x), sqrt_flush(v[h][j].y)};
      const F2 d = fma2(root[h][j], both(o.root), both(o.eps));
      const F2 step = mul2(mul2(m[h][j], {rcp_flush(d.x), rcp_flush(d.y)}), both(-o.size));
      pv[h][j] = add2(mul2(pv[h][j], both(o.keep)), step);
      if (BITS == 8) {
        big = max_nan(big, m[h][j].x, m[h][j].y);
        most = max_nan(most, v[h][j].x, v[h][j].y);
      }
    }
    const int i = h * 128 + lane * 4;
    put4(p + i, left - i, whole, pv[h]);
  }
  if (BITS == 8) {
#pragma unroll
    for (int k = 16; k; k >>= 1) {
      big = max_nan(big, big, __shfl_xor_sync(0xffffffffu, big, k));
      most = max_nan(most, most, __shfl_xor_sync(0xffffffffu, most, k));
    }
    // a scale below the normal range counts as zero; NaN and infinity stay and
    // mark the whole block
    if (big < FLT_MIN) big = 0.f;
    if (most < FLT_MIN) most = 0.f;
    const float im = big > 0.f ? __frcp_rn(big) : 0.f, iv = most > 0.f ? __frcp_rn(most) : 0.f;
    // y^(1/4) = sqrt(sqrt(v) sqrt(255^4 / V))
    const F2 up = both(sqrtf(iv) * (65025.f * kAbove));
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const long long i = off + h * 128 + lane * 4;
      const uint32_t x0 = (static_cast<uint32_t>(i) + o.key) * kGolden;
      F2 mc[2], vc[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint32_t x = noise(x0 + 2 * j * kGolden), y = noise(x0 + (2 * j + 1) * kGolden);
        const F2 t = mul2(root[h][j], up);
        mc[j] = m_code(m[h][j], im, add2({big_half(x, 1), big_half(y, 1)}, both(-kBig)));
        vc[j] = v_code(v[h][j], iv, {sqrt_flush(t.x), sqrt_flush(t.y)},
                       add2({big_half(x, 0), big_half(y, 0)}, both(-kBig)));
      }
      *reinterpret_cast<uint32_t*>(static_cast<int8_t*>(s.m) + i) =
          pack4(mc[0], mc[1]) ^ 0x80808080u;
      *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(s.v) + i) = pack4(vc[0], vc[1]);
    }
    if (lane == 0) {
      s.ms[off / kBlock] = big;
      s.vs[off / kBlock] = most;
    }
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const long long i = off + h * 128 + lane * 4;
      put4(static_cast<float*>(s.m) + i, 4, true, m[h]);
      put4(static_cast<float*>(s.v) + i, 4, true, v[h]);
    }
  }
}

// The values 8-bit moments stand for; one thread per 4 elements.
__global__ void __launch_bounds__(256)
    adamw_values_kernel(long long quads, const int8_t* __restrict__ m, const uint8_t* __restrict__ v,
                        const float* __restrict__ ms, const float* __restrict__ vs,
                        float* __restrict__ mo, float* __restrict__ vo) {
  const long long q = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (q >= quads) return;
  const long long i = q * 4;
  const float a = ms[i / kBlock], b = vs[i / kBlock];
  const uint32_t mc = *reinterpret_cast<const uint32_t*>(m + i) ^ 0x80808080u;
  const uint32_t vc = *reinterpret_cast<const uint32_t*>(v + i);
  put4(mo + i, 4, true, {m_value(mc, 0, a), m_value(mc, 2, a)});
  put4(vo + i, 4, true, {v_value(vc, 0, b), v_value(vc, 2, b)});
}

// The tensors of a call: arrays of `count`.
struct Tensors {
  int count;
  void* const* p;
  const void* const* g;
  const int64_t *n, *off;
};

template <typename PT, typename GT, int BITS>
int launch(const Tensors& t, const State& s, cudaStream_t st) {
  const int pb = sizeof(PT), gb = sizeof(GT);
  for (int a = 0; a < t.count;) {
    Table<kLargeTable> tab;
    tab.count = 0;
    long long ctas = 0;
    for (; a < t.count && tab.count < kLargeTable; ++a) {
      if (t.n[a] == 0) continue;
      const long long own = (t.n[a] + kChunk - 1) / kChunk;
      if (ctas + own > 0x7fffffffLL) {
        if (tab.count == 0) return fail(VCB_ERR_UNSUPPORTED, "vcb_adamw: tensor %d too large", a);
        break;
      }
      const bool vec = reinterpret_cast<uintptr_t>(t.p[a]) % (4 * pb) == 0 &&
                       reinterpret_cast<uintptr_t>(t.g[a]) % (4 * gb) == 0;
      tab.e[tab.count++] = {t.p[a], t.g[a], t.n[a], t.off[a], static_cast<int>(ctas), vec};
      ctas += own;
    }
    if (tab.count == 0) break;
    if (tab.count <= kSmallTable) {
      Table<kSmallTable> small;
      small.count = tab.count;
      for (int i = 0; i < tab.count; ++i) small.e[i] = tab.e[i];
      adamw_kernel<PT, GT, BITS, kSmallTable>
          <<<static_cast<unsigned>(ctas), kWarps * 32, 0, st>>>(small, s);
    } else {
      adamw_kernel<PT, GT, BITS, kLargeTable>
          <<<static_cast<unsigned>(ctas), kWarps * 32, 0, st>>>(tab, s);
    }
    const int rc = check_launch("vcb_adamw");
    if (rc) return rc;
  }
  return VCB_OK;
}

template <int BITS>
int dispatch(const Tensors& t, int pt, int gt, const State& s, cudaStream_t st) {
  if (pt == VCB_F32) return launch<float, float, BITS>(t, s, st);
  if (pt == VCB_BF16)
    return gt == VCB_F32 ? launch<__nv_bfloat16, float, BITS>(t, s, st)
                         : launch<__nv_bfloat16, __nv_bfloat16, BITS>(t, s, st);
  return gt == VCB_F32 ? launch<__half, float, BITS>(t, s, st)
                       : launch<__half, __half, BITS>(t, s, st);
}

}  // namespace
}  // namespace vcb

using namespace vcb;

extern "C" int vcb_adamw(int32_t count, void* const* p, const void* const* g, const int64_t* n,
                         const int64_t* off, int32_t p_type, int32_t g_type, int32_t state_bits,
                         void* m, void* v, float* m_scale, float* v_scale,
                         const vcb_adamw_opts* opts, void* stream) {
  if (count < 0 || (count > 0 && (!p || !g || !n || !off)) || !opts || !valid_dtype(p_type) ||
      !(g_type == p_type || g_type == VCB_F32) || (state_bits != 8 && state_bits != 32))
    return fail(VCB_ERR_INVALID, "vcb_adamw: count=%d p_type=%d g_type=%d state_bits=%d", count,
                p_type, g_type, state_bits);
  bool any = false;
  for (int i = 0; i < count; ++i) {
    if (n[i] < 0 || off[i] < 0 || off[i] % kBlock || (n[i] > 0 && (!p[i] || !g[i])) ||
        reinterpret_cast<uintptr_t>(p[i]) % dtype_bytes(p_type) ||
        reinterpret_cast<uintptr_t>(g[i]) % dtype_bytes(g_type))
      return fail(VCB_ERR_INVALID, "vcb_adamw: tensor %d: n=%lld off=%lld", i,
                  static_cast<long long>(n[i]), static_cast<long long>(off[i]));
    any |= n[i] > 0;
  }
  if (!any) return VCB_OK;
  auto off16 = [](const void* q) { return reinterpret_cast<uintptr_t>(q) % 16 != 0; };
  if (!m || !v || off16(m) || off16(v) || (state_bits == 8 && (!m_scale || !v_scale)))
    return fail(VCB_ERR_INVALID, "vcb_adamw: the state must be there and 16-byte aligned");
  const Tensors t{count, p, g, n, off};
  const State s{m, v, m_scale, v_scale, *opts};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return state_bits == 8 ? dispatch<8>(t, p_type, g_type, s, st)
                         : dispatch<32>(t, p_type, g_type, s, st);
}

extern "C" int vcb_adamw_values(int64_t n, const void* m, const void* v, const float* m_scale,
                                const float* v_scale, float* m_out, float* v_out, void* stream) {
  if (n < 0 || n % kBlock) return fail(VCB_ERR_INVALID, "vcb_adamw_values: n=%lld", (long long)n);
  if (n == 0) return VCB_OK;
  auto off16 = [](const void* q) { return !q || reinterpret_cast<uintptr_t>(q) % 16 != 0; };
  if (off16(m) || off16(v) || !m_scale || !v_scale || off16(m_out) || off16(v_out))
    return fail(VCB_ERR_INVALID, "vcb_adamw_values: NULL or misaligned pointer");
  const long long ctas = (n / 4 + 255) / 256;
  if (ctas > 0x7fffffffLL) return fail(VCB_ERR_UNSUPPORTED, "vcb_adamw_values: n=%lld", (long long)n);
  adamw_values_kernel<<<static_cast<unsigned>(ctas), 256, 0, static_cast<cudaStream_t>(stream)>>>(
      n / 4, static_cast<const int8_t*>(m), static_cast<const uint8_t*>(v), m_scale, v_scale, m_out,
      v_out);
  return check_launch("vcb_adamw_values");
}
