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

__device__ __forceinline__ float sqrt_fast(float x) {
  float y;
  asm("sqrt.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Larger of the two, NaN when either is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

// 32 noise bits of an element: three multiply-xorshift rounds (multiplicative
// hashing) with the fractional bits of the golden ratio, sqrt 2 and sqrt 3.
__device__ __forceinline__ uint32_t noise(uint32_t index, uint32_t key) {
  uint32_t x = (index + key) * 0x9E3779B9u;
  x = (x ^ (x >> 16)) * 0x6A09E667u;
  x = (x ^ (x >> 15)) * 0xBB67AE85u;
  return x ^ (x >> 16);
}

__device__ __forceinline__ float four(float c) {
  const float q = __fmul_rn(c, c);
  return __fmul_rn(q, q);
}

__device__ __forceinline__ float m_value(int8_t code, float scale) {
  const float c = code;
  return __fmul_rn(scale, __fmul_rn(__fmul_rn(c, fabsf(c)), 1.f / 16129.f));
}

__device__ __forceinline__ float v_value(uint8_t code, float scale) {
  return __fmul_rn(scale, __fmul_rn(four(code), static_cast<float>(1.0 / 4228250625.0)));
}

// The largest c with c^2 <= y, or the next one with the probability
// (y - c^2) / (2c + 1): the approximate root is off by one at most.
__device__ __forceinline__ int8_t m_code(float m, float inv, float r) {
  const float y = __fmul_rn(__fmul_rn(fabsf(m), inv), 16129.f);
  float c = fminf(floorf(sqrt_fast(y)), 126.f);
  if (c * c > y) c -= 1.f;
  if ((c + 1.f) * (c + 1.f) <= y && c < 126.f) c += 1.f;
  if (__fmul_rn(r, 2.f * c + 1.f) < __fsub_rn(y, c * c)) c += 1.f;
  return static_cast<int8_t>(m < 0.f ? -static_cast<int>(c) : static_cast<int>(c));
}

__device__ __forceinline__ uint8_t v_code(float v, float inv, float r) {
  const float y = __fmul_rn(__fmul_rn(v, inv), 4228250625.f);
  float c = fminf(floorf(sqrt_fast(sqrt_fast(y))), 254.f);
  if (four(c) > y) c -= 1.f;
  if (four(c + 1.f) <= y && c < 254.f) c += 1.f;
  const float lo = four(c);
  if (__fmul_rn(r, __fsub_rn(four(c + 1.f), lo)) < __fsub_rn(y, lo)) c += 1.f;
  if (y > 0.f && c < 1.f) c = 1.f;
  return static_cast<uint8_t>(c);
}

template <typename T>
__device__ __forceinline__ void get4(const T* p, int live, bool vec, float (&v)[4]) {
  if (vec && live >= 4) {
    load4(p, v);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i < live ? to_f32(p[i]) : 0.f;
  }
}

template <typename T>
__device__ __forceinline__ void put4(T* p, int live, bool vec, const float (&v)[4]) {
  if (vec && live >= 4) {
    store4(p, v);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < live) p[i] = from_f32<T>(v[i]);
  }
}

template <typename PT, typename GT, int BITS, int CAP>
__global__ void __launch_bounds__(kWarps * 32)
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
  const bool vec = e.vec;
  PT* p = static_cast<PT*>(e.p) + at;
  const GT* g = static_cast<const GT*>(e.g) + at;
  const long long off = e.off + at;  // of this block in the state
  const long long left = e.n - at;
  int live[2];
  float pv[2][4], gv[2][4], m[2][4], v[2][4];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int i = h * 128 + lane * 4;
    live[h] = static_cast<int>(max(0LL, min(4LL, left - i)));
    get4(p + i, live[h], vec, pv[h]);
    get4(g + i, live[h], vec, gv[h]);
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
      const char4 mc = *reinterpret_cast<const char4*>(static_cast<const int8_t*>(s.m) + i);
      const uchar4 vc = *reinterpret_cast<const uchar4*>(static_cast<const uint8_t*>(s.v) + i);
      m[h][0] = m_value(mc.x, ms), m[h][1] = m_value(mc.y, ms);
      m[h][2] = m_value(mc.z, ms), m[h][3] = m_value(mc.w, ms);
      v[h][0] = v_value(vc.x, vs), v[h][1] = v_value(vc.y, vs);
      v[h][2] = v_value(vc.z, vs), v[h][3] = v_value(vc.w, vs);
    } else {
      load4(static_cast<const float*>(s.m) + i, m[h]);
      load4(static_cast<const float*>(s.v) + i, v[h]);
    }
  }
  const vcb_adamw_opts& o = s.o;
  float big = 0.f, most = 0.f;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float gj = gv[h][j];
      // each product and sum rounded by itself: the codes of an 8-bit state
      // do not depend on how a compiler contracts them
      m[h][j] = __fadd_rn(__fmul_rn(m[h][j], o.b1), __fmul_rn(gj, o.c1));
      v[h][j] = __fadd_rn(__fmul_rn(v[h][j], o.b2), __fmul_rn(__fmul_rn(gj, o.c2), gj));
      const float d = __fdividef(m[h][j], sqrt_fast(v[h][j]) * o.root + o.eps);
      pv[h][j] = __fsub_rn(__fmul_rn(pv[h][j], o.keep), __fmul_rn(d, o.size));
      if (BITS == 8) {
        big = max_nan(big, fabsf(m[h][j]));
        most = max_nan(most, v[h][j]);
      }
    }
    put4(p + h * 128 + lane * 4, live[h], vec, pv[h]);
  }
  if (BITS == 8) {
#pragma unroll
    for (int k = 16; k; k >>= 1) {
      big = max_nan(big, __shfl_xor_sync(0xffffffffu, big, k));
      most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, k));
    }
    // a scale below the normal range counts as zero; NaN and infinity stay and
    // mark the whole block
    if (big < FLT_MIN) big = 0.f;
    if (most < FLT_MIN) most = 0.f;
    const float im = big > 0.f ? __frcp_rn(big) : 0.f, iv = most > 0.f ? __frcp_rn(most) : 0.f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const long long i = off + h * 128 + lane * 4;
      int8_t mc[4];
      uint8_t vc[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t x = noise(static_cast<uint32_t>(i + j), o.key);
        mc[j] = m_code(m[h][j], im, static_cast<float>(x >> 16) * (1.f / 65536.f));
        vc[j] = v_code(v[h][j], iv, static_cast<float>(x & 0xFFFFu) * (1.f / 65536.f));
      }
      *reinterpret_cast<char4*>(static_cast<int8_t*>(s.m) + i) =
          make_char4(mc[0], mc[1], mc[2], mc[3]);
      *reinterpret_cast<uchar4*>(static_cast<uint8_t*>(s.v) + i) =
          make_uchar4(vc[0], vc[1], vc[2], vc[3]);
    }
    if (lane == 0) {
      s.ms[off / kBlock] = big;
      s.vs[off / kBlock] = most;
    }
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const long long i = off + h * 128 + lane * 4;
      store4(static_cast<float*>(s.m) + i, m[h]);
      store4(static_cast<float*>(s.v) + i, v[h]);
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
  const char4 mc = *reinterpret_cast<const char4*>(m + i);
  const uchar4 vc = *reinterpret_cast<const uchar4*>(v + i);
  store4(mo + i, {m_value(mc.x, a), m_value(mc.y, a), m_value(mc.z, a), m_value(mc.w, a)});
  store4(vo + i, {v_value(vc.x, b), v_value(vc.y, b), v_value(vc.z, b), v_value(vc.w, b)});
}

template <typename PT, typename GT, int BITS>
int launch(const vcb_adamw_tensor* t, int count, const State& s, cudaStream_t st) {
  const int pb = sizeof(PT), gb = sizeof(GT);
  for (int a = 0; a < count;) {
    Table<kLargeTable> tab;
    tab.count = 0;
    long long ctas = 0;
    for (; a < count && tab.count < kLargeTable; ++a) {
      if (t[a].n == 0) continue;
      const long long own = (t[a].n + kChunk - 1) / kChunk;
      if (ctas + own > 0x7fffffffLL) {
        if (tab.count == 0) return fail(VCB_ERR_UNSUPPORTED, "vcb_adamw: tensor %d too large", a);
        break;
      }
      const bool vec = reinterpret_cast<uintptr_t>(t[a].p) % (4 * pb) == 0 &&
                       reinterpret_cast<uintptr_t>(t[a].g) % (4 * gb) == 0;
      tab.e[tab.count++] = {t[a].p, t[a].g, t[a].n, t[a].off, static_cast<int>(ctas), vec};
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
int dispatch(const vcb_adamw_tensor* t, int count, int pt, int gt, const State& s,
             cudaStream_t st) {
  if (pt == VCB_F32) return launch<float, float, BITS>(t, count, s, st);
  if (pt == VCB_BF16)
    return gt == VCB_F32 ? launch<__nv_bfloat16, float, BITS>(t, count, s, st)
                         : launch<__nv_bfloat16, __nv_bfloat16, BITS>(t, count, s, st);
  return gt == VCB_F32 ? launch<__half, float, BITS>(t, count, s, st)
                       : launch<__half, __half, BITS>(t, count, s, st);
}

}  // namespace
}  // namespace vcb

using namespace vcb;

extern "C" int vcb_adamw(int32_t count, const vcb_adamw_tensor* tensors, int32_t p_type,
                         int32_t g_type, int32_t state_bits, void* m, void* v, float* m_scale,
                         float* v_scale, const vcb_adamw_opts* opts, void* stream) {
  if (count < 0 || (count > 0 && !tensors) || !opts || !valid_dtype(p_type) ||
      !(g_type == p_type || g_type == VCB_F32) || (state_bits != 8 && state_bits != 32))
    return fail(VCB_ERR_INVALID, "vcb_adamw: count=%d p_type=%d g_type=%d state_bits=%d", count,
                p_type, g_type, state_bits);
  bool any = false;
  for (int i = 0; i < count; ++i) {
    const vcb_adamw_tensor& t = tensors[i];
    if (t.n < 0 || t.off < 0 || t.off % kBlock || (t.n > 0 && (!t.p || !t.g)) ||
        reinterpret_cast<uintptr_t>(t.p) % dtype_bytes(p_type) ||
        reinterpret_cast<uintptr_t>(t.g) % dtype_bytes(g_type))
      return fail(VCB_ERR_INVALID, "vcb_adamw: tensor %d: n=%lld off=%lld", i,
                  static_cast<long long>(t.n), static_cast<long long>(t.off));
    any |= t.n > 0;
  }
  if (!any) return VCB_OK;
  auto off16 = [](const void* q) { return reinterpret_cast<uintptr_t>(q) % 16 != 0; };
  if (!m || !v || off16(m) || off16(v) || (state_bits == 8 && (!m_scale || !v_scale)))
    return fail(VCB_ERR_INVALID, "vcb_adamw: the state must be there and 16-byte aligned");
  const State s{m, v, m_scale, v_scale, *opts};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return state_bits == 8 ? dispatch<8>(tensors, count, p_type, g_type, s, st)
                         : dispatch<32>(tensors, count, p_type, g_type, s, st);
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
