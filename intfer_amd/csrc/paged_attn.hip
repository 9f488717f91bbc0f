// Attention of new rows over a caller-owned paged cache (fp16, int8 or int4
// pages), with optional score cap, distance bias and per-row visible range.
//
//   a = scale q.k;  a = cap tanh(a / cap);  a -= slope_h |pos - t|
//   o = sum_t softmax(a)_t v_t over the t in [lo, hi) of the row
//
// A column is (new row, head of the kv head's group).  S^T = K Q^T and
// O^T = V^T P^T, so the columns are the MFMA's columns, the running maximum
// and sum of a column live in its lanes, and P leaves the first product in the
// lanes the second one wants it in (paged_vtok gives V that token order).
// Quantized codes become the fp16 values that they stand for in registers:
// from there on all formats are the same kernel.
//
// Places that a row does not see: their scores are replaced, not added to, and
// in pages that some row sees only in part ("edge" pages) V is cleared where no
// column looks and where it is not finite; what a column sees of the latter
// goes into that column's result alone.
#include "ifr_dev.h"
#include "ifr_paged.h"

#include <type_traits>

namespace ifrk {
namespace {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef float v16f __attribute__((ext_vector_type(16)));

constexpr float kLog2e = 1.44269504088896340736f;

__device__ __forceinline__ h2 as_h2(uint32_t x) { return __builtin_bit_cast(h2, x); }
__device__ __forceinline__ uint32_t as_u(h2 x) { return __builtin_bit_cast(uint32_t, x); }
__device__ __forceinline__ h2 both(uint16_t x) { return as_h2((uint32_t)x | ((uint32_t)x << 16)); }

// 8 int4 codes -> fp16 pairs of neighbours, exact: a nibble under the exponent
// 0x64 is 1024 + c, one four bits higher 1024 + 16 c.
__device__ __forceinline__ void codes4(uint32_t w, h2 (&c)[4]) {
  const h2 k1024 = {(_Float16)1024.0f, (_Float16)1024.0f};
  const h2 k16 = {(_Float16)0.0625f, (_Float16)0.0625f}, k64 = {(_Float16)-64.0f, (_Float16)-64.0f};
  const uint32_t v = w >> 8;
  c[0] = as_h2((w & 0x000F000Fu) | 0x64006400u) - k1024;
  c[1] = __builtin_elementwise_fma(as_h2((w & 0x00F000F0u) | 0x64006400u), k16, k64);
  c[2] = as_h2((v & 0x000F000Fu) | 0x64006400u) - k1024;
  c[3] = __builtin_elementwise_fma(as_h2((v & 0x00F000F0u) | 0x64006400u), k16, k64);
}
// 4 int8 codes -> fp16 pairs, exact: b ^ 0x80 = b + 128 under 0x64 is 1024 + b + 128.
__device__ __forceinline__ void codes8(uint32_t w, h2& lo, h2& hi) {
  const h2 bias = {(_Float16)1152.0f, (_Float16)1152.0f};
  const uint32_t u = w ^ 0x80808080u;
  lo = as_h2(__builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) - bias;
  hi = as_h2(__builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) - bias;
}
__device__ __forceinline__ v8h join8(h2 a, h2 b, h2 c, h2 d) {
  return __builtin_bit_cast(v8h, (u4){as_u(a), as_u(b), as_u(c), as_u(d)});
}
// 8 dims of one token: one scale and minimum
template <int FMT>
__device__ __forceinline__ v8h k_values(const uint32_t* w, uint32_t sz) {
  if constexpr (FMT == IFR_KV_FP16) {
    return __builtin_bit_cast(v8h, (u4){w[0], w[1], w[2], w[3]});
  } else if constexpr (FMT == IFR_KV_INT8) {
    h2 c[4];
    codes8(w[0], c[0], c[1]);
    codes8(w[1], c[2], c[3]);
    const h2 s = both((uint16_t)sz);
    return join8(c[0] * s, c[1] * s, c[2] * s, c[3] * s);
  } else {
    h2 c[4];
    codes4(w[0], c);
    const h2 s = both((uint16_t)sz), z = both((uint16_t)(sz >> 16));
    return join8(__builtin_elementwise_fma(c[0], s, z), __builtin_elementwise_fma(c[1], s, z),
                 __builtin_elementwise_fma(c[2], s, z), __builtin_elementwise_fma(c[3], s, z));
  }
}
// 8 tokens of one dim: a scale and minimum each
template <int FMT>
__device__ __forceinline__ v8h v_values(const uint32_t* w, const uint32_t* s, const uint32_t* z) {
  if constexpr (FMT == IFR_KV_FP16) {
    return __builtin_bit_cast(v8h, (u4){w[0], w[1], w[2], w[3]});
  } else if constexpr (FMT == IFR_KV_INT8) {
    h2 c[4];
    codes8(w[0], c[0], c[1]);
    codes8(w[1], c[2], c[3]);
    return join8(c[0] * as_h2(s[0]), c[1] * as_h2(s[1]), c[2] * as_h2(s[2]), c[3] * as_h2(s[3]));
  } else {
    h2 c[4];
    codes4(w[0], c);
    return join8(__builtin_elementwise_fma(c[0], as_h2(s[0]), as_h2(z[0])),
                 __builtin_elementwise_fma(c[1], as_h2(s[1]), as_h2(z[1])),
                 __builtin_elementwise_fma(c[2], as_h2(s[2]), as_h2(z[2])),
                 __builtin_elementwise_fma(c[3], as_h2(s[3]), as_h2(z[3])));
  }
}

template <int N>
__device__ __forceinline__ void load_dwords(const uint8_t* p, uint32_t* w) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const u4 x = reinterpret_cast<const u4*>(p)[i];
      w[4 * i] = x[0]; w[4 * i + 1] = x[1]; w[4 * i + 2] = x[2]; w[4 * i + 3] = x[3];
    }
  } else if constexpr (N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const u2 x = reinterpret_cast<const u2*>(p)[i];
      w[2 * i] = x[0]; w[2 * i + 1] = x[1];
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = reinterpret_cast<const uint32_t*>(p)[i];
  }
}

// What a score becomes: in x[C] q.k, out the score times log2 e.
//
// cap tanh(z), z = scale q.k / cap, keeps errors relative to the result, so that
// small scores keep their bits.  While every |z| of the wave is at most 1/2
// (scores hardly ever come near their cap) it is z P(z^2), P the Chebyshev
// interpolation of tanh(z) / z in z^2 on [0, 1/4]: of degree 4 (1.4e-8 off) for
// fp32 outputs, 3 (6e-7, where the rounding of P and of the output is 2e-4) for
// fp16 ones, with every factor inside the coefficients: 5 or 6 operations a
// score.  Else, and where a power of scale / cap would leave fp32, 1 - 2 / (e^2z
// + 1) above 1/2.  The bias takes |pos - t| in fp32, exact up to 2^24; far(j) is
// pos - t of score j.
struct Scoring {
  float scale2;           // scale log2 e
  float inv, cap2;        // scale / cap, cap log2 e; inv 0: no cap
  float limit;            // |q.k| up to which f holds (negative: none)
  float f[5];             // cap2 P, times the powers of inv
  bool mod;               // cap or bias
};
constexpr float kTanh4[5] = {0.99999999f, -0.333330679f, 0.133247505f, -0.0529842388f, 0.0171313444f};
constexpr float kTanh3[5] = {0.999999451f, -0.333262842f, 0.131899394f, -0.0443927384f, 0.0f};
template <bool FINE>
__device__ __forceinline__ Scoring scoring(const PagedAttnArgs& a) {
  Scoring s;
  s.scale2 = a.scale * kLog2e;
  s.inv = a.cap != 0.0f ? a.scale / a.cap : 0.0f;
  s.cap2 = a.cap * kLog2e;
  s.limit = s.inv >= 1e-4f && s.inv <= 1e3f ? 0.5f / s.inv : -1.0f;
  float w = s.cap2 * s.inv;
#pragma unroll
  for (int i = 0; i < 5; ++i) {
    s.f[i] = (FINE ? kTanh4[i] : kTanh3[i]) * w;
    w *= s.inv * s.inv;
  }
  s.mod = a.cap != 0.0f || a.slopes != nullptr;
  return s;
}
template <bool FINE, int C, typename Far>
__device__ __forceinline__ void modify(float (&x)[C], const Scoring& s, bool biased, float slope2, Far far) {
  if (s.inv != 0.0f) {
    float big = 0.0f;
#pragma unroll
    for (int j = 0; j < C; ++j) big = fmaxf(big, fabsf(x[j]));
    if (__all(!(big > s.limit))) {
#pragma unroll
      for (int j = 0; j < C; ++j) {
        const float y = x[j] * x[j];
        float p = fmaf(s.f[3], y, s.f[2]);
        if constexpr (FINE) p = fmaf(fmaf(s.f[4], y, s.f[3]), y, s.f[2]);
        x[j] *= fmaf(fmaf(p, y, s.f[1]), y, s.f[0]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < C; ++j) {
        const float z = x[j] * s.inv, y = z * z;
        const float e = __builtin_amdgcn_exp2f(fabsf(z) * (2.0f * kLog2e));
        const float t = __builtin_copysignf(1.0f - 2.0f * __builtin_amdgcn_rcpf(e + 1.0f), z);
        const float p = fmaf(fmaf(fmaf(fmaf(kTanh4[4], y, kTanh4[3]), y, kTanh4[2]), y, kTanh4[1]), y, kTanh4[0]);
        x[j] = (fabsf(z) > 0.5f ? t : z * p) * s.cap2;
        __builtin_amdgcn_sched_barrier(0);  // (one at a time: the seldom case is to hold few registers)
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < C; ++j) x[j] *= s.scale2;
  }
  if (biased) {
#pragma unroll
    for (int j = 0; j < C; ++j) x[j] = fmaf(-slope2, fabsf(far(j)), x[j]);
  }
}

__device__ __forceinline__ uint32_t nonfinite2(uint32_t x) {  // of two fp16
  return ((x & 0x7C007C00u) + 0x04000400u) & 0x80008000u;
}

__device__ __forceinline__ int wave_max_i(int v) {  // uniform, in a scalar register
  v = max(v, ifrd::dpp_i<ifrd::kQuadXor1>(v));
  v = max(v, ifrd::dpp_i<ifrd::kQuadXor2>(v));
  v = max(v, ifrd::dpp_i<ifrd::kRowRor4>(v));
  v = max(v, ifrd::dpp_i<ifrd::kRowRor8>(v));
  return max(max(__builtin_amdgcn_readlane(v, 0), __builtin_amdgcn_readlane(v, 16)),
             max(__builtin_amdgcn_readlane(v, 32), __builtin_amdgcn_readlane(v, 48)));
}

// ---- V of edge pages ----
// Tokens that no column sees are cleared, and so are values that are not
// finite: a product with a weight of zero must stay zero.  What a column does
// see of the latter is noted per element of O (Unbounded) and put into the
// result.  fp16 is judged value by value, a quantized token by its scale.
template <int FMT>
__device__ __forceinline__ bool not_finite(uint32_t s, uint32_t z) {  // (low halves)
  return (s & 0x7C00u) == 0x7C00u || (FMT == IFR_KV_INT4 && (z & 0x7C00u) == 0x7C00u);
}
// fp16: a run of 8 tokens
__device__ __forceinline__ void edge_run(uint32_t* x, const u4& keep, uint32_t& bad) {
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    x[q] &= keep[q];
    const uint32_t nf = nonfinite2(x[q]);
    bad |= nf;
    x[q] &= ~((nf >> 15) * 0xFFFFu);
  }
}
// int8, int4: the scales (and minima) of 8 tokens
template <int FMT>
__device__ __forceinline__ void edge_scales(uint32_t* s, uint32_t* z, const u4& keep, uint32_t& bad) {
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    s[q] &= keep[q];
    uint32_t nf = nonfinite2(s[q]);
    if constexpr (FMT == IFR_KV_INT4) {
      z[q] &= keep[q];
      nf |= nonfinite2(z[q]);
    }
    bad |= nf;
    const uint32_t in = ~((nf >> 15) * 0xFFFFu);
    s[q] &= in;
    if constexpr (FMT == IFR_KV_INT4) z[q] &= in;
  }
}
// Elements of a lane's O that got +infinity, -infinity (both: NaN).
template <int N>
struct Unbounded {
  uint64_t up[(N + 63) / 64], down[(N + 63) / 64];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < (N + 63) / 64; ++i) up[i] = down[i] = 0;
  }
  // V element (group g, element j, dim d) of the part p, seen by this lane's column, to element k
  template <int HD, int FMT>
  __device__ __forceinline__ void add(const uint8_t* p, int g, int j, int d, int k) {
    bool hi, lo;
    if constexpr (FMT == IFR_KV_FP16) {
      const uint32_t x = reinterpret_cast<const uint16_t*>(p)[paged_vrun(FMT, HD, g, d) * 8 + j];
      const bool nan = (x & 0x7FFFu) > 0x7C00u;
      hi = x == 0x7C00u || nan;
      lo = x == 0xFC00u || nan;
    } else {
      constexpr int kCodes = FMT == IFR_KV_INT8 ? 32 * HD : 16 * HD;
      const uint16_t* sc = reinterpret_cast<const uint16_t*>(p + kCodes) +
                           (FMT == IFR_KV_INT8 ? g * 8 + j : (g * (HD / kPgGroup) + d / kPgGroup) * 16 + j);
      hi = lo = not_finite<FMT>(sc[0], FMT == IFR_KV_INT4 ? sc[8] : 0);
    }
#pragma unroll
    for (int i = 0; i < (N + 63) / 64; ++i) {
      const uint64_t bit = k / 64 == i ? (uint64_t)1 << (k & 63) : 0;
      if (hi) up[i] |= bit;
      if (lo) down[i] |= bit;
    }
  }
  __device__ __forceinline__ bool any() const {
    uint64_t x = 0;
#pragma unroll
    for (int i = 0; i < (N + 63) / 64; ++i) x |= up[i] | down[i];
    return x != 0;
  }
  __device__ __forceinline__ float value(int k, float x) const {
    if ((up[k / 64] >> (k & 63)) & 1) x += INFINITY;
    if ((down[k / 64] >> (k & 63)) & 1) x -= INFINITY;
    return x;
  }
};
// Tokens of lane group g's run (from position t0) that lie in [lo, hi)
__device__ __forceinline__ u4 kept(int t0, int g, int lo, int hi) {
  u4 keep = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int t = t0 + paged_vtok(g, j);
    if (t >= lo && t < hi) keep[j >> 1] |= j & 1 ? 0xFFFF0000u : 0x0000FFFFu;
  }
  return keep;
}
// ---- the splits of a column, in ascending order ------------------------------------------------
// HD / 4 lanes a column, 4 dims each: a wave takes 256 / HD columns (a wave a
// column read 4 bytes a lane: 32000 columns of 64 dims 16.4 us).  A launch of
// its own: a unit that finds itself the last of its tile and joins in place needs
// the device's L2 caches written back and dropped by every unit, which made 64
// rows of 2048 int4 tokens 116 us instead of 43.
template <int HD>
__global__ __launch_bounds__(256) void paged_join_kernel(const PagedJoin* joins, PagedAttnArgs a, PagedPool kv) {
  constexpr int LPC = HD / 4;
  const PagedJoin j = joins[blockIdx.x];
  const int i = threadIdx.x / LPC, d = (threadIdx.x % LPC) * 4;
  if (i >= j.n) return;
  const float2* ml = reinterpret_cast<const float2*>(a.part_ml);
  const int64_t base = (int64_t)j.base + i;
  float m = -INFINITY, l = 0.0f;
  v4f x = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = 0; s0 < j.ns; s0 += 8) {
    float2 q[8];
    v4f p[8];
    float mr = m;
#pragma unroll
    for (int k = 0; k < 8; ++k) {  // (clamped, unconditional: one latency a round)
      const int64_t e = base + (int64_t)min(s0 + k, j.ns - 1) * j.stride;
      q[k] = ml[e];
      p[k] = *reinterpret_cast<const v4f*>(a.part_o + e * HD + d);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) mr = fmaxf(mr, q[k].x);
    const float mu = mr == -INFINITY ? 0.0f : mr;
    const float al = __builtin_amdgcn_exp2f(m - mu);
    l *= al;
    x *= al;
    m = mr;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (s0 + k >= j.ns) continue;  // (a split without a finite score: 0, or a NaN that is to stay)
      const float f = __builtin_amdgcn_exp2f(q[k].x - mu);
      l += f * q[k].y;
      x += p[k] * f;
    }
  }
  const int G = kv.nq / kv.nkv, col = j.col0 + i;
  const PagedRow row = a.rows[j.row0 + col / G];
  x *= l != 0.0f ? 1.0f / l : row.lo < row.hi ? NAN : 0.0f;
  const int64_t at = (int64_t)(j.row0 + col / G) * a.out_stride + (int64_t)(j.kvh * G + col % G) * HD + d;
  if (a.out_f32)
    *reinterpret_cast<v4f*>(static_cast<float*>(a.out) + at) = x;
  else
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + at) =
        make_uint2(ifrd::f2h(x[0]) | ((uint32_t)ifrd::f2h(x[1]) << 16),
                   ifrd::f2h(x[2]) | ((uint32_t)ifrd::f2h(x[3]) << 16));
}

// ---- few columns: the waves of a workgroup take the pages in turn --------------------------------
//
// A wave holds NT tiles of 16 columns.  The next page's K is loaded once the
// first product has read this one's, its V once the second product has.  At
// the end the waves' (m, l, O) meet in LDS.
//
// HL: P enters the second product as an fp16 high + low pair (22 bits), for
// outputs in fp32.  An fp16 output takes P rounded to fp16, which is off like
// the output's own rounding and saves 5 % (64 rows of 2048 int4 tokens, with
// the first plan, 60.2 -> 57.3 us, 16 of 32000 160.6 -> 152.3).  Bound by its VALU work at 4 bits:
// 13 operations turn a dword of codes into 8 values; the 64 rows take 40 to 44 us
// where their bytes would take 32, the 16 rows 117 to 126 of 104.  (Two K buffers and both
// steps unrolled spilled at 192 VGPRs: 142.8 and 467 us.)
template <int HD, int FMT, int NT, int NW, bool HL>
__global__ __launch_bounds__(64 * NW, paged_narrow_waves(FMT, HD, NT)) void paged_narrow_kernel(PagedAttnArgs a, PagedPool kv) {
  constexpr int I = HD / 32, N = HD / 16, U = HD / kPgGroup;
  constexpr int W = FMT == IFR_KV_FP16 ? 4 : FMT == IFR_KV_INT8 ? 2 : 1;  // dwords of 8 elements
  constexpr size_t kPart = paged_part(FMT, HD);
  constexpr int kCodes = FMT == IFR_KV_INT8 ? 32 * HD : 16 * HD;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  const PagedUnit un = a.units[blockIdx.x];
  const int G = kv.nq / kv.nkv;
  const Scoring sco = scoring<HL>(a);
  const float sl = sco.mod ? 1.0f : sco.scale2;  // what turns a score into powers of two

  v8h qf[NT][I];
  int lo[NT], hi[NT], pos[NT], lo_max = 0, hi_min = 0x7FFFFFFF, lo_min = 0x7FFFFFFF, hi_max = 0;
  float slope[NT];
  bool on[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int i = 16 * t + c;
    on[t] = i < un.ncol;
    const int col = un.col0 + (on[t] ? i : 0), row = un.row0 + col / G, h = un.kvh * G + col % G;
    const PagedRow r = a.rows[row];
    // a split's unit sees its own pages only
    lo[t] = max(r.lo, un.p0 * kPgTok);
    hi[t] = on[t] ? min(r.hi, un.p1 * kPgTok) : 0;
    pos[t] = r.pos;
    slope[t] = a.slopes ? a.slopes[h] * kLog2e : 0.0f;
    if (on[t]) {
      lo_max = max(lo_max, lo[t]);
      hi_min = min(hi_min, hi[t]);
      lo_min = min(lo_min, lo[t]);
      hi_max = max(hi_max, hi[t]);
    }
    const uint16_t* qp = a.q + (int64_t)row * a.q_stride + (int64_t)h * HD + 8 * g;
#pragma unroll
    for (int k = 0; k < I; ++k) {
      const v8h x = *reinterpret_cast<const v8h*>(qp + 32 * k);
      qf[t][k] = on[t] ? x : (v8h){0, 0, 0, 0, 0, 0, 0, 0};
    }
  }
  lo_max = wave_max_i(lo_max);
  hi_max = wave_max_i(hi_max);
  hi_min = -wave_max_i(-hi_min);
  lo_min = -wave_max_i(-lo_min);

  float m_run[NT], l_run[NT];
  v4f o[NT][N];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    m_run[t] = -INFINITY;
    l_run[t] = 0.0f;
#pragma unroll
    for (int n = 0; n < N; ++n) o[t][n] = (v4f){0.f, 0.f, 0.f, 0.f};
  }
  Unbounded<4 * N> ub[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) ub[t].clear();

  struct {  // a lane's part of a page
    uint32_t k[2][I * W];
    uint32_t sz[FMT == IFR_KV_INT4 ? 2 * U : 1];  // int4 [u][h]: scale | minimum; int8: both tiles' scales
    uint32_t v[N * W];
    uint32_t s[FMT == IFR_KV_INT4 ? U * 8 : 4];   // int4 [u]: 8 scales, 8 minima; int8: 8 scales
  } rb;
  const int32_t* tab = a.table + un.tab;
  const size_t page_bytes = paged_page(FMT, HD, kv.nkv), head = (size_t)un.kvh * 2 * kPart;
  // every load is unconditional (the page clamped to the unit's last one)
  auto block_of = [&](int i) -> const uint8_t* { return kv.pool + (size_t)tab[min(i, un.p1 - 1)] * page_bytes + head; };
  auto load_k = [&](const uint8_t* p) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if constexpr (FMT == IFR_KV_FP16) {
#pragma unroll
        for (int k = 0; k < I; ++k) load_dwords<4>(p + ((4 * k + g) * 32 + 16 * h + c) * 16, &rb.k[h][4 * k]);
      } else {
        load_dwords<I * W>(p + ((16 * h + c) * 4 + g) * (I * W * 4), rb.k[h]);
      }
    }
    if constexpr (FMT == IFR_KV_INT8) load_dwords<1>(p + kCodes + c * 4, rb.sz);
    if constexpr (FMT == IFR_KV_INT4) load_dwords<2 * U>(p + kCodes + c * (8 * U), rb.sz);
  };
  auto load_v = [&](const uint8_t* p) {
    p += kPart;
    if constexpr (FMT == IFR_KV_FP16) {
#pragma unroll
      for (int n = 0; n < N; ++n) load_dwords<4>(p + (g * HD + 16 * n + c) * 16, &rb.v[4 * n]);
    } else {
      load_dwords<N * W>(p + (g * 16 + c) * (N * W * 4), rb.v);
      load_dwords<(FMT == IFR_KV_INT4 ? U * 8 : 4)>(p + kCodes + g * (FMT == IFR_KV_INT4 ? U * 32 : 16), rb.s);
    }
  };

  const int i0 = un.p0 + w;
  if (i0 < un.p1) {
    load_k(block_of(i0));
    load_v(block_of(i0));
  }
#pragma unroll 1
  for (int i = i0; i < un.p1; i += NW) {
    const uint8_t* const nxt = block_of(i + NW);
    const int t0 = i * kPgTok;
    v4f s[NT][2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (h) __builtin_amdgcn_sched_barrier(0);  // (the scheduler would keep every value of the page in registers)
#pragma unroll
      for (int k = 0; k < I; ++k) {
        uint32_t sz = 0;
        if constexpr (FMT == IFR_KV_INT8) sz = h ? rb.sz[0] >> 16 : rb.sz[0];
        if constexpr (FMT == IFR_KV_INT4) sz = rb.sz[(k / 2) * 2 + h];
        const v8h kf = k_values<FMT>(&rb.k[h][k * W], sz);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          if (k == 0) s[t][h] = (v4f){0.f, 0.f, 0.f, 0.f};
          s[t][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[t][k], s[t][h], 0, 0, 0);
        }
      }
    }
    load_k(nxt);
    const bool inner = t0 >= lo_max && t0 + kPgTok <= hi_min;  // every column sees the whole page
    v8h phi[NT], plo[NT];
    uint32_t seen[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float x[8], mt = -INFINITY;
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = s[t][j >> 2][j & 3];
      if (sco.mod) {
        const float d = (float)(pos[t] - t0 - 4 * g);
        modify<HL>(x, sco, a.slopes != nullptr, slope[t], [&](int j) { return d - (float)(16 * (j >> 2) + (j & 3)); });
      }
      seen[t] = 0xFFu;
      if (!inner) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int tk = t0 + 16 * (j >> 2) + 4 * g + (j & 3);
          if (tk < lo[t] || tk >= hi[t]) {
            x[j] = -INFINITY;
            seen[t] &= ~(1u << j);
          }
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) mt = fmaxf(mt, x[j]);
      mt = fmaxf(mt, ifrd::lane_xor<16>(mt));
      mt = fmaxf(mt, ifrd::lane_xor<32>(mt)) * sl;
      // The reference point of a column's powers moves only when some column's
      // maximum has passed its own by 2^8: P stays below 2^8 and O is rescaled
      // in few pages.
      if (!__all(!(mt > m_run[t] + 8.0f))) {
        const float m_new = fmaxf(m_run[t], mt);
        const float al = m_run[t] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m_run[t] - m_new);
        m_run[t] = m_new;
        l_run[t] *= al;
#pragma unroll
        for (int n = 0; n < N; ++n) o[t][n] *= al;
      }
      const float mu = m_run[t] == -INFINITY ? 0.0f : m_run[t];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float p = __builtin_amdgcn_exp2f(fmaf(x[j], sl, -mu));
        l_run[t] += p;  // this lane's tokens; the groups meet at the end
        const _Float16 hh = (_Float16)p;
        phi[t][j] = hh;
        if constexpr (HL) plo[t][j] = (_Float16)(p - (float)hh);
      }
    }
    uint32_t bad = 0;
    constexpr int S = FMT == IFR_KV_INT4 ? 8 : 0;
    if (!inner) {
      const u4 keep = kept(t0, g, lo_min, hi_max);
      if constexpr (FMT == IFR_KV_FP16) {
#pragma unroll
        for (int n = 0; n < N; ++n) edge_run(&rb.v[4 * n], keep, bad);
      } else {
#pragma unroll
        for (int u = 0; u < (S ? U : 1); ++u) edge_scales<FMT>(&rb.s[u * S], &rb.s[u * S + S / 2], keep, bad);
      }
    }
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int u = n / 4;
      const v8h vf = v_values<FMT>(&rb.v[n * W], &rb.s[u * S], &rb.s[u * S + S / 2]);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        o[t][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, phi[t], o[t][n], 0, 0, 0);
        if constexpr (HL) o[t][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, plo[t], o[t][n], 0, 0, 0);
      }
    }
    load_v(nxt);
    if (!__all(bad == 0)) {  // rare: a cached infinity or NaN where some column looks
#pragma unroll 1
      for (int e = 0; e < 32; ++e) {  // group e / 8, element e % 8
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const int sb = __shfl((int)(seen[t] >> (e & 7)) & 1, (e >> 3) * 16 + c, 64);
          if (!sb) continue;
#pragma unroll 1
          for (int k = 0; k < 4 * N; ++k)
            ub[t].template add<HD, FMT>(block_of(i) + kPart, e >> 3, e & 7, 16 * (k >> 2) + 4 * g + (k & 3), k);
        }
      }
    }
  }
#pragma unroll
  for (int t = 0; t < NT; ++t)
    if (!__all(!ub[t].any()))
#pragma unroll
      for (int k = 0; k < 4 * N; ++k) o[t][k >> 2][k & 3] = ub[t].value(k, o[t][k >> 2][k & 3]);

  // ---- the waves' parts: the columns' common maximum first, then O in
  // slices of 64 dims
  constexpr int kRow = 68;  // floats of a column in a slice (16 lanes' stores on 64 banks)
  __shared__ __align__(16) float slab[NW][16 * NT * kRow];
  __shared__ float ml[NW][16 * NT][2];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    l_run[t] += ifrd::lane_xor<16>(l_run[t]);
    l_run[t] += ifrd::lane_xor<32>(l_run[t]);
    if (g == 0) {
      ml[w][16 * t + c][0] = m_run[t];
      ml[w][16 * t + c][1] = l_run[t];
    }
  }
  __syncthreads();
  float f[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    float m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int q = 0; q < NW; ++q) m = fmaxf(m, ml[q][16 * t + c][0]);
    const float mu = m == -INFINITY ? 0.0f : m;
#pragma unroll
    for (int q = 0; q < NW; ++q) l += __builtin_amdgcn_exp2f(ml[q][16 * t + c][0] - mu) * ml[q][16 * t + c][1];
    f[t] = __builtin_amdgcn_exp2f(m_run[t] - mu);
    if (un.part < 0) {
      // a row that sees nothing: zeros; only scores of -infinity: not a number
      f[t] = l != 0.0f ? f[t] / l : lo[t] < hi[t] ? NAN : 0.0f;
    } else if (w == 0 && g == 0 && on[t]) {
      float* p = a.part_ml + ((int64_t)un.part + 16 * t + c) * 2;
      p[0] = m;
      p[1] = l;
    }
  }
  const int tid = threadIdx.x;
#pragma unroll
  for (int q = 0; q < N / 4; ++q) {
    if (q) __syncthreads();
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int n = 0; n < 4; ++n)
        *reinterpret_cast<v4f*>(&slab[w][(16 * t + c) * kRow + 16 * n + 4 * g]) = o[t][4 * q + n] * f[t];
    __syncthreads();
    // 16 lanes a column, 4 dims each; NW x 4 columns at once
#pragma unroll
    for (int t = 0; t < (4 * NT + NW - 1) / NW; ++t) {
      const int i = 4 * NW * t + tid / 16, d = (tid % 16) * 4;
      if (i >= un.ncol) continue;
      v4f x = *reinterpret_cast<const v4f*>(&slab[0][i * kRow + d]);
#pragma unroll
      for (int k = 1; k < NW; ++k) x += *reinterpret_cast<const v4f*>(&slab[k][i * kRow + d]);
      if (un.part >= 0) {
        *reinterpret_cast<v4f*>(a.part_o + ((int64_t)un.part + i) * HD + 64 * q + d) = x;
      } else {
        const int col = un.col0 + i;
        const int64_t at = (int64_t)(un.row0 + col / G) * a.out_stride + (int64_t)(un.kvh * G + col % G) * HD + 64 * q + d;
        if (a.out_f32) {
          *reinterpret_cast<v4f*>(static_cast<float*>(a.out) + at) = x;
        } else {
          *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + at) =
              make_uint2(ifrd::f2h(x[0]) | ((uint32_t)ifrd::f2h(x[1]) << 16),
                         ifrd::f2h(x[2]) | ((uint32_t)ifrd::f2h(x[3]) << 16));
        }
      }
    }
  }
}

// ---- many columns: the four waves of a workgroup take 32 columns each and share the pages ------
//
// The workgroup turns NP pages a step into fp16 in LDS, two buffers in turn:
// the next step's codes are in flight while this one is computed, one barrier
// a step.  32x32x16 MFMAs: K row rho of a page is token wide_tok(rho), so that
// the scores a lane gets are the P elements that it holds of V's runs.  The
// 16-byte runs of a dim block (K) or of 16 dims (V) are rotated against each
// other by an exclusive or, which spreads both the quantized formats' stores
// and the reads over the banks.
//
// Bound by its matrix products and the softmax's VALU work between them: 8000
// causal fp16 rows of 16/8 heads of 128 take 311 us (840 TFLOP/s), over 4-bit
// pages 342; two-tile units 349 and 468.  With a cap and four documents 167.
// Heads of 256 leave LDS for one such workgroup a CU, and two-tile units win:
// 4000 causal fp16 rows of 8/2 heads 244 us here, 114 there, 4-bit 289 and 166.
__device__ __forceinline__ int wide_tok(int rho) {
  return 8 * (rho >> 4) + 4 * ((rho >> 2) & 1) + 16 * ((rho >> 3) & 1) + (rho & 3);
}
__device__ __forceinline__ int wide_row(int t) {
  return 16 * ((t >> 3) & 1) + 8 * (t >> 4) + 4 * ((t >> 2) & 1) + (t & 3);
}
__device__ __forceinline__ int k_run(int blk, int rho) { return blk * 32 + (rho ^ (blk & 15)); }
template <int HD>
__device__ __forceinline__ int v_run(int g, int d) { return g * HD + (d ^ ((d >> 4) & 15)); }

template <int HD, int FMT, bool HL>
__global__ __launch_bounds__(256, kPgWideGroups) void paged_wide_kernel(PagedAttnArgs a, PagedPool kv) {
  constexpr int NP = 2;
  static_assert(HD <= kPgWideDim, "LDS for two workgroups a CU");
  constexpr int I = HD / 32, N = HD / 16, U = HD / kPgGroup, KS = HD / 16, D = HD / 32;
  constexpr int RUNS = 4 * HD;  // 16-byte runs of a page's K (or V) in LDS
  constexpr size_t kPart = paged_part(FMT, HD);
  constexpr int kCodes = FMT == IFR_KV_INT8 ? 32 * HD : 16 * HD;
  __shared__ __align__(16) u4 lds[2][2][NP * RUNS];  // [buffer][K, V]
  __shared__ int aside[2];                           // step + 1 of the last one in this buffer that set V aside
  __shared__ int range[4][4];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 31, hl = lane >> 5;
  const PagedUnit un = a.units[blockIdx.x];
  const int G = kv.nq / kv.nkv;
  const Scoring sco = scoring<HL>(a);
  const float sl = sco.mod ? 1.0f : sco.scale2;

  // this lane's column
  const int ci = 32 * w + c;
  const bool on = ci < un.ncol;
  const int col = un.col0 + (on ? ci : 0), row = un.row0 + col / G, h = un.kvh * G + col % G;
  const PagedRow pr = a.rows[row];
  const int lo = max(pr.lo, un.p0 * kPgTok), hi = on ? min(pr.hi, un.p1 * kPgTok) : 0, pos = pr.pos;
  const float slope = a.slopes ? a.slopes[h] * kLog2e : 0.0f;
  const int lo_max = wave_max_i(on ? lo : 0), hi_max = wave_max_i(on ? hi : 0);
  const int hi_min = -wave_max_i(on ? -hi : -0x7FFFFFFF), lo_min = -wave_max_i(on ? -lo : -0x7FFFFFFF);
  // ... and of the workgroup's columns
  if (tid < 2) aside[tid] = 0;
  if (lane == 0) {
    range[w][0] = lo_min;
    range[w][1] = -lo_max;
    range[w][2] = -hi_max;
    range[w][3] = hi_min;
  }
  __syncthreads();
  auto least = [&](int i) {
    return __builtin_amdgcn_readfirstlane(min(min(range[0][i], range[1][i]), min(range[2][i], range[3][i])));
  };
  const int wg_lo = least(0), wg_lo_max = -least(1), wg_hi = -least(2), wg_hi_min = least(3);
  v8h qf[KS];
  {
    const uint16_t* qp = a.q + (int64_t)row * a.q_stride + (int64_t)h * HD + 8 * hl;
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      const v8h x = *reinterpret_cast<const v8h*>(qp + 16 * k);
      qf[k] = on ? x : (v8h){0, 0, 0, 0, 0, 0, 0, 0};
    }
  }
  float m_run = -INFINITY, l_run = 0.0f;
  v16f o[D];
#pragma unroll
  for (int d = 0; d < D; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[d][r] = 0.0f;
  Unbounded<16 * D> ub;
  ub.clear();

  // ---- staging: what a thread holds of a step
  constexpr int FR = FMT == IFR_KV_FP16 ? NP * RUNS / 256 : 1;
  constexpr int KD = FMT == IFR_KV_INT8 ? 2 * I : I;              // dwords of a K item (token, group)
  constexpr int VD = FMT == IFR_KV_INT8 ? 8 : 4;                  // dwords of a V item (group, c, 64 dims)
  constexpr int K_ITEMS = NP * 128, V_ITEMS = NP * 64 * U;        // at most 256 each
  struct {
    u4 kf[FR], vf[FR];                                            // fp16
    uint32_t k[KD], ks[FMT == IFR_KV_INT4 ? U : 1], v[VD], vs[8]; // int8, int4
  } sg;
  const int32_t* tab = a.table + un.tab;
  const size_t page_bytes = paged_page(FMT, HD, kv.nkv), head = (size_t)un.kvh * 2 * kPart;
  auto block_of = [&](int st, int ps) -> const uint8_t* {
    return kv.pool + (size_t)tab[min(un.p0 + NP * st + ps, un.p1 - 1)] * page_bytes + head;
  };
  auto load_stage = [&](int st) {
    if constexpr (FMT == IFR_KV_FP16) {
#pragma unroll
      for (int r = 0; r < FR; ++r) {
        const int e = tid + 256 * r, ps = 256 * r / RUNS, i = e % RUNS;
        const uint8_t* p = block_of(st, ps);
        sg.kf[r] = reinterpret_cast<const u4*>(p)[(i & ~31) + wide_tok(i & 31)];
        sg.vf[r] = reinterpret_cast<const u4*>(p + kPart)[i];
      }
    } else {
      if (w * 64 < K_ITEMS) {
        const uint8_t* p = block_of(st, w * 64 / 128);
        const int i = tid % 128, t = i >> 2;
        load_dwords<KD>(p + i * (KD * 4), sg.k);
        const uint8_t* sc = p + kCodes;
        if constexpr (FMT == IFR_KV_INT8) {
          sg.ks[0] = reinterpret_cast<const uint16_t*>(sc)[(t & 15) * 2 + (t >> 4)];
        } else {
#pragma unroll
          for (int u = 0; u < U; ++u) sg.ks[u] = reinterpret_cast<const uint32_t*>(sc)[((t & 15) * U + u) * 2 + (t >> 4)];
        }
      }
      if (w * 64 < V_ITEMS) {
        const uint8_t* p = block_of(st, w * 64 / (64 * U)) + kPart;
        const int i = tid % (64 * U), u = i % U, gc = i / U;  // (group, c), 64 dims u
        load_dwords<VD>(p + ((size_t)gc * N + 4 * u) * (VD), sg.v);
        if constexpr (FMT == IFR_KV_INT8) load_dwords<4>(p + kCodes + (gc >> 4) * 16, sg.vs);
        else load_dwords<8>(p + kCodes + ((gc >> 4) * U + u) * 32, sg.vs);
      }
    }
  };
  auto store_stage = [&](int b, int st) {
    const int t0 = (un.p0 + NP * st) * kPgTok;
    if (t0 < wg_lo_max || t0 + NP * kPgTok > wg_hi_min) {  // an edge step of some column
      uint32_t bad = 0;
      if constexpr (FMT == IFR_KV_FP16) {
#pragma unroll
        for (int r = 0; r < FR; ++r) {
          const int e = tid + 256 * r;
          uint32_t* x = reinterpret_cast<uint32_t*>(&sg.vf[r]);
          edge_run(x, kept(t0 + 32 * (256 * r / RUNS), e % RUNS / HD, wg_lo, wg_hi), bad);
        }
      } else if (w * 64 < V_ITEMS) {
        edge_scales<FMT>(sg.vs, sg.vs + 4, kept(t0 + 32 * (tid / (64 * U)), tid % (64 * U) / U >> 4, wg_lo, wg_hi), bad);
      }
      if (bad) aside[b] = st + 1;
    }
    if constexpr (FMT == IFR_KV_FP16) {
#pragma unroll
      for (int r = 0; r < FR; ++r) {
        const int e = tid + 256 * r, ps = 256 * r / RUNS, i = e % RUNS;
        lds[b][0][ps * RUNS + k_run(i >> 5, i & 31)] = sg.kf[r];
        lds[b][1][ps * RUNS + v_run<HD>(i / HD, i % HD)] = sg.vf[r];
      }
    } else {
      if (w * 64 < K_ITEMS) {
        const int i = tid % 128, ps = tid / 128, rho = wide_row(i >> 2), g = i & 3;
#pragma unroll
        for (int k = 0; k < I; ++k)
          lds[b][0][ps * RUNS + k_run(4 * k + g, rho)] = __builtin_bit_cast(
              u4, k_values<FMT>(&sg.k[k * KD / I], sg.ks[FMT == IFR_KV_INT4 ? k / 2 : 0]));
      }
      if (w * 64 < V_ITEMS) {
        const int i = tid % (64 * U), ps = tid / (64 * U), u = i % U, gc = i / U;
#pragma unroll
        for (int n = 0; n < 4; ++n)
          lds[b][1][ps * RUNS + v_run<HD>(gc >> 4, 16 * (4 * u + n) + (gc & 15))] =
              __builtin_bit_cast(u4, v_values<FMT>(&sg.v[n * VD / 4], sg.vs, sg.vs + 4));
      }
    }
  };

  // page q of the step in buffer b
  auto page = [&](int b, int st, int q) {
    const int t0 = (un.p0 + NP * st + q) * kPgTok;
    if (t0 >= hi_max || t0 + kPgTok <= lo_min) return;  // (the whole wave)
    const u4* lk = &lds[b][0][q * RUNS];
    const u4* lv = &lds[b][1][q * RUNS];
    v16f s;
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = 0.0f;
#pragma unroll
    for (int k = 0; k < KS; ++k)
      s = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, lk[k_run(2 * k + hl, c)]), qf[k], s, 0, 0, 0);
    const bool inner = t0 >= lo_max && t0 + kPgTok <= hi_min;
    float x[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) x[r] = s[r];
    if (sco.mod) {
      const float d = (float)(pos - t0 - 4 * hl);
      modify<HL>(x, sco, a.slopes != nullptr, slope, [&](int r) { return d - (float)wide_tok(8 * (r >> 2) + (r & 3)); });
    }
    uint32_t seen = 0xFFFFu;
    if (!inner) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int tk = t0 + wide_tok(8 * (r >> 2) + 4 * hl + (r & 3));
        if (tk < lo || tk >= hi) {
          x[r] = -INFINITY;
          seen &= ~(1u << r);
        }
      }
    }
    float mt = -INFINITY;
#pragma unroll
    for (int r = 0; r < 16; ++r) mt = fmaxf(mt, x[r]);
    mt = fmaxf(mt, ifrd::lane_xor<32>(mt)) * sl;
    if (!__all(!(mt > m_run + 8.0f))) {  // (as in the narrow kernel)
      const float m_new = fmaxf(m_run, mt);
      const float al = m_run == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m_run - m_new);
      m_run = m_new;
      l_run *= al;
#pragma unroll
      for (int d = 0; d < D; ++d) o[d] *= al;
    }
    const float mu = m_run == -INFINITY ? 0.0f : m_run;
    v8h phi[2], plo[2];
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const float p = __builtin_amdgcn_exp2f(fmaf(x[r], sl, -mu));
      l_run += p;
      const _Float16 hh = (_Float16)p;
      phi[r >> 3][r & 7] = hh;
      if constexpr (HL) plo[r >> 3][r & 7] = (_Float16)(p - (float)hh);
    }
#pragma unroll
    for (int z = 0; z < 2; ++z)
#pragma unroll
      for (int d = 0; d < D; ++d) {
        const v8h vf = __builtin_bit_cast(v8h, lv[v_run<HD>(2 * z + hl, 32 * d + c)]);
        o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, phi[z], o[d], 0, 0, 0);
        if constexpr (HL) o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, plo[z], o[d], 0, 0, 0);
      }
    if (__builtin_amdgcn_readfirstlane(aside[b]) == st + 1) {  // rare (as in the narrow kernel)
      const uint8_t* vp = block_of(st, q) + kPart;
#pragma unroll 1
      for (int e = 0; e < 32; ++e) {
        const int sb = __shfl((int)(seen >> (8 * (e >> 4) + (e & 7))) & 1, 32 * ((e >> 3) & 1) + c, 64);
        if (!sb) continue;
#pragma unroll 1
        for (int k = 0; k < 16 * D; ++k)
          ub.template add<HD, FMT>(vp, e >> 3, e & 7, 32 * (k >> 4) + 8 * ((k >> 2) & 3) + 4 * hl + (k & 3), k);
      }
    }
  };

  const int nst = (un.p1 - un.p0 + NP - 1) / NP;
  if (nst > 0) {
    load_stage(0);
    store_stage(0, 0);
  }
  __syncthreads();
#pragma unroll 1
  for (int st = 0; st < nst; ++st) {
    const bool more = st + 1 < nst;
    if (more) load_stage(st + 1);
#pragma unroll 1
    for (int q = 0; q < NP; ++q) page(st & 1, st, q);
    if (more) store_stage((st + 1) & 1, st + 1);  // last read before the barrier of step st - 1
    __syncthreads();
  }
  if (!__all(!ub.any()))
#pragma unroll
    for (int k = 0; k < 16 * D; ++k) o[k >> 4][k & 15] = ub.value(k, o[k >> 4][k & 15]);
  const float l = l_run + ifrd::lane_xor<32>(l_run);
  if (!on) return;
  float f = 1.0f;
  if (un.part < 0) {
    f = l != 0.0f ? 1.0f / l : lo < hi ? NAN : 0.0f;
  } else if (hl == 0) {
    float* p = a.part_ml + ((int64_t)un.part + ci) * 2;
    p[0] = m_run;
    p[1] = l;
  }
  const int64_t at = (int64_t)row * a.out_stride + (int64_t)h * HD;
#pragma unroll
  for (int d = 0; d < D; ++d)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int e = 32 * d + 8 * q + 4 * hl;
      const v4f x = (v4f){o[d][4 * q], o[d][4 * q + 1], o[d][4 * q + 2], o[d][4 * q + 3]} * f;
      if (un.part >= 0)
        *reinterpret_cast<v4f*>(a.part_o + ((int64_t)un.part + ci) * HD + e) = x;
      else if (a.out_f32)
        *reinterpret_cast<v4f*>(static_cast<float*>(a.out) + at + e) = x;
      else
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + at + e) =
            make_uint2(ifrd::f2h(x[0]) | ((uint32_t)ifrd::f2h(x[1]) << 16),
                       ifrd::f2h(x[2]) | ((uint32_t)ifrd::f2h(x[3]) << 16));
    }
}

template <int HD, int FMT, int NT, int NW>
hipError_t narrow_shape(const PagedAttnArgs& a, const PagedPool& kv, hipStream_t st) {
  const dim3 grid(a.n_units), block(64 * NW);
  if (a.out_f32) hipLaunchKernelGGL((paged_narrow_kernel<HD, FMT, NT, NW, true>), grid, block, 0, st, a, kv);
  else hipLaunchKernelGGL((paged_narrow_kernel<HD, FMT, NT, NW, false>), grid, block, 0, st, a, kv);
  return hipGetLastError();
}

template <int HD, int FMT>
hipError_t narrow_fmt(const PagedAttnArgs& a, const PagedPool& kv, int tiles, int waves, hipStream_t st) {
  if (tiles == 1 && waves == 4) return narrow_shape<HD, FMT, 1, 4>(a, kv, st);
  if (tiles == 2 && waves == 4) return narrow_shape<HD, FMT, 2, 4>(a, kv, st);
  if constexpr (HD == 128)
    if (tiles == 2 && waves == 8) return narrow_shape<HD, FMT, 2, 8>(a, kv, st);
  return hipErrorInvalidValue;
}

template <int HD, int FMT>
hipError_t wide_fmt(const PagedAttnArgs& a, const PagedPool& kv, hipStream_t st) {
  if constexpr (HD > kPgWideDim) {
    return hipErrorInvalidValue;
  } else {
    const dim3 grid(a.n_units), block(256);
    if (a.out_f32) hipLaunchKernelGGL((paged_wide_kernel<HD, FMT, true>), grid, block, 0, st, a, kv);
    else hipLaunchKernelGGL((paged_wide_kernel<HD, FMT, false>), grid, block, 0, st, a, kv);
    return hipGetLastError();
  }
}

}  // namespace

#define IFR_PAGED_DIMS(F, FMT, ...)                     \
  do {                                                  \
    if (kv.hd == 64) return F<64, FMT>(__VA_ARGS__);    \
    if (kv.hd == 128) return F<128, FMT>(__VA_ARGS__);  \
    if (kv.hd == 256) return F<256, FMT>(__VA_ARGS__);  \
    return hipErrorInvalidValue;                        \
  } while (0)

#if defined(IFR_PAGED_FMT)
// compiled once per format: that format's kernels
template <int FMT>
hipError_t paged_narrow_of(const PagedAttnArgs& a, const PagedPool& kv, int tiles, int waves, hipStream_t st) {
  IFR_PAGED_DIMS(narrow_fmt, FMT, a, kv, tiles, waves, st);
}
template <int FMT>
hipError_t paged_wide_of(const PagedAttnArgs& a, const PagedPool& kv, hipStream_t st) {
  IFR_PAGED_DIMS(wide_fmt, FMT, a, kv, st);
}
template hipError_t paged_narrow_of<IFR_PAGED_FMT>(const PagedAttnArgs&, const PagedPool&, int, int, hipStream_t);
template hipError_t paged_wide_of<IFR_PAGED_FMT>(const PagedAttnArgs&, const PagedPool&, hipStream_t);
#else
// and once without: the joins and the dispatch
template <int FMT>
hipError_t paged_narrow_of(const PagedAttnArgs& a, const PagedPool& kv, int tiles, int waves, hipStream_t st);
template <int FMT>
hipError_t paged_wide_of(const PagedAttnArgs& a, const PagedPool& kv, hipStream_t st);
#define IFR_PAGED_EXTERN(FMT)                                                                              \
  extern template hipError_t paged_narrow_of<FMT>(const PagedAttnArgs&, const PagedPool&, int, int, hipStream_t); \
  extern template hipError_t paged_wide_of<FMT>(const PagedAttnArgs&, const PagedPool&, hipStream_t)
IFR_PAGED_EXTERN(IFR_KV_FP16);
IFR_PAGED_EXTERN(IFR_KV_INT8);
IFR_PAGED_EXTERN(IFR_KV_INT4);

hipError_t launch_paged_narrow(const PagedAttnArgs& a, const PagedPool& kv, int tiles, int waves, hipStream_t st) {
  if (a.n_units <= 0) return hipSuccess;
  if (kv.fmt == IFR_KV_FP16) return paged_narrow_of<IFR_KV_FP16>(a, kv, tiles, waves, st);
  if (kv.fmt == IFR_KV_INT8) return paged_narrow_of<IFR_KV_INT8>(a, kv, tiles, waves, st);
  if (kv.fmt == IFR_KV_INT4) return paged_narrow_of<IFR_KV_INT4>(a, kv, tiles, waves, st);
  return hipErrorInvalidValue;
}

hipError_t launch_paged_wide(const PagedAttnArgs& a, const PagedPool& kv, hipStream_t st) {
  if (a.n_units <= 0) return hipSuccess;
  if (kv.fmt == IFR_KV_FP16) return paged_wide_of<IFR_KV_FP16>(a, kv, st);
  if (kv.fmt == IFR_KV_INT8) return paged_wide_of<IFR_KV_INT8>(a, kv, st);
  if (kv.fmt == IFR_KV_INT4) return paged_wide_of<IFR_KV_INT4>(a, kv, st);
  return hipErrorInvalidValue;
}

hipError_t launch_paged_join(const PagedJoin* joins, int n, const PagedAttnArgs& a, const PagedPool& kv,
                             hipStream_t st) {
  if (n <= 0) return hipSuccess;
  const dim3 grid(n), block(256);
  if (kv.hd == 64) hipLaunchKernelGGL(paged_join_kernel<64>, grid, block, 0, st, joins, a, kv);
  else if (kv.hd == 128) hipLaunchKernelGGL(paged_join_kernel<128>, grid, block, 0, st, joins, a, kv);
  else if (kv.hd == 256) hipLaunchKernelGGL(paged_join_kernel<256>, grid, block, 0, st, joins, a, kv);
  else return hipErrorInvalidValue;
  return hipGetLastError();
}
#endif

}  // namespace ifrk
