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
// pages that some row sees only in part ("edge" pages) take V with every token
// that no column sees cleared; if a non-finite V is left there, its products
// are added only to the columns that see it.
#include "ifr_dev.h"
#include "ifr_paged.h"

namespace ifrk {
namespace {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));

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

// cap tanh(a / cap) with errors relative to the result, so that small scores
// keep their bits: tanh x = x (135135 + 17325 y + 378 y^2 + y^3) /
// (135135 + 62370 y + 3150 y^2 + 28 y^3), y = x^2, the seventh convergent of
// Lambert's continued fraction (below 2e-8 off for |x| < 1), and
// 1 - 2 / (e^2x + 1) from there on.
__device__ __forceinline__ float capped(float a, float cap, float inv_cap) {
  const float x = a * inv_cap, y = x * x;
  const float n = fmaf(fmaf(fmaf(y, 1.0f, 378.0f), y, 17325.0f), y, 135135.0f);
  const float d = fmaf(fmaf(fmaf(28.0f, y, 3150.0f), y, 62370.0f), y, 135135.0f);
  float r = a * n * __builtin_amdgcn_rcpf(d);
  if (!(y < 1.0f)) {
    const float e = __builtin_amdgcn_exp2f(fabsf(x) * (2.0f * kLog2e));
    r = __builtin_copysignf(cap * (1.0f - 2.0f * __builtin_amdgcn_rcpf(e + 1.0f)), a);
    if (a != a) r = a;
  }
  return r;
}

__device__ __forceinline__ uint32_t nonfinite2(uint32_t x) {  // of two fp16
  return ((x & 0x7C007C00u) + 0x04000400u) & 0x80008000u;
}

// One V element: token paged_vtok(g, j), dim d.
template <int HD, int FMT>
__device__ __forceinline__ float v_at(const uint8_t* p, int g, int j, int d) {
  const int e = paged_vrun(FMT, HD, g, d) * 8 + j;
  if constexpr (FMT == IFR_KV_FP16) {
    return ifrd::h2f(reinterpret_cast<const uint16_t*>(p)[e]);
  } else if constexpr (FMT == IFR_KV_INT8) {
    const _Float16 s = __builtin_bit_cast(_Float16, reinterpret_cast<const uint16_t*>(p + 32 * HD)[g * 8 + j]);
    return (float)((_Float16)(float)(int8_t)p[e] * s);
  } else {
    const uint16_t* sc = reinterpret_cast<const uint16_t*>(p + 16 * HD) + (g * (HD / kPgGroup) + d / kPgGroup) * 16 + j;
    const int n = (e & ~7) + paged_nibble(e & 7);
    return (float)__builtin_elementwise_fma((_Float16)(float)((p[n >> 1] >> (4 * (n & 1))) & 15),
                                            __builtin_bit_cast(_Float16, sc[0]), __builtin_bit_cast(_Float16, sc[8]));
  }
}

__device__ __forceinline__ int wave_max_i(int v) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) v = max(v, __shfl_xor(v, m, 64));
  return v;
}

// ---- few columns: the four waves of a workgroup take every fourth page ------------------------
//
// A wave holds NT tiles of 16 columns.  The next page's K is loaded once the
// first product has read this one's, its V once the second product has.  At
// the end the waves' (m, l, O) meet in LDS.
//
// HL: P enters the second product as an fp16 high + low pair (22 bits), for
// outputs in fp32.  An fp16 output takes P rounded to fp16, which is off like
// the output's own rounding and saves 5 % (64 rows of 2048 int4 tokens 60.2 ->
// 57.3 us, 16 of 32000 160.6 -> 152.3).  Bound by its VALU work at 4 bits:
// 13 operations turn a dword of codes into 8 values.  (Two K buffers and both
// steps unrolled spilled at 192 VGPRs: 142.8 and 467 us.)
template <int HD, int FMT, int NT, bool HL>
__global__ __launch_bounds__(256) void paged_narrow_kernel(PagedAttnArgs a, PagedPool kv) {
  constexpr int I = HD / 32, N = HD / 16, U = HD / kPgGroup;
  constexpr int W = FMT == IFR_KV_FP16 ? 4 : FMT == IFR_KV_INT8 ? 2 : 1;  // dwords of 8 elements
  constexpr size_t kPart = paged_part(FMT, HD);
  constexpr int kCodes = FMT == IFR_KV_INT8 ? 32 * HD : 16 * HD;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  const PagedUnit un = a.units[blockIdx.x];
  const int G = kv.nq / kv.nkv;
  const bool mod = a.cap != 0.0f || a.slopes != nullptr;
  const float inv_cap = a.cap != 0.0f ? 1.0f / a.cap : 0.0f;
  const float sl = mod ? 1.0f : a.scale * kLog2e;  // what turns a score into powers of two

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
    slope[t] = a.slopes ? a.slopes[h] : 0.0f;
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

  struct {
    uint32_t k[2][I * W];
    uint32_t sz[FMT == IFR_KV_INT4 ? 2 * U : 1];  // int4 [u][h]: scale | minimum; int8: both tiles' scales
  } kb;
  struct {
    uint32_t v[N * W];
    uint32_t s[FMT == IFR_KV_INT4 ? U * 8 : 4];   // int4 [u]: 8 scales, 8 minima; int8: 8 scales
  } vb;
  const int32_t* tab = a.table + un.tab;
  const size_t page_bytes = paged_page(FMT, HD, kv.nkv), head = (size_t)un.kvh * 2 * kPart;
  // every load is unconditional (the page clamped to the unit's last one)
  auto block_of = [&](int i) -> const uint8_t* { return kv.pool + (size_t)tab[min(i, un.p1 - 1)] * page_bytes + head; };
  auto load_k = [&](const uint8_t* p) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if constexpr (FMT == IFR_KV_FP16) {
#pragma unroll
        for (int k = 0; k < I; ++k) load_dwords<4>(p + ((4 * k + g) * 32 + 16 * h + c) * 16, &kb.k[h][4 * k]);
      } else {
        load_dwords<I * W>(p + ((16 * h + c) * 4 + g) * (I * W * 4), kb.k[h]);
      }
    }
    if constexpr (FMT == IFR_KV_INT8) load_dwords<1>(p + kCodes + c * 4, kb.sz);
    if constexpr (FMT == IFR_KV_INT4) load_dwords<2 * U>(p + kCodes + c * (8 * U), kb.sz);
  };
  auto load_v = [&](const uint8_t* p) {
    p += kPart;
    if constexpr (FMT == IFR_KV_FP16) {
#pragma unroll
      for (int n = 0; n < N; ++n) load_dwords<4>(p + (g * HD + 16 * n + c) * 16, &vb.v[4 * n]);
    } else {
      load_dwords<N * W>(p + (g * 16 + c) * (N * W * 4), vb.v);
      load_dwords<(FMT == IFR_KV_INT4 ? U * 8 : 4)>(p + kCodes + g * (FMT == IFR_KV_INT4 ? U * 32 : 16), vb.s);
    }
  };

  const int i0 = un.p0 + w;
  const uint8_t *cur = nullptr, *nxt = nullptr;
  if (i0 < un.p1) {
    cur = block_of(i0);
    nxt = block_of(i0 + 4);
    load_k(cur);
    load_v(cur);
  }
#pragma unroll 1
  for (int i = i0; i < un.p1; i += 4) {
    const uint8_t* after = block_of(i + 8);  // its table entry is there when it is wanted
    const int t0 = i * kPgTok;
    v4f s[NT][2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int k = 0; k < I; ++k) {
        uint32_t sz = 0;
        if constexpr (FMT == IFR_KV_INT8) sz = h ? kb.sz[0] >> 16 : kb.sz[0];
        if constexpr (FMT == IFR_KV_INT4) sz = kb.sz[(k / 2) * 2 + h];
        const v8h kf = k_values<FMT>(&kb.k[h][k * W], sz);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          if (k == 0) s[t][h] = (v4f){0.f, 0.f, 0.f, 0.f};
          s[t][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[t][k], s[t][h], 0, 0, 0);
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
      if (mod) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          x[j] *= a.scale;
          if (a.cap != 0.0f) x[j] = capped(x[j], a.cap, inv_cap);
          x[j] -= slope[t] * (float)abs(pos[t] - (t0 + 16 * (j >> 2) + 4 * g + (j & 3)));
          x[j] *= kLog2e;
        }
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
    // an edge page: V of tokens that no column sees and non-finite V are cleared
    u4 keep = {~0u, ~0u, ~0u, ~0u};
    uint32_t bad = 0;
    if (!inner) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int tk = t0 + 16 * (j >> 2) + 4 * g + (j & 3);
        if (tk < lo_min || tk >= hi_max) keep[j >> 1] &= j & 1 ? 0x0000FFFFu : 0xFFFF0000u;
      }
    }
#pragma unroll
    for (int n = 0; n < N; ++n) {
      constexpr int S = FMT == IFR_KV_INT4 ? 8 : 0;
      const int u = n / 4;
      v8h vf = v_values<FMT>(&vb.v[n * W], &vb.s[u * S], &vb.s[u * S + (FMT == IFR_KV_INT4 ? 4 : 0)]);
      if (!inner) {
        u4 x = __builtin_bit_cast(u4, vf) & keep;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const uint32_t nf = nonfinite2(x[q]);
          bad |= nf;
          x[q] &= ~((nf >> 15) * 0xFFFFu);
        }
        vf = __builtin_bit_cast(v8h, x);
      }
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        o[t][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, phi[t], o[t][n], 0, 0, 0);
        if constexpr (HL) o[t][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, plo[t], o[t][n], 0, 0, 0);
      }
    }
    load_v(nxt);
    if (!__all(bad == 0)) {
      // cached infinities or NaN where a column looks: their products, read
      // again one by one, go to the columns that see them
      const uint8_t* vp = cur + kPart;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
#pragma unroll 1
        for (int e = 0; e < 32; ++e) {
          const int src = (e >> 3) * 16 + c, j = e & 7;
          float pj = 0.0f;
#pragma unroll
          for (int q = 0; q < 8; ++q)
            if (q == j) pj = (float)phi[t][q];
          const float p = __shfl(pj, src, 64);
          const int sb = __shfl((int)(seen[t] >> j) & 1, src, 64);
#pragma unroll
          for (int n = 0; n < N; ++n)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const float v = v_at<HD, FMT>(vp, e >> 3, j, 16 * n + 4 * g + r);
              if (sb && (__builtin_bit_cast(uint32_t, v) & 0x7F800000u) == 0x7F800000u) o[t][n][r] += p * v;
            }
        }
      }
    }
    cur = nxt;
    nxt = after;
  }

  // ---- the four waves' parts: the columns' common maximum first, then O in
  // slices of 64 dims
  constexpr int kRow = 68;  // floats of a column in a slice (16 lanes' stores on 64 banks)
  __shared__ __align__(16) float slab[4][16 * NT * kRow];
  __shared__ float ml[4][16 * NT][2];
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
    for (int q = 0; q < 4; ++q) m = fmaxf(m, ml[q][16 * t + c][0]);
    const float mu = m == -INFINITY ? 0.0f : m;
#pragma unroll
    for (int q = 0; q < 4; ++q) l += __builtin_amdgcn_exp2f(ml[q][16 * t + c][0] - mu) * ml[q][16 * t + c][1];
    f[t] = __builtin_amdgcn_exp2f(m_run[t] - mu);
    if (un.part < 0) {
      f[t] = l == 0.0f ? 0.0f : f[t] / l;  // a row that sees nothing: zeros
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
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int i = 16 * t + tid / 16, d = (tid % 16) * 4;
      if (i >= un.ncol) continue;
      v4f x = *reinterpret_cast<const v4f*>(&slab[0][i * kRow + d]);
#pragma unroll
      for (int k = 1; k < 4; ++k) x += *reinterpret_cast<const v4f*>(&slab[k][i * kRow + d]);
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

// ---- the splits of a column, in ascending order ------------------------------------------------
template <int HD>
__global__ __launch_bounds__(256) void paged_join_kernel(const PagedJoin* joins, PagedAttnArgs a, PagedPool kv) {
  constexpr int E = HD / 64;  // dims of a lane
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const PagedJoin j = joins[blockIdx.x];
  if (w >= j.n) return;
  const int G = kv.nq / kv.nkv;
  const float2* ml = reinterpret_cast<const float2*>(a.part_ml);
  const int64_t base = (int64_t)j.base + w;
  float m = -INFINITY;
  for (int s = 0; s < j.ns; ++s) m = fmaxf(m, ml[base + (int64_t)s * j.stride].x);
  const float mu = m == -INFINITY ? 0.0f : m;
  float l = 0.0f, x[E];
#pragma unroll
  for (int e = 0; e < E; ++e) x[e] = 0.0f;
  for (int s0 = 0; s0 < j.ns; s0 += 8) {
    float2 q[8];
    float p[8][E];
#pragma unroll
    for (int k = 0; k < 8; ++k) {  // (clamped, unconditional: one latency a round)
      const int64_t i = base + (int64_t)min(s0 + k, j.ns - 1) * j.stride;
      q[k] = ml[i];
#pragma unroll
      for (int e = 0; e < E; ++e) p[k][e] = a.part_o[i * HD + lane * E + e];
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (s0 + k >= j.ns || q[k].x == -INFINITY) continue;
      const float f = __builtin_amdgcn_exp2f(q[k].x - mu);
      l += f * q[k].y;
#pragma unroll
      for (int e = 0; e < E; ++e) x[e] += f * p[k][e];
    }
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  const int col = j.col0 + w;
  const int64_t at = (int64_t)(j.row0 + col / G) * a.out_stride + (int64_t)(j.kvh * G + col % G) * HD + lane * E;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    if (a.out_f32) static_cast<float*>(a.out)[at + e] = x[e] * inv;
    else static_cast<uint16_t*>(a.out)[at + e] = ifrd::f2h(x[e] * inv);
  }
}

template <int HD, int FMT>
hipError_t narrow_fmt(const PagedAttnArgs& a, const PagedPool& kv, int tiles, hipStream_t st) {
  const dim3 grid(a.n_units), block(256);
  if (tiles == 1 && a.out_f32) hipLaunchKernelGGL((paged_narrow_kernel<HD, FMT, 1, true>), grid, block, 0, st, a, kv);
  else if (tiles == 1) hipLaunchKernelGGL((paged_narrow_kernel<HD, FMT, 1, false>), grid, block, 0, st, a, kv);
  else if (tiles == 2 && a.out_f32) hipLaunchKernelGGL((paged_narrow_kernel<HD, FMT, 2, true>), grid, block, 0, st, a, kv);
  else if (tiles == 2) hipLaunchKernelGGL((paged_narrow_kernel<HD, FMT, 2, false>), grid, block, 0, st, a, kv);
  else return hipErrorInvalidValue;
  return hipGetLastError();
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
hipError_t paged_narrow_of(const PagedAttnArgs& a, const PagedPool& kv, int tiles, hipStream_t st) {
  IFR_PAGED_DIMS(narrow_fmt, FMT, a, kv, tiles, st);
}
template hipError_t paged_narrow_of<IFR_PAGED_FMT>(const PagedAttnArgs&, const PagedPool&, int, hipStream_t);
#else
// and once without: the joins and the dispatch
template <int FMT>
hipError_t paged_narrow_of(const PagedAttnArgs& a, const PagedPool& kv, int tiles, hipStream_t st);
extern template hipError_t paged_narrow_of<IFR_KV_FP16>(const PagedAttnArgs&, const PagedPool&, int, hipStream_t);
extern template hipError_t paged_narrow_of<IFR_KV_INT8>(const PagedAttnArgs&, const PagedPool&, int, hipStream_t);
extern template hipError_t paged_narrow_of<IFR_KV_INT4>(const PagedAttnArgs&, const PagedPool&, int, hipStream_t);

hipError_t launch_paged_narrow(const PagedAttnArgs& a, const PagedPool& kv, int tiles, hipStream_t st) {
  if (a.n_units <= 0) return hipSuccess;
  if (kv.fmt == IFR_KV_FP16) return paged_narrow_of<IFR_KV_FP16>(a, kv, tiles, st);
  if (kv.fmt == IFR_KV_INT8) return paged_narrow_of<IFR_KV_INT8>(a, kv, tiles, st);
  if (kv.fmt == IFR_KV_INT4) return paged_narrow_of<IFR_KV_INT4>(a, kv, tiles, st);
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
