// Rows of K and V into the pages of a caller-owned cache, with the rotation of
// K and Q on the way, and cached rows back as fp16.
//
// Rotation (rotate-half over the first `rotary` dims, fp32 tables):
//   x'_d = x_d cos_d - x_{d+r/2} sin_d,  x'_{d+r/2} = x_{d+r/2} cos_d + x_d sin_d
// with every product and the sum rounded to fp32.  K is stored from that fp32
// value, so the only rounding after it is the format's own:
//   fp16  fp16(x)
//   int8  s = fp16(max|x| / 127) per (token, head), c = half-away(x * (1 / s))
//   int4  z = fp16(min), s = fp16((max - min) / 15) per (token, head, 64 dims),
//         c = rint((x - z) * (1 / s)) in 0 .. 15; it stands for fp16(c s + z)
// A group that holds a NaN or an infinity gets a NaN scale and reads back as
// NaN; the codes of a group whose scale rounds to zero are zero.  A scale whose
// largest code would round to infinity is the next smaller one (int8: 515.5 at
// most), so that no finite row reads back as infinite.
#include "ifr_dev.h"
#include "ifr_paged.h"

namespace ifrk {
namespace {

constexpr float kMaxHalf = 65504.0f;

__device__ __forceinline__ bool finite_f(float x) {
  return (__builtin_bit_cast(uint32_t, x) & 0x7F800000u) != 0x7F800000u;
}

// Reductions over the 8, 16 or 32 consecutive lanes that share a token (all
// lanes of the wave take part).
template <int LPT>
__device__ __forceinline__ float group_max(float v) {
  v = fmaxf(v, ifrd::lane_xor<1>(v));
  v = fmaxf(v, ifrd::lane_xor<2>(v));
  v = fmaxf(v, ifrd::lane_xor<4>(v));
  if constexpr (LPT >= 16) v = fmaxf(v, ifrd::lane_xor<8>(v));
  if constexpr (LPT >= 32) v = fmaxf(v, ifrd::lane_xor<16>(v));
  return v;
}

// Quantize a lane's 8 consecutive dims.  int8: the scale of the whole head row
// (LPT lanes); int4: of its 64 dims (8 lanes).  Codes as bytes.
template <int FMT, int LPT>
__device__ __forceinline__ void quantize8(const float (&x)[8], uint32_t (&code)[2], uint16_t& scale, uint16_t& zero) {
  code[0] = code[1] = 0u;
  float bad = 0.0f;
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (!finite_f(x[e])) bad = 1.0f;
  if constexpr (FMT == IFR_KV_INT8) {
    float a = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) a = fmaxf(a, fabsf(x[e]));
    a = group_max<LPT>(a);
    bad = group_max<LPT>(bad);
    scale = bad != 0.0f ? (uint16_t)0x7E00u : ifrd::f2h(fminf(a / 127.0f, 515.5f));
    const float s = ifrd::h2f(scale);
    const float inv = s > 0.0f && bad == 0.0f ? 1.0f / s : 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float v = bad != 0.0f ? 0.0f : x[e];
      code[e >> 2] |= ((uint32_t)ifrd::quant_half_away(v, inv) & 0xFFu) << (8 * (e & 3));
    }
  } else if constexpr (FMT == IFR_KV_INT4) {
    float hi = -INFINITY, lo = INFINITY;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      hi = fmaxf(hi, x[e]);
      lo = fminf(lo, x[e]);
    }
    hi = group_max<8>(hi);
    lo = -group_max<8>(-lo);
    bad = group_max<8>(bad);
    lo = fminf(fmaxf(lo, -kMaxHalf), kMaxHalf);  // (a rotated value can pass fp16's range)
    hi = fminf(fmaxf(hi, -kMaxHalf), kMaxHalf);
    scale = ifrd::f2h((hi - lo) / 15.0f);
    zero = ifrd::f2h(lo);
    if (15.0f * ifrd::h2f(scale) + ifrd::h2f(zero) >= 65520.0f) scale -= 1;  // code 15 would round to infinity
    if (bad != 0.0f) {
      scale = 0x7E00u;
      zero = 0u;
    }
    const float s = ifrd::h2f(scale), z = ifrd::h2f(zero);
    const float inv = s > 0.0f && bad == 0.0f ? 1.0f / s : 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float v = bad != 0.0f ? 0.0f : (x[e] - z) * inv;
      const int c = (int)fminf(fmaxf(__builtin_rintf(v), 0.0f), 15.0f);
      code[e >> 2] |= (uint32_t)c << (8 * (e & 3));
    }
  }
}

__device__ __forceinline__ void load8(const uint16_t* p, float (&x)[8]) {
  const v8h h = *reinterpret_cast<const v8h*>(p);
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = (float)h[e];
}
__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) w[e] = (uint32_t)ifrd::f2h(x[2 * e]) | ((uint32_t)ifrd::f2h(x[2 * e + 1]) << 16);
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Bytes of codes -> the int4 dword of 8 elements.
__device__ __forceinline__ uint32_t pack_nibbles(const uint32_t (&b)[2]) {
  uint32_t w = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) w |= ((b[e >> 2] >> (8 * (e & 3))) & 15u) << (4 * paged_nibble(e));
  return w;
}

// One wave per (run, kv head): up to 32 tokens of one page.  HD / 8 lanes hold
// a token, 8 dims each.  K goes straight to its place; V, whose 8-element runs
// are 8 tokens of one dim, crosses through LDS.  A run of V that the tokens
// cover whole is stored whole, else element by element (fp16, int8) or as a
// read-modify-write of its dword (int4; a batch writes a page from one run
// only, so nobody else has that dword).  The blocks past the runs rotate Q.
template <int HD, int FMT>
__global__ __launch_bounds__(256) void paged_append_kernel(PagedAppendArgs a, PagedPool kv, int kv_blocks) {
  constexpr int LPT = HD / 8, TPI = 64 / LPT, U = HD / kPgGroup;
  constexpr int ES = FMT == IFR_KV_FP16 ? 2 : 1;   // bytes of an element in LDS
  constexpr int LROW = HD * ES + 16;
  __shared__ __align__(16) uint8_t stage[4][kPgTok * LROW];
  const int half = a.r.rotary / 2;
  if ((int)blockIdx.x >= kv_blocks) {
    // Q: an item is 8 dims and their partners, or 8 dims past the rotation
    const int np = half / 8, ni = np + (HD - a.r.rotary) / 8;
    const int64_t item = ((int64_t)blockIdx.x - kv_blocks) * 256 + threadIdx.x;
    if (item >= (int64_t)a.M * kv.nq * ni) return;
    const int p = (int)(item % ni);
    const int64_t mh = item / ni;
    const int h = (int)(mh % kv.nq), m = (int)(mh / kv.nq);
    const uint16_t* src = a.r.q_d + (int64_t)m * a.r.q_stride + (int64_t)h * HD;
    uint16_t* dst = a.r.q_out_d + (int64_t)m * a.r.q_out_stride + (int64_t)h * HD;
    if (p >= np) {
      const int d = a.r.rotary + 8 * (p - np);
      *reinterpret_cast<uint4*>(dst + d) = *reinterpret_cast<const uint4*>(src + d);
      return;
    }
    const int64_t t = (int64_t)a.rows[m].pos * half + 8 * p;
    float x[8], y[8], u[8], v[8];
    load8(src + 8 * p, x);
    load8(src + half + 8 * p, y);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float c = a.r.cos_d[t + e], s = a.r.sin_d[t + e];
      u[e] = x[e] * c - y[e] * s;
      v[e] = y[e] * c + x[e] * s;
    }
    *reinterpret_cast<uint4*>(dst + 8 * p) = pack8(u);
    *reinterpret_cast<uint4*>(dst + half + 8 * p) = pack8(v);
    return;
  }
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t item = (int64_t)blockIdx.x * 4 + w;
  if (item >= (int64_t)a.n_runs * kv.nkv) return;
  const PagedRun run = a.runs[item / kv.nkv];
  const int kvh = (int)(item % kv.nkv);
  uint8_t* kpart = kv.pool + (size_t)run.page * paged_page(FMT, HD, kv.nkv) + (size_t)kvh * 2 * paged_part(FMT, HD);
  uint8_t* vpart = kpart + paged_part(FMT, HD);
  constexpr size_t codes = FMT == IFR_KV_FP16 ? 0 : FMT == IFR_KV_INT8 ? 32 * HD : 16 * HD;
  uint16_t* kscale = reinterpret_cast<uint16_t*>(kpart + codes);
  uint16_t* vscale = reinterpret_cast<uint16_t*>(vpart + codes);
  uint8_t* st = stage[w];
  const int sub = lane / LPT, d0 = (lane % LPT) * 8, u = d0 / kPgGroup;
  for (int b = 0; b < run.n; b += TPI) {
    const int i = b + sub, t = run.t0 + i;
    const bool on = i < run.n;
    const int64_t m = run.row + (on ? i : 0);
    const uint16_t* kr = a.r.k_d + m * a.r.k_stride + (int64_t)kvh * HD;
    const uint16_t* vr = a.r.v_d + m * a.r.v_stride + (int64_t)kvh * HD;
    float x[8], y[8];
    load8(kr + d0, x);
    load8(vr + d0, y);
    if (d0 < a.r.rotary) {
      const int ds = d0 < half ? d0 : d0 - half;
      float p[8];
      load8(kr + (d0 < half ? d0 + half : ds), p);
      const int64_t tb = (int64_t)a.rows[m].pos * half + ds;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float c = a.r.cos_d[tb + e], s = a.r.sin_d[tb + e];
        const float xc = x[e] * c, ps = p[e] * s;
        x[e] = d0 < half ? xc - ps : xc + ps;
      }
    }
    if constexpr (FMT == IFR_KV_FP16) {
      if (on) {
        *reinterpret_cast<uint4*>(kpart + (size_t)paged_koff(FMT, HD, t, d0) * 2) = pack8(x);
        *reinterpret_cast<uint4*>(st + t * LROW + d0 * 2) = pack8(y);
      }
    } else {
      uint32_t kc[2], vc[2];
      uint16_t ks, kz, vs, vz;
      quantize8<FMT, LPT>(x, kc, ks, kz);
      quantize8<FMT, LPT>(y, vc, vs, vz);
      if (on) {
        *reinterpret_cast<uint2*>(st + t * LROW + d0) = make_uint2(vc[0], vc[1]);
        if constexpr (FMT == IFR_KV_INT8) {
          *reinterpret_cast<uint2*>(kpart + paged_koff(FMT, HD, t, d0)) = make_uint2(kc[0], kc[1]);
          if (d0 == 0) {
            kscale[paged_kscale(FMT, HD, t, 0)] = ks;
            vscale[paged_vscale(FMT, HD, t, 0)] = vs;
          }
        } else {
          *reinterpret_cast<uint32_t*>(kpart + paged_koff(FMT, HD, t, d0) / 2) = pack_nibbles(kc);
          if (d0 % kPgGroup == 0) {
            *reinterpret_cast<uint32_t*>(kscale + paged_kscale(FMT, HD, t, u)) = (uint32_t)ks | ((uint32_t)kz << 16);
            vscale[paged_vscale(FMT, HD, t, u)] = vs;
            vscale[paged_vscale(FMT, HD, t, u) + 8] = vz;
          }
        }
      }
    }
  }
  ifrd::wave_sync();
  const int t1 = run.t0 + run.n;
  // run r of 8 tokens: group g, dim d; only groups that hold a token of ours
  for (int r = lane; r < 4 * HD; r += 64) {
    const int g = r / HD;
    const int d = FMT == IFR_KV_FP16 ? r % HD : (r % (HD / 16)) * 16 + (r % HD) / (HD / 16);
    uint32_t mine = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int t = paged_vtok(g, j);
      if (t >= run.t0 && t < t1) mine |= 1u << j;
    }
    if (!mine) continue;
    if constexpr (FMT == IFR_KV_FP16) {
      uint16_t x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = (mine >> j) & 1 ? *reinterpret_cast<const uint16_t*>(st + paged_vtok(g, j) * LROW + d * 2) : 0;
      uint16_t* dst = reinterpret_cast<uint16_t*>(vpart) + (size_t)r * 8;
      if (mine == 0xFFu) {
        *reinterpret_cast<uint4*>(dst) =
            make_uint4(x[0] | ((uint32_t)x[1] << 16), x[2] | ((uint32_t)x[3] << 16), x[4] | ((uint32_t)x[5] << 16),
                       x[6] | ((uint32_t)x[7] << 16));
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if ((mine >> j) & 1) dst[j] = x[j];
      }
    } else {
      uint32_t x[2] = {0u, 0u};
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if ((mine >> j) & 1) x[j >> 2] |= (uint32_t)st[paged_vtok(g, j) * LROW + d] << (8 * (j & 3));
      if constexpr (FMT == IFR_KV_INT8) {
        uint8_t* dst = vpart + (size_t)r * 8;
        if (mine == 0xFFu) {
          *reinterpret_cast<uint2*>(dst) = make_uint2(x[0], x[1]);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if ((mine >> j) & 1) dst[j] = (uint8_t)(x[j >> 2] >> (8 * (j & 3)));
        }
      } else {
        uint32_t* dst = reinterpret_cast<uint32_t*>(vpart) + r;
        uint32_t keep = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (!((mine >> j) & 1)) keep |= 15u << (4 * paged_nibble(j));
        const uint32_t nw = pack_nibbles(x);
        *dst = keep ? (*dst & keep) | nw : nw;
      }
    }
  }
}

// fp16 value of one code (int4: the one rounding of c s + z, as the attention
// kernels have it).
template <int FMT>
__device__ __forceinline__ uint16_t value_of(int c, uint16_t s, uint16_t z) {
  if constexpr (FMT == IFR_KV_INT8) {
    return ifrd::f2h((float)c * ifrd::h2f(s));
  } else {
    const _Float16 v = __builtin_elementwise_fma((_Float16)c, __builtin_bit_cast(_Float16, s), __builtin_bit_cast(_Float16, z));
    return __builtin_bit_cast(uint16_t, v);
  }
}

// One wave per (run, kv head): the inverse of the append, into [M][nkv][HD].
// Whole 8-token runs of V are read (they are inside the page), the tokens of
// the run are written.
template <int HD, int FMT>
__global__ __launch_bounds__(256) void paged_read_kernel(const PagedRun* runs, int n_runs, uint16_t* k, uint16_t* v,
                                                         PagedPool kv) {
  constexpr int LPT = HD / 8, TPI = 64 / LPT;
  constexpr int LROW = HD * 2 + 16;
  __shared__ __align__(16) uint8_t stage[4][kPgTok * LROW];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t item = (int64_t)blockIdx.x * 4 + w;
  if (item >= (int64_t)n_runs * kv.nkv) return;
  const PagedRun run = runs[item / kv.nkv];
  const int kvh = (int)(item % kv.nkv);
  const uint8_t* kpart =
      kv.pool + (size_t)run.page * paged_page(FMT, HD, kv.nkv) + (size_t)kvh * 2 * paged_part(FMT, HD);
  const uint8_t* vpart = kpart + paged_part(FMT, HD);
  constexpr size_t codes = FMT == IFR_KV_FP16 ? 0 : FMT == IFR_KV_INT8 ? 32 * HD : 16 * HD;
  const uint16_t* kscale = reinterpret_cast<const uint16_t*>(kpart + codes);
  const uint16_t* vscale = reinterpret_cast<const uint16_t*>(vpart + codes);
  uint8_t* st = stage[w];
  const int t1 = run.t0 + run.n;
  for (int r = lane; r < 4 * HD; r += 64) {
    const int g = r / HD;
    const int d = FMT == IFR_KV_FP16 ? r % HD : (r % (HD / 16)) * 16 + (r % HD) / (HD / 16);
    uint32_t x[4];
    if constexpr (FMT == IFR_KV_FP16) {
      const uint4 q = reinterpret_cast<const uint4*>(vpart)[r];
      x[0] = q.x; x[1] = q.y; x[2] = q.z; x[3] = q.w;
    } else if constexpr (FMT == IFR_KV_INT8) {
      const uint2 q = reinterpret_cast<const uint2*>(vpart)[r];
      x[0] = q.x; x[1] = q.y;
    } else {
      x[0] = reinterpret_cast<const uint32_t*>(vpart)[r];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int t = paged_vtok(g, j);
      if (t < run.t0 || t >= t1) continue;
      uint16_t y;
      if constexpr (FMT == IFR_KV_FP16) {
        y = (uint16_t)(x[j >> 1] >> (16 * (j & 1)));
      } else if constexpr (FMT == IFR_KV_INT8) {
        y = value_of<FMT>((int)(int8_t)(x[j >> 2] >> (8 * (j & 3))), vscale[paged_vscale(FMT, HD, t, 0)], 0);
      } else {
        const int i = paged_vscale(FMT, HD, t, d / kPgGroup);
        y = value_of<FMT>((int)((x[0] >> (4 * paged_nibble(j))) & 15u), vscale[i], vscale[i + 8]);
      }
      *reinterpret_cast<uint16_t*>(st + t * LROW + d * 2) = y;
    }
  }
  ifrd::wave_sync();
  const int sub = lane / LPT, d0 = (lane % LPT) * 8;
  for (int b = 0; b < run.n; b += TPI) {
    const int i = b + sub, t = run.t0 + i;
    if (i >= run.n) continue;
    const int64_t o = ((int64_t)(run.row + i) * kv.nkv + kvh) * HD + d0;
    uint4 kw;
    if constexpr (FMT == IFR_KV_FP16) {
      kw = *reinterpret_cast<const uint4*>(kpart + (size_t)paged_koff(FMT, HD, t, d0) * 2);
    } else {
      uint16_t y[8];
      if constexpr (FMT == IFR_KV_INT8) {
        const uint2 c = *reinterpret_cast<const uint2*>(kpart + paged_koff(FMT, HD, t, d0));
        const uint32_t cw[2] = {c.x, c.y};
        const uint16_t s = kscale[paged_kscale(FMT, HD, t, 0)];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = value_of<FMT>((int)(int8_t)(cw[e >> 2] >> (8 * (e & 3))), s, 0);
      } else {
        const uint32_t c = *reinterpret_cast<const uint32_t*>(kpart + paged_koff(FMT, HD, t, d0) / 2);
        const int si = paged_kscale(FMT, HD, t, d0 / kPgGroup);
        const uint16_t s = kscale[si], z = kscale[si + 1];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = value_of<FMT>((int)((c >> (4 * paged_nibble(e))) & 15u), s, z);
      }
      kw = make_uint4(y[0] | ((uint32_t)y[1] << 16), y[2] | ((uint32_t)y[3] << 16), y[4] | ((uint32_t)y[5] << 16),
                      y[6] | ((uint32_t)y[7] << 16));
    }
    *reinterpret_cast<uint4*>(k + o) = kw;
    *reinterpret_cast<uint4*>(v + o) = *reinterpret_cast<const uint4*>(st + t * LROW + d0 * 2);
  }
}

constexpr int64_t kMaxBlocks = 0x7FFFFFFF;

template <int HD, int FMT>
hipError_t append_fmt(const PagedAppendArgs& a, const PagedPool& kv, hipStream_t st) {
  const int64_t kvb = ((int64_t)a.n_runs * kv.nkv + 3) / 4;
  const int64_t items = a.r.q_d ? (int64_t)a.M * kv.nq * (a.r.rotary / 16 + (HD - a.r.rotary) / 8) : 0;
  const int64_t blocks = kvb + (items + 255) / 256;
  if (blocks <= 0) return hipSuccess;
  if (blocks > kMaxBlocks) return hipErrorInvalidValue;
  hipLaunchKernelGGL((paged_append_kernel<HD, FMT>), dim3((unsigned)blocks), dim3(256), 0, st, a, kv, (int)kvb);
  return hipGetLastError();
}

template <int HD, int FMT>
hipError_t read_fmt(const PagedRun* runs, int n, uint16_t* k, uint16_t* v, const PagedPool& kv, hipStream_t st) {
  const int64_t blocks = ((int64_t)n * kv.nkv + 3) / 4;
  if (blocks <= 0) return hipSuccess;
  if (blocks > kMaxBlocks) return hipErrorInvalidValue;
  hipLaunchKernelGGL((paged_read_kernel<HD, FMT>), dim3((unsigned)blocks), dim3(256), 0, st, runs, n, k, v, kv);
  return hipGetLastError();
}

}  // namespace

#define IFR_PAGED_BY_FORMAT(F, ...)                                  \
  do {                                                               \
    if (kv.hd == 64 && kv.fmt == IFR_KV_FP16) return F<64, IFR_KV_FP16>(__VA_ARGS__);   \
    if (kv.hd == 64 && kv.fmt == IFR_KV_INT8) return F<64, IFR_KV_INT8>(__VA_ARGS__);   \
    if (kv.hd == 64 && kv.fmt == IFR_KV_INT4) return F<64, IFR_KV_INT4>(__VA_ARGS__);   \
    if (kv.hd == 128 && kv.fmt == IFR_KV_FP16) return F<128, IFR_KV_FP16>(__VA_ARGS__); \
    if (kv.hd == 128 && kv.fmt == IFR_KV_INT8) return F<128, IFR_KV_INT8>(__VA_ARGS__); \
    if (kv.hd == 128 && kv.fmt == IFR_KV_INT4) return F<128, IFR_KV_INT4>(__VA_ARGS__); \
    if (kv.hd == 256 && kv.fmt == IFR_KV_FP16) return F<256, IFR_KV_FP16>(__VA_ARGS__); \
    if (kv.hd == 256 && kv.fmt == IFR_KV_INT8) return F<256, IFR_KV_INT8>(__VA_ARGS__); \
    if (kv.hd == 256 && kv.fmt == IFR_KV_INT4) return F<256, IFR_KV_INT4>(__VA_ARGS__); \
    return hipErrorInvalidValue;                                     \
  } while (0)

hipError_t launch_paged_append(const PagedAppendArgs& a, const PagedPool& kv, hipStream_t st) {
  IFR_PAGED_BY_FORMAT(append_fmt, a, kv, st);
}
hipError_t launch_paged_read(const PagedRun* runs, int n, uint16_t* k, uint16_t* v, const PagedPool& kv, hipStream_t st) {
  IFR_PAGED_BY_FORMAT(read_fmt, runs, n, k, v, kv, st);
}

}  // namespace ifrk
