// Rows of K and V into the pages of a caller-owned cache, with the rotation of
// K and Q on the way, and cached rows back as fp16.
//
// Rotation (rotate-half over the first `rotary` dims, fp32 tables):
//   x'_d = x_d cos_d - x_{d+r/2} sin_d,  x'_{d+r/2} = x_{d+r/2} cos_d + x_d sin_d
// with every product and the sum rounded to fp32.  K is stored from that fp32
// value, so the only rounding after it is the format's own:
//   fp16  fp16(x)
//   int8  s = fp16(max|x| * (1 / 127)) per (token, head),
//         c = half-away(x * (1 / s))
//   int4  z = fp16(min), s = fp16((max - min) * (1 / 15)) per (token, head, 64
//         dims), c = rint((x - z) * (1 / s)) in 0 .. 15; it stands for
//         fp16(c s + z)
// (reciprocals and products rounded to fp32 each).
// A group that holds a NaN or an infinity gets a NaN scale and reads back as
// NaN; the codes of a group whose scale rounds to zero are zero.  A scale whose
// largest code would round to infinity is the next smaller one (int8: 515.5 at
// most), so that no finite row reads back as infinite.
#include "ifr_dev.h"
#include "ifr_paged.h"

namespace ifrk {
namespace {

constexpr float kMaxHalf = 65504.0f;
constexpr int kHalfMirror = 0x141;  // DPP: lane i of 8 reads lane 7 - i

// Reductions over the 8, 16 or 32 consecutive lanes that share a token (all
// lanes of the wave take part).
template <int LPT>
__device__ __forceinline__ float group_max(float v) {
  v = fmaxf(v, ifrd::lane_xor<1>(v));
  v = fmaxf(v, ifrd::lane_xor<2>(v));
  v = fmaxf(v, ifrd::dpp_f<kHalfMirror>(v));  // (the quads are uniform: any lane of the other one)
  if constexpr (LPT >= 16) v = fmaxf(v, ifrd::lane_xor<8>(v));
  if constexpr (LPT >= 32) v = fmaxf(v, ifrd::lane_xor<16>(v));
  return v;
}
// Whether one of the lanes' values is a NaN or an infinity (0 x is 0 of none else).
template <int LPT>
__device__ __forceinline__ bool group_bad(const float (&x)[8]) {
  float t = 0.0f;
#pragma unroll
  for (int e = 0; e < 8; ++e) t = fmaf(x[e], 0.0f, t);
  constexpr uint64_t kLanes = LPT >= 32 ? 0xFFFFFFFFull : (1ull << LPT) - 1;
  return (__ballot(t != t) >> (threadIdx.x & 63 & ~(LPT - 1)) & kLanes) != 0;
}

// Quantize a lane's 8 consecutive dims.  int8: the scale of the whole head row
// (LPT lanes); int4: of its 64 dims (8 lanes).  Codes as bytes or, NIBBLES, as
// the int4 dword of 8 elements.
template <int FMT, int LPT, bool NIBBLES>
__device__ __forceinline__ void quantize8(const float (&x)[8], uint32_t (&code)[2], uint16_t& scale, uint16_t& zero) {
  if constexpr (FMT == IFR_KV_INT8) {
    const bool bad = group_bad<LPT>(x);
    float a = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) a = fmaxf(a, fabsf(x[e]));
    a = group_max<LPT>(a);
    scale = bad ? (uint16_t)0x7E00u : ifrd::f2h(fminf(a * (1.0f / 127.0f), 515.5f));
    const float s = ifrd::h2f(scale);
    const float inv = s > 0.0f && !bad ? 1.0f / s : 0.0f;
    code[0] = code[1] = 0u;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float v = bad ? 0.0f : x[e];
      code[e >> 2] |= ((uint32_t)ifrd::quant_half_away(v, inv) & 0xFFu) << (8 * (e & 3));
    }
  } else if constexpr (FMT == IFR_KV_INT4) {
    const bool bad = group_bad<8>(x);
    float hi = -INFINITY, lo = INFINITY;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      hi = fmaxf(hi, x[e]);
      lo = fminf(lo, x[e]);
    }
    hi = group_max<8>(hi);
    lo = -group_max<8>(-lo);
    lo = fminf(fmaxf(lo, -kMaxHalf), kMaxHalf);  // (a rotated value can pass fp16's range)
    hi = fminf(fmaxf(hi, -kMaxHalf), kMaxHalf);
    scale = ifrd::f2h((hi - lo) * (1.0f / 15.0f));
    zero = ifrd::f2h(lo);
    if (15.0f * ifrd::h2f(scale) + ifrd::h2f(zero) >= 65520.0f) scale -= 1;  // code 15 would round to infinity
    if (bad) {
      scale = 0x7E00u;
      zero = 0u;
    }
    const float s = ifrd::h2f(scale), z = ifrd::h2f(zero);
    const float inv = s > 0.0f && !bad ? 1.0f / s : 0.0f;
    float c[8];  // (the clamp also turns the NaN of a bad group's infinity times zero into a code)
#pragma unroll
    for (int e = 0; e < 8; ++e) c[e] = fminf(fmaxf(__builtin_rintf((x[e] - z) * inv), 0.0f), 15.0f);
    // codes side by side by exact fp32 sums: 16 bits at a time
    if constexpr (NIBBLES) {
      const float even = fmaf(c[6], 4096.0f, fmaf(c[4], 256.0f, fmaf(c[2], 16.0f, c[0])));
      const float odd = fmaf(c[7], 4096.0f, fmaf(c[5], 256.0f, fmaf(c[3], 16.0f, c[1])));
      code[0] = (uint32_t)even | ((uint32_t)odd << 16);
      code[1] = 0u;
    } else {
#pragma unroll
      for (int q = 0; q < 2; ++q)
        code[q] = (uint32_t)fmaf(c[4 * q + 1], 256.0f, c[4 * q]) | ((uint32_t)fmaf(c[4 * q + 3], 256.0f, c[4 * q + 2]) << 16);
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

// 8 values of a rotation table (16-byte aligned rows: half is a multiple of 8)
__device__ __forceinline__ void load_table(const float* p, float (&x)[8]) {
  const v4f u = reinterpret_cast<const v4f*>(p)[0], v = reinterpret_cast<const v4f*>(p)[1];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    x[e] = u[e];
    x[4 + e] = v[e];
  }
}

// Rows a workgroup rotates of Q, about four items a thread.
__host__ __device__ inline int q_rows(int items) { return items >= 1024 ? 1 : 1024 / items; }

// One workgroup per (run, kv head): up to 32 tokens of one page.  HD / 8 lanes
// hold a token, 8 dims each, so 2048 / HD tokens are in hand at once and a page
// is one to four such passes (loading all of them ahead took 126 registers at
// 256 dims and left the blocks that rotate Q three waves a SIMD).  K goes
// straight to its place; V, whose 8-element runs are 8 tokens of one dim, crosses
// through LDS.  A run of V that the tokens cover whole is stored whole, else
// element by element (fp16, int8) or as a read-modify-write of its dword (int4; a
// batch writes a page from one run only, so nobody else has that dword).  The
// blocks past the runs rotate Q.
template <int HD, int FMT>
__global__ __launch_bounds__(256) void paged_append_kernel(PagedAppendArgs a, PagedPool kv, int kv_blocks) {
  constexpr int LPT = HD / 8, TP = 256 / LPT, PASSES = kPgTok / TP, U = HD / kPgGroup;
  constexpr int ES = FMT == IFR_KV_FP16 ? 2 : 1;   // bytes of an element in LDS
  constexpr int LROW = HD * ES + 16;
  __shared__ __align__(16) uint8_t st[kPgTok * LROW];
  const int half = a.r.rotary / 2, tid = threadIdx.x;
  if ((int)blockIdx.x >= kv_blocks) {
    // Q: an item is 8 dims and their partners, or 8 dims past the rotation
    const unsigned np = half / 8, ni = np + (HD - a.r.rotary) / 8, per = ni * kv.nq, nr = q_rows((int)per);
    const int m0 = ((int)blockIdx.x - kv_blocks) * (int)nr;
    const unsigned n = min((int)nr, a.M - m0) * per;
    for (unsigned i = tid; i < n; i += 256) {
      const unsigned r = i / per, hp = i - r * per, h = hp / ni, p = hp - h * ni;
      const int m = m0 + (int)r;
      const uint16_t* src = a.r.q_d + (int64_t)m * a.r.q_stride + (int64_t)h * HD;
      uint16_t* dst = a.r.q_out_d + (int64_t)m * a.r.q_out_stride + (int64_t)h * HD;
      if (p >= np) {
        const int d = a.r.rotary + 8 * (int)(p - np);
        *reinterpret_cast<uint4*>(dst + d) = *reinterpret_cast<const uint4*>(src + d);
        continue;
      }
      const int64_t t = (int64_t)a.rows[m].pos * half + 8 * p;
      float x[8], y[8], c[8], s[8], u[8], v[8];
      load8(src + 8 * p, x);
      load8(src + half + 8 * p, y);
      load_table(a.r.cos_d + t, c);
      load_table(a.r.sin_d + t, s);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        u[e] = x[e] * c[e] - y[e] * s[e];
        v[e] = y[e] * c[e] + x[e] * s[e];
      }
      *reinterpret_cast<uint4*>(dst + 8 * p) = pack8(u);
      *reinterpret_cast<uint4*>(dst + half + 8 * p) = pack8(v);
    }
    return;
  }
  const unsigned item = blockIdx.x, ri = item / (unsigned)kv.nkv;
  const PagedRun run = a.runs[ri];
  const int kvh = (int)(item - ri * kv.nkv);
  uint8_t* kpart = kv.pool + (size_t)run.page * paged_page(FMT, HD, kv.nkv) + (size_t)kvh * 2 * paged_part(FMT, HD);
  uint8_t* vpart = kpart + paged_part(FMT, HD);
  constexpr size_t codes = FMT == IFR_KV_FP16 ? 0 : FMT == IFR_KV_INT8 ? 32 * HD : 16 * HD;
  uint16_t* kscale = reinterpret_cast<uint16_t*>(kpart + codes);
  uint16_t* vscale = reinterpret_cast<uint16_t*>(vpart + codes);
  const int sub = tid / LPT, d0 = (tid % LPT) * 8, u = d0 / kPgGroup;
  const bool turns = d0 < a.r.rotary;
  const int ds = d0 < half ? d0 : d0 - half;  // where the pair's table values are
#pragma unroll 1
  for (int q = 0; q < PASSES; ++q) {
    if (q * TP >= run.n) break;
    const int i = q * TP + sub, t = run.t0 + i;
    const bool on = i < run.n;
    const int64_t m = run.row + (on ? i : 0);
    const uint16_t* kr = a.r.k_d + m * a.r.k_stride + (int64_t)kvh * HD;
    float x[8], y[8];
    load8(kr + d0, x);
    load8(a.r.v_d + m * a.r.v_stride + (int64_t)kvh * HD + d0, y);
    if (turns) {
      float p[8], c[8], s[8];
      load8(kr + (d0 < half ? d0 + half : ds), p);
      const int64_t tb = (int64_t)(run.pos + (on ? i : 0)) * half + ds;
      load_table(a.r.cos_d + tb, c);
      load_table(a.r.sin_d + tb, s);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float xc = x[e] * c[e], ps = p[e] * s[e];
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
      quantize8<FMT, LPT, FMT == IFR_KV_INT4>(x, kc, ks, kz);
      quantize8<FMT, LPT, false>(y, vc, vs, vz);
      if (on) {
        *reinterpret_cast<uint2*>(st + t * LROW + d0) = make_uint2(vc[0], vc[1]);
        if constexpr (FMT == IFR_KV_INT8) {
          *reinterpret_cast<uint2*>(kpart + paged_koff(FMT, HD, t, d0)) = make_uint2(kc[0], kc[1]);
          if (d0 == 0) {
            kscale[paged_kscale(FMT, HD, t, 0)] = ks;
            vscale[paged_vscale(FMT, HD, t, 0)] = vs;
          }
        } else {
          *reinterpret_cast<uint32_t*>(kpart + paged_koff(FMT, HD, t, d0) / 2) = kc[0];
          if (d0 % kPgGroup == 0) {
            *reinterpret_cast<uint32_t*>(kscale + paged_kscale(FMT, HD, t, u)) = (uint32_t)ks | ((uint32_t)kz << 16);
            vscale[paged_vscale(FMT, HD, t, u)] = vs;
            vscale[paged_vscale(FMT, HD, t, u) + 8] = vz;
          }
        }
      }
    }
  }
  __syncthreads();
  const int t1 = run.t0 + run.n;
  // A thread takes 4 bytes of each of a group's 8 tokens, 2 or 4 dims, and turns
  // them into those dims' runs; only groups that hold a token of ours.
  constexpr int DPI = 4 / ES;
  for (int i = tid; i < 4 * HD / DPI; i += 256) {
    const int g = i / (HD / DPI), d = i % (HD / DPI) * DPI;
    uint32_t mine = 0, w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int t = paged_vtok(g, j);
      const bool in = t >= run.t0 && t < t1;
      mine |= (uint32_t)in << j;
      w[j] = in ? *reinterpret_cast<const uint32_t*>(st + t * LROW + d * ES) : 0u;
    }
    if (!mine) continue;
    if constexpr (FMT == IFR_KV_FP16) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint32_t sel = e ? 0x07060302u : 0x05040100u;  // the e-th halves of two dwords
        uint16_t* dst = reinterpret_cast<uint16_t*>(vpart) + (size_t)(g * HD + d + e) * 8;
        uint32_t x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = __builtin_amdgcn_perm(w[2 * j + 1], w[2 * j], sel);
        if (mine == 0xFFu) {
          *reinterpret_cast<uint4*>(dst) = make_uint4(x[0], x[1], x[2], x[3]);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if ((mine >> j) & 1) dst[j] = (uint16_t)(x[j >> 1] >> (16 * (j & 1)));
        }
      }
    } else if constexpr (FMT == IFR_KV_INT8) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        uint8_t* dst = vpart + (size_t)paged_vrun(FMT, HD, g, d + e) * 8;
        const uint32_t sel = 0x0C0C0400u + e * 0x0101u;  // byte e of two dwords
        uint32_t x[2];
#pragma unroll
        for (int q = 0; q < 2; ++q)
          x[q] = __builtin_amdgcn_perm(w[4 * q + 1], w[4 * q], sel) | (__builtin_amdgcn_perm(w[4 * q + 3], w[4 * q + 2], sel) << 16);
        if (mine == 0xFFu) {
          *reinterpret_cast<uint2*>(dst) = make_uint2(x[0], x[1]);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if ((mine >> j) & 1) dst[j] = (uint8_t)(x[j >> 2] >> (8 * (j & 3)));
        }
      }
    } else {
      // even tokens' nibbles side by side, then odd ones' (paged_nibble)
      const uint32_t p = w[0] | (w[2] << 4), q = w[4] | (w[6] << 4), r = w[1] | (w[3] << 4), u2 = w[5] | (w[7] << 4);
      uint32_t keep = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (!((mine >> j) & 1)) keep |= 15u << (4 * paged_nibble(j));
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        uint32_t* dst = reinterpret_cast<uint32_t*>(vpart) + paged_vrun(FMT, HD, g, d + e);
        const uint32_t sel = 0x0C0C0400u + e * 0x0101u;
        const uint32_t nw = __builtin_amdgcn_perm(q, p, sel) | (__builtin_amdgcn_perm(u2, r, sel) << 16);
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

// One workgroup per (run, kv head): the inverse of the append, into
// [M][nkv][HD].  Whole 8-token runs of V are read (they are inside the page), the
// tokens of the run are written.
template <int HD, int FMT>
__global__ __launch_bounds__(256) void paged_read_kernel(const PagedRun* runs, uint16_t* k, uint16_t* v, PagedPool kv) {
  constexpr int LPT = HD / 8, TP = 256 / LPT, PASSES = kPgTok / TP, VR = HD / 64;
  constexpr int LROW = HD * 2 + 16;
  __shared__ __align__(16) uint8_t st[kPgTok * LROW];
  const int tid = threadIdx.x;
  const unsigned item = blockIdx.x, ri = item / (unsigned)kv.nkv;
  const PagedRun run = runs[ri];
  const int kvh = (int)(item - ri * kv.nkv);
  const uint8_t* kpart =
      kv.pool + (size_t)run.page * paged_page(FMT, HD, kv.nkv) + (size_t)kvh * 2 * paged_part(FMT, HD);
  const uint8_t* vpart = kpart + paged_part(FMT, HD);
  constexpr size_t codes = FMT == IFR_KV_FP16 ? 0 : FMT == IFR_KV_INT8 ? 32 * HD : 16 * HD;
  const uint16_t* kscale = reinterpret_cast<const uint16_t*>(kpart + codes);
  const uint16_t* vscale = reinterpret_cast<const uint16_t*>(vpart + codes);
  const int t1 = run.t0 + run.n;
  const int sub = tid / LPT, d0 = (tid % LPT) * 8;
  // K of all passes is on its way while V crosses
  uint4 kq[PASSES];
  uint32_t ks[PASSES];
#pragma unroll
  for (int q = 0; q < PASSES; ++q) {
    if (q * TP >= run.n) break;
    const int t = run.t0 + min(q * TP + sub, run.n - 1);
    if constexpr (FMT == IFR_KV_FP16) {
      kq[q] = *reinterpret_cast<const uint4*>(kpart + (size_t)paged_koff(FMT, HD, t, d0) * 2);
    } else if constexpr (FMT == IFR_KV_INT8) {
      const uint2 w = *reinterpret_cast<const uint2*>(kpart + paged_koff(FMT, HD, t, d0));
      kq[q] = make_uint4(w.x, w.y, 0u, 0u);
      ks[q] = kscale[paged_kscale(FMT, HD, t, 0)];
    } else {
      kq[q] = make_uint4(*reinterpret_cast<const uint32_t*>(kpart + paged_koff(FMT, HD, t, d0) / 2), 0u, 0u, 0u);
      ks[q] = *reinterpret_cast<const uint32_t*>(kscale + paged_kscale(FMT, HD, t, d0 / kPgGroup));
    }
  }
#pragma unroll
  for (int b = 0; b < VR; ++b) {
    const int r = tid + 256 * b, g = r / HD;
    const int d = FMT == IFR_KV_FP16 ? r % HD : (r % (HD / 16)) * 16 + (r % HD) / (HD / 16);
    uint32_t x[4];
    uint4 s = make_uint4(0u, 0u, 0u, 0u), z = s;
    if constexpr (FMT == IFR_KV_FP16) {
      const uint4 q = reinterpret_cast<const uint4*>(vpart)[r];
      x[0] = q.x; x[1] = q.y; x[2] = q.z; x[3] = q.w;
    } else if constexpr (FMT == IFR_KV_INT8) {
      const uint2 q = reinterpret_cast<const uint2*>(vpart)[r];
      x[0] = q.x; x[1] = q.y;
      s = reinterpret_cast<const uint4*>(vscale)[g];
    } else {
      x[0] = reinterpret_cast<const uint32_t*>(vpart)[r];
      const uint4* sz = reinterpret_cast<const uint4*>(vscale) + (g * (HD / kPgGroup) + d / kPgGroup) * 2;
      s = sz[0];
      z = sz[1];
    }
    const uint32_t sw[4] = {s.x, s.y, s.z, s.w}, zw[4] = {z.x, z.y, z.z, z.w};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int t = paged_vtok(g, j);
      if (t < run.t0 || t >= t1) continue;
      const uint16_t sj = (uint16_t)(sw[j >> 1] >> (16 * (j & 1))), zj = (uint16_t)(zw[j >> 1] >> (16 * (j & 1)));
      uint16_t y;
      if constexpr (FMT == IFR_KV_FP16) y = (uint16_t)(x[j >> 1] >> (16 * (j & 1)));
      else if constexpr (FMT == IFR_KV_INT8) y = value_of<FMT>((int)(int8_t)(x[j >> 2] >> (8 * (j & 3))), sj, 0);
      else y = value_of<FMT>((int)((x[0] >> (4 * paged_nibble(j))) & 15u), sj, zj);
      *reinterpret_cast<uint16_t*>(st + t * LROW + d * 2) = y;
    }
  }
  __syncthreads();
#pragma unroll
  for (int q = 0; q < PASSES; ++q) {
    const int i = q * TP + sub, t = run.t0 + i;
    if (i >= run.n) break;
    const int64_t o = ((int64_t)(run.row + i) * kv.nkv + kvh) * HD + d0;
    uint4 kw = kq[q];
    if constexpr (FMT != IFR_KV_FP16) {
      uint16_t y[8];
      const uint16_t s = (uint16_t)ks[q], z = (uint16_t)(ks[q] >> 16);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        y[e] = FMT == IFR_KV_INT8
                   ? value_of<FMT>((int)(int8_t)((e < 4 ? kw.x : kw.y) >> (8 * (e & 3))), s, 0)
                   : value_of<FMT>((int)((kw.x >> (4 * paged_nibble(e))) & 15u), s, z);
      kw = make_uint4(y[0] | ((uint32_t)y[1] << 16), y[2] | ((uint32_t)y[3] << 16), y[4] | ((uint32_t)y[5] << 16),
                      y[6] | ((uint32_t)y[7] << 16));
    }
    *reinterpret_cast<uint4*>(k + o) = kw;
    *reinterpret_cast<uint4*>(v + o) = *reinterpret_cast<const uint4*>(st + t * LROW + d0 * 2);
  }
}

constexpr int64_t kMaxBlocks = 0xFFFFFF;  // of 256 threads

template <int HD, int FMT>
hipError_t append_fmt(const PagedAppendArgs& a, const PagedPool& kv, hipStream_t st) {
  const int64_t kvb = (int64_t)a.n_runs * kv.nkv, items = (int64_t)kv.nq * (a.r.rotary / 16 + (HD - a.r.rotary) / 8);
  const int64_t nr = items < kMaxBlocks ? q_rows((int)items) : 1;
  const int64_t blocks = kvb + (a.r.q_d ? (a.M + nr - 1) / nr : 0);
  if (blocks <= 0) return hipSuccess;
  if (blocks > kMaxBlocks || items > kMaxBlocks) return hipErrorInvalidValue;
  hipLaunchKernelGGL((paged_append_kernel<HD, FMT>), dim3((unsigned)blocks), dim3(256), 0, st, a, kv, (int)kvb);
  return hipGetLastError();
}

template <int HD, int FMT>
hipError_t read_fmt(const PagedRun* runs, int n, uint16_t* k, uint16_t* v, const PagedPool& kv, hipStream_t st) {
  const int64_t blocks = (int64_t)n * kv.nkv;
  if (blocks <= 0) return hipSuccess;
  if (blocks > kMaxBlocks) return hipErrorInvalidValue;
  hipLaunchKernelGGL((paged_read_kernel<HD, FMT>), dim3((unsigned)blocks), dim3(256), 0, st, runs, k, v, kv);
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
