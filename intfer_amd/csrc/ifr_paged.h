// Caller-owned paged KV cache: page layout and the launchers of its kernels
// (paged.hip: append and read; paged_attn.hip: attention).  The plan that
// fills these structs from a batch is paged.cpp.
#pragma once
#include <hip/hip_runtime.h>
#include <cstddef>
#include <cstdint>

#include "intfer_amd.h"

namespace ifrk {

constexpr int kPgTok = 32;    // tokens per page
constexpr int kPgGroup = 64;  // dims of one int4 scale and minimum

// Bytes of the K (or the V) part of one (page, kv head) block, and of a page.
__host__ __device__ constexpr size_t paged_part(int fmt, int hd) {
  return fmt == IFR_KV_FP16 ? 64 * (size_t)hd : fmt == IFR_KV_INT8 ? 32 * (size_t)hd + 64 : 18 * (size_t)hd;
}
__host__ __device__ constexpr size_t paged_page(int fmt, int hd, int nkv) { return 2 * paged_part(fmt, hd) * nkv; }

// Element order inside a part (token t of the page, dim d).  A lane of a
// 16x16x32 MFMA takes 8 consecutive elements: K rows are tokens 16 h + c and
// the lane group g holds dims 32 i + 8 g ..; V rows are dims 16 n + c and the
// lane group g holds tokens 4 g .. and 16 + 4 g .., which are the tokens whose
// scores K's product leaves in that group, so P moves between no lanes.
// fp16 lanes read 16 bytes per fragment; the narrower formats keep all of a
// lane's fragments together, so that a lane's read stays 8 to 32 bytes wide.
__host__ __device__ constexpr int paged_koff(int fmt, int hd, int t, int d) {
  return fmt == IFR_KV_FP16 ? ((d >> 3) * 32 + t) * 8 + (d & 7)
                            : ((t * 4 + ((d >> 3) & 3)) * (hd / 32) + (d >> 5)) * 8 + (d & 7);
}
__host__ __device__ constexpr int paged_vgroup(int t) { return (t & 15) >> 2; }
__host__ __device__ constexpr int paged_vslot(int t) { return 4 * (t >> 4) + (t & 3); }
__host__ __device__ constexpr int paged_vtok(int g, int j) { return 16 * (j >> 2) + 4 * g + (j & 3); }
// 8-element run of (group, dim) in V
__host__ __device__ constexpr int paged_vrun(int fmt, int hd, int g, int d) {
  return fmt == IFR_KV_FP16 ? g * hd + d : (g * 16 + (d & 15)) * (hd / 16) + (d >> 4);
}
// int4: nibble of element e in its 8-element dword (the order in which two
// masks and a shift yield fp16 pairs of neighbours)
__host__ __device__ constexpr int paged_nibble(int e) { return (e & 1) * 4 + (e >> 1); }
// fp16 index of a scale behind the codes (int4: the scale; its minimum is
// +1 in K and +8 in V)
__host__ __device__ constexpr int paged_kscale(int fmt, int hd, int t, int u) {
  return fmt == IFR_KV_INT8 ? (t & 15) * 2 + (t >> 4) : (((t & 15) * (hd / kPgGroup) + u) * 2 + (t >> 4)) * 2;
}
__host__ __device__ constexpr int paged_vscale(int fmt, int hd, int t, int u) {
  return fmt == IFR_KV_INT8 ? paged_vgroup(t) * 8 + paged_vslot(t)
                            : (paged_vgroup(t) * (hd / kPgGroup) + u) * 16 + paged_vslot(t);
}

struct PagedPool {
  uint8_t* pool;
  int fmt, nkv, hd, nq;
};

struct PagedRow {       // one row of the batch: it sees positions [lo, hi)
  int lo, hi, pos, seq;
};
struct PagedRun {       // rows [row, row + n) are tokens [t0, t0 + n) of a page, positions from pos
  int page, t0, n, row, pos, pad[3];
};
// One workgroup of attention: columns [col0, col0 + ncol) of a sequence (column
// = new row * G + head of the kv head's group) over its pages [p0, p1).
struct PagedUnit {
  int row0;   // batch row of the sequence's first new row
  int kvh;
  int col0, ncol;
  int tab;    // the sequence's first entry in the page table
  int p0, p1;
  int part;   // first partial column, or -1: the unit writes the output itself
};
// Partials of columns [col0, col0 + n), at most 1024 / hd of them: split s of
// column i is partial column base + s * stride + i.
struct PagedJoin {
  int row0, kvh, col0, n, base, stride, ns, pad;
};

struct PagedAppendArgs {
  const PagedRun* runs;
  int n_runs;
  const PagedRow* rows;
  int M;
  ifr_paged_rows r;
};
hipError_t launch_paged_append(const PagedAppendArgs& a, const PagedPool& kv, hipStream_t st);
hipError_t launch_paged_read(const PagedRun* runs, int n_runs, uint16_t* k, uint16_t* v, const PagedPool& kv,
                             hipStream_t st);

struct PagedAttnArgs {
  const PagedUnit* units;   // of this launch
  int n_units;
  const PagedRow* rows;
  const int32_t* table;
  const uint16_t* q;
  int64_t q_stride;
  void* out;
  int64_t out_stride;
  int out_f32;
  float scale;              // of q . k
  float cap;                // 0: none
  const float* slopes;      // null: none
  float* part_o;            // [columns][hd]
  float* part_ml;           // [columns][2]
};
// narrow units: up to 16 * tiles columns (tiles 1 or 2) by workgroups of 4
// waves, or 8 (two tiles, heads of 128); wide units: up to kPgWide columns, heads
// of up to kPgWideDim.
constexpr int kPgWide = 128, kPgWideDim = 128;
// Waves a SIMD that a narrow kernel's registers leave (o, q and the raw page),
// and workgroups a CU of a wide one.
constexpr int paged_narrow_waves(int fmt, int hd, int nt) {
  return fmt == IFR_KV_FP16 && hd >= 128 ? (hd == 128 ? 2 : 1)
                                         : hd * nt <= 64 ? 4 : hd * nt <= 128 ? 3 : hd * nt <= 256 ? 2 : 1;
}
constexpr int kPgWideGroups = 2;
hipError_t launch_paged_narrow(const PagedAttnArgs& a, const PagedPool& kv, int tiles, int waves, hipStream_t st);
hipError_t launch_paged_wide(const PagedAttnArgs& a, const PagedPool& kv, hipStream_t st);
hipError_t launch_paged_join(const PagedJoin* joins, int n, const PagedAttnArgs& a, const PagedPool& kv,
                             hipStream_t st);

}  // namespace ifrk
