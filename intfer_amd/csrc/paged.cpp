// The plan of a caller-owned paged KV cache (ifr_paged_*): checks a batch on
// the host, cuts it into work for the kernels of paged.hip and
// paged_attn.hip, and keeps what they need on the device.  One plan serves
// every layer of an iteration.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <new>
#include <vector>

#include "host_model.h"
#include "ifr_kernels.h"
#include "ifr_paged.h"

using ifrh::fail;
using ifrk::kPgTok;

namespace {

#define PGCHK(expr)                                                                            \
  do {                                                                                         \
    hipError_t e_ = (expr);                                                                    \
    if (e_ != hipSuccess)                                                                      \
      return fail(e_ == hipErrorInvalidValue ? IFR_EINVAL : IFR_EDEVICE, "%s: %s (%s:%d)", #expr, \
                  hipGetErrorString(e_), __FILE__, __LINE__);                                  \
  } while (0)

constexpr int64_t kMaxRows = 1 << 24;      // rows of a batch
constexpr int64_t kMaxTokens = 1 << 30;    // tokens of a sequence
constexpr int64_t kMaxStride = (int64_t)1 << 32;
constexpr int64_t kMaxUnits = 1 << 22;     // attention tiles of all kv heads (a launch has fewer than 2^32 threads)

// scale, cap and scale / cap: products with log2 e and a zero score stay finite.
constexpr float kMaxFactor = 1e30f;

// Kinds of attention unit, by the columns and the waves of their workgroups:
// narrow ones of one and two column tiles, wide ones, and narrow ones of two
// tiles by eight waves.
constexpr int kKinds = 4, kWide = 2, kEight = 3;
constexpr int kWidth[kKinds] = {16, 32, ifrk::kPgWide, 32}, kTiles[kKinds] = {1, 2, 0, 2}, kWaves[kKinds] = {4, 4, 4, 8};

// The fewest pages of a wide split (256 tokens) and what one is a multiple of (a
// step's two pages); narrow: a page for each wave.
constexpr int kWideMin = 8, kWideGrain = 2;
constexpr int kCUs = 256;
// A narrow tile of so few pages a wave is not split: its waves' turns cost less
// than the launch that joins splits (one row, four waves, us: 250 tokens whole
// 5.6, in two 7.6; 500 tokens whole 8.9, in four 8.4).
constexpr int kWhole = 3;
// Sequences of more than 32 columns take wide units where the batch has so many
// pages of wide tiles: below, there are too few of them to hide their longer
// start, and narrow units, four times as many, win although they turn the pages
// into fp16 four times (16/8 heads of 128, int4, us narrow / wide: 64 rows on 500
// tokens 10.9 / 16.0, 256 on 2000, 2112 pages, 23.0 / 27.2, 512 on 2000, 4544,
// 33.8 / 34.2, 256 on 8000, 8128, 45.8 / 43.1).  Over fp16 pages, which need no
// turning, they have to fill the CUs besides (us narrow / wide: 4000 causal rows,
// 504 tiles, 101 / 109; 8000, 1000 tiles, 349 / 311; 4000 of 32/4 heads 198 / 164).
constexpr int64_t kWidePages = 16 * kCUs;
// A batch with units of two tiles takes its sequences of one tile in such units
// too, if these have few pages: their second tile is idle, but they run beside
// the others and not in a launch before them (16/8 heads of 128, int4, us two
// launches / one: 24 decode rows on 1000 tokens and a chunk of 512 32.4 / 28.2, 8
// on 1300 and 72 24.3 / 14.5, 8 on 4000 and 256 35.3 / 28.8, 64 on 1000 and 64,
// 20 thousand pages, 33.4 / 34.2).
constexpr int64_t kMergePages = 64 * kCUs;
// Two-tile units of heads of 128 leave a CU eight waves.  One workgroup of all
// of them takes whole tiles where two of four would need splits and a join: if
// the CUs hold all tiles at once and the longest is not far over the mean, or is
// whole for eight waves and not for four (16/8 heads of 128, int4: 512 rows on 500
// tokens 20.9 -> 15.9 us, 128 on 500 13.9 -> 11.2; but 28 x 5 verify rows on ragged
// contexts, the longest twice the mean, 28.0 -> 34.7).
constexpr double kEven = 1.5;

// The context's device is current while a call runs, the caller's afterwards.
struct OnDevice {
  int was = -1;
  explicit OnDevice(int dev) {
    if (hipGetDevice(&was) != hipSuccess) was = -1;
    if (was != dev) (void)hipSetDevice(dev);
    else was = -1;
  }
  ~OnDevice() {
    if (was >= 0) (void)hipSetDevice(was);
  }
};

bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// Whether rows a[M][wa] (stride sa) and b[M][wb] (stride sb), in bytes, share one.
bool overlap(const void* a, int64_t sa, int64_t wa, const void* b, int64_t sb, int64_t wb, int64_t M) {
  const int64_t x = (int64_t)reinterpret_cast<uintptr_t>(a), y = (int64_t)reinterpret_cast<uintptr_t>(b);
  if (x + (M - 1) * sa + wa <= y || y + (M - 1) * sb + wb <= x) return false;
  if (sa != sb || M == 1) return true;
  // equal strides (slices of one buffer): the columns decide
  int64_t d = (y - x) % sa;
  if (d < 0) d += sa;
  return !(d >= wa && d + wb <= sa);
}

}  // namespace

struct ifr_paged {
  ifr_ctx* ctx = nullptr;
  int device = 0;
  hipStream_t st = nullptr;
  ifr_paged_cfg cfg{};
  bool set = false, frozen = false, appendable = true;
  int M = 0, max_pos = -1;
  // what the kernels read, one allocation
  uint8_t* meta = nullptr;
  size_t meta_cap = 0;
  uint8_t* stage = nullptr;  // pinned; reused once the copy before has left it
  size_t stage_cap = 0;
  hipEvent_t copied = nullptr;
  bool copying = false;
  size_t o_rows = 0, o_runs = 0, o_units[kKinds] = {}, o_joins = 0, o_table = 0;
  int n_runs = 0, n_units[kKinds] = {}, n_joins = 0;
  float* part = nullptr;     // [columns][hd], then [columns][2]
  int64_t part_cap = 0, part_cols = 0;
};

namespace {

struct Tile {
  int kind, seq, col0, ncol, p0, p1;
};

int grow(ifr_paged* p, size_t meta, int64_t cols) {
  if (meta > p->meta_cap) {
    PGCHK(hipStreamSynchronize(p->st));
    if (p->meta) hipFree(p->meta);
    p->meta = nullptr;
    p->meta_cap = 0;
    const size_t n = std::max(meta + meta / 2, (size_t)65536);
    if (hipMalloc((void**)&p->meta, n) != hipSuccess) return fail(IFR_ENOMEM, "paged plan: %zu bytes", n);
    p->meta_cap = n;
  }
  if (meta > p->stage_cap) {
    if (p->copying) PGCHK(hipEventSynchronize(p->copied));
    p->copying = false;
    if (p->stage) hipHostFree(p->stage);
    p->stage = nullptr;
    p->stage_cap = 0;
    const size_t n = std::max(meta + meta / 2, (size_t)65536);
    if (hipHostMalloc((void**)&p->stage, n, 0) != hipSuccess) return fail(IFR_ENOMEM, "paged plan: %zu pinned bytes", n);
    p->stage_cap = n;
  }
  if (cols > p->part_cap) {
    PGCHK(hipStreamSynchronize(p->st));
    if (p->part) hipFree(p->part);
    p->part = nullptr;
    p->part_cap = 0;
    const int64_t n = std::max(cols + cols / 2, (int64_t)1024);
    if (hipMalloc((void**)&p->part, (size_t)n * (p->cfg.head_dim + 2) * sizeof(float)) != hipSuccess)
      return fail(IFR_ENOMEM, "paged plan: partials of %lld columns", (long long)n);
    p->part_cap = n;
  }
  return IFR_OK;
}

int set_batch(ifr_paged* p, const ifr_paged_batch* b) {
  const ifr_paged_cfg& c = p->cfg;
  const int S = b->n_seqs, G = c.n_heads / c.n_kv;
  if (S < 0) return fail(IFR_EINVAL, "n_seqs=%d", S);
  if (S && (!b->rows || !b->len || !b->table)) return fail(IFR_EINVAL, "paged batch: rows, len or table is null");
  int64_t M = 0;
  for (int s = 0; s < S; ++s) {
    if (b->rows[s] == 0) continue;
    if (b->rows[s] < 0 || b->len[s] < b->rows[s] || b->len[s] > kMaxTokens)
      return fail(IFR_EINVAL, "sequence %d: %d new rows of %d tokens", s, b->rows[s], b->len[s]);
    const int np = (b->len[s] + kPgTok - 1) / kPgTok;
    if (np > b->table_stride) return fail(IFR_EINVAL, "sequence %d: %d pages, table rows of %d", s, np, b->table_stride);
    for (int i = 0; i < np; ++i) {
      const int pg = b->table[(size_t)s * b->table_stride + i];
      if (pg < 0 || pg >= c.n_pages) return fail(IFR_EINVAL, "sequence %d: page %d is %d of %d", s, i, pg, c.n_pages);
    }
    if (b->prefix && b->prefix[s] < 0) return fail(IFR_EINVAL, "sequence %d: prefix %d", s, b->prefix[s]);
    M += b->rows[s];
    if (M > kMaxRows || M * G > kMaxTokens) return fail(IFR_EINVAL, "more than %lld rows", (long long)kMaxRows);
  }

  std::vector<ifrk::PagedRow> rows((size_t)M);
  std::vector<ifrk::PagedRun> runs;
  std::vector<int32_t> table;
  std::vector<Tile> tiles;
  std::vector<int> row0(S), tab(S);
  std::vector<int> written;
  int max_pos = -1;
  int64_t m = 0;
  for (int s = 0; s < S; ++s) {
    const int n = b->len[s], r = b->rows[s];
    row0[s] = (int)m;
    tab[s] = (int)table.size();
    if (r == 0) continue;
    if ((int64_t)table.size() + n / kPgTok + 1 > kMaxTokens) return fail(IFR_EINVAL, "page tables too long");
    const int32_t* t = b->table + (size_t)s * b->table_stride;
    table.insert(table.end(), t, t + (n + kPgTok - 1) / kPgTok);
    const int prefix = b->prefix ? b->prefix[s] : 0;
    for (int i = 0; i < r; ++i) {
      const int pos = n - r + i;
      rows[(size_t)(m + i)] = {b->first ? std::max(b->first[m + i], 0) : 0, std::min(std::max(pos + 1, prefix), n), pos, s};
    }
    max_pos = std::max(max_pos, n - 1);
    for (int pos = n - r; pos < n;) {
      const int t0 = pos % kPgTok, k = std::min(kPgTok - t0, n - pos), pg = t[pos / kPgTok];
      written.push_back(pg);
      runs.push_back({pg, t0, k, (int)(m + pos - (n - r)), pos, {0, 0, 0}});
      pos += k;
    }
    m += r;
  }
  std::sort(written.begin(), written.end());
  const bool appendable = std::adjacent_find(written.begin(), written.end()) == written.end();
  // The pages that columns [c0, c0 + n) of sequence s look at.
  const auto tile_of = [&](int kind, int s, int64_t c0, int n) {
    int lo = 0x7FFFFFFF, hi = 0;
    for (int64_t i = c0 / G; i <= (c0 + n - 1) / G; ++i) {
      const ifrk::PagedRow& x = rows[(size_t)(row0[s] + i)];
      if (x.lo >= x.hi) continue;
      lo = std::min(lo, x.lo);
      hi = std::max(hi, x.hi);
    }
    Tile t{kind, s, (int)c0, n, 0, 0};
    if (lo < hi) {
      t.p0 = lo / kPgTok;
      t.p1 = (hi + kPgTok - 1) / kPgTok;
    }
    return t;
  };
  const auto cut = [&](int kind, int s, std::vector<Tile>& to) {
    const int64_t n = (int64_t)b->rows[s] * G;
    for (int64_t c0 = 0; c0 < n; c0 += kWidth[kind])
      to.push_back(tile_of(kind, s, c0, (int)std::min<int64_t>(kWidth[kind], n - c0)));
  };
  std::vector<Tile> wide;
  int64_t wide_pages = 0;
  for (int s = 0; s < S; ++s)
    if ((int64_t)b->rows[s] * G > kWidth[1]) cut(kWide, s, wide);
  for (const Tile& t : wide) wide_pages += (int64_t)(t.p1 - t.p0) * c.n_kv;
  constexpr int64_t wide_slots = (int64_t)kCUs * ifrk::kPgWideGroups;
  const bool use_wide = c.head_dim <= ifrk::kPgWideDim && wide_pages >= kWidePages &&
                        (c.format != IFR_KV_FP16 || (int64_t)wide.size() * c.n_kv >= wide_slots);
  if (use_wide) tiles = wide;
  for (int s = 0; s < S; ++s) {
    const int64_t n = (int64_t)b->rows[s] * G;
    if (n == 0 || (n > kWidth[1] && use_wide)) continue;
    cut(n <= kWidth[0] ? 0 : 1, s, tiles);
  }
  if ((int64_t)tiles.size() * c.n_kv > kMaxUnits || (int64_t)runs.size() * c.n_kv >= 4 * kMaxUnits)
    return fail(IFR_EINVAL, "%lld rows of %d kv heads are too many for one batch", (long long)M, c.n_kv);
  int64_t pages[kKinds] = {}, n_tiles[kKinds] = {}, most[kKinds] = {};
  for (const Tile& t : tiles) {
    pages[t.kind] += t.p1 - t.p0;
    most[t.kind] = std::max<int64_t>(most[t.kind], t.p1 - t.p0);
    ++n_tiles[t.kind];
  }
  if (n_tiles[1] > 0 && pages[0] * c.n_kv < kMergePages) {
    for (Tile& t : tiles)
      if (t.kind == 0) t.kind = 1;
    pages[1] += pages[0];
    most[1] = std::max(most[0], most[1]);
    n_tiles[1] += n_tiles[0];
    pages[0] = most[0] = n_tiles[0] = 0;
  }
  const int64_t eight = kCUs * ifrk::paged_narrow_waves(c.format, c.head_dim, 2) / 2;  // workgroups at once
  if (c.head_dim == 128 && n_tiles[1] * c.n_kv <= eight &&
      ((double)most[1] * eight <= kEven * (double)pages[1] * c.n_kv ||
       (most[1] > 4 * kWhole && most[1] <= 8 * kWhole))) {
    for (Tile& t : tiles)
      if (t.kind == 1) t.kind = kEight;
    std::swap(pages[1], pages[kEight]);
    std::swap(most[1], most[kEight]);
    std::swap(n_tiles[1], n_tiles[kEight]);
  }
  // Pages of a unit: the fewest for which the batch's units all run at once,
  // so that no CU waits for a last round of few; with more tiles than that, the
  // share of a workgroup.
  int wants[kKinds], grains[kKinds];
  for (int k = 0; k < kKinds; ++k) {
    const int64_t slots = k == kWide ? wide_slots
                                     : kCUs * ifrk::paged_narrow_waves(c.format, c.head_dim, kTiles[k]) * 4 / kWaves[k];
    const int g = grains[k] = k == kWide ? kWideGrain : kWaves[k], least = k == kWide ? kWideMin : kWaves[k];
    const auto grain = [&](int64_t n) { return (int)std::max<int64_t>(least, (n + g - 1) / g * g); };
    const int64_t share = (pages[k] * c.n_kv + slots - 1) / slots;
    int lo = grain(share), hi = std::max(lo, grain(most[k]));
    if (n_tiles[k] * c.n_kv <= slots)
      while (lo < hi) {
        const int mid = lo + (hi - lo) / g / 2 * g;
        int64_t units = 0;
        for (const Tile& t : tiles)
          if (t.kind == k) units += std::max(1, (t.p1 - t.p0 + mid - 1) / mid);
        if (units * c.n_kv <= slots) hi = mid;
        else lo = mid + g;
      }
    // A causal prompt's tiles differ in length up to its own.  Where they all run
    // at once unsplit, those of more than three quarters of the longest are split
    // (4000 rows over 4-bit pages, 16/8 heads of 128, 129.9 -> 113.0 us).
    if (k == kWide && lo >= most[k] && 5 * share <= 3 * most[k]) lo = grain(most[k] * 3 / 4);
    wants[k] = lo;
  }
  std::vector<ifrk::PagedUnit> units[kKinds];
  std::vector<ifrk::PagedJoin> joins;
  int64_t cols = 0;
  for (const Tile& t : tiles) {
    const int want = wants[t.kind], np = t.p1 - t.p0;
    const int cuts = t.kind != kWide && np <= kWhole * grains[t.kind] ? 1 : std::max(1, (np + want - 1) / want);
    const int g = grains[t.kind], step = cuts == 1 ? std::max(np, 1) : ((np + cuts - 1) / cuts + g - 1) / g * g;
    const int ns = std::max(1, (np + step - 1) / step);
    // (heads inside splits: with 8 kv heads a head's units run on one XCD)
    const int64_t base = cols;
    for (int s = 0; s < ns; ++s)
      for (int h = 0; h < c.n_kv; ++h) {
        const int p0 = t.p0 + s * step, p1 = std::min(t.p1, p0 + step);
        const int64_t part = base + ((int64_t)h * ns + s) * t.ncol;
        units[t.kind].push_back({row0[t.seq], h, t.col0, t.ncol, tab[t.seq], p0, p1, ns == 1 ? -1 : (int)part});
      }
    if (ns > 1) {
      cols += (int64_t)c.n_kv * ns * t.ncol;
      if (cols > kMaxTokens) return fail(IFR_EINVAL, "too many partial columns");
      for (int h = 0; h < c.n_kv; ++h)
        for (int i = 0, n = 1024 / c.head_dim; i < t.ncol; i += n)
          joins.push_back({row0[t.seq], h, t.col0 + i, std::min(n, t.ncol - i),
                           (int)(base + (int64_t)h * ns * t.ncol) + i, t.ncol, ns, 0});
    }
  }
  // the longest first, for short ones to fill the end
  for (auto& u : units)
    std::stable_sort(u.begin(), u.end(),
                     [](const ifrk::PagedUnit& x, const ifrk::PagedUnit& y) { return x.p1 - x.p0 > y.p1 - y.p0; });
  // Of wide units a CU takes one of the first 256 and one of the next: these in
  // rising order put a short one beside a long one (8000 rows capped, in four
  // documents, 175 -> 166 us; 2 x 1000 on 2777 63.5 -> 60.9).  Eight at a time,
  // the heads' XCDs as they were.
  if (auto& u = units[kWide]; u.size() > (size_t)kCUs) {
    const size_t n = std::min<size_t>(u.size() - kCUs, kCUs) / 8;
    for (size_t i = 0; i < n / 2; ++i)
      std::swap_ranges(u.begin() + kCUs + 8 * i, u.begin() + kCUs + 8 * (i + 1), u.begin() + kCUs + 8 * (n - 1 - i));
  }
  size_t at = 0;
  auto room = [&](size_t bytes) {
    const size_t o = at;
    at = (at + bytes + 255) & ~(size_t)255;
    return o;
  };
  const size_t o_rows = room(rows.size() * sizeof(rows[0])), o_runs = room(runs.size() * sizeof(runs[0]));
  size_t o_units[kKinds];
  for (int k = 0; k < kKinds; ++k) o_units[k] = room(units[k].size() * sizeof(ifrk::PagedUnit));
  const size_t o_joins = room(joins.size() * sizeof(ifrk::PagedJoin)), o_table = room(table.size() * 4);
  p->set = false;
  if (int r = grow(p, at, cols)) return r;
  if (p->copying) PGCHK(hipEventSynchronize(p->copied));
  p->copying = false;
  auto put = [&](size_t o, const void* src, size_t n) {
    if (n) std::memcpy(p->stage + o, src, n);
  };
  put(o_rows, rows.data(), rows.size() * sizeof(rows[0]));
  put(o_runs, runs.data(), runs.size() * sizeof(runs[0]));
  for (int k = 0; k < kKinds; ++k) put(o_units[k], units[k].data(), units[k].size() * sizeof(ifrk::PagedUnit));
  put(o_joins, joins.data(), joins.size() * sizeof(ifrk::PagedJoin));
  put(o_table, table.data(), table.size() * 4);
  if (at) {
    PGCHK(hipMemcpyAsync(p->meta, p->stage, at, hipMemcpyHostToDevice, p->st));
    PGCHK(hipEventRecord(p->copied, p->st));
    p->copying = true;
  }
  p->o_rows = o_rows;
  p->o_runs = o_runs;
  p->o_joins = o_joins;
  p->o_table = o_table;
  p->n_runs = (int)runs.size();
  for (int k = 0; k < kKinds; ++k) {
    p->o_units[k] = o_units[k];
    p->n_units[k] = (int)units[k].size();
  }
  p->n_joins = (int)joins.size();
  p->part_cols = cols;
  p->M = (int)M;
  p->max_pos = max_pos;
  p->appendable = appendable;
  p->set = true;
  return IFR_OK;
}

// What every call on a batch needs: a set plan, a pool; notes a capture.
int begin(ifr_paged* p, const void* pool) {
  if (!p) return fail(IFR_EINVAL, "paged plan is null");
  if (!p->set) return fail(IFR_ESTATE, "ifr_paged_set has not set a batch");
  if (!pool || !aligned(pool, 16)) return fail(IFR_EINVAL, "pool: null, or not on 16 bytes");
  return IFR_OK;
}

int note_capture(ifr_paged* p) {
  hipStreamCaptureStatus cs = hipStreamCaptureStatusNone;
  PGCHK(hipStreamIsCapturing(p->st, &cs));
  if (cs != hipStreamCaptureStatusNone) p->frozen = true;
  return IFR_OK;
}

size_t pool_bytes(const ifr_paged_cfg& c) {
  return ifrk::paged_page(c.format, c.head_dim, c.n_kv) * (size_t)c.n_pages;
}

ifrk::PagedPool pool_of(const ifr_paged* p, const void* pool) {
  return {static_cast<uint8_t*>(const_cast<void*>(pool)), p->cfg.format, p->cfg.n_kv, p->cfg.head_dim, p->cfg.n_heads};
}

// Rows of `width` elements of `size` bytes: not null, on 16 bytes, wide enough.
int rows_ok(const char* name, const void* d, int64_t stride, int64_t width, int size) {
  if (!d) return fail(IFR_EINVAL, "%s is null", name);
  if (!aligned(d, 16) || stride < width || stride * size % 16 != 0 || stride > kMaxStride)
    return fail(IFR_EINVAL, "%s: rows of %lld elements need 16-byte alignment and a stride that keeps it (stride %lld)",
                name, (long long)width, (long long)stride);
  return IFR_OK;
}

int cfg_ok(const ifr_paged_cfg* c) {
  if (!c) return fail(IFR_EINVAL, "paged cfg is null");
  if (c->format < IFR_KV_FP16 || c->format > IFR_KV_INT4) return fail(IFR_EINVAL, "cache format %d", c->format);
  if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
    return fail(IFR_EDECLINE, "head_dim %d: 64, 128 or 256", c->head_dim);
  if (c->n_kv <= 0 || c->n_heads <= 0 || c->n_heads % c->n_kv != 0 || c->n_heads > 65536)
    return fail(IFR_EINVAL, "%d heads over %d kv heads", c->n_heads, c->n_kv);
  if (c->n_pages <= 0) return fail(IFR_EINVAL, "n_pages=%d", c->n_pages);
  return IFR_OK;
}

}  // namespace

extern "C" {

size_t ifr_paged_bytes(const ifr_paged_cfg* c) { return cfg_ok(c) == IFR_OK ? pool_bytes(*c) : 0; }

int ifr_paged_create(ifr_ctx* ctx, const ifr_paged_cfg* cfg, ifr_paged** out) {
  if (!out) return fail(IFR_EINVAL, "out is null");
  *out = nullptr;
  if (!ctx) return fail(IFR_EINVAL, "ctx null");
  if (int r = cfg_ok(cfg)) return r;
  auto* p = new (std::nothrow) ifr_paged();
  if (!p) return fail(IFR_ENOMEM, "paged plan");
  p->ctx = ctx;
  p->device = ifrh::ctx_device(ctx);
  p->st = static_cast<hipStream_t>(ifr_ctx_stream(ctx));
  p->cfg = *cfg;
  OnDevice od(p->device);
  if (hipEventCreateWithFlags(&p->copied, hipEventDisableTiming) != hipSuccess) {
    delete p;
    return fail(IFR_EDEVICE, "hipEventCreate");
  }
  *out = p;
  return IFR_OK;
}

int ifr_paged_destroy(ifr_paged* p) {
  if (!p) return IFR_OK;
  OnDevice od(p->device);
  (void)hipStreamSynchronize(p->st);
  if (p->meta) hipFree(p->meta);
  if (p->part) hipFree(p->part);
  if (p->stage) hipHostFree(p->stage);
  if (p->copied) hipEventDestroy(p->copied);
  delete p;
  return IFR_OK;
}

int ifr_paged_set(ifr_paged* p, const ifr_paged_batch* b) {
  if (!p || !b) return fail(IFR_EINVAL, "null arg");
  OnDevice od(p->device);
  hipStreamCaptureStatus cs = hipStreamCaptureStatusNone;
  PGCHK(hipStreamIsCapturing(p->st, &cs));
  if (cs != hipStreamCaptureStatusNone) return fail(IFR_ESTATE, "ifr_paged_set inside a stream capture");
  if (p->frozen) return fail(IFR_ESTATE, "the plan's calls were captured into a graph: make another plan");
  try {
    return set_batch(p, b);
  } catch (const std::exception& e) {
    return fail(IFR_ENOMEM, "paged plan: %s", e.what());
  }
}

int ifr_paged_append(ifr_paged* p, void* pool_d, const ifr_paged_rows* r) {
  if (int e = begin(p, pool_d)) return e;
  if (!r) return fail(IFR_EINVAL, "rows are null");
  const ifr_paged_cfg& c = p->cfg;
  if (!p->appendable) return fail(IFR_EINVAL, "two runs of the batch write one page");
  if (r->rotary < 0 || r->rotary > c.head_dim || r->rotary % 16 != 0)
    return fail(IFR_EINVAL, "rotary %d: a multiple of 16 up to the head's %d dims", r->rotary, c.head_dim);
  if (p->M == 0) return IFR_OK;
  const int64_t kw = (int64_t)c.n_kv * c.head_dim, qw = (int64_t)c.n_heads * c.head_dim;
  if (int e = rows_ok("k_d", r->k_d, r->k_stride, kw, 2)) return e;
  if (int e = rows_ok("v_d", r->v_d, r->v_stride, kw, 2)) return e;
  if (!r->q_d != !r->q_out_d) return fail(IFR_EINVAL, "q_d and q_out_d go together");
  if (r->rotary && (!r->cos_d || !r->sin_d || !aligned(r->cos_d, 16) || !aligned(r->sin_d, 16)))
    return fail(IFR_EINVAL, "rotary %d: its tables are null or not on 16 bytes", r->rotary);
  if (r->rotary && p->max_pos >= r->max_pos)
    return fail(IFR_EINVAL, "position %d, tables of %d positions", p->max_pos, r->max_pos);
  const int64_t pb = (int64_t)pool_bytes(c);
  if (overlap(pool_d, pb, pb, r->k_d, pb, (p->M - 1) * r->k_stride * 2 + kw * 2, 1) ||
      overlap(pool_d, pb, pb, r->v_d, pb, (p->M - 1) * r->v_stride * 2 + kw * 2, 1))
    return fail(IFR_EINVAL, "k_d or v_d inside the pool");
  if (r->q_d) {
    if (int e = rows_ok("q_d", r->q_d, r->q_stride, qw, 2)) return e;
    if (int e = rows_ok("q_out_d", r->q_out_d, r->q_out_stride, qw, 2)) return e;
    const bool in_place = r->q_d == r->q_out_d && r->q_stride == r->q_out_stride;
    if (!in_place && overlap(r->q_out_d, r->q_out_stride * 2, qw * 2, r->q_d, r->q_stride * 2, qw * 2, p->M))
      return fail(IFR_EINVAL, "q_out_d overlaps q_d and is not q_d itself");
    if (overlap(r->q_out_d, r->q_out_stride * 2, qw * 2, r->k_d, r->k_stride * 2, kw * 2, p->M) ||
        overlap(r->q_out_d, r->q_out_stride * 2, qw * 2, r->v_d, r->v_stride * 2, kw * 2, p->M) ||
        overlap(pool_d, pb, pb, r->q_out_d, pb, (p->M - 1) * r->q_out_stride * 2 + qw * 2, 1))
      return fail(IFR_EINVAL, "q_out_d overlaps k_d, v_d or the pool");
    const int64_t tb = (int64_t)r->max_pos * (r->rotary / 2) * 4, ob = (p->M - 1) * r->q_out_stride * 2 + qw * 2;
    if (r->rotary && (overlap(r->q_out_d, ob, ob, r->cos_d, tb, tb, 1) || overlap(r->q_out_d, ob, ob, r->sin_d, tb, tb, 1)))
      return fail(IFR_EINVAL, "q_out_d overlaps the rotation's tables");
  }
  OnDevice od(p->device);
  if (int e = note_capture(p)) return e;
  ifrk::PagedAppendArgs a{};
  a.runs = reinterpret_cast<const ifrk::PagedRun*>(p->meta + p->o_runs);
  a.n_runs = p->n_runs;
  a.rows = reinterpret_cast<const ifrk::PagedRow*>(p->meta + p->o_rows);
  a.M = p->M;
  a.r = *r;
  PGCHK(ifrk::launch_paged_append(a, pool_of(p, pool_d), p->st));
  return IFR_OK;
}

int ifr_paged_read(ifr_paged* p, const void* pool_d, uint16_t* k_d, uint16_t* v_d) {
  if (int e = begin(p, pool_d)) return e;
  if (p->M == 0) return IFR_OK;
  const ifr_paged_cfg& c = p->cfg;
  const int64_t kw = (int64_t)c.n_kv * c.head_dim, pb = (int64_t)pool_bytes(c), ob = kw * 2 * p->M;
  if (int e = rows_ok("k_d", k_d, kw, kw, 2)) return e;
  if (int e = rows_ok("v_d", v_d, kw, kw, 2)) return e;
  if (overlap(k_d, ob, ob, v_d, ob, ob, 1) || overlap(pool_d, pb, pb, k_d, pb, ob, 1) ||
      overlap(pool_d, pb, pb, v_d, pb, ob, 1))
    return fail(IFR_EINVAL, "k_d, v_d and the pool overlap");
  OnDevice od(p->device);
  if (int e = note_capture(p)) return e;
  PGCHK(ifrk::launch_paged_read(reinterpret_cast<const ifrk::PagedRun*>(p->meta + p->o_runs), p->n_runs, k_d, v_d,
                                pool_of(p, pool_d), p->st));
  return IFR_OK;
}

int ifr_paged_attention(ifr_paged* p, const void* pool_d, const ifr_paged_query* q) {
  if (int e = begin(p, pool_d)) return e;
  if (!q) return fail(IFR_EINVAL, "query is null");
  const ifr_paged_cfg& c = p->cfg;
  if (!(q->scale >= 0.0f && q->scale <= kMaxFactor)) return fail(IFR_EINVAL, "scale %g", q->scale);
  const float scale = q->scale > 0.0f ? q->scale : 1.0f / std::sqrt((float)c.head_dim);
  if (!(q->softcap >= 0.0f && q->softcap <= kMaxFactor) || (q->softcap > 0.0f && !(scale / q->softcap <= kMaxFactor)))
    return fail(IFR_EINVAL, "softcap %g", q->softcap);
  if (q->out_f32 != 0 && q->out_f32 != 1) return fail(IFR_EINVAL, "out_f32 %d", q->out_f32);
  if (p->M == 0) return IFR_OK;
  const int64_t w = (int64_t)c.n_heads * c.head_dim, pb = (int64_t)pool_bytes(c);
  const int os = q->out_f32 ? 4 : 2;
  if (int e = rows_ok("q_d", q->q_d, q->q_stride, w, 2)) return e;
  if (int e = rows_ok("out_d", q->out_d, q->out_stride, w, os)) return e;
  if (overlap(q->out_d, q->out_stride * os, w * os, q->q_d, q->q_stride * 2, w * 2, p->M) ||
      overlap(pool_d, pb, pb, q->out_d, pb, (p->M - 1) * q->out_stride * os + w * os, 1))
    return fail(IFR_EINVAL, "out_d overlaps q_d or the pool");
  if (const int64_t ob = (p->M - 1) * q->out_stride * os + w * os;
      q->slopes_d && overlap(q->out_d, ob, ob, q->slopes_d, 4 * c.n_heads, 4 * c.n_heads, 1))
    return fail(IFR_EINVAL, "out_d overlaps the slopes");
  OnDevice od(p->device);
  if (int e = note_capture(p)) return e;
  ifrk::PagedAttnArgs a{};
  a.rows = reinterpret_cast<const ifrk::PagedRow*>(p->meta + p->o_rows);
  a.table = reinterpret_cast<const int32_t*>(p->meta + p->o_table);
  a.q = q->q_d;
  a.q_stride = q->q_stride;
  a.out = q->out_d;
  a.out_stride = q->out_stride;
  a.out_f32 = q->out_f32;
  a.scale = scale;
  a.cap = q->softcap;
  a.slopes = q->slopes_d;
  a.part_o = p->part;
  a.part_ml = p->part ? p->part + p->part_cols * c.head_dim : nullptr;
  const ifrk::PagedPool kv = pool_of(p, pool_d);
  for (int k = 0; k < kKinds; ++k) {
    a.units = reinterpret_cast<const ifrk::PagedUnit*>(p->meta + p->o_units[k]);
    a.n_units = p->n_units[k];
    PGCHK(k == kWide ? ifrk::launch_paged_wide(a, kv, p->st)
                     : ifrk::launch_paged_narrow(a, kv, kTiles[k], kWaves[k], p->st));
  }
  PGCHK(ifrk::launch_paged_join(reinterpret_cast<const ifrk::PagedJoin*>(p->meta + p->o_joins), p->n_joins, a, kv,
                                p->st));
  return IFR_OK;
}

}  // extern "C"
