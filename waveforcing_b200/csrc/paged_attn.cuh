// Shared by the kernels of paged_attn.cu and paged_tile.cu: what a launch
// attends to, which keys a row sees, and how a call is cut.
//
// A row at position p of a sequence of len keys sees the keys below hi and,
// with a window, of those only the last `window` and the first `sink`; hi and
// lo = hi - window do not fall from one row to the next, so the keys a run of
// rows sees together are [0, sink of the last) and [lo of the first, hi of the
// last).  Cross attention is the same sum over one page, the entry's states.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <climits>

#include "host_util.h"
#include "paged.cuh"
#include "sm100.cuh"

namespace wfk {
namespace paged {

// Where the K/V rows of every sequence lie.
struct Keys {
  const void *k, *v;
  const float *ks, *vs;
  int64_t k_str[3], v_str[3];    // page, head, row, in elements
  int64_t ks_str[2], vs_str[2];  // page, head
  const int32_t* table;          // page ids of sequence b; NULL: page b, or 0 of a single one
  int64_t table_stride;
  const int32_t* lens;           // by sequence, or by state (page) for cross attention; NULL: page_size
  const uint8_t* mask;           // cross attention: [state, key]; NULL: all keys
  int64_t mask_stride;
  int64_t n_pages;
  int page_size, max_pages, dtype;
  bool cross;
};

// The query rows.
struct Queries {
  const __nv_bfloat16* q;
  __nv_bfloat16* o;
  float* lse;
  int64_t q_str[3], o_str[3];  // batch entry (cross attention), row, head
  const int32_t* cu;           // NULL: Lq rows to an entry
  int seqs, rows, Lq, H, group;
  int block, window, sink;
  float scale_log2;            // softmax scale times log2(e)
};

struct Span {  // one sequence's queries and keys
  int first, n;  // packed rows
  int len;       // keys
  int pos0;      // position of the first row
  int state;     // cross attention: the page, -1 when the index is bad
};

__device__ __forceinline__ Span span_of(const Keys& ky, const Queries& qr, int b) {
  Span s;
  if (ky.cross) {
    s.first = b * qr.Lq;
    s.n = qr.Lq;
    s.state = ky.table ? __ldg(ky.table + b) : (ky.n_pages == 1 ? 0 : b);
    if (s.state < 0 || s.state >= ky.n_pages) {
      status_raise(ST_PAGE_ID);
      s.state = -1;
    }
    s.len = s.state < 0 ? 0 : ky.lens ? min(max(__ldg(ky.lens + s.state), 0), ky.page_size) : ky.page_size;
    s.pos0 = 0;
  } else {
    s.first = min(max(__ldg(qr.cu + b), 0), qr.rows);
    s.n = min(max(__ldg(qr.cu + b + 1), s.first), qr.rows) - s.first;
    const int len = max(__ldg(ky.lens + b), 0);
    s.pos0 = len - s.n;
    s.len = min(len, ky.max_pages * ky.page_size);
    if (s.len < len) status_raise(ST_PAGE_ID);
    s.state = -1;
  }
  return s;
}

struct Sees {  // keys [0, sink) and [lo, hi)
  int hi, lo, sink;
};
__device__ __forceinline__ Sees sees(const Queries& qr, const Span& s, int i) {
  const int p = s.pos0 + i;
  Sees v;
  v.hi = s.len;
  if (qr.block > 0 && p >= 0) v.hi = (int)min((long long)s.len, (p / qr.block + 1ll) * qr.block);
  if (p < 0) v.hi = 0;
  v.lo = qr.window > 0 ? max(v.hi - qr.window, 0) : 0;
  v.sink = min(qr.sink, v.lo);
  return v;
}

// Page of the keys [j * page_size, ...) of sequence b, unchecked.
__device__ __forceinline__ int page_id(const Keys& ky, const Span& s, int b, int j) {
  return ky.cross ? s.state : __ldg(ky.table + b * ky.table_stride + j);
}

// How the keys of a sequence fall into tiles of BN rows, and those into boxes (one
// TMA copy each, a multiple of the swizzle's 8 rows, in one page).  Page sizes
// that are multiples of 8 give dense tiles of BN consecutive positions, in boxes
// of the largest power of two that divides the page size (one box where the
// whole tile lies in a page).  Others leave holes: pages of at least BN rows
// give ceil(page_size / BN) tiles each, smaller ones share a tile, a page to a
// box.
struct Tiling {
  uint32_t mul, shift;              // x / ps = x * mul >> shift for 0 <= x < 2^31
  int ps, dense, tpp, boxes, rows;  // page size; tiles per page (large, not dense); boxes of a tile, their rows
  int tq, splits, even, wide;       // paged_tile.cu: tokens of a sub-tile, runs of keys, whether items are dealt
                                    // evenly, whether rows of O begin on 32-byte boundaries
};
inline Tiling tiling_of(int ps, int bn, bool dense = true) {
  Tiling t{0, 31, ps, dense && ps % 8 == 0, (ps + bn - 1) / bn, 1, bn, 0, 1, 0, 0};
  if (t.dense)
    while (ps % t.rows) t.rows /= 2;
  else if (ps < bn)
    t.rows = (ps + 7) & ~7;
  t.boxes = bn / t.rows;
  while ((1ll << (t.shift - 31)) < ps) ++t.shift;  // mul = ceil(2^shift / ps): off by less than x / 2^shift < 1 / ps
  t.mul = (uint32_t)(((1ull << t.shift) + ps - 1) / ps);
  return t;
}
__device__ __forceinline__ int page_of(const Tiling& tl, int pos) { return (int)((uint64_t)pos * tl.mul >> tl.shift); }
template <int BN>
__device__ __forceinline__ int tile_of(const Tiling& tl, int pos) {
  if (tl.dense) return pos / BN;
  const int j = page_of(tl, pos);
  return tl.ps < BN ? j / tl.boxes : j * tl.tpp + (pos - j * tl.ps) / BN;
}
struct TileAt {
  int page, row, base;  // page and row of the tile's first key, its position
};
template <int BN>
__device__ __forceinline__ TileAt tile_at(const Tiling& tl, int t) {
  TileAt a;
  if (tl.dense) {
    a.base = t * BN;
    a.page = page_of(tl, a.base);
    a.row = a.base - a.page * tl.ps;
    return a;
  }
  if (tl.ps < BN) {
    a.page = t * tl.boxes;
    a.row = 0;
  } else {
    a.page = t / tl.tpp;
    a.row = (t - a.page * tl.tpp) * BN;
  }
  a.base = a.page * tl.ps + a.row;
  return a;
}
// Tile rows whose position is below x.
template <int BN>
__device__ __forceinline__ int rows_below(const Tiling& tl, const TileAt& a, int x) {
  const int d = x - a.base;
  if (d <= 0) return 0;
  if (tl.dense) return min(d, BN);
  if (tl.ps >= BN) return min(d, min(BN, tl.ps - a.row));
  const int j = page_of(tl, d);
  return min(j, tl.boxes) * tl.rows + (j < tl.boxes ? d - j * tl.ps : 0);
}
// The tile after a (of consecutive tiles).
template <int BN>
__device__ __forceinline__ void next_tile(const Tiling& tl, TileAt& a) {
  a.base += BN;
  a.row += BN;
  if (tl.dense) {
    while (a.row >= tl.ps) a.row -= tl.ps, ++a.page;
  } else if (tl.ps < BN) {
    a.page += tl.boxes;
    a.row = 0;
    a.base = a.page * tl.ps;
  } else if (a.row >= tl.ps) {
    a.row = 0;
    ++a.page;
    a.base = a.page * tl.ps;
  }
}
// Whether the tile lies in one page and one copy of BN rows fetches it.
template <int BN>
__device__ __forceinline__ bool one_box(const Tiling& tl, const TileAt& a) {
  return tl.boxes == 1 || (tl.dense && a.row + BN <= tl.ps);
}
struct Box {
  int page, row, pos;  // page (of the sequence), row in it, position of the box's first key
};
template <int BN>
__device__ __forceinline__ Box box_at(const Tiling& tl, const TileAt& a, int i) {
  Box x{a.page, a.row, a.base};
  if (tl.dense) {
    x.pos += i * tl.rows;
    x.page = page_of(tl, x.pos);
    x.row = x.pos - x.page * tl.ps;
  } else if (tl.ps < BN) {
    x.page += i;
    x.pos += i * tl.ps;
  }
  return x;
}
// Bits [a, b) of a 32-bit word that starts at bit `at`.
__device__ __forceinline__ uint32_t bit_range(int a, int b, int at) {
  const int lo = min(max(a - at, 0), 32), hi = min(max(b - at, 0), 32);
  if (hi <= lo) return 0;
  return (0xFFFFFFFFu >> (32 - (hi - lo))) << lo;
}

// The keys that tokens [i0, i1] of a sequence see, and the list of their tiles:
// n_sink tiles from the first, then those from t_lo on.
struct Range {
  int hi, lo, sink;              // seen by some token: [0, sink) and [lo, hi)
  int hi_min, lo_max, sink_min;  // and by every one
  int n_sink, t_lo, n;
};
template <int BN>
__device__ __forceinline__ Range range_of(const Queries& qr, const Span& sp, const Tiling& tl, int i0, int i1) {
  const Sees last = sees(qr, sp, i1);
  const Sees first = sees(qr, sp, max(i0, min(-sp.pos0, i1)));  // earlier rows have no position
  Range r;
  r.hi = last.hi;
  r.lo = first.lo;
  r.sink = min(last.sink, r.hi);
  r.hi_min = i0 + sp.pos0 < 0 ? 0 : first.hi;
  r.lo_max = last.lo;
  r.sink_min = first.sink;
  r.n_sink = r.t_lo = r.n = 0;
  if (r.hi > 0) {
    r.t_lo = tile_of<BN>(tl, r.lo);
    r.n_sink = r.sink > 0 ? min(tile_of<BN>(tl, r.sink - 1) + 1, r.t_lo) : 0;
    r.n = r.n_sink + tile_of<BN>(tl, r.hi - 1) + 1 - r.t_lo;
  }
  return r;
}
__device__ __forceinline__ int nth_tile(const Range& r, int i) { return i < r.n_sink ? i : i - r.n_sink + r.t_lo; }
// Whether some token sees a key of [pos, pos + rows).
__device__ __forceinline__ bool needed(const Range& r, int pos, int rows) {
  return (pos < r.hi && pos + rows > r.lo) || pos < r.sink;
}
// Walks the tiles of a list from its i-th on.
template <int BN>
struct Walk {
  const Range& r;
  const Tiling& tl;
  int i;
  TileAt a;
  __device__ __forceinline__ Walk(const Range& r, const Tiling& tl, int i)
      : r(r), tl(tl), i(i), a(tile_at<BN>(tl, nth_tile(r, i))) {}
  __device__ __forceinline__ void next() {
    if (++i == r.n_sink)
      a = tile_at<BN>(tl, r.t_lo);
    else
      next_tile<BN>(tl, a);
  }
};
// Whether every key of a one-box tile is seen by some token.
template <int BN>
__device__ __forceinline__ bool inside(const Range& r, const TileAt& a) {
  return (a.base >= r.lo && a.base + BN <= r.hi) || a.base + BN <= r.sink;
}
__device__ __forceinline__ bool seen(const Range& r, int pos) { return (pos < r.hi && pos >= r.lo) || pos < r.sink; }

// Whether some tokens see keys that others do not, and whether of a tile.  There a V
// row of bf16 pages may hold a NaN or an infinity that its P of 0 would hand to the
// others: such elements are taken out and given to the rows that see them.
__device__ __forceinline__ bool rows_differ(const Range& r) {
  return r.hi != r.hi_min || r.lo != r.lo_max || r.sink != r.sink_min;
}
template <int BN>
__device__ __forceinline__ bool mixed(const Range& r, const TileAt& a) {
  return rows_differ(r) && !(a.base + BN <= r.hi_min && (a.base >= r.lo_max || a.base + BN <= r.sink_min));
}
__device__ __forceinline__ uint32_t fma_bf16x2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
// Bits 15 and 31: which of two bf16 are not finite.
__device__ __forceinline__ uint32_t not_finite2(uint32_t w) { return ((w & 0x7F807F80u) + 0x00800080u) & 0x80008000u; }
// The pair with what is not finite made 0.
__device__ __forceinline__ uint32_t finite2(uint32_t w) { return w & ~((not_finite2(w) >> 15) * 0xFFFFu); }

__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort, uint32_t code) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity & 1, abort, code));
}
// Maximum of two or three, NaN if one is NaN (a NaN score must reach the row's result).
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// Over 8-bit pages P is rounded to f16, which ends at 2^-24 where weights do not: with
// P of 1 for a row's largest score, keys 17 nats below it were lost, all there is where
// the largest belongs to a sink without V.  So P is 2^(s - m + bias), up to 2^15; the
// sum l holds the same power, which leaves the quotient as it was.  Maxima beyond 2^16
// take none: there m - bias would round.
__device__ __forceinline__ float p_base(float m, float bias) { return fabsf(m) < 0x1p16f ? m - bias : m; }
__device__ __forceinline__ uint32_t f16x2(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ void cp4(uint32_t dst, const void* src, bool take) {  // zero when not taken
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(take ? 4 : 0) : "memory");
}
// Power of two at or above x (> 0), between 2^-122 and 2^122 (a row scale is below 2^122).
__device__ __forceinline__ float pow2_above(float x) {
  const uint32_t e = ((__float_as_uint(x) + 0x7FFFFFu) >> 23) << 23;
  return fminf(fmaxf(__uint_as_float(e), 0x1p-122f), 0x1p122f);
}

// What the host knows of a call: the rows and lengths' upper bounds, from which
// it cuts the work (and sizes the workspace of the cut).
struct Shape {
  int64_t rows, keys;  // packed rows; keys an item of work may see
  int64_t max_new;
  int seqs, H, group, page_size, Lq;
  bool cross, kv8;
};
constexpr int SMS = 148;  // B200
inline int64_t tiles_of_keys(const Shape& sh, int bn, bool dense = true) {
  const Tiling tl = tiling_of(sh.page_size, bn, dense);
  if (tl.dense) return (sh.keys + bn - 1) / bn;
  const int64_t pages = (sh.keys + sh.page_size - 1) / sh.page_size;
  return sh.page_size >= bn ? pages * tl.tpp : (pages + tl.boxes - 1) / tl.boxes;
}

// Many rows to a K/V head (paged_tile.cu); few (paged_rows.cu).  `parts`: f32
// rows of 128 + 1 that the workspace holds (0: none).
namespace tile {
int64_t parts(const Shape& sh);
int launch(const Keys& ky, const Queries& qr, const Shape& sh, void* workspace, cudaStream_t st);
}  // namespace tile
namespace rows {
int64_t parts(const Shape& sh);
int launch(const Keys& ky, const Queries& qr, const Shape& sh, void* workspace, cudaStream_t st);
}  // namespace rows
// Tensor maps of the K and V pages: boxes of the tiling's rows of one page and
// head, and of whole tiles (64 bf16 or 128 codes wide, 128-byte swizzle).
struct PageMaps {
  CUtensorMap k, v, k_tile, v_tile;
};
int page_maps(PageMaps* m, const Keys& ky, int kv_heads, const Tiling& tl, int bn);
int join(const Keys& ky, const Queries& qr, const float* part_o, const float* part_l, int splits, cudaStream_t st);

}  // namespace paged
}  // namespace wfk
