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
  if (qr.block > 0) v.hi = (int)min((long long)s.len, ((long long)p / qr.block + 1) * qr.block);
  if (p < 0) v.hi = 0;
  v.lo = qr.window > 0 ? max(v.hi - qr.window, 0) : 0;
  v.sink = min(qr.sink, v.lo);
  return v;
}

// Page of the keys [j * page_size, ...) of sequence b, unchecked.
__device__ __forceinline__ int page_id(const Keys& ky, const Span& s, int b, int j) {
  return ky.cross ? s.state : __ldg(ky.table + b * ky.table_stride + j);
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

// Many rows to a K/V head (paged_tile.cu); few (paged_rows.cu).  `splits`: runs
// of keys whose partial rows the workspace holds for `join` (1: none).
namespace tile {
int splits(const Shape& sh);
int launch(const Keys& ky, const Queries& qr, const Shape& sh, void* workspace, cudaStream_t st);
}  // namespace tile
namespace rows {
int splits(const Shape& sh);
int launch(const Keys& ky, const Queries& qr, const Shape& sh, void* workspace, cudaStream_t st);
}  // namespace rows
int join(const Keys& ky, const Queries& qr, const float* part_o, const float* part_l, int splits, cudaStream_t st);

}  // namespace paged
}  // namespace wfk
