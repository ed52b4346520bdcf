// What the paged-cache kernels share: where a position of a sequence lies in
// the pool of pages, which sequence a packed row belongs to, and which keys a
// query sees.  Everything the device reads from the caller's integer tensors
// (page ids, offsets, lengths) is clamped or checked here before it becomes an
// address: a bad page id raises the status word and counts as absent.
#pragma once

#include <cstdint>

#include "../../include/wfk.h"
#include "wfk_status.cuh"

namespace wfk {
namespace paged {

constexpr int HD = 128;  // head dim of every attention kernel of this library

// A batch of sequences: packed rows [cu[b], cu[b + 1]) are the last rows of
// sequence b, whose total length is lens[b].
struct Batch {
  const int32_t* table;  // [seqs, max_pages] page ids
  const int32_t* cu;     // [seqs + 1]
  const int32_t* lens;   // [seqs]
  int64_t table_stride;
  int seqs, max_pages, rows;
};

struct Seq {
  int first, n;  // packed rows
};

__device__ __forceinline__ Seq seq_of(const Batch& bt, int b) {
  Seq s;
  s.first = min(max(__ldg(bt.cu + b), 0), bt.rows);
  s.n = min(max(__ldg(bt.cu + b + 1), s.first), bt.rows) - s.first;
  return s;
}

// The sequence of packed row r: the last b with cu[b] <= r; -1 behind the last sequence.
__device__ __forceinline__ int seq_of_row(const Batch& bt, int r) {
  if (bt.seqs == 0 || r >= __ldg(bt.cu + bt.seqs) || r < __ldg(bt.cu)) return -1;
  int lo = 0, hi = bt.seqs;  // cu[lo] <= r < cu[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(bt.cu + mid) <= r)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

}  // namespace paged
}  // namespace wfk
