// The paged K/V cache's write and read-back (HBM-bound).
//
// Write: the row x[0..127] of one token and head becomes, for 8-bit pages,
//     a     = max(max|x|, 2^-100)          scale = a / Q   (Q = 448 e4m3, 127 s8)
//     code  = the e4m3 value or integer nearest to x * Q / a, ties to even
// and is copied for bf16 pages.  A row that holds a NaN or an infinity gets
// scale NaN and codes 0, so it reads back as NaN and reaches the attention as
// NaN through its scale, whatever the codes are.
//
// Exact codes from one multiply: y = x * RN(Q / a) is within 2^-23 (relative)
// of x * Q / a.  x and a are bf16 (8-bit significands X, A), so x * Q / a =
// (X / A) * Q up to a power of two, and a rounding midpoint is t * 2^j with t
// of at most 5 bits (e4m3) or 8 bits (integers below 128 and a half).  If
// they differ, |X * Q / A - t * 2^j| is at least 2^j / A, i.e. 1 / (A t) >=
// 2^-16 relative.  Rounding y to 18 significant bits moves it by at most
// 2^-18: a y within 2^-23 of a midpoint lands on it, any other stays on its
// side, so the code is the one of the exact quotient.
//
// Read: bf16(code * scale), one rounding.
//
// Half a warp holds a row (8 elements a lane): lanes 0-15 take K, 16-31 V.  A
// block takes 16 packed rows and 4 heads at a time, all their loads in flight
// before the first use, then the next 4 heads, loaded under the stores of the
// last: the rows' slots are looked up once (28080 rows of 40 heads, e4m3: 320 us
// with a block to every 4 heads).  The maxima of a half warp's 8 rows are folded
// together so that two divisions serve all of them; with two divisions and four
// shuffles a row the write took 301 us, bound by instructions.
//
// Measured: that write 194 us, 4.5 TB/s or 0.70 of the HBM copy rate; 23400
// rows of 12 heads read back in 45 us, 4.8 TB/s.
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>

#include "host_util.h"
#include "paged.cuh"
#include "quant_rows.cuh"

namespace wfk {
namespace paged {

constexpr int RUN = 16;             // packed rows of a block
constexpr int HEADS = 4;            // heads of a block
constexpr int THREADS = 256;
constexpr int STEP = THREADS / 32;  // (row, head) pairs a pass over the block covers
constexpr int NPAIR = RUN * HEADS / STEP;
constexpr int SMS = 148;  // B200

struct Pool {
  void *k, *v;
  float *ks, *vs;
  int64_t k_str[3], v_str[3];    // page, head, row, in elements
  int64_t ks_str[2], vs_str[2];  // page, head
  int64_t n_pages;
  int page_size, heads;
};
struct Rows {  // packed bf16 rows: read by the write, written by the read
  void *k, *v;
  int64_t k_str[2], v_str[2];  // row, head
};

// Slot of each of the block's rows: page id (-1: none), row in the page (-1:
// behind the last sequence), and where it lies in K and V pages (-1: nowhere)
// and their scales, without the head.
struct Slots {
  int page[RUN], row[RUN];
  int64_t at[2][RUN], scale[2][RUN];
};

__device__ __forceinline__ void find_slots(Slots& sl, const Batch& bt, const Pool& pool, int r0) {
  if (threadIdx.x < RUN) {
    const int r = r0 + threadIdx.x;
    int page = -1, row = 0;
    const int b = r < bt.rows ? seq_of_row(bt, r) : -1;
    if (b >= 0) {
      const int n_total = __ldg(bt.lens + b);
      const Seq s = seq_of(bt, b);
      const int pos = n_total - s.n + (r - s.first);
      if (pos >= 0) {
        const int j = pos / pool.page_size;
        const int id = j < bt.max_pages ? __ldg(bt.table + b * bt.table_stride + j) : -1;
        if (id >= 0 && id < pool.n_pages) {
          page = id;
          row = pos - j * pool.page_size;
        } else {
          status_raise(ST_PAGE_ID);
        }
      }
    } else {
      row = -1;  // behind the last sequence
    }
    const int t = threadIdx.x;
    sl.page[t] = page;
    sl.row[t] = row;
    sl.at[0][t] = page < 0 ? -1 : page * pool.k_str[0] + row * pool.k_str[2];
    sl.at[1][t] = page < 0 ? -1 : page * pool.v_str[0] + row * pool.v_str[2];
    sl.scale[0][t] = page * pool.ks_str[0] + row;
    sl.scale[1][t] = page * pool.vs_str[0] + row;
  }
}

// Drops the block's rows whose slot a later packed row also lands in (pages
// listed twice): the last row wins, whole.  All written pages of the batch are
// looked at once per block, `w` threads to a sequence.
__device__ __forceinline__ void drop_overwritten(Slots& sl, const Batch& bt, const Pool& pool, int r0) {
  const int ps = pool.page_size;
  int w = 1;
  while (w * 2 * bt.seqs <= THREADS) w *= 2;
  for (int b = threadIdx.x / w; b < bt.seqs; b += THREADS / w) {
    const int total = __ldg(bt.lens + b);
    const Seq s = seq_of(bt, b);
    const int base = total - s.n;  // position of the sequence's first packed row
    if (s.n == 0 || total <= 0 || s.first + s.n - 1 <= r0) continue;  // none of its rows is later than the block's first
    const int j1 = min((total - 1) / ps, bt.max_pages - 1);
    for (int j = max(base, 0) / ps + (threadIdx.x & (w - 1)); j <= j1; j += w) {
      const int id = __ldg(bt.table + b * bt.table_stride + j);
#pragma unroll
      for (int i = 0; i < RUN; ++i) {
        if (id == sl.page[i] && id >= 0) {
          const int pos = j * ps + sl.row[i];
          if (pos >= base && pos < total && s.first + (pos - base) > r0 + i) sl.at[0][i] = sl.at[1][i] = -1;
        }
      }
    }
  }
}

__device__ __forceinline__ float snap18(float y) {
  return __uint_as_float((__float_as_uint(y) + 0x20u) & ~0x3Fu);
}

// Calls fetch(buffer, h) and put(buffer, h) for h = h0, h0 + HEADS, ... below h1,
// each fetch before the put that precedes its own (two buffers by turns).
template <class Buf, class Fetch, class Look, class Put>
__device__ __forceinline__ void by_heads(int h0, int h1, Fetch fetch, Look look, Put put) {
  Buf a, b;
  fetch(a, h0);
  look();
  for (int h = h0; h < h1; h += 2 * HEADS) {
    if (h + HEADS < h1) fetch(b, h + HEADS);
    put(a, h);
    if (h + HEADS >= h1) break;
    if (h + 2 * HEADS < h1) fetch(a, h + 2 * HEADS);
    put(b, h + HEADS);
  }
}

template <int DT>
__global__ void __launch_bounds__(THREADS) write_kernel(const __grid_constant__ Batch bt,
                                                        const __grid_constant__ Pool pool,
                                                        const __grid_constant__ Rows src, int heads) {
  __shared__ Slots sl;
  const int r0 = blockIdx.x * RUN, h_lo = blockIdx.y * heads, h_hi = min(h_lo + heads, pool.heads);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = lane & 15;
  const int i0 = warp / HEADS, dh = warp % HEADS;  // row i0 + p * STEP / HEADS, head h + dh of pair p
  const bool is_v = lane >= 16;
  const __nv_bfloat16* x = static_cast<const __nv_bfloat16*>(is_v ? src.v : src.k) + c * 8;
  const int64_t* xs = is_v ? src.v_str : src.k_str;
  struct Buf {
    uint4 v[NPAIR];
  };
  auto fetch = [&](Buf& f, int h) {
    const __nv_bfloat16* at = x + (int64_t)(r0 + i0) * xs[0] + (h + dh) * xs[1];
#pragma unroll
    for (int p = 0; p < NPAIR; ++p) {
      f.v[p] = make_uint4(0, 0, 0, 0);
      if (r0 + i0 + p * (STEP / HEADS) < bt.rows && h + dh < h_hi)
        f.v[p] = __ldg(reinterpret_cast<const uint4*>(at + p * (STEP / HEADS) * xs[0]));
    }
  };
  auto look = [&]() {
    find_slots(sl, bt, pool, r0);
    __syncthreads();
    drop_overwritten(sl, bt, pool, r0);
    __syncthreads();
  };
  const int64_t hs = (is_v ? pool.v_str : pool.k_str)[1], shs = (is_v ? pool.vs_str : pool.ks_str)[1];
  float* scales = is_v ? pool.vs : pool.ks;
  constexpr float Q = DT == WF_DTYPE_E4M3 ? 448.f : 127.f;
  auto put = [&](const Buf& f, int h4) {
    const int h = h4 + dh;
    if (h >= h_hi) return;
    float inv = 0.f;  // Q / a of pair c / 2's row; 0 where it is not finite
    if constexpr (DT != WF_DTYPE_BF16) {
      // Maxima of the 8 rows over the half warp, rows and lanes folded together:
      // lane c ends with row c / 2's, so that one division serves 8 rows.
      uint32_t m[NPAIR];
#pragma unroll
      for (int p = 0; p < NPAIR; ++p) m[p] = quant::amax8_bits(f.v[p], 0u);
#pragma unroll
      for (int n = NPAIR / 2, o = 8; n > 0; n /= 2, o /= 2) {
#pragma unroll
        for (int p = 0; p < n; ++p) {
          const uint32_t give = (c & o) ? m[p] : m[p + n], keep = (c & o) ? m[p + n] : m[p];
          m[p] = quant::vmax_u16x2(keep, __shfl_xor_sync(0xffffffffu, give, o));
        }
      }
      m[0] = quant::vmax_u16x2(m[0], __shfl_xor_sync(0xffffffffu, m[0], 1));
      const uint32_t top = max(m[0] & 0xFFFFu, m[0] >> 16);
      const bool finite = top < 0x7F80u;
      const float a = fmaxf(__uint_as_float(top << 16), 0x1p-100f);
      inv = finite ? __fdiv_rn(Q, a) : 0.f;
      const int i = i0 + (c >> 1) * (STEP / HEADS);
      if (!(c & 1) && sl.at[is_v][i] >= 0)
        scales[sl.scale[is_v][i] + h * shs] = finite ? __fdiv_rn(a, Q) : __uint_as_float(0x7FC00000u);
    }
    const int64_t to = h * hs + c * 8;
#pragma unroll
    for (int p = 0; p < NPAIR; ++p) {
      const int64_t at = sl.at[is_v][i0 + p * (STEP / HEADS)];
      if constexpr (DT == WF_DTYPE_BF16) {
        if (at >= 0)
          *reinterpret_cast<uint4*>((is_v ? static_cast<__nv_bfloat16*>(pool.v) : static_cast<__nv_bfloat16*>(pool.k)) +
                                    at + to) = f.v[p];
      } else {
        const float mul = __shfl_sync(0xffffffffu, inv, 2 * p, 16);
        const uint32_t w[4] = {f.v[p].x, f.v[p].y, f.v[p].z, f.v[p].w};
        uint32_t codes[2] = {0, 0};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float y0 = snap18(__uint_as_float(w[e] << 16) * mul);
          const float y1 = snap18(__uint_as_float(w[e] & 0xFFFF0000u) * mul);
          uint32_t two;
          if constexpr (DT == WF_DTYPE_E4M3)
            two = quant::e4m3x2_hw(y0, y1);
          else
            two = (static_cast<uint32_t>(__float2int_rn(y0)) & 0xFFu) |
                  ((static_cast<uint32_t>(__float2int_rn(y1)) & 0xFFu) << 8);
          codes[e >> 1] |= two << ((e & 1) * 16);
        }
        if (mul == 0.f) codes[0] = codes[1] = 0;
        uint8_t* base = static_cast<uint8_t*>(is_v ? pool.v : pool.k);
        if (at >= 0) *reinterpret_cast<uint2*>(base + at + to) = make_uint2(codes[0], codes[1]);
      }
    }
  };
  by_heads<Buf>(h_lo, h_hi, fetch, look, put);
}

template <int DT>
__global__ void __launch_bounds__(THREADS) read_kernel(const __grid_constant__ Batch bt,
                                                       const __grid_constant__ Pool pool,
                                                       const __grid_constant__ Rows dst, int heads) {
  __shared__ Slots sl;
  const int r0 = blockIdx.x * RUN, h_lo = blockIdx.y * heads, h_hi = min(h_lo + heads, pool.heads);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = lane & 15;
  const int i0 = warp / HEADS, dh = warp % HEADS;
  const bool is_v = lane >= 16;
  find_slots(sl, bt, pool, r0);
  __syncthreads();
  const int64_t hs = (is_v ? pool.v_str : pool.k_str)[1], shs = (is_v ? pool.vs_str : pool.ks_str)[1];
  const float* scales = is_v ? pool.vs : pool.ks;
  constexpr bool WIDE = DT == WF_DTYPE_BF16;
  struct Buf {
    uint4 w[WIDE ? NPAIR : 1];
    uint2 q[WIDE ? 1 : NPAIR];
    float s;  // scale of pair c / 2's row
  };
  auto fetch = [&](Buf& f, int h4) {
    const int h = h4 + dh;
    if constexpr (!WIDE) {
      const int i = i0 + (c >> 1) * (STEP / HEADS);
      f.s = sl.at[is_v][i] >= 0 && h < h_hi ? __ldg(scales + sl.scale[is_v][i] + h * shs) : 0.f;
    }
    const int64_t from = h * hs + c * 8;
#pragma unroll
    for (int p = 0; p < NPAIR; ++p) {
      const int64_t at = sl.at[is_v][i0 + p * (STEP / HEADS)] + from;
      const bool live = at >= from && h < h_hi;
      if constexpr (WIDE) {
        f.w[p] = make_uint4(0, 0, 0, 0);
        if (live)
          f.w[p] = __ldg(reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(is_v ? pool.v : pool.k) + at));
      } else {
        f.q[p] = make_uint2(0, 0);
        if (live) f.q[p] = __ldg(reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(is_v ? pool.v : pool.k) + at));
      }
    }
  };
  __nv_bfloat16* y = static_cast<__nv_bfloat16*>(is_v ? dst.v : dst.k) + c * 8;
  const int64_t* ys = is_v ? dst.v_str : dst.k_str;
  auto put = [&](const Buf& f, int h4) {
    const int h = h4 + dh;
    if (h >= h_hi) return;
#pragma unroll
    for (int p = 0; p < NPAIR; ++p) {
      const int i = i0 + p * (STEP / HEADS);
      const float scale = WIDE ? 1.f : __shfl_sync(0xffffffffu, f.s, 2 * p, 16);
      if (sl.row[i] < 0) continue;  // behind the last sequence: left as it was
      uint4 o;
      if constexpr (WIDE) {
        o = f.w[p];
      } else if constexpr (DT == WF_DTYPE_E4M3) {
        o = quant::dequant8(f.q[p], scale);
      } else {
        uint32_t u[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t two = (e < 2 ? f.q[p].x : f.q[p].y) >> ((e & 1) * 16);
          u[e] = pack_bf16x2(static_cast<float>(static_cast<int8_t>(two & 0xFF)) * scale,
                             static_cast<float>(static_cast<int8_t>((two >> 8) & 0xFF)) * scale);
        }
        o = make_uint4(u[0], u[1], u[2], u[3]);
      }
      *reinterpret_cast<uint4*>(y + (int64_t)(r0 + i) * ys[0] + h * ys[1]) = o;
    }
  };
  by_heads<Buf>(h_lo, h_hi, fetch, [] {}, put);
}

// ------------------------------------------------------------------- host
int check_pages(const char* who, const wf_kv_pages* p) {
  if (!p) return fail(WF_ERR_INVALID_ARG, "%s: null pages", who);
  const bool bf = p->dtype == WF_DTYPE_BF16;
  if (!bf && p->dtype != WF_DTYPE_E4M3 && p->dtype != WF_DTYPE_S8)
    return fail(WF_ERR_UNSUPPORTED, "%s: page dtype %d unsupported (bf16, e4m3 or s8)", who, p->dtype);
  if (p->head_dim != HD) return fail(WF_ERR_UNSUPPORTED, "%s: head_dim %d unsupported (only 128)", who, p->head_dim);
  if (p->n_pages < 1 || p->n_pages > INT_MAX || p->page_size < 1 || p->heads < 1 || p->heads > 65535)
    return fail(WF_ERR_INVALID_ARG, "%s: bad pool sizes (%lld pages of %d rows, %d heads)", who,
                (long long)p->n_pages, p->page_size, p->heads);
  if (!p->k || !p->v || !aligned16(p->k) || !aligned16(p->v))
    return fail(WF_ERR_INVALID_ARG, "%s: K/V pages null or not 16-byte aligned", who);
  const int unit = bf ? 8 : 16;
  for (const int64_t* st : {p->k_stride, p->v_stride})
    for (int i = 0; i < 3; ++i)
      if (st[i] <= 0 || st[i] % unit)
        return fail(WF_ERR_INVALID_ARG, "%s: page strides must be positive multiples of 16 bytes", who);
  if (bf ? (p->k_scale || p->v_scale) : (!p->k_scale || !p->v_scale))
    return fail(WF_ERR_INVALID_ARG, "%s: 8-bit pages need k_scale and v_scale, bf16 pages take none", who);
  if (!bf)
    for (const int64_t* st : {p->k_scale_stride, p->v_scale_stride})
      for (int i = 0; i < 2; ++i)
        if (st[i] <= 0) return fail(WF_ERR_INVALID_ARG, "%s: scale strides must be positive", who);
  return WF_OK;
}

int check_batch(const char* who, const wf_kv_batch* b, int page_size) {
  if (!b || b->seqs < 0 || b->seqs > (1 << 24) || b->max_pages < 1 || b->rows < 0 || b->rows > INT_MAX - 1024)
    return fail(WF_ERR_INVALID_ARG, "%s: bad batch sizes", who);
  if ((int64_t)b->max_pages * page_size > INT_MAX - 4096)
    return fail(WF_ERR_INVALID_ARG, "%s: %d pages of %d rows pass 2^31 positions", who, b->max_pages, page_size);
  if (b->seqs > 0 && (!b->table || !b->cu || !b->lens || b->table_stride < 0))
    return fail(WF_ERR_INVALID_ARG, "%s: null page table, offsets or lengths", who);
  return WF_OK;
}

static Batch make_batch(const wf_kv_batch* b) {
  return Batch{b->table, b->cu, b->lens, b->table_stride, b->seqs, b->max_pages, (int)b->rows};
}

static Pool make_pool(const wf_kv_pages* p) {
  Pool q{p->k, p->v, p->k_scale, p->v_scale, {}, {}, {}, {}, p->n_pages, p->page_size, p->heads};
  for (int i = 0; i < 3; ++i) q.k_str[i] = p->k_stride[i], q.v_str[i] = p->v_stride[i];
  for (int i = 0; i < 2; ++i) q.ks_str[i] = p->k_scale_stride[i], q.vs_str[i] = p->v_scale_stride[i];
  return q;
}

static int run(const char* who, const wf_kv_pages* pages, const wf_kv_batch* batch, void* k, void* v,
               const int64_t* ks, const int64_t* vs, void* stream, bool write) {
  int rc;
  if ((rc = check_pages(who, pages)) != WF_OK) return rc;
  if ((rc = check_batch(who, batch, pages->page_size)) != WF_OK) return rc;
  if (batch->rows == 0 || batch->seqs == 0) return WF_OK;
  if (!k || !v || !ks || !vs || !aligned16(k) || !aligned16(v))
    return fail(WF_ERR_INVALID_ARG, "%s: packed K/V null or not 16-byte aligned", who);
  for (int i = 0; i < 2; ++i)
    if (ks[i] < (write ? 0 : 1) || vs[i] < (write ? 0 : 1) || ks[i] % 8 || vs[i] % 8)
      return fail(WF_ERR_INVALID_ARG, "%s: packed strides must be multiples of 8 elements", who);
  const Batch bt = make_batch(batch);
  const Pool pool = make_pool(pages);
  const Rows rows{k, v, {ks[0], ks[1]}, {vs[0], vs[1]}};
  // Heads of a block: as many as leave the blocks that run at once, two to an SM.
  const int64_t runs = (batch->rows + RUN - 1) / RUN, groups = (pages->heads + HEADS - 1) / HEADS;
  const int heads = HEADS * (int)std::clamp<int64_t>((runs * groups + 2 * SMS - 1) / (2 * SMS), 1, groups);
  const dim3 grid((unsigned)runs, (unsigned)((pages->heads + heads - 1) / heads));
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto pick = [&](auto bf, auto e4, auto s8) {
    return pages->dtype == WF_DTYPE_BF16 ? bf : pages->dtype == WF_DTYPE_E4M3 ? e4 : s8;
  };
  auto kern = write ? pick(write_kernel<WF_DTYPE_BF16>, write_kernel<WF_DTYPE_E4M3>, write_kernel<WF_DTYPE_S8>)
                    : pick(read_kernel<WF_DTYPE_BF16>, read_kernel<WF_DTYPE_E4M3>, read_kernel<WF_DTYPE_S8>);
  kern<<<grid, THREADS, 0, st>>>(bt, pool, rows, heads);
  WFK_CUDA_TRY(cudaGetLastError());
  return WF_OK;
}

}  // namespace paged
}  // namespace wfk

extern "C" int wf_paged_kv_write(const wf_kv_pages* pages, const wf_kv_batch* batch, const void* k, const void* v,
                                 const int64_t* k_stride, const int64_t* v_stride, void* stream) {
  return wfk::paged::run("wf_paged_kv_write", pages, batch, const_cast<void*>(k), const_cast<void*>(v), k_stride,
                         v_stride, stream, true);
}

extern "C" int wf_paged_kv_read(const wf_kv_pages* pages, const wf_kv_batch* batch, void* k, void* v,
                                const int64_t* k_stride, const int64_t* v_stride, void* stream) {
  return wfk::paged::run("wf_paged_kv_read", pages, batch, k, v, k_stride, v_stride, stream, false);
}

extern "C" unsigned int wfk_status_take_paged_kv(void) { return wfk::status_take_local(); }
