// Attention of packed query rows over K/V rows that lie in pages, and cross
// attention to an encoder's states (each state set is one page).
//
// Simplest form: a warp per (row, head) walks the keys the row sees with a
// running maximum and sum; lane l holds dims 4l..4l+3.
#include <cuda_runtime.h>

#include <climits>
#include <cmath>

#include "host_util.h"
#include "paged.cuh"
#include "sm100.cuh"

namespace wfk {
namespace paged {

int check_pages(const char* who, const wf_kv_pages* p);
int check_batch(const char* who, const wf_kv_batch* b, int page_size);
Batch make_batch(const wf_kv_batch* b);

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

// Page of the keys [j * page_size, ...) of sequence b, -1 when its id is bad.
__device__ __forceinline__ int page_of(const Keys& ky, const Span& s, int b, int j) {
  if (ky.cross) return s.state;
  const int id = __ldg(ky.table + b * ky.table_stride + j);
  if (id >= 0 && id < ky.n_pages) return id;
  status_raise(ST_PAGE_ID);
  return -1;
}

template <int DT>
__device__ __forceinline__ float4 load4(const void* base, int64_t at) {
  if constexpr (DT == WF_DTYPE_BF16) {
    const uint2 w = __ldg(reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(base) + at));
    return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xFFFF0000u), __uint_as_float(w.y << 16),
                       __uint_as_float(w.y & 0xFFFF0000u));
  } else {
    const uint32_t w = __ldg(reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(base) + at));
    if constexpr (DT == WF_DTYPE_S8) {
      return make_float4((float)(int8_t)(w & 0xFF), (float)(int8_t)(w >> 8 & 0xFF), (float)(int8_t)(w >> 16 & 0xFF),
                         (float)(int8_t)(w >> 24));
    } else {
      uint32_t a, b;
      asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(a) : "h"(static_cast<uint16_t>(w & 0xFFFF)));
      asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(b) : "h"(static_cast<uint16_t>(w >> 16)));
      auto f = [](uint32_t h) { return __half2float(__ushort_as_half(static_cast<unsigned short>(h))); };
      return make_float4(f(a & 0xFFFF), f(a >> 16), f(b & 0xFFFF), f(b >> 16));
    }
  }
}

template <int DT>
__global__ void __launch_bounds__(128) simple_kernel(const __grid_constant__ Keys ky,
                                                     const __grid_constant__ Queries qr) {
  const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (unit >= (int64_t)qr.rows * qr.H) return;
  const int r = unit / qr.H, h = unit % qr.H, hk = h / qr.group;
  int b;
  if (ky.cross) {
    b = r / qr.Lq;
  } else {
    Batch bt{nullptr, qr.cu, nullptr, 0, qr.seqs, 0, qr.rows};
    b = seq_of_row(bt, r);
    if (b < 0) return;
  }
  const Span s = span_of(ky, qr, b);
  const int i = r - s.first;
  const int64_t row = ky.cross ? b * qr.q_str[0] + i * qr.q_str[1] : r * qr.q_str[1];
  const float4 q = load4<WF_DTYPE_BF16>(qr.q, row + h * qr.q_str[2] + lane * 4);
  const Sees se = sees(qr, s, i);
  float m = -INFINITY, l = 0.f;
  float4 o = make_float4(0, 0, 0, 0);
  int page = -1;
  for (int k = 0; k < se.hi; ++k) {
    if (k == se.sink && k < se.lo) k = se.lo;
    const int j = k / ky.page_size, off = k - j * ky.page_size;
    page = page_of(ky, s, b, j);
    if (page < 0) continue;
    if (ky.mask && !__ldg(ky.mask + page * ky.mask_stride + k)) continue;
    const float4 kk = load4<DT>(ky.k, page * ky.k_str[0] + hk * ky.k_str[1] + off * ky.k_str[2] + lane * 4);
    float d = q.x * kk.x + q.y * kk.y + q.z * kk.z + q.w * kk.w;
#pragma unroll
    for (int w = 16; w > 0; w >>= 1) d += __shfl_xor_sync(0xffffffffu, d, w);
    float vs = 1.f;
    if constexpr (DT != WF_DTYPE_BF16) {
      d *= __ldg(ky.ks + page * ky.ks_str[0] + hk * ky.ks_str[1] + off);
      vs = __ldg(ky.vs + page * ky.vs_str[0] + hk * ky.vs_str[1] + off);
    }
    d *= qr.scale_log2;
    const float mn = d != d ? d : fmaxf(m, d);
    const float c = m == mn ? 1.f : exp2f(m - mn), p = d == mn ? 1.f : exp2f(d - mn);
    const float4 v = load4<DT>(ky.v, page * ky.v_str[0] + hk * ky.v_str[1] + off * ky.v_str[2] + lane * 4);
    const float pv = p * vs;
    o.x = o.x * c + pv * v.x;
    o.y = o.y * c + pv * v.y;
    o.z = o.z * c + pv * v.z;
    o.w = o.w * c + pv * v.w;
    l = l * c + p;
    m = mn;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int64_t orow = ky.cross ? b * qr.o_str[0] + i * qr.o_str[1] : r * qr.o_str[1];
  *reinterpret_cast<uint2*>(qr.o + orow + h * qr.o_str[2] + lane * 4) =
      make_uint2(pack_bf16x2(o.x * inv, o.y * inv), pack_bf16x2(o.z * inv, o.w * inv));
  if (qr.lse && lane == 0) qr.lse[(int64_t)r * qr.H + h] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
}

static int launch(const Keys& ky, const Queries& qr, void* stream) {
  const int64_t units = (int64_t)qr.rows * qr.H;
  if (units == 0) return WF_OK;
  if (units > (int64_t)INT_MAX * 4) return fail(WF_ERR_INVALID_ARG, "paged attention: too many rows");
  auto kern = ky.dtype == WF_DTYPE_BF16 ? simple_kernel<WF_DTYPE_BF16>
              : ky.dtype == WF_DTYPE_E4M3 ? simple_kernel<WF_DTYPE_E4M3>
                                          : simple_kernel<WF_DTYPE_S8>;
  kern<<<(unsigned)((units + 3) / 4), 128, 0, static_cast<cudaStream_t>(stream)>>>(ky, qr);
  WFK_CUDA_TRY(cudaGetLastError());
  return WF_OK;
}

static int check_rows(const char* who, const void* q, const void* o, const int64_t* qs, const int64_t* os, int n,
                      float scale) {
  if (!q || !o || !qs || !os || !aligned16(q) || !aligned16(o))
    return fail(WF_ERR_INVALID_ARG, "%s: q or o null or not 16-byte aligned", who);
  for (int i = 0; i < n; ++i)
    if (qs[i] <= 0 || qs[i] % 8 || os[i] <= 0 || os[i] % 8)
      return fail(WF_ERR_INVALID_ARG, "%s: q and o strides must be positive multiples of 8 elements", who);
  if (!(scale > 0.f) || !std::isfinite(scale))
    return fail(WF_ERR_INVALID_ARG, "%s: softmax_scale must be positive", who);
  return WF_OK;
}

static int check_heads(const char* who, int H, int kv_heads) {
  if (H < 1 || H > 65535 || kv_heads < 1 || H % kv_heads || H / kv_heads > 128)
    return fail(WF_ERR_INVALID_ARG, "%s: %d query heads over %d K/V heads (a multiple of at most 128 needed)", who, H,
                kv_heads);
  return WF_OK;
}

}  // namespace paged
}  // namespace wfk

extern "C" int64_t wf_paged_attn_workspace(const wf_kv_pages* pages, const wf_kv_batch* batch, int H, int64_t max_new,
                                           int64_t max_len) {
  using namespace wfk::paged;
  if (check_pages("wf_paged_attn_workspace", pages) || check_batch("wf_paged_attn_workspace", batch, pages->page_size) ||
      check_heads("wf_paged_attn_workspace", H, pages->heads))
    return -1;
  return 0;
}

extern "C" int wf_paged_attn(const wf_kv_pages* pages, const wf_kv_batch* batch, const void* q,
                             const int64_t* q_stride, void* o, const int64_t* o_stride, float* lse, int H, int block,
                             int window, int sink, int64_t max_new, int64_t max_len, float softmax_scale,
                             void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace wfk;
  using namespace wfk::paged;
  static const char* who = "wf_paged_attn";
  int rc;
  if ((rc = check_pages(who, pages)) != WF_OK) return rc;
  if ((rc = check_batch(who, batch, pages->page_size)) != WF_OK) return rc;
  if ((rc = check_heads(who, H, pages->heads)) != WF_OK) return rc;
  if (block < 0 || window < 0 || sink < 0 || (sink > 0 && window == 0) || max_new < 0 || max_len < 0)
    return fail(WF_ERR_INVALID_ARG, "%s: block, window, sink, max_new and max_len must not be negative, a sink needs a "
                "window", who);
  if (batch->rows == 0 || batch->seqs == 0) return WF_OK;
  if ((rc = check_rows(who, q, o, q_stride, o_stride, 2, softmax_scale)) != WF_OK) return rc;
  Keys ky{pages->k, pages->v, pages->k_scale, pages->v_scale, {}, {}, {}, {}, batch->table, batch->table_stride,
          batch->lens, nullptr, 0, pages->n_pages, pages->page_size, batch->max_pages, pages->dtype, false};
  for (int i = 0; i < 3; ++i) ky.k_str[i] = pages->k_stride[i], ky.v_str[i] = pages->v_stride[i];
  for (int i = 0; i < 2; ++i) ky.ks_str[i] = pages->k_scale_stride[i], ky.vs_str[i] = pages->v_scale_stride[i];
  const Queries qr{static_cast<const __nv_bfloat16*>(q), static_cast<__nv_bfloat16*>(o), lse,
                   {0, q_stride[0], q_stride[1]}, {0, o_stride[0], o_stride[1]}, batch->cu, batch->seqs,
                   (int)batch->rows, 0, H, H / pages->heads, block, window, sink, softmax_scale * 1.4426950408889634f};
  return launch(ky, qr, stream);
}

extern "C" int64_t wf_cross_attn_workspace(int batch, int Lq, int states, int Lk, int H, int kv_heads) {
  using namespace wfk::paged;
  if (batch < 0 || Lq < 0 || states < 1 || Lk < 1 || check_heads("wf_cross_attn_workspace", H, kv_heads)) return -1;
  return 0;
}

extern "C" int wf_cross_attn(const void* q, const void* k, const void* v, void* o, float* lse, int batch, int Lq,
                             int states, int Lk, int H, int kv_heads, int D, const int64_t* q_stride,
                             const int64_t* k_stride, const int64_t* v_stride, const int64_t* o_stride,
                             const int32_t* kv_index, const int32_t* kv_lens, const uint8_t* key_mask,
                             int64_t mask_stride, float softmax_scale, void* workspace, int64_t workspace_bytes,
                             void* stream) {
  using namespace wfk;
  using namespace wfk::paged;
  static const char* who = "wf_cross_attn";
  int rc;
  if (D != HD) return fail(WF_ERR_UNSUPPORTED, "%s: head_dim %d unsupported (only 128)", who, D);
  if ((rc = check_heads(who, H, kv_heads)) != WF_OK) return rc;
  if (batch < 0 || Lq < 0 || states < 1 || Lk < 1 || batch > 65535 || (int64_t)batch * Lq > INT_MAX - 1024 ||
      Lk > INT_MAX - 1024)
    return fail(WF_ERR_INVALID_ARG, "%s: bad sizes batch=%d Lq=%d states=%d Lk=%d", who, batch, Lq, states, Lk);
  if (!kv_index && states != 1 && states != batch)
    return fail(WF_ERR_INVALID_ARG, "%s: %d states for %d query entries need kv_index", who, states, batch);
  if (batch == 0 || Lq == 0) return WF_OK;
  if ((rc = check_rows(who, q, o, q_stride, o_stride, 3, softmax_scale)) != WF_OK) return rc;
  if (!k || !v || !k_stride || !v_stride || !aligned16(k) || !aligned16(v))
    return fail(WF_ERR_INVALID_ARG, "%s: k or v null or not 16-byte aligned", who);
  for (int i = 0; i < 3; ++i)
    if (k_stride[i] <= 0 || k_stride[i] % 8 || v_stride[i] <= 0 || v_stride[i] % 8)
      return fail(WF_ERR_INVALID_ARG, "%s: k and v strides must be positive multiples of 8 elements", who);
  if (key_mask && mask_stride < 0) return fail(WF_ERR_INVALID_ARG, "%s: negative mask stride", who);
  const Keys ky{k, v, nullptr, nullptr, {k_stride[0], k_stride[2], k_stride[1]},
                {v_stride[0], v_stride[2], v_stride[1]}, {0, 0}, {0, 0}, kv_index, 1, kv_lens, key_mask, mask_stride,
                states, Lk, 1, WF_DTYPE_BF16, true};
  const Queries qr{static_cast<const __nv_bfloat16*>(q), static_cast<__nv_bfloat16*>(o), lse,
                   {q_stride[0], q_stride[1], q_stride[2]}, {o_stride[0], o_stride[1], o_stride[2]}, nullptr, batch,
                   batch * Lq, Lq, H, H / kv_heads, 0, 0, 0, softmax_scale * 1.4426950408889634f};
  return launch(ky, qr, stream);
}

extern "C" unsigned int wfk_status_take_paged_attn(void) { return wfk::status_take_local(); }
