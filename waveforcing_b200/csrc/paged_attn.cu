// Entry points of the attention over pages and of cross attention to an
// encoder's states (each state set is one page): argument checks, and the
// choice of kernel.
#include <cuda_runtime.h>

#include <cmath>

#include "paged_attn.cuh"

namespace wfk {
namespace paged {

// ------------------------------------------------------------------- joining
// One warp to an output row: the splits' outputs weighted by their sums.
__global__ void __launch_bounds__(256) join_kernel(const __grid_constant__ Keys ky, const __grid_constant__ Queries qr,
                                                   const float* __restrict__ part_o,
                                                   const float* __restrict__ part_l, int splits) {
  const int64_t n = (int64_t)qr.rows * qr.H;
  const int64_t at = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (at >= n) return;
  const int r = (int)(at / qr.H), h = (int)(at - (int64_t)r * qr.H);
  int64_t orow;
  if (ky.cross) {
    const int b = r / qr.Lq;
    orow = b * qr.o_str[0] + (r - b * qr.Lq) * qr.o_str[1];
  } else {
    if (r < __ldg(qr.cu) || r >= __ldg(qr.cu + qr.seqs)) return;  // behind the last sequence
    orow = r * qr.o_str[1];
  }
  float m = -INFINITY;
  for (int s = 0; s < splits; ++s) m = max_nan(m, part_l[s * n + at]);
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  float l = 0.f;
  if (m != -INFINITY)
    for (int s = 0; s < splits; ++s) {
      const float ls = part_l[s * n + at];
      if (ls == -INFINITY) continue;  // its output was not written
      const float w = exp2f(ls - m);
      const float4 x = __ldcs(reinterpret_cast<const float4*>(part_o + (s * n + at) * HD) + lane);
      o.x += w * x.x, o.y += w * x.y, o.z += w * x.z, o.w += w * x.w;
      l += w;
    }
  const float inv = m == -INFINITY ? 0.f : 1.f / l;
  *reinterpret_cast<uint2*>(qr.o + orow + h * qr.o_str[2] + lane * 4) =
      make_uint2(pack_bf16x2(o.x * inv, o.y * inv), pack_bf16x2(o.z * inv, o.w * inv));
  if (qr.lse && lane == 0) qr.lse[at] = m == -INFINITY ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
}

int join(const Keys& ky, const Queries& qr, const float* part_o, const float* part_l, int splits, cudaStream_t st) {
  join_kernel<<<(unsigned)(((int64_t)qr.rows * qr.H + 7) / 8), 256, 0, st>>>(ky, qr, part_o, part_l, splits);
  WFK_CUDA_TRY(cudaGetLastError());
  return WF_OK;
}

int page_maps(PageMaps* m, const Keys& ky, int kv_heads, const Tiling& tl, int bn) {
  const bool kv8 = ky.dtype != WF_DTYPE_BF16;
  const uint64_t dim[4] = {HD, (uint64_t)ky.page_size, (uint64_t)kv_heads, (uint64_t)ky.n_pages};
  const uint64_t elem = kv8 ? 1 : 2;
  for (int i = 0; i < 2; ++i) {
    const int64_t* s = i ? ky.v_str : ky.k_str;
    const uint64_t str[3] = {(uint64_t)s[2] * elem, (uint64_t)s[1] * elem, (uint64_t)s[0] * elem};
    for (int rows : {bn, tl.rows}) {
      CUtensorMap* to = rows == bn ? (i ? &m->v_tile : &m->k_tile) : (i ? &m->v : &m->k);
      const uint32_t box[4] = {kv8 ? 128u : 64u, (uint32_t)rows, 1, 1};
      const int rc = encode_tiled(to, kv8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
                                  i ? ky.v : ky.k, dim, str, box, CU_TENSOR_MAP_SWIZZLE_128B);
      if (rc != WF_OK) return rc;
      if (tl.rows == bn) {
        (i ? m->v : m->k) = *to;
        break;
      }
    }
  }
  return WF_OK;
}

// ------------------------------------------------------------- entry points
// Up to 16 rows to a K/V head read K and V once; more would read them again for
// each 16, where the tile kernel takes 128 rows at a time.
static bool few_rows(const Shape& sh) { return sh.max_new * sh.group <= 16; }

static int64_t workspace_need(const Shape& sh) {
  return (few_rows(sh) ? rows::parts(sh) : tile::parts(sh)) * (HD + 1) * 4;
}

int check_pages(const char* who, const wf_kv_pages* p);
int check_batch(const char* who, const wf_kv_batch* b, int page_size);

static int launch(const char* who, const Keys& ky, const Queries& qr, const Shape& sh, void* workspace,
                  int64_t workspace_bytes, void* stream) {
  const int64_t need = workspace_need(sh);
  if (need > 0 && (workspace_bytes < need || !workspace || !aligned16(workspace)))
    return fail(WF_ERR_INVALID_ARG, "%s: %lld bytes of 16-byte aligned workspace needed, %lld given", who,
                (long long)need, (long long)workspace_bytes);
  return (few_rows(sh) ? rows::launch : tile::launch)(ky, qr, sh, workspace, static_cast<cudaStream_t>(stream));
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

static Shape paged_shape(const wf_kv_pages* pages, const wf_kv_batch* batch, int H, int window, int sink,
                         int64_t max_new, int64_t max_len) {
  Shape sh{};
  sh.rows = batch->rows;
  sh.seqs = batch->seqs;
  sh.max_new = max_new < batch->rows ? max_new : batch->rows;
  sh.H = H;
  sh.group = H / pages->heads;
  sh.page_size = pages->page_size;
  const int64_t cap = (int64_t)batch->max_pages * pages->page_size;
  sh.keys = max_len < cap ? max_len : cap;
  if (window > 0 && (int64_t)window + sink + 256 < sh.keys) sh.keys = (int64_t)window + sink + 256;
  if (sh.keys < 1) sh.keys = 1;
  sh.kv8 = pages->dtype != WF_DTYPE_BF16;
  return sh;
}

static Shape cross_shape(int batch, int Lq, int Lk, int H, int kv_heads) {
  Shape sh{};
  sh.rows = (int64_t)batch * Lq;
  sh.seqs = batch;
  sh.max_new = sh.Lq = Lq;
  sh.H = H;
  sh.group = H / kv_heads;
  sh.page_size = Lk;
  sh.keys = Lk;
  sh.cross = true;
  return sh;
}

static int check_heads(const char* who, int H, int kv_heads) {
  if (H < 1 || H > 65535 || kv_heads < 1 || H % kv_heads || H / kv_heads > 128)
    return fail(WF_ERR_INVALID_ARG, "%s: %d query heads over %d K/V heads (a multiple of at most 128 needed)", who, H,
                kv_heads);
  return WF_OK;
}

}  // namespace paged
}  // namespace wfk

extern "C" int64_t wf_paged_attn_workspace(const wf_kv_pages* pages, const wf_kv_batch* batch, int H, int window, int sink,
                                           int64_t max_new,
                                           int64_t max_len) {
  using namespace wfk::paged;
  static const char* who = "wf_paged_attn_workspace";
  if (check_pages(who, pages) || check_batch(who, batch, pages->page_size) || check_heads(who, H, pages->heads) ||
      window < 0 || sink < 0 || max_new < 0 || max_len < 0)
    return -1;
  if (batch->rows == 0 || batch->seqs == 0) return 0;
  return workspace_need(paged_shape(pages, batch, H, window, sink, max_new, max_len));
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
  return launch(who, ky, qr, paged_shape(pages, batch, H, window, sink, max_new, max_len), workspace, workspace_bytes,
                stream);
}

extern "C" int64_t wf_cross_attn_workspace(int batch, int Lq, int states, int Lk, int H, int kv_heads) {
  using namespace wfk::paged;
  if (batch < 0 || Lq < 0 || states < 1 || Lk < 1 || check_heads("wf_cross_attn_workspace", H, kv_heads)) return -1;
  if (batch == 0 || Lq == 0) return 0;
  return workspace_need(cross_shape(batch, Lq, Lk, H, kv_heads));
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
  return launch(who, ky, qr, cross_shape(batch, Lq, Lk, H, kv_heads), workspace, workspace_bytes, stream);
}

extern "C" unsigned int wfk_status_take_paged_attn(void) { return wfk::status_take_local(); }
