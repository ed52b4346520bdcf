// Attention over pages for few query rows to a K/V head (single tokens, short
// runs of them): bound by reading K and V once from HBM.
//
// Rows of one K/V head (tokens x the query heads that share it) come in tiles
// of 16, the height of mma.sync's A operand, which here only has to keep up
// with the loads: 32 instructions to 8 KB of K and V.  A cluster of up to 8
// CTAs takes one tile of rows, each CTA a share of the keys, each warp every
// fourth chunk of that share: its K and V rows arrive by cp.async in a ring of
// its own (no CTA barrier in the loop, 2 x 8 KB a warp in flight, 128 KB an
// SM), are multiplied straight from shared memory, and the warps' and CTAs'
// sums are joined through (distributed) shared memory at the end.
//
// A contraction does not mind in which order its dimension is taken, so a
// thread loads 16 consecutive bytes of a K row and feeds them to the k indices
// it owns, with Q's fragments gathered in the same order; for 8-bit V it takes
// 16 consecutive dims of four keys, and byte j of each makes output tile j.
// 8-bit pages: codes are exact in f16; a key's scale multiplies its score and
// its P in f32 before P is rounded to f16 (2^-11), V's scales relative to the
// largest power of two so far; Q rows are scaled by powers of two to f16.
#include <cuda_fp16.h>

#include <cmath>

#include "paged_attn.cuh"

namespace wfk {
namespace paged {
namespace rows {

constexpr int WARPS = 4, THREADS = WARPS * 32, ST = 3, MAX_CLUSTER = 8;
constexpr int KV_BYTES = 8192;             // K and V rows of a chunk
constexpr int META_BYTES = 2 * 32 * 4 + 128;  // scales of K and V, the live keys
constexpr int STAGE = KV_BYTES + META_BYTES;
constexpr int O_PITCH = 132;               // floats of a row of partial sums, off the banks of the next
constexpr int SMEM = WARPS * ST * STAGE + 128;
static_assert(16 * (O_PITCH + 3) * 4 <= ST * STAGE, "a warp's sums fit its ring");

__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool take) {  // zeros when not taken
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(take ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp4(uint32_t dst, const void* src, bool take) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(take ? 4 : 0) : "memory");
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// Two codes (low halves' bytes 0 and 1) -> f16x2, exact.
template <int DT>
__device__ __forceinline__ uint32_t codes_f16(uint32_t two) {
  uint32_t r;
  if constexpr (DT == WF_DTYPE_E4M3) {
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(static_cast<uint16_t>(two)));
  } else {  // 1024 + (c + 128) by its bits, minus 1152
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(__byte_perm(two ^ 0x8080u, 0x64646464u, 0x4140)), "r"(0x64806480u));
  }
  return r;
}
__device__ __forceinline__ float pow2_above(float x) {  // power of two at or above x (> 0), within 2^+-122
  const uint32_t e = ((__float_as_uint(x) + 0x7FFFFFu) >> 23) << 23;
  return fminf(fmaxf(__uint_as_float(e), 0x1p-122f), 0x1p122f);
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float cluster_load(uint32_t saddr, uint32_t rank) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(mapa_shared(saddr, rank)) : "memory");
  return v;
}

struct Cut {
  int cluster, outer;  // CTAs of a cluster; clusters to a tile of rows (joined through the workspace)
  int row_tiles;       // tiles of rows that the grid has to a sequence and K/V head
};

template <int DT>
__global__ void __launch_bounds__(THREADS, 2)
    rows_kernel(const __grid_constant__ Keys ky, const __grid_constant__ Queries qr, const __grid_constant__ Cut cut,
                float* part_o, float* part_l) {
  constexpr bool KV8 = DT != WF_DTYPE_BF16;
  constexpr int KC = KV8 ? 32 : 16;        // keys of a chunk
  constexpr int ROWB = KV8 ? 128 : 256;    // bytes of a row
  constexpr int NT = KC / 8;               // score tiles of a chunk
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const uint32_t rank = cut.cluster > 1 ? cluster_ctarank() : 0;
  const int item = blockIdx.x / cut.cluster;
  const int G = qr.H / qr.group;
  const int rt0 = item % cut.row_tiles, hk = item / cut.row_tiles % G, b = item / cut.row_tiles / G;
  const Span sp = span_of(ky, qr, b);
  uint8_t* ring = smem + warp * ST * STAGE;
  const uint32_t ring_s = smem_u32(ring);
  const int ps = ky.page_size;

  for (int rt = rt0; rt * 16 < sp.n * qr.group; rt += cut.row_tiles) {
    // This thread's two rows, g and g + 8.
    int tok[2], head[2];
    bool has[2];
    Sees se[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = rt * 16 + g + e * 8;
      tok[e] = r / qr.group;
      head[e] = hk * qr.group + r - tok[e] * qr.group;
      has[e] = tok[e] < sp.n;
      if (!has[e]) tok[e] = sp.n - 1;
      se[e] = sees(qr, sp, tok[e]);
    }
    // Q fragments, dims in the order in which K is read.
    uint32_t a[8][4];
    float q_pow[2] = {1.f, 1.f};
    {
      uint2 v[8][2];
      float top[2] = {0.f, 0.f};
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int64_t at = ky.cross ? b * qr.q_str[0] + tok[e] * qr.q_str[1] : (int64_t)(sp.first + tok[e]) * qr.q_str[1];
        const __nv_bfloat16* q = qr.q + at + (has[e] ? head[e] : hk * qr.group) * qr.q_str[2];
#pragma unroll
        for (int s = 0; s < 8; ++s) {
          const int d = KV8 ? (s >> 2) * 64 + t * 16 + (s & 3) * 4 : (t + 4 * (s >> 1)) * 8 + (s & 1) * 4;
          v[s][e] = __ldg(reinterpret_cast<const uint2*>(q + d));
          if (KV8)
            top[e] = fmaxf(fmaxf(top[e], fmaxf(fabsf(__uint_as_float(v[s][e].x << 16)), fabsf(__uint_as_float(v[s][e].x & 0xFFFF0000u)))),
                           fmaxf(fabsf(__uint_as_float(v[s][e].y << 16)), fabsf(__uint_as_float(v[s][e].y & 0xFFFF0000u))));
        }
        if (KV8) {
          top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 1));
          top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 2));
          q_pow[e] = pow2_above(fminf(top[e], 0x1p122f));
        }
      }
#pragma unroll
      for (int s = 0; s < 8; ++s)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          if constexpr (KV8) {
            const float inv = 1.f / q_pow[e];
            a[s][e] = pack_f16(__uint_as_float(v[s][e].x << 16) * inv, __uint_as_float(v[s][e].x & 0xFFFF0000u) * inv);
            a[s][2 + e] = pack_f16(__uint_as_float(v[s][e].y << 16) * inv, __uint_as_float(v[s][e].y & 0xFFFF0000u) * inv);
          } else {
            a[s][e] = v[s][e].x;
            a[s][2 + e] = v[s][e].y;
          }
        }
    }
    // The keys that the tile's rows see together, in chunks of consecutive
    // positions, and this warp's share of them.
    const int i0 = rt * 16 / qr.group, i1 = min((rt * 16 + 15) / qr.group, sp.n - 1);
    const Sees first = sees(qr, sp, max(i0, min(-sp.pos0, i1))), last = sees(qr, sp, i1);
    const int hi = last.hi, lo = first.lo, sink = min(last.sink, hi);
    const int hi_min = i0 + sp.pos0 < 0 ? 0 : first.hi, lo_max = last.lo, sink_min = first.sink;
    const int n_rows = min(16, sp.n * qr.group - rt * 16);
    const float q_scale[2] = {q_pow[0] * qr.scale_log2, q_pow[1] * qr.scale_log2};
    int n_sink = 0, c_lo = 0, n = 0;
    if (hi > 0) {
      c_lo = lo / KC;
      n_sink = sink > 0 ? min((sink - 1) / KC + 1, c_lo) : 0;
      n = n_sink + (hi - 1) / KC + 1 - c_lo;
    }
    const int parts = cut.cluster * cut.outer, part = blockIdx.y * cut.cluster + rank;
    const int p0 = (int)((long long)n * part / parts) + warp, p1 = (int)((long long)n * (part + 1) / parts);

    // Key lane % KC of a chunk: page and row, fetched a chunk ahead of its loads.
    int nx_id = -1, nx_off = 0;
    bool nx_in = false;
    auto look = [&](int i) {
      nx_in = false;
      nx_id = -1;
      if (i < p1) {
        const int pos = (i < n_sink ? i : i - n_sink + c_lo) * KC + (lane % KC);
        if ((pos < hi && pos >= lo) || pos < sink) {
          const int j = pos / ps;
          nx_off = pos - j * ps;
          nx_id = page_id(ky, sp, b, j);
          nx_in = !(ky.mask && nx_id >= 0) || __ldg(ky.mask + nx_id * ky.mask_stride + pos) != 0;
        }
      }
    };
    auto issue = [&](int i, int stage) {
      const uint32_t at = ring_s + stage * STAGE;
      if (i < p1) {
        int id = nx_id;
        const int off = nx_off;
        if (nx_in && (id < 0 || id >= ky.n_pages)) {
          status_raise(ST_PAGE_ID);
          id = -1;
        }
        if (!nx_in) id = -1;
        const uint32_t live = __ballot_sync(0xffffffffu, id >= 0);
        if (lane == 0) *reinterpret_cast<uint32_t*>(ring + stage * STAGE + KV_BYTES + 256) = live;
        if constexpr (KV8) {
          cp4(at + KV_BYTES + lane * 4, ky.ks + (id >= 0 ? id * ky.ks_str[0] + hk * ky.ks_str[1] + off : 0), id >= 0);
          cp4(at + KV_BYTES + 128 + lane * 4, ky.vs + (id >= 0 ? id * ky.vs_str[0] + hk * ky.vs_str[1] + off : 0),
              id >= 0);
        }
        // Row offsets (bytes) of this lane's key, then each lane's share of 16-byte pieces.
        constexpr int CH = ROWB / 16, RPI = 32 / CH;  // pieces of a row, rows that an instruction covers
        constexpr int ES = KV8 ? 1 : 2;
        const int64_t kr = id >= 0 ? (id * ky.k_str[0] + hk * ky.k_str[1] + off * ky.k_str[2]) * ES : -1;
        const int64_t vr = (id * ky.v_str[0] + hk * ky.v_str[1] + off * ky.v_str[2]) * ES;
        const int c = lane % CH;
        const uint8_t *kb = static_cast<const uint8_t*>(ky.k) + c * 16, *vb = static_cast<const uint8_t*>(ky.v) + c * 16;
#pragma unroll
        for (int k = 0; k < KC / RPI; ++k) {
          const int r = k * RPI + lane / CH;
          const int64_t ko = __shfl_sync(0xffffffffu, kr, r), vo = __shfl_sync(0xffffffffu, vr, r);
          const bool take = ko >= 0;
          cp16(at + r * ROWB + ((c ^ ((r & 1) << 2)) << 4), kb + (take ? ko : 0), take);
          cp16(at + KC * ROWB + r * ROWB + ((c ^ (r & 7)) << 4), vb + (take ? vo : 0), take);
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };

    float o[16][4];
#pragma unroll
    for (int k = 0; k < 16; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[k][e] = 0.f;
    float m_run[2] = {-INFINITY, -INFINITY}, m_use[2] = {0.f, 0.f}, l_run[2] = {0.f, 0.f}, v_top = 0.f;

    look(p0);
#pragma unroll
    for (int k = 0; k < ST - 1; ++k) {
      issue(p0 + k * WARPS, k);
      look(p0 + (k + 1) * WARPS);
    }
    int stage = 0;
    for (int i = p0; i < p1; i += WARPS) {
      asm volatile("cp.async.wait_group %0;" ::"n"(ST - 2) : "memory");
      __syncwarp();
      // the stage that the last chunk used is free: all lanes are past it
      issue(i + (ST - 1) * WARPS, stage == 0 ? ST - 1 : stage - 1);
      look(i + ST * WARPS);
      const uint8_t* K = ring + stage * STAGE;
      const uint8_t* V = K + KC * ROWB;
      const float* scale = reinterpret_cast<const float*>(K + KV_BYTES);
      const uint32_t live = *reinterpret_cast<const uint32_t*>(K + KV_BYTES + 256);

      float s[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int e = 0; e < 4; ++e) s[nt][e] = 0.f;
        const int r = nt * 8 + g;
#pragma unroll
        for (int c = 0; c < ROWB / 64; ++c) {
          const uint4 w = *reinterpret_cast<const uint4*>(K + r * ROWB + (((t + 4 * c) ^ ((r & 1) << 2)) << 4));
          if constexpr (KV8) {
            const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int k = 0; k < 4; ++k)
              mma_f16(s[nt], a[c * 4 + k], codes_f16<DT>(x[k] & 0xFFFFu), codes_f16<DT>(x[k] >> 16));
          } else {
            mma_bf16(s[nt], a[2 * c], w.x, w.y);
            mma_bf16(s[nt], a[2 * c + 1], w.z, w.w);
          }
        }
      }
      // Scores in log2 units, -inf where the row does not see the key.
      const int pos0 = (i < n_sink ? i : i - n_sink + c_lo) * KC;
      const bool whole = live == (KC == 32 ? 0xFFFFFFFFu : (1u << (KC & 31)) - 1) && pos0 + KC <= hi_min &&
                         (pos0 >= lo_max || pos0 + KC <= sink_min);
      float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float2 ks = KV8 ? *reinterpret_cast<const float2*>(scale + nt * 8 + 2 * t) : make_float2(1.f, 1.f);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[nt][e] *= KV8 ? q_scale[e >> 1] * ((e & 1) ? ks.y : ks.x) : qr.scale_log2;
          if (!whole) {
            const int k = nt * 8 + 2 * t + (e & 1), pos = pos0 + k;
            const Sees& v = se[e >> 1];
            if (!((live >> k & 1) && pos < v.hi && (pos >= v.lo || pos < v.sink))) s[nt][e] = -INFINITY;
          }
          mx[e >> 1] = max_nan(mx[e >> 1], s[nt][e]);
        }
      }
      bool grow = false;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        mx[e] = max_nan(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 1));
        mx[e] = max_nan(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 2));
        grow |= !(mx[e] <= m_run[e] + 8.f);
      }
      float v_new = v_top;
      if constexpr (KV8) {
        float top = live >> lane & 1 ? fabsf(scale[32 + lane]) : 0.f;
        if (!(top < INFINITY)) top = 0.f;
        top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));
        if (v_top == 0.f || top > v_top) v_new = pow2_above(top) * 8.f;
      }
      // Sums are rescaled only when a row's maximum grows by more than 2^8, or
      // V's largest scale does; a NaN or +inf score makes its row NaN.
      if (__any_sync(0xffffffffu, grow) || v_new != v_top) {
        float al[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          al[e] = 1.f;
          if (!(mx[e] <= m_run[e] + 8.f)) {
            const float m_new = mx[e] < INFINITY ? mx[e] : __uint_as_float(0x7FC00000u);
            al[e] = exp2f(m_run[e] - m_new);
            l_run[e] *= al[e];
            m_run[e] = m_use[e] = m_new;
          }
          if (KV8) al[e] *= v_top / v_new;
        }
        v_top = v_new;
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          o[k][0] *= al[0], o[k][1] *= al[0];
          o[k][2] *= al[1], o[k][3] *= al[1];
        }
      }
      const float v_inv = KV8 ? 1.f / v_top : 1.f;
      uint32_t p[NT / 2][4];  // as the A operand of P V: [rows g | g + 8][keys 2t | 2t + 8]
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[e] = ex2_approx(s[nt][e] - m_use[e >> 1]);
          l_run[e >> 1] += x[e];
        }
        if constexpr (KV8) {
          const float2 vs = *reinterpret_cast<const float2*>(scale + 32 + nt * 8 + 2 * t);
#pragma unroll
          for (int e = 0; e < 4; ++e)  // a key that is not seen does not count, whatever its scale
            x[e] = s[nt][e] == -INFINITY ? 0.f : x[e] * (((e & 1) ? vs.y : vs.x) * v_inv);
          p[nt >> 1][(nt & 1) * 2] = pack_f16(x[0], x[1]);
          p[nt >> 1][(nt & 1) * 2 + 1] = pack_f16(x[2], x[3]);
        } else {
          p[nt >> 1][(nt & 1) * 2] = pack_bf16x2(x[0], x[1]);
          p[nt >> 1][(nt & 1) * 2 + 1] = pack_bf16x2(x[2], x[3]);
        }
      }
#pragma unroll
      for (int k16 = 0; k16 < NT / 2; ++k16) {
        if constexpr (KV8) {
          uint4 w[4];  // dims 16 g .. 16 g + 15 of keys 2t, 2t + 1, 2t + 8, 2t + 9
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int r = k16 * 16 + 2 * t + (e & 1) + (e >> 1) * 8;
            w[e] = *reinterpret_cast<const uint4*>(V + r * ROWB + ((g ^ (r & 7)) << 4));
          }
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            auto word = [&](const uint4& x) { return k < 4 ? x.x : k < 8 ? x.y : k < 12 ? x.z : x.w; };
            const uint32_t sel = (k & 3) | ((4 + (k & 3)) << 4);
            mma_f16(o[k], p[k16], codes_f16<DT>(__byte_perm(word(w[0]), word(w[1]), sel) & 0xFFFFu),
                    codes_f16<DT>(__byte_perm(word(w[2]), word(w[3]), sel) & 0xFFFFu));
          }
        } else {
          const int mat = lane >> 3, r = (lane & 7) + (mat & 1) * 8;
#pragma unroll
          for (int d = 0; d < 8; ++d) {
            uint32_t v0, v1, v2, v3;
            asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                         : "=r"(v0), "=r"(v1), "=r"(v2), "=r"(v3)
                         : "r"(smem_u32(V + r * ROWB + (((2 * d + (mat >> 1)) ^ (r & 7)) << 4)))
                         : "memory");
            mma_bf16(o[2 * d], p[0], v0, v1);
            mma_bf16(o[2 * d + 1], p[0], v2, v3);
          }
        }
      }
      stage = stage + 1 == ST ? 0 : stage + 1;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncwarp();
    // ---- the warps' sums: O [16][O_PITCH], then m[16], l[16], over the ring
    float* mine = reinterpret_cast<float*>(ring);
    if (KV8 && v_top == 0.f) v_top = 1.f;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      l_run[e] += __shfl_xor_sync(0xffffffffu, l_run[e], 1);
      l_run[e] += __shfl_xor_sync(0xffffffffu, l_run[e], 2);
      if (g + e * 8 >= n_rows) continue;
      if (t == 0) {
        mine[16 * O_PITCH + g + e * 8] = m_run[e];
        mine[16 * O_PITCH + 16 + g + e * 8] = l_run[e];
      }
#pragma unroll
      for (int k = 0; k < 16; ++k)
#pragma unroll
        for (int f = 0; f < 2; ++f) {
          const int d = KV8 ? (2 * t + f) * 16 + k : k * 8 + 2 * t + f;
          mine[(g + e * 8) * O_PITCH + d] = KV8 ? o[k][2 * e + f] * v_top : o[k][2 * e + f];
        }
    }
    __syncthreads();
    // The CTA's sums, into warp 0's place: first each row's maximum, l and the
    // warps' weights (in place of their maxima), then thread x dim x of the rows.
    constexpr int PITCH_W = ST * STAGE / 4;
    float* base = reinterpret_cast<float*>(smem);
    const int dim = threadIdx.x;
    if (dim < n_rows) {
      float* at = base + 16 * O_PITCH + dim;
      float m = -INFINITY, l = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) m = max_nan(m, at[w * PITCH_W]);
      const float mu = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        const float wt = exp2f(at[w * PITCH_W] - mu);
        l += wt * at[w * PITCH_W + 16];
        at[w * PITCH_W] = wt;
      }
      at[16] = l;
      at[32] = m;
    }
    __syncthreads();
#pragma unroll 2
    for (int r = 0; r < n_rows; ++r) {
      float x = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w)
        x += base[w * PITCH_W + 16 * O_PITCH + r] * base[w * PITCH_W + r * O_PITCH + dim];
      base[r * O_PITCH + dim] = x;
    }
    if (cut.cluster > 1)
      cluster_sync();
    else
      __syncthreads();
    // CTA `rank` finishes rows rank, rank + cluster, ...: the CTAs' sums joined.
    for (int r = rank; r < n_rows; r += cut.cluster) {
      const int rg = rt * 16 + r, i = rg / qr.group;
      const int h = hk * qr.group + rg - i * qr.group;
      const uint32_t am = smem_u32(base + 16 * O_PITCH + 32 + r), ao = smem_u32(base + r * O_PITCH + dim);
      float m = -INFINITY, l = 0.f, x = 0.f;
      if (cut.cluster > 1) {
        for (int c = 0; c < cut.cluster; ++c) m = max_nan(m, cluster_load(am, c));
        const float mu = m == -INFINITY ? 0.f : m;
        for (int c = 0; c < cut.cluster; ++c) {
          const float wt = exp2f(cluster_load(am, c) - mu);
          l += wt * cluster_load(am - 64, c);
          x += wt * cluster_load(ao, c);
        }
      } else {
        m = base[16 * O_PITCH + 32 + r];
        l = base[16 * O_PITCH + 16 + r];
        x = base[r * O_PITCH + dim];
      }
      const bool none = m == -INFINITY;
      const float inv = none ? 0.f : m != m ? m : 1.f / l;
      const float lse2 = none ? -INFINITY : m + log2f(l);
      const int64_t packed = (int64_t)(sp.first + i) * qr.H + h;
      if (cut.outer > 1) {
        const int64_t at = (int64_t)blockIdx.y * qr.rows * qr.H + packed;
        part_o[at * HD + dim] = x * inv;
        if (dim == 0) part_l[at] = lse2;
      } else {
        const int64_t orow = ky.cross ? b * qr.o_str[0] + i * qr.o_str[1] : (int64_t)(sp.first + i) * qr.o_str[1];
        qr.o[orow + h * qr.o_str[2] + dim] = __float2bfloat16_rn(none ? 0.f : x * inv);
        if (qr.lse && dim == 0) qr.lse[packed] = lse2 * 0.6931471805599453f;
      }
    }
    // the others may still read this CTA's sums
    if (cut.cluster > 1)
      cluster_sync();
    else
      __syncthreads();
  }
}

// --------------------------------------------------------------------- host
// Enough CTAs for every SM's two places, as long as each keeps two chunks to a
// warp; what a cluster cannot give, clusters joined afterwards do as far as one
// CTA to each SM.
static Cut cut_of(const Shape& sh, bool kv8) {
  const int64_t chunk = kv8 ? 32 : 16;
  Cut c{1, 1, (int)((sh.max_new * sh.group + 15) / 16)};
  if (c.row_tiles < 1) c.row_tiles = 1;
  const int64_t seqs = sh.seqs < sh.rows ? sh.seqs : sh.rows;
  const int64_t items = seqs * (sh.H / sh.group) * c.row_tiles, most = sh.keys / (chunk * WARPS * 2);
  while (c.cluster < MAX_CLUSTER && items * c.cluster < 2 * SMS && 2 * c.cluster <= most) c.cluster *= 2;
  if (c.cluster == MAX_CLUSTER)
    while (c.outer < 16 && items * c.cluster * c.outer < SMS && 2 * c.outer * c.cluster <= most) c.outer *= 2;
  return c;
}

int splits(const Shape& sh) { return cut_of(sh, sh.kv8).outer; }

template <int DT>
static int start(const Keys& ky, const Queries& qr, const Cut& cut, float* part_o, float* part_l, cudaStream_t st) {
  static thread_local int configured = -1;
  int dev = 0;
  WFK_CUDA_TRY(cudaGetDevice(&dev));
  if (configured != dev) {
    WFK_CUDA_TRY(cudaFuncSetAttribute(rows_kernel<DT>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM));
    configured = dev;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)((int64_t)qr.seqs * (qr.H / qr.group) * cut.row_tiles * cut.cluster), (unsigned)cut.outer);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = SMEM;
  cfg.stream = st;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim = {(unsigned)cut.cluster, 1, 1};
  cfg.attrs = &at;
  cfg.numAttrs = cut.cluster > 1 ? 1 : 0;
  WFK_CUDA_TRY(cudaLaunchKernelEx(&cfg, rows_kernel<DT>, ky, qr, cut, part_o, part_l));
  return WF_OK;
}

int launch(const Keys& ky, const Queries& qr, const Shape& sh, void* workspace, cudaStream_t st) {
  const Cut cut = cut_of(sh, sh.kv8);
  if ((int64_t)qr.seqs * (qr.H / qr.group) * cut.row_tiles * cut.cluster > INT_MAX)
    return fail(WF_ERR_INVALID_ARG, "attention: too many rows");
  float *part_o = nullptr, *part_l = nullptr;
  if (cut.outer > 1) {
    part_o = static_cast<float*>(workspace);
    part_l = part_o + (int64_t)cut.outer * qr.rows * qr.H * HD;
  }
  const int rc = ky.dtype == WF_DTYPE_BF16   ? start<WF_DTYPE_BF16>(ky, qr, cut, part_o, part_l, st)
                 : ky.dtype == WF_DTYPE_E4M3 ? start<WF_DTYPE_E4M3>(ky, qr, cut, part_o, part_l, st)
                                             : start<WF_DTYPE_S8>(ky, qr, cut, part_o, part_l, st);
  if (rc != WF_OK || cut.outer == 1) return rc;
  return join(ky, qr, part_o, part_l, cut.outer, st);
}

}  // namespace rows
}  // namespace paged
}  // namespace wfk

extern "C" unsigned int wfk_status_take_paged_rows(void) { return wfk::status_take_local(); }
