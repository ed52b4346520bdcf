// Attention over pages for few query rows to a K/V head (single tokens, short
// runs of them): bound by reading K and V once from HBM.
//
// Rows of one K/V head (tokens x the query heads that share it) come in tiles
// of 16, the height of mma.sync's A operand, which here only has to keep up
// with the loads: 32 instructions to 8 KB of K and V.  A cluster of up to 8
// CTAs takes one tile of rows, each CTA a share of the key tiles.  Warp 4 loads
// tiles by TMA into a ring of three (64 KB in flight, two CTAs to an SM); warps
// 0-3 take a quarter of a tile's keys each, multiply them straight from shared
// memory and keep sums of their own, which are joined through (distributed)
// shared memory at the end.  (With every warp loading its own chunks, issuing
// four TMA copies cost 600 of 1700 clocks a chunk.)
//
// A contraction does not mind in which order its dimension is taken, so a
// thread loads 16 consecutive bytes of a K row and feeds them to the k indices
// it owns, with Q's fragments gathered in the same order; for 8-bit V it takes
// 16 consecutive dims of four keys, and byte j of each makes output tile j.
// Column n of a score tile is key n ^ 4 (n & 1): with the 128-byte swizzle the
// eight lanes of a 16-byte read then meet eight bank groups for K and for V.
// 8-bit pages: codes are exact in f16; a key's scale multiplies its score and
// its P in f32 before P is rounded to f16 (2^-11), V's scales relative to the
// largest power of two so far; Q rows are scaled by powers of two to f16.
#include <cuda_fp16.h>

#include <cmath>

#include "paged_attn.cuh"

namespace wfk {
namespace paged {
namespace rows {

constexpr int WARPS = 4, THREADS = (WARPS + 1) * 32, ST = 3, MAX_CLUSTER = 8;
constexpr int STAGE = 32768;               // a tile's K and V rows
constexpr int MAX_BN = 128;
constexpr int META = 2 * MAX_BN * 4 + 32;  // scales of K and V, live keys, whether every row sees all, the tile
constexpr int O_PITCH = 132;               // floats of a row of partial sums, off the banks of the next
constexpr int PART = 16 * (O_PITCH + 3) * 4;  // a warp's sums: O, m, l, and the CTA's m
constexpr int SMEM = 1024 + ST * (STAGE + META + 16) + 16;
static_assert(WARPS * PART <= ST * STAGE, "the sums lie over the ring");

// Key of column n of an 8-key score tile.
__device__ __forceinline__ int key_of(int n) { return n ^ ((n & 1) << 2); }

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
__device__ __forceinline__ float cluster_load(uint32_t saddr, uint32_t rank) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(mapa_shared(saddr, rank)) : "memory");
  return v;
}

struct Cut {
  Tiling tl;
  int cluster, outer;  // CTAs of a cluster; clusters to a tile of rows (joined through the workspace)
  int row_tiles;       // tiles of rows that the grid has to a sequence and K/V head
};

template <int DT>
__global__ void __launch_bounds__(THREADS, 2)
    rows_kernel(const __grid_constant__ PageMaps tm,
                const __grid_constant__ Keys ky, const __grid_constant__ Queries qr, const __grid_constant__ Cut cut,
                float* part_o, float* part_l) {
  constexpr bool KV8 = DT != WF_DTYPE_BF16;
  constexpr int BN = KV8 ? 128 : 64;       // keys of a tile
  constexpr int KC = BN / WARPS;           // keys of a warp
  constexpr int ROWB = KV8 ? 128 : 256;    // bytes of a row
  constexpr int NT = KC / 8;               // score tiles of a warp
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const uint32_t rank = cut.cluster > 1 ? cluster_ctarank() : 0;
  const int item = blockIdx.x / cut.cluster;
  const int G = qr.H / qr.group;
  const int rt0 = item % cut.row_tiles, hk = item / cut.row_tiles % G, b = item / cut.row_tiles / G;
  // The page table's row comes to L2 while the sequence's length is on its way.
  if (!ky.cross && threadIdx.x * 32 < ky.max_pages)
    asm volatile("prefetch.global.L2 [%0];" ::"l"(ky.table + b * ky.table_stride + threadIdx.x * 32));
  const Span sp = span_of(ky, qr, b);
  const Tiling& tl = cut.tl;
  const int ps = tl.ps;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + ST * (STAGE + META));
  uint64_t* empty = full + ST;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(empty + ST);
  if (threadIdx.x == 0) {
    for (int k = 0; k < ST; ++k) {
      mbar_init(&full[k], KV8 ? 33 : 1);
      mbar_init(&empty[k], WARPS);
    }
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tm.k_tile);
    tma_prefetch_desc(&tm.v_tile);
  }
  __syncthreads();
  uint32_t done = 0;  // tiles through the ring

  for (int rt = rt0; rt * 16 < sp.n * qr.group; rt += cut.row_tiles) {
    const int i0 = rt * 16 / qr.group, i1 = min((rt * 16 + 15) / qr.group, sp.n - 1);
    const Range rg = range_of<BN>(qr, sp, tl, i0, i1);
    const int n_rows = min(16, sp.n * qr.group - rt * 16);
    const int parts = cut.cluster * cut.outer, part = blockIdx.y * cut.cluster + rank;
    const int p0 = (int)((long long)rg.n * part / parts), p1 = (int)((long long)rg.n * (part + 1) / parts);
    if (warp == WARPS) {
      // ---------------------------------------------------------- producer
      // A tile's page ids (a lane to a box) are fetched a tile ahead; scales go
      // to shared memory by cp.async: no latency lies between the waits.
      constexpr int KL = BN / 32;
      int sub[KL], at_row[KL];  // of key c * 32 + lane: its box, and the row in it
#pragma unroll
      for (int c = 0; c < KL; ++c) {
        const int r = c * 32 + lane;
        sub[c] = min(r / tl.rows, tl.boxes);  // behind the last box: a hole
        at_row[c] = r - sub[c] * tl.rows;
      }
      Box nx{};             // the next tile, or this lane's box of it
      int nx_id = INT_MIN;  // and its page, as the table has it (INT_MIN: not needed)
      auto look = [&](const TileAt& a) {
        const bool one = one_box<BN>(tl, a);
        nx = one ? Box{a.page, a.row, a.base} : box_at<BN>(tl, a, lane);
        nx_id = one || (lane < tl.boxes && needed(rg, nx.pos, min(tl.rows, ps - nx.row))) ? page_id(ky, sp, b, nx.page)
                                                                                          : INT_MIN;
      };
      Walk<BN> walk(rg, tl, min(p0, max(p1 - 1, 0)));
      if (p0 < p1) look(walk.a);
      for (int i = p0; i < p1; ++i, ++done) {
        const TileAt a = walk.a;
        const bool bad = nx_id != INT_MIN && (nx_id < 0 || nx_id >= ky.n_pages), one = one_box<BN>(tl, a);
        if (bad) status_raise(ST_PAGE_ID);
        const int box = bad || nx_id == INT_MIN ? -1 : nx_id;
        const Box x = nx;
        if (i + 1 < p1) {
          walk.next();
          look(walk.a);
        }
        const uint32_t st = done % ST, turn = done / ST;
        if (turn > 0 && !warp_wait(&empty[st], turn - 1, abort_flag, ST_PAGED_ROWS)) break;
        uint8_t *at = smem + st * STAGE, *mt = smem + ST * STAGE + st * META;
        const uint32_t to = smem_u32(mt) + lane * 4;
        uint32_t all = 0xFFFFFFFFu;
        const int64_t ko = KV8 ? box * ky.ks_str[0] + hk * ky.ks_str[1] + x.row : 0;
        const int64_t vo = KV8 ? box * ky.vs_str[0] + hk * ky.vs_str[1] + x.row : 0;
        const bool easy = __all_sync(0xffffffffu, (one || lane < tl.boxes) ? box >= 0 : true) && inside<BN>(rg, a) &&
                          !ky.mask && (tl.dense || (one && x.row + BN <= ps));  // every key of the tile
#pragma unroll
        for (int c = 0; c < KL; ++c) {
          const int src = one ? 0 : sub[c] & 31, ar = one ? c * 32 + lane : at_row[c];
          bool in = true;
          if (!easy) {
            const int id = __shfl_sync(0xffffffffu, box, src);
            const int off = __shfl_sync(0xffffffffu, x.row, src) + ar;
            const int pos = __shfl_sync(0xffffffffu, x.pos, src) + ar;
            in = id >= 0 && (one || sub[c] < tl.boxes) && off < ps && seen(rg, pos);
            if (ky.mask && in) in = __ldg(ky.mask + id * ky.mask_stride + off) != 0;
            const uint32_t word = __ballot_sync(0xffffffffu, in);
            all &= word;
            if (lane == c) reinterpret_cast<uint32_t*>(mt + 2 * MAX_BN * 4)[c] = word;
          }
          if constexpr (KV8) {
            const int64_t k = __shfl_sync(0xffffffffu, ko, src), v = __shfl_sync(0xffffffffu, vo, src);
            cp4(to + c * 128, ky.ks + (in ? k + ar : 0), in);
            cp4(to + MAX_BN * 4 + c * 128, ky.vs + (in ? v + ar : 0), in);
          }
        }
        if (easy && lane < KL) reinterpret_cast<uint32_t*>(mt + 2 * MAX_BN * 4)[lane] = 0xFFFFFFFFu;
        if constexpr (KV8) asm volatile("cp.async.mbarrier.arrive.noinc.shared.b64 [%0];" ::"r"(smem_u32(&full[st])) : "memory");
        // BN live keys lie at consecutive positions, whatever the page size
        const bool whole = all == 0xFFFFFFFFu && a.base + BN <= rg.hi_min &&
                           (a.base >= rg.lo_max || a.base + BN <= rg.sink_min);
        if (lane == 4) *reinterpret_cast<uint2*>(mt + 2 * MAX_BN * 4 + 16) = make_uint2(whole, nth_tile(rg, i));
        __syncwarp();
        auto copy = [&](const CUtensorMap* mk, const CUtensorMap* mv, uint8_t* k, int row, int id) {
          tma_load_4d(k, mk, &full[st], 0, row, hk, id);
          if constexpr (!KV8) tma_load_4d(k + STAGE / 4, mk, &full[st], 64, row, hk, id);
          tma_load_4d(k + STAGE / 2, mv, &full[st], 0, row, hk, id);
          if constexpr (!KV8) tma_load_4d(k + 3 * STAGE / 4, mv, &full[st], 64, row, hk, id);
        };
        if (one) {  // operands in uniform registers
          const int id = __shfl_sync(0xffffffffu, box, 0);
          const int row = __shfl_sync(0xffffffffu, a.row, 0);
          if (elect_one()) {
            mbar_arrive_expect_tx(&full[st], id >= 0 ? STAGE : 0);
            if (id >= 0) copy(&tm.k_tile, &tm.v_tile, at, row, id);
          }
        } else {
          const uint32_t boxes = __ballot_sync(0xffffffffu, box >= 0), bytes = (uint32_t)tl.rows * 128;
          if (lane == 0) mbar_arrive_expect_tx(&full[st], __popc(boxes) * bytes * (KV8 ? 2 : 4));
          __syncwarp();
          if (box >= 0) copy(&tm.k, &tm.v, at + lane * bytes, x.row, box);
        }
        __syncwarp();
      }
      if (*abort_flag && lane == 0) {  // let the loads in flight land before their place is used again
        const uint64_t t0 = globaltimer_ns();
        for (uint32_t k = done > ST ? done - ST : 0; k < done; ++k)
          while (!mbar_try_wait(&full[k % ST], (k / ST) & 1) && globaltimer_ns() - t0 < 200000000ull) {
          }
      }
      __syncwarp();
    } else {
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
            a[s][e] = f16x2(__uint_as_float(v[s][e].x << 16) * inv, __uint_as_float(v[s][e].x & 0xFFFF0000u) * inv);
            a[s][2 + e] = f16x2(__uint_as_float(v[s][e].y << 16) * inv, __uint_as_float(v[s][e].y & 0xFFFF0000u) * inv);
          } else {
            a[s][e] = v[s][e].x;
            a[s][2 + e] = v[s][e].y;
          }
        }
    }
    const float q_scale[2] = {q_pow[0] * qr.scale_log2, q_pow[1] * qr.scale_log2};

    float o[16][4];
#pragma unroll
    for (int k = 0; k < 16; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[k][e] = 0.f;
    float m_run[2] = {-INFINITY, -INFINITY}, m_use[2] = {0.f, 0.f}, l_run[2] = {0.f, 0.f}, v_top = 0.f;

    for (int i = p0; i < p1; ++i, ++done) {
      const uint32_t st = done % ST;
      if (!warp_wait(&full[st], done / ST, abort_flag, ST_PAGED_ROWS)) break;
      uint8_t* K = smem + st * STAGE + warp * KC * 128;
      uint8_t* V = K + STAGE / 2;
      const uint8_t* mt = smem + ST * STAGE + st * META;
      const float* scale = reinterpret_cast<const float*>(mt) + warp * KC;
      const uint2 mark = *reinterpret_cast<const uint2*>(mt + 2 * MAX_BN * 4 + 16);
      const bool whole = mark.x != 0;
      uint32_t keep[2] = {~0u, ~0u}, live = ~0u;  // by key of this warp
      if (!whole) {
        const int k0 = warp * KC;
        live = reinterpret_cast<const uint32_t*>(mt + 2 * MAX_BN * 4)[k0 >> 5] >> (k0 & 31);
        const TileAt a = tile_at<BN>(tl, mark.y);
#pragma unroll
        for (int e = 0; e < 2; ++e)
          keep[e] = live & (bit_range(rows_below<BN>(tl, a, se[e].lo), rows_below<BN>(tl, a, se[e].hi), k0) |
                            bit_range(0, rows_below<BN>(tl, a, se[e].sink), k0));
        // V rows that no query sees may hold NaN
        constexpr int PER = ROWB / 16;  // 16-byte pieces of a row
        for (int r = lane / PER; r < KC; r += 32 / PER)
          if (!(live >> r & 1))
            *reinterpret_cast<uint4*>(V + (lane % PER / 8) * (STAGE / 4) + r * 128 + (lane & 7) * 16) = make_uint4(0, 0, 0, 0);
        fence_proxy_async_smem();  // the ring's next TMA comes after these writes
        __syncwarp();
      }

      float s[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float c0[4] = {0.f, 0.f, 0.f, 0.f}, c1[4] = {0.f, 0.f, 0.f, 0.f};  // two chains to a tile
        const int r = nt * 8 + key_of(g);
#pragma unroll
        for (int c = 0; c < ROWB / 64; ++c) {
          const uint4 w = *reinterpret_cast<const uint4*>(K + (c >> 1) * (STAGE / 4) + r * 128 +
                                                          (((t + 4 * (c & 1)) ^ (r & 7)) << 4));
          if constexpr (KV8) {
            const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int k = 0; k < 4; ++k)
              mma_f16(k & 1 ? c1 : c0, a[c * 4 + k], codes_f16<DT>(x[k] & 0xFFFFu), codes_f16<DT>(x[k] >> 16));
          } else {
            mma_bf16(c0, a[2 * c], w.x, w.y);
            mma_bf16(c1, a[2 * c + 1], w.z, w.w);
          }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) s[nt][e] = c0[e] + c1[e];
      }
      // Scores in log2 units, -inf where the row does not see the key.
      float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int k = nt * 8 + key_of(2 * t + (e & 1));
          s[nt][e] *= KV8 ? q_scale[e >> 1] * scale[k] : qr.scale_log2;
          if (!whole && !(keep[e >> 1] >> k & 1)) s[nt][e] = -INFINITY;
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
        float top = fabsf(scale[MAX_BN + lane]);  // 0 where a key is not seen at all
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
#pragma unroll
          for (int e = 0; e < 4; ++e)  // a key that is not seen does not count, whatever its scale
            x[e] = s[nt][e] == -INFINITY ? 0.f : x[e] * (scale[MAX_BN + nt * 8 + key_of(2 * t + (e & 1))] * v_inv);
          p[nt >> 1][(nt & 1) * 2] = f16x2(x[0], x[1]);
          p[nt >> 1][(nt & 1) * 2 + 1] = f16x2(x[2], x[3]);
        } else {
          p[nt >> 1][(nt & 1) * 2] = pack_bf16x2(x[0], x[1]);
          p[nt >> 1][(nt & 1) * 2 + 1] = pack_bf16x2(x[2], x[3]);
        }
      }
#pragma unroll
      for (int k16 = 0; k16 < NT / 2; ++k16) {
        if constexpr (KV8) {
          uint4 w[4];  // dims 16 g .. 16 g + 15 of the keys of columns 2t, 2t + 1, 2t + 8, 2t + 9
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int r = k16 * 16 + key_of(2 * t + (e & 1)) + (e >> 1) * 8;
            w[e] = *reinterpret_cast<const uint4*>(V + r * 128 + ((g ^ (r & 7)) << 4));
          }
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            auto word = [&](const uint4& x) { return k < 4 ? x.x : k < 8 ? x.y : k < 12 ? x.z : x.w; };
            const uint32_t sel = (k & 3) | ((4 + (k & 3)) << 4);
            mma_f16(o[k], p[k16], codes_f16<DT>(__byte_perm(word(w[0]), word(w[1]), sel) & 0xFFFFu),
                    codes_f16<DT>(__byte_perm(word(w[2]), word(w[3]), sel) & 0xFFFFu));
          }
        } else {
          const int mat = lane >> 3, r = key_of(lane & 7) + (mat & 1) * 8;
#pragma unroll
          for (int d = 0; d < 8; ++d) {
            uint32_t v0, v1, v2, v3;
            asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                         : "=r"(v0), "=r"(v1), "=r"(v2), "=r"(v3)
                         : "r"(smem_u32(V + (d >> 2) * (STAGE / 4) + r * 128 +
                                        (((2 * (d & 3) + (mat >> 1)) ^ (r & 7)) << 4)))
                         : "memory");
            mma_bf16(o[2 * d], p[0], v0, v1);
            mma_bf16(o[2 * d + 1], p[0], v2, v3);
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[st]);
    }
    named_bar_sync(1, WARPS * 32);  // the sums lie over the ring: every warp is past it
    // ---- the warps' sums: O [16][O_PITCH], then m[16], l[16], over the ring
    float* mine = reinterpret_cast<float*>(smem + warp * PART);
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
    }
    __syncthreads();
    // The CTA's sums, into warp 0's place: first each row's maximum, l and the
    // warps' weights (in place of their maxima), then thread x dim x of the rows.
    constexpr int PITCH_W = PART / 4;
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
    if (dim < HD)
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
    for (int r = rank; r < n_rows && dim < HD; r += cut.cluster) {
      const int row = rt * 16 + r, i = row / qr.group;
      const int h = hk * qr.group + row - i * qr.group;
      const uint32_t am = smem_u32(base + 16 * O_PITCH + 32 + r), ao = smem_u32(base + r * O_PITCH + dim);
      float m = -INFINITY, l = 0.f, x = 0.f;
      if (cut.cluster > 1) {
        float mc[MAX_CLUSTER], lc[MAX_CLUSTER], xc[MAX_CLUSTER];  // all in flight at once
#pragma unroll
        for (int c = 0; c < MAX_CLUSTER; ++c) {
          const int from = min(c, cut.cluster - 1);
          mc[c] = cluster_load(am, from);
          lc[c] = cluster_load(am - 64, from);
          xc[c] = cluster_load(ao, from);
        }
#pragma unroll
        for (int c = 0; c < MAX_CLUSTER; ++c) m = max_nan(m, mc[c]);
        const float mu = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int c = 0; c < MAX_CLUSTER; ++c) {
          const float wt = c < cut.cluster ? exp2f(mc[c] - mu) : 0.f;
          l += c < cut.cluster ? wt * lc[c] : 0.f;
          x += c < cut.cluster ? wt * xc[c] : 0.f;
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
    // the others may still read this CTA's sums; the next rows' TMA comes after
    fence_proxy_async_smem();
    if (cut.cluster > 1)
      cluster_sync();
    else
      __syncthreads();
  }
}

// --------------------------------------------------------------------- host
// The cut of the keys with the least estimated time, in tiles: those of all
// waves of CTAs with about six for a CTA's
// start and end, half of one CTA's again because sequences differ in length,
// and four for the join of clusters.
static int places(int cluster) { return cluster <= 2 ? 2 * SMS : cluster == 4 ? 284 : 264; }  // CTAs that run at once
static Cut cut_of(const Shape& sh, bool kv8) {
  const int bn = kv8 ? 128 : 64;
  Cut c{tiling_of(sh.page_size, bn), 1, 1, (int)((sh.max_new * sh.group + 15) / 16)};
  if (c.row_tiles < 1) c.row_tiles = 1;
  const int64_t seqs = sh.seqs < sh.rows ? sh.seqs : sh.rows;
  const int64_t items = seqs * (sh.H / sh.group) * c.row_tiles;
  const int64_t n = tiles_of_keys(sh, bn);
  double best = 1e30;
  for (int cluster = 1; cluster <= MAX_CLUSTER; cluster *= 2)
    for (int outer = 1; outer <= 16; ++outer) {
      if (cluster * outer > 1 && n < (int64_t)cluster * outer * 2) break;
      const double rounds = (double)((n + cluster * outer - 1) / (cluster * outer));
      const double cost = (double)((items * cluster * outer + places(cluster) - 1) / places(cluster)) * (rounds + 6) + 0.5 * rounds +
                          (outer > 1 ? 4 : 0);
      if (cost < best) best = cost, c.cluster = cluster, c.outer = outer;
    }
  return c;
}

int64_t parts(const Shape& sh) {
  const int outer = cut_of(sh, sh.kv8).outer;
  return outer > 1 ? (int64_t)outer * sh.rows * sh.H : 0;
}

template <int DT>
static int start(const PageMaps& tm, const Keys& ky, const Queries& qr, const Cut& cut, float* part_o, float* part_l, cudaStream_t st) {
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
  WFK_CUDA_TRY(cudaLaunchKernelEx(&cfg, rows_kernel<DT>, tm, ky, qr, cut, part_o, part_l));
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
  PageMaps tm;
  int rc;
  if ((rc = page_maps(&tm, ky, qr.H / qr.group, cut.tl, sh.kv8 ? 128 : 64)) != WF_OK) return rc;
  rc = ky.dtype == WF_DTYPE_BF16   ? start<WF_DTYPE_BF16>(tm, ky, qr, cut, part_o, part_l, st)
       : ky.dtype == WF_DTYPE_E4M3 ? start<WF_DTYPE_E4M3>(tm, ky, qr, cut, part_o, part_l, st)
                                   : start<WF_DTYPE_S8>(tm, ky, qr, cut, part_o, part_l, st);
  if (rc != WF_OK || cut.outer == 1) return rc;
  return join(ky, qr, part_o, part_l, cut.outer, st);
}

}  // namespace rows
}  // namespace paged
}  // namespace wfk

extern "C" unsigned int wfk_status_take_paged_rows(void) { return wfk::status_take_local(); }
