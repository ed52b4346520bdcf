// Attention over pages on tcgen05 for calls with many query rows.
//
// Work item = two sub-tiles of 128 query rows of one K/V head (rows of a
// sub-tile: TQ = 128 / group tokens x the group's query heads) against a run
// of 128-key tiles.  K and V tiles are loaded once for both sub-tiles.
//   warp 0       TMA producer (a lane to a page of a tile)
//   warp 1       MMA issue: S_u = Q_u K_j^T (M=N=K=128), O_u += P_u V_j
//   warp 2       marks the live keys of each tile, zeroes the V rows of the
//                others (their P is 0, but 0 * NaN is not), fetches scales
//   warps 4-11   softmax; warpgroup u owns sub-tile u, a thread a row
//   warps 12-15  (8-bit pages) expand codes to bf16
// TMEM columns: S_0 [0,128) S_1 [128,256) O_0 [256,384) O_1 [384,512); P_u
// (bf16) overwrites the first half of S_u, which its warpgroup holds in
// registers by then.  The tensor pipe runs in issue order, PV_0(j) QK_0(j+1)
// PV_1(j) QK_1(j+1) ..., so QK_u(j+1) overwrites P_u(j) only after PV_u(j) has
// read it, and S_u(j+1) complete means that PV_u(j) is: O_u may be rescaled.
// While one sub-tile's products run, the other's exponentials do.
#include <cmath>

#include "paged_attn.cuh"

namespace wfk {
namespace paged {
namespace tile {

constexpr int BM = 128;  // rows of a sub-tile
constexpr int BN = 128;  // keys of a tile
constexpr int HALF = 16384;       // 128 rows x 64 bf16
constexpr int SLOT = 2 * HALF;    // a K or V tile, or a Q sub-tile: [d 0-63][d 64-127]
constexpr int META = 4;           // tiles whose marks (and scales) are kept
constexpr uint32_t COL_S = 0, COL_O = 256;

constexpr int WORK_BYTES = 80;
template <bool KV8>
struct Cfg {
  static constexpr int NS = KV8 ? 4 : 5;  // ring slots
  static constexpr int THREADS = KV8 ? 512 : 384;
  static constexpr int NBARS = (3 * NS + 10 + 1 + 1) & ~1;  // even: what follows is 16-byte aligned
  static constexpr int META_BYTES = META * (16 + (KV8 ? 2 * BN * 4 : 0) + 4);
  static constexpr int SMEM = 1024 + 2 * SLOT + NS * SLOT + NBARS * 8 + META_BYTES + 16 + 8 * WORK_BYTES;
  static_assert(SMEM <= 232448, "shared memory of one CTA");
};

// How the keys of a sequence fall into tiles: pages of at least 128 rows give
// ceil(page_size / 128) tiles each, smaller ones share a tile, a page on every
// `rows` tile rows (page_size rounded up to the swizzle's 8).
struct Tiling {
  int ps, tpp, ppt, rows;  // tiles per page (large pages), pages per tile (small), tile rows of a page
  int tq;                  // tokens of a sub-tile
  int splits;
};
__device__ __forceinline__ int tile_of(const Tiling& tl, int pos) {
  const int j = pos / tl.ps;
  return tl.ps < BN ? j / tl.ppt : j * tl.tpp + (pos - j * tl.ps) / BN;
}
struct TileAt {
  int page, row, base;  // first page, row in it, position of the tile's first key
};
__device__ __forceinline__ TileAt tile_at(const Tiling& tl, int t) {
  TileAt a;
  if (tl.ps < BN) {
    a.page = t * tl.ppt;
    a.row = 0;
  } else {
    a.page = t / tl.tpp;
    a.row = (t - a.page * tl.tpp) * BN;
  }
  a.base = a.page * tl.ps + a.row;
  return a;
}
// Tile rows whose position is below x.
__device__ __forceinline__ int rows_below(const Tiling& tl, const TileAt& a, int x) {
  const int d = x - a.base;
  if (d <= 0) return 0;
  if (tl.ps >= BN) return min(d, min(BN, tl.ps - a.row));
  const int j = d / tl.ps;
  return min(j, tl.ppt) * tl.rows + (j < tl.ppt ? d - j * tl.ps : 0);
}

struct Work {
  int b, hk, split;
  int i0, nsub;  // first token, sub-tiles with rows
  Span sp;
  int hi, lo, sink;  // keys the item's rows see: [0, sink) and [lo, hi)
  int n_sink, t_lo;  // tiles of the sink range; first tile of the other
  int t0, t1;        // this item's share of the tile list
};

static_assert(sizeof(Work) <= WORK_BYTES, "a softmax warp's item");

// Query tiles of the launch over all sequences (one warp).
__device__ __forceinline__ int count_tiles(const Keys& ky, const Queries& qr, const Tiling& tl, int lane) {
  if (ky.cross) return qr.seqs * ((qr.Lq + 2 * tl.tq - 1) / (2 * tl.tq));
  int n = 0;
  for (int b = lane; b < qr.seqs; b += 32) {
    const int first = min(max(__ldg(qr.cu + b), 0), qr.rows);
    n += (min(max(__ldg(qr.cu + b + 1), first), qr.rows) - first + 2 * tl.tq - 1) / (2 * tl.tq);
  }
  return __reduce_add_sync(0xffffffffu, n);
}

// Item `it` of the launch (one warp, same result in every lane).
__device__ __forceinline__ bool find_work(Work& w, const Keys& ky, const Queries& qr, const Tiling& tl, int n_tiles,
                                          int G, long long it, int lane) {
  if (n_tiles == 0 || it >= (long long)n_tiles * G * tl.splits) return false;
  int tile = (int)(it % n_tiles);
  const int rest = (int)(it / n_tiles);
  w.hk = rest % G;
  w.split = rest / G;
  int nq = 0;
  if (ky.cross) {
    nq = (qr.Lq + 2 * tl.tq - 1) / (2 * tl.tq);
    w.b = tile / nq;
    tile -= w.b * nq;
  } else {
    for (int b0 = 0;; b0 += 32) {
      int n = 0;
      if (b0 + lane < qr.seqs) {
        const int first = min(max(__ldg(qr.cu + b0 + lane), 0), qr.rows);
        n = (min(max(__ldg(qr.cu + b0 + lane + 1), first), qr.rows) - first + 2 * tl.tq - 1) / (2 * tl.tq);
      }
      int sum = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += t;
      }
      const uint32_t over = __ballot_sync(0xffffffffu, sum > tile);
      if (over) {
        const int src = __ffs(over) - 1;
        nq = __shfl_sync(0xffffffffu, n, src);
        tile -= __shfl_sync(0xffffffffu, sum, src) - nq;
        w.b = b0 + src;
        break;
      }
      tile -= __shfl_sync(0xffffffffu, sum, 31);
    }
  }
  tile = nq - 1 - tile;  // a causal sequence's longest rows first
  w.sp = span_of(ky, qr, w.b);
  w.i0 = tile * 2 * tl.tq;
  const int i1 = min(w.i0 + 2 * tl.tq, w.sp.n) - 1;  // last token
  w.nsub = i1 >= w.i0 + tl.tq ? 2 : 1;
  const Sees last = sees(qr, w.sp, i1);
  const Sees first = sees(qr, w.sp, max(w.i0, min(-w.sp.pos0, i1)));  // earlier rows have no position
  w.hi = last.hi;
  w.lo = first.lo;
  w.sink = min(last.sink, w.hi);
  int n = 0;
  w.n_sink = w.t_lo = 0;
  if (w.hi > 0) {
    const int t_hi = tile_of(tl, w.hi - 1) + 1;
    w.t_lo = tile_of(tl, w.lo);
    w.n_sink = w.sink > 0 ? min(tile_of(tl, w.sink - 1) + 1, w.t_lo) : 0;
    n = w.n_sink + t_hi - w.t_lo;
  }
  w.t0 = (int)((long long)n * w.split / tl.splits);
  w.t1 = (int)((long long)n * (w.split + 1) / tl.splits);
  return true;
}
__device__ __forceinline__ int nth_tile(const Work& w, int i) { return i < w.n_sink ? i : i - w.n_sink + w.t_lo; }

// Page j of the item's sequence if some row of the item sees one of its keys: its id, or -1.
__device__ __forceinline__ int needed_page(const Keys& ky, const Work& w, const Tiling& tl, int j) {
  const long long p0 = (long long)j * tl.ps;
  if (!((p0 < w.hi && p0 + tl.ps > w.lo) || p0 < w.sink)) return -1;
  return page_of(ky, w.sp, w.b, j);
}

__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort, uint32_t code) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity & 1, abort, code));
}
__device__ __forceinline__ bool drain(uint64_t* bar, uint32_t parity, uint64_t ns) {
  const uint64_t t0 = globaltimer_ns();
  while (!mbar_try_wait(bar, parity & 1))
    if (globaltimer_ns() - t0 > ns) {
      status_raise(ST_DRAIN_TIMEOUT);
      return false;
    }
  return true;
}

// Maximum of three, NaN if one is NaN (a NaN score must reach the row's result).
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Two e4m3 codes in the high bytes of t's halves -> bf16x2, exactly: the
// code's exponent and mantissa moved into bf16's fields are the value times
// 2^-120 (subnormal codes become subnormal bf16 and stay exact).  The NaN
// codes come out as +-480; a row that holds NaN has a NaN scale instead.
__device__ __forceinline__ uint32_t e4m3x2_bf16x2(uint32_t t) {
  const uint32_t u = (t & 0x80008000u) | ((t >> 4) & 0x07F007F0u);
  uint32_t r;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(u), "r"(0x7B807B80u));
  return r;
}
// Two signed bytes in the low bytes of t's halves -> bf16x2, exactly: (128 +
// low 7 bits) - (128, or 256 for a negative byte).
__device__ __forceinline__ uint32_t s8x2_bf16x2(uint32_t t) {
  const uint32_t a = (t & 0x007F007Fu) | 0x43004300u, b = (t & 0x00800080u) | 0x43004300u;
  uint32_t r;
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <int DT>
__device__ __forceinline__ void expand4(uint32_t w, uint32_t& lo, uint32_t& hi) {  // 4 codes -> 4 bf16
  if constexpr (DT == WF_DTYPE_E4M3) {
    lo = e4m3x2_bf16x2(__byte_perm(w, 0, 0x1404));
    hi = e4m3x2_bf16x2(__byte_perm(w, 0, 0x3424));
  } else {
    lo = s8x2_bf16x2(__byte_perm(w, 0, 0x4140));
    hi = s8x2_bf16x2(__byte_perm(w, 0, 0x4342));
  }
}

// Expands the 32 rows of one converter warp of a code tile (128 bytes a row,
// swizzled, in the slot's upper half) in place to two halves of bf16 rows.  A
// code row shares its line with the upper bf16 row: the eight lanes of a row
// read all of it before any of them writes.  Lanes 4-7 of a row write their
// odd chunk first, so that a row's eight stores meet eight bank groups.
template <int DT>
__device__ __forceinline__ void expand_rows(uint8_t* slot, int row0, int lane) {
  const int c = lane & 7, hi = c >> 2;
#pragma unroll 1
  for (int i = 0; i < 32; i += 8) {
    uint32_t h[2][8];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int r = row0 + i + 4 * t + (lane >> 3);
      const uint4 raw = *reinterpret_cast<const uint4*>(slot + HALF + r * 128 + ((c ^ (r & 7)) << 4));
      const uint32_t w[4] = {hi ? raw.z : raw.x, hi ? raw.w : raw.y, hi ? raw.x : raw.z, hi ? raw.y : raw.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) expand4<DT>(w[k], h[t][2 * k], h[t][2 * k + 1]);
    }
    __syncwarp();
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int r = row0 + i + 4 * t + (lane >> 3);
      uint8_t* row = slot + hi * HALF + r * 128;
      const int first = ((2 * (c & 3)) ^ (r & 7)) ^ hi;
      *reinterpret_cast<uint4*>(row + (first << 4)) = make_uint4(h[t][0], h[t][1], h[t][2], h[t][3]);
      *reinterpret_cast<uint4*>(row + ((first ^ 1) << 4)) = make_uint4(h[t][4], h[t][5], h[t][6], h[t][7]);
    }
  }
}

// Bits [a, b) of a 32-bit word that starts at bit `at`.
__device__ __forceinline__ uint32_t bit_range(int a, int b, int at) {
  const int lo = min(max(a - at, 0), 32), hi = min(max(b - at, 0), 32);
  if (hi <= lo) return 0;
  return (0xFFFFFFFFu >> (32 - (hi - lo))) << lo;
}

template <int DT>
__global__ void __launch_bounds__(Cfg<DT != WF_DTYPE_BF16>::THREADS, 1)
    tile_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                const __grid_constant__ CUtensorMap tmV, const __grid_constant__ Keys ky,
                const __grid_constant__ Queries qr, const __grid_constant__ Tiling tl, float* part_o, float* part_l) {
  constexpr bool KV8 = DT != WF_DTYPE_BF16;
  constexpr int NS = Cfg<KV8>::NS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  uint8_t* sQ = smem;                // 2 sub-tiles
  uint8_t* ring = sQ + 2 * SLOT;     // K_0 V_0 K_1 V_1 ...
  uint64_t* raw = reinterpret_cast<uint64_t*>(ring + NS * SLOT);  // [NS] TMA landed
  uint64_t* full = raw + NS;         // [NS] ready for the tensor pipe
  uint64_t* empty = full + NS;       // [NS] read by it
  uint64_t* q_full = empty + NS;     // [2]
  uint64_t* q_empty = q_full + 2;    // [2] the item's last QK_u has completed
  uint64_t* bar_s = q_empty + 2;     // [2] S_u complete
  uint64_t* bar_p = bar_s + 2;       // [2] P_u written
  uint64_t* o_full = bar_p + 2;      // [2] the item's last PV_u has completed
  uint64_t* bar_fin = o_full + 2;
  uint32_t* live = reinterpret_cast<uint32_t*>(raw + Cfg<KV8>::NBARS);  // [META][4] live keys of a tile
  float* scales = reinterpret_cast<float*>(live + META * 4);            // [META][2][BN], 8-bit pages
  int* first_key = reinterpret_cast<int*>(scales + (KV8 ? META * 2 * BN : 0));  // [META] position of its first key
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(reinterpret_cast<uint8_t*>(live) + Cfg<KV8>::META_BYTES);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = qr.H / qr.group;

  if (threadIdx.x == 0) {
    for (int s = 0; s < NS; ++s) {
      mbar_init(&raw[s], 1);
      mbar_init(&full[s], KV8 ? 129 : 1);
      mbar_init(&empty[s], 1);
    }
    for (int u = 0; u < 2; ++u) {
      mbar_init(&q_full[u], 1);
      mbar_init(&q_empty[u], 1);
      mbar_init(&bar_s[u], 1);
      mbar_init(&bar_p[u], 128);
      mbar_init(&o_full[u], 1);
    }
    mbar_init(bar_fin, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tbase = *tmem_slot;
  const int n_tiles = count_tiles(ky, qr, tl, lane);

  auto teardown = [&]() {
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
      tc_fence_after();
      tmem_dealloc(tbase, 512);
    }
  };
  // Registers: 384 threads launch with 168 each (64,512 = 128 * 72 + 256 *
  // 216); 512 with 128 (65,536 = 256 * 64 + 256 * 192).
  if (warp < 4) {
    if constexpr (KV8)
      asm volatile("setmaxnreg.dec.sync.aligned.u32 64;\n" ::: "memory");
    else
      asm volatile("setmaxnreg.dec.sync.aligned.u32 72;\n" ::: "memory");
    Work w;
    if (warp == 0) {
      // ------------------------------------------------------------ producer
      uint32_t slot_n = 0;        // ring slots filled
      uint32_t qn[2] = {0, 0};    // Q sub-tiles loaded
      bool ok = true;
      const int sub = lane;       // a lane to a page of the tile
      auto page_for = [&](int t, int& row) -> int {
        const TileAt a = tile_at(tl, t);
        row = a.row;
        return sub < tl.ppt ? needed_page(ky, w, tl, a.page + sub) : -1;
      };
      auto load = [&](const CUtensorMap* map, int id, int row) -> bool {
        const uint32_t s = slot_n % NS, n = slot_n / NS;
        if (n > 0 && !warp_wait(&empty[s], n - 1, abort_flag, ST_PAGED_PRODUCER)) return false;
        uint8_t* dst = ring + s * SLOT;
        const uint32_t box = (uint32_t)tl.rows * 128;
        const uint32_t pages = __popc(__ballot_sync(0xffffffffu, id >= 0));
        if (lane == 0) mbar_arrive_expect_tx(&raw[s], pages * box * (KV8 ? 1 : 2));
        __syncwarp();
        if (id >= 0) {
          if constexpr (KV8) {
            tma_load_4d(dst + HALF + sub * box, map, &raw[s], 0, row, w.hk, id);
          } else {
            tma_load_4d(dst + sub * box, map, &raw[s], 0, row, w.hk, id);
            tma_load_4d(dst + HALF + sub * box, map, &raw[s], 64, row, w.hk, id);
          }
        }
        ++slot_n;
        return true;
      };
      for (long long it = blockIdx.x; ok && find_work(w, ky, qr, tl, n_tiles, G, it, lane); it += gridDim.x) {
        if (w.t1 <= w.t0) continue;
        for (int u = 0; ok && u < w.nsub; ++u) {
          if (qn[u] > 0 && !(ok = warp_wait(&q_empty[u], qn[u] - 1, abort_flag, ST_PAGED_PRODUCER))) break;
          if (lane == 0) {
            mbar_arrive_expect_tx(&q_full[u], 2 * tl.tq * qr.group * 128);
            const int i = w.i0 + u * tl.tq, row = ky.cross ? i : w.sp.first + i, entry = ky.cross ? w.b : 0;
            tma_load_4d(sQ + u * SLOT, &tmQ, &q_full[u], 0, w.hk * qr.group, row, entry);
            tma_load_4d(sQ + u * SLOT + HALF, &tmQ, &q_full[u], 64, w.hk * qr.group, row, entry);
          }
          ++qn[u];
        }
        int row, next_row = 0, id, next_id = page_for(nth_tile(w, w.t0), next_row);
        for (int i = w.t0; ok && i < w.t1; ++i) {
          id = next_id;
          row = next_row;
          if (i + 1 < w.t1) next_id = page_for(nth_tile(w, i + 1), next_row);
          ok = load(&tmK, id, row) && load(&tmV, id, row);
        }
      }
      if (*abort_flag && lane == 0) {
        // let the copies in flight land before the CTA exits
        for (int u = 0; u < 2; ++u)
          if (qn[u] > 0) drain(&q_full[u], qn[u] - 1, 200000000ull);
        for (uint32_t n = slot_n > NS ? slot_n - NS : 0; n < slot_n; ++n) drain(&raw[n % NS], n / NS, 200000000ull);
      }
    } else if (warp == 1) {
      // ----------------------------------------------------------------- MMA
      constexpr uint32_t idesc_qk = make_idesc(1, FMT_BF16, FMT_BF16, 0, BM, BN);
      constexpr uint32_t idesc_pv = make_idesc(1, FMT_BF16, FMT_BF16, 1, BM, HD);
      uint32_t slot_n = 0, items[2] = {0, 0}, pn[2] = {0, 0};
      bool ok = true;
      auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
        ok = ok && warp_wait(bar, parity, abort_flag, ST_PAGED_MMA);
        return ok;
      };
      auto qk = [&](int u, uint32_t slot) {
        const uint64_t dQ = desc_sw128(smem_u32(sQ + u * SLOT), 16, 1024);
        const uint64_t dK = desc_sw128(smem_u32(ring + (slot % NS) * SLOT), 16, 1024);
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < HD / 16; ++kk) {
            const uint32_t off = ((kk >> 2) * HALF + (kk & 3) * 32) >> 4;
            umma_f16_ss(tbase + COL_S + u * BN, dQ + off, dK + off, idesc_qk, kk > 0);
          }
          umma_commit(&bar_s[u]);
        }
        __syncwarp();
      };
      for (long long it = blockIdx.x; ok && find_work(w, ky, qr, tl, n_tiles, G, it, lane); it += gridDim.x) {
        const int nt = w.t1 - w.t0;
        if (nt <= 0) continue;
        const int last_u = w.nsub - 1;
        if (!wait(&full[slot_n % NS], slot_n / NS)) break;
        for (int u = 0; u < w.nsub; ++u) {
          if (!wait(&q_full[u], items[u])) break;
          tc_fence_after();
          qk(u, slot_n);
          if (nt == 1 && elect_one()) umma_commit(&q_empty[u]);
        }
        if (!ok) break;
        if (elect_one()) umma_commit(&empty[slot_n % NS]);
        ++slot_n;
        for (int j = 0; ok && j < nt; ++j) {
          const uint32_t sv = slot_n, sk = slot_n + 1;
          const bool more = j + 1 < nt;
          if (!wait(&full[sv % NS], sv / NS)) break;
          for (int u = 0; u < w.nsub; ++u) {
            if (!wait(&bar_p[u], pn[u])) break;
            ++pn[u];
            // P_u of an item's first tile also says that the last item's O_u has been read
            tc_fence_after();
            const uint64_t dV = desc_sw128(smem_u32(ring + (sv % NS) * SLOT), HALF, 1024);
            if (elect_one()) {
#pragma unroll
              for (int kk = 0; kk < BN / 16; ++kk)
                umma_f16_ts(tbase + COL_O + u * HD, tbase + COL_S + u * BN + kk * 8, dV + kk * 128, idesc_pv,
                            (j > 0 || kk > 0) ? 1u : 0u);
              if (u == last_u) umma_commit(&empty[sv % NS]);
              if (!more) umma_commit(&o_full[u]);
            }
            __syncwarp();
            if (more) {
              if (u == 0 && !wait(&full[sk % NS], sk / NS)) break;
              tc_fence_after();
              qk(u, sk);
              if (elect_one()) {
                if (j + 2 == nt) umma_commit(&q_empty[u]);
                if (u == last_u) umma_commit(&empty[sk % NS]);
              }
            }
          }
          slot_n += more ? 2 : 1;
        }
        for (int u = 0; u < w.nsub; ++u) ++items[u];
      }
      // nothing of ours may still be running when TMEM is released
      if (elect_one()) {
        umma_commit(bar_fin);
        drain(bar_fin, 0, 200000000ull);
      }
    } else if (warp == 2) {
      // --------------------------------------------------------------- marks
      uint32_t slot_n = 0, tiles = 0;
      bool ok = true;
      for (long long it = blockIdx.x; ok && find_work(w, ky, qr, tl, n_tiles, G, it, lane); it += gridDim.x) {
        for (int i = w.t0; ok && i < w.t1; ++i, ++tiles) {
          const TileAt a = tile_at(tl, nth_tile(w, i));
          uint32_t words[4];
          float sk[KV8 ? 4 : 1], sv[KV8 ? 4 : 1];
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int r = c * 32 + lane;
            int off = a.row + r, j = a.page;
            bool in = off < tl.ps;
            if (tl.ps < BN) {
              const int p = r / tl.rows;
              off = r - p * tl.rows;
              j += p;
              in = off < tl.ps && p < tl.ppt;
            }
            const int pos = j * tl.ps + off;
            in = in && ((pos < w.hi && pos >= w.lo) || pos < w.sink);
            const int id = in ? page_of(ky, w.sp, w.b, j) : -1;
            in = in && id >= 0;
            if (in && ky.mask) in = __ldg(ky.mask + id * ky.mask_stride + pos) != 0;
            if constexpr (KV8) {
              sk[c] = in ? __ldg(ky.ks + id * ky.ks_str[0] + w.hk * ky.ks_str[1] + off) : 0.f;
              sv[c] = in ? __ldg(ky.vs + id * ky.vs_str[0] + w.hk * ky.vs_str[1] + off) : 0.f;
            }
            words[c] = __ballot_sync(0xffffffffu, in);
          }
          // The marks of tile n - META are dead: its V slot (and with it its
          // P, which was formed with them) has been released before this
          // tile's K could land.
          uint32_t s = slot_n % NS;
          if (!(ok = warp_wait(&raw[s], slot_n / NS, abort_flag, ST_PAGED_MARK))) break;
          const uint32_t m = tiles % META;
          if (lane < 4) live[m * 4 + lane] = lane < 2 ? (lane ? words[1] : words[0]) : (lane & 1 ? words[3] : words[2]);
          if (lane == 4) first_key[m] = a.base;
          if constexpr (KV8) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              scales[m * 2 * BN + c * 32 + lane] = sk[c];
              scales[m * 2 * BN + BN + c * 32 + lane] = sv[c];
            }
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&full[s]);
          ++slot_n;
          s = slot_n % NS;
          if (!(ok = warp_wait(&raw[s], slot_n / NS, abort_flag, ST_PAGED_MARK))) break;
          if constexpr (!KV8) {
            if ((words[0] & words[1] & words[2] & words[3]) != 0xFFFFFFFFu) {
              uint8_t* v = ring + s * SLOT + (lane >> 4) * 128 + ((lane >> 3) & 1) * HALF + (lane & 7) * 16;
#pragma unroll 1
              for (int c = 0; c < 4; ++c) {
                const uint32_t word = c < 2 ? (c ? words[1] : words[0]) : (c & 1 ? words[3] : words[2]);
                if (word == 0xFFFFFFFFu) continue;
#pragma unroll 1
                for (int r = lane >> 4; r < 32; r += 2)  // half a warp to a row, 16 bytes a lane
                  if (!(word >> r & 1))
                    *reinterpret_cast<uint4*>(v + (c * 32 + r - (lane >> 4)) * 128) = make_uint4(0, 0, 0, 0);
              }
              fence_proxy_async_smem();
              __syncwarp();
            }
          }
          if (lane == 0) mbar_arrive(&full[s]);
          ++slot_n;
        }
      }
    }
    __syncwarp();
    teardown();
  } else if (warp < 12) {
    // ------------------------------------------------------------- softmax
    if constexpr (KV8)
      asm volatile("setmaxnreg.inc.sync.aligned.u32 192;\n" ::: "memory");
    else
      asm volatile("setmaxnreg.inc.sync.aligned.u32 216;\n" ::: "memory");
    const int u = (warp - 4) >> 2;
    const int row = (warp & 3) * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tS = tbase + lane_off + COL_S + u * BN, tO = tbase + lane_off + COL_O + u * HD;
    uint32_t sn = 0, items = 0, tiles = 0;  // S_u consumed, items with keys, tiles of the CTA
    bool ok = true;
    // The item lies in shared memory: the loop over its tiles has no registers to spare.
    Work& w = *reinterpret_cast<Work*>(reinterpret_cast<uint8_t*>(tmem_slot) + 16 + (warp - 4) * WORK_BYTES);
    for (long long it = blockIdx.x; ok; it += gridDim.x) {
      {
        Work next;
        if (!find_work(next, ky, qr, tl, n_tiles, G, it, lane)) break;
        __syncwarp();
        if (lane == 0) w = next;
        __syncwarp();
      }
      const int nt = w.t1 - w.t0;
      if (u >= w.nsub) {
        tiles += max(nt, 0);
        continue;
      }
      const int i = w.i0 + u * tl.tq + row / qr.group, h = w.hk * qr.group + row % qr.group;
      const bool has_row = row < tl.tq * qr.group && i < w.sp.n;
      const Sees se = sees(qr, w.sp, min(i, w.sp.n - 1));
      float m_run = -INFINITY, l_run = 0.f;
      for (int j = 0; j < nt; ++j, ++sn, ++tiles) {
        ok = warp_wait(&bar_s[u], sn, abort_flag, ST_PAGED_SOFTMAX);
        if (!ok) break;
        tc_fence_after();
        const uint32_t m = tiles % META;
        const uint4 lv = *reinterpret_cast<const uint4*>(live + m * 4);
        const int k0 = first_key[m];
        float s[BN];
        {
          uint32_t r[64];
          tmem_ld32x32b_x64(tS, r);
#pragma unroll
          for (int k = 0; k < 64; ++k) s[k] = __uint_as_float(r[k]);
          tmem_ld32x32b_x64(tS + 64, r);
#pragma unroll
          for (int k = 0; k < 64; ++k) s[64 + k] = __uint_as_float(r[k]);
        }
        if constexpr (KV8) {
          const float4* ks = reinterpret_cast<const float4*>(scales + m * 2 * BN);
#pragma unroll
          for (int k = 0; k < BN / 4; ++k) {
            const float4 x = ks[k];
            const float2 a = fmul2(make_float2(s[4 * k], s[4 * k + 1]), make_float2(x.x, x.y));
            const float2 b = fmul2(make_float2(s[4 * k + 2], s[4 * k + 3]), make_float2(x.z, x.w));
            s[4 * k] = a.x, s[4 * k + 1] = a.y, s[4 * k + 2] = b.x, s[4 * k + 3] = b.y;
          }
        }
        // Which of the tile's keys this row sees.  128 live keys lie at
        // consecutive positions, whatever the page size.
        const bool whole = (lv.x & lv.y & lv.z & lv.w) == 0xFFFFFFFFu && k0 + BN <= se.hi &&
                           (k0 >= se.lo || k0 + BN <= se.sink);
        const bool masked = !__all_sync(0xffffffffu, whole);
        uint32_t keep[4] = {lv.x, lv.y, lv.z, lv.w};
        if (masked) {
          const TileAt at = tile_at(tl, nth_tile(w, w.t0 + j));
          const int b_hi = rows_below(tl, at, se.hi), b_lo = rows_below(tl, at, se.lo);
          const int b_sink = rows_below(tl, at, se.sink);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            keep[c] &= bit_range(b_lo, b_hi, c * 32) | bit_range(0, b_sink, c * 32);
#pragma unroll
            for (int k = 0; k < 32; ++k)
              if (!(keep[c] >> k & 1)) s[c * 32 + k] = -INFINITY;
          }
        }
        // Row maximum, in four chains.
        float mx;
        {
          float mc[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) mc[c] = max3_nan(s[c], s[4 + c], s[4 + c]);
#pragma unroll
          for (int k = 8; k < BN; k += 8)
#pragma unroll
            for (int c = 0; c < 4; ++c) mc[c] = max3_nan(mc[c], s[k + c], s[k + 4 + c]);
          mx = max3_nan(max3_nan(mc[0], mc[1], mc[2]), mc[3], mc[3]);
        }
        const float mx2 = mx * qr.scale_log2;
        // O is rescaled only when the maximum grows by more than 2^8; l and O
        // use the same stale maximum, so the quotient does not change.
        float m_new = m_run;
        bool grow = false;
        if (mx2 > m_run + 8.f || (m_run == -INFINITY && mx2 > -INFINITY)) {
          m_new = mx2;
          grow = true;
        }
        if (!(mx2 < INFINITY)) m_new = __uint_as_float(0x7FC00000u);  // NaN or +inf score: the row is NaN from here on
        const float m_use = m_new == -INFINITY ? 0.f : m_new;         // nothing seen yet
        const float2 sc2 = make_float2(qr.scale_log2, qr.scale_log2);
        const float2 nm2 = make_float2(-m_use, -m_use);
        float2 sum[4] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        uint32_t pk[BN / 2];
        float4 vs;
        // P = 2^(s * scale - m), 3 of 8 pairs on the FMA pipe's polynomial, the
        // rest on MUFU; l sums P before its rounding to bf16.
#pragma unroll
        for (int k = 0; k < BN / 2; ++k) {
          const float2 x = ffma2(make_float2(s[2 * k], s[2 * k + 1]), sc2, nm2);
          float2 p;
          if ((k & 7) < 3) {
            p = exp2_poly2(x);
          } else {
            p.x = ex2_approx(x.x);
            p.y = ex2_approx(x.y);
          }
          sum[k & 3] = fadd2(sum[k & 3], p);
          if constexpr (KV8) {
            if ((k & 1) == 0) vs = *reinterpret_cast<const float4*>(scales + m * 2 * BN + BN + 2 * k);
            p = fmul2(p, (k & 1) ? make_float2(vs.z, vs.w) : make_float2(vs.x, vs.y));
          }
          pk[k] = pack_bf16x2(p.x, p.y);
        }
        if (masked) {  // the polynomial's smallest value, and a NaN scale, must not count
#pragma unroll
          for (int k = 0; k < BN / 2; ++k) {
            const uint32_t two = keep[k >> 4] >> ((2 * k) & 31) & 3;
            pk[k] &= ((two & 1) ? 0xFFFFu : 0u) | ((two & 2) ? 0xFFFF0000u : 0u);
          }
        }
        const float2 s2 = fadd2(fadd2(sum[0], sum[1]), fadd2(sum[2], sum[3]));
        const float alpha = grow ? ex2_approx(m_run - m_new) : 1.f;
        if (j > 0 && __any_sync(0xffffffffu, grow)) {
#pragma unroll
          for (int c = 0; c < HD; c += 32) {
            uint32_t r[32];
            tmem_ld32x32b_x32(tO + c, r);
#pragma unroll
            for (int k = 0; k < 32; ++k) r[k] = __float_as_uint(__uint_as_float(r[k]) * alpha);
            tmem_st32x32b_x32(tO + c, r);
          }
        }
        l_run = l_run * alpha + (s2.x + s2.y);
        m_run = m_new;
        tmem_st32x32b_x64(tS, pk);
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(&bar_p[u]);
      }
      if (!ok) break;
      if (nt > 0) {
        ok = warp_wait(&o_full[u], items, abort_flag, ST_PAGED_SOFTMAX);
        if (!ok) break;
        ++items;
        tc_fence_after();
      }
      const bool none = m_run == -INFINITY;
      const float inv = none ? 0.f : m_run != m_run ? m_run : 1.f / l_run;
      const int64_t packed = (int64_t)(w.sp.first + i) * qr.H + h;
      const float lse2 = none ? -INFINITY : m_run + log2f(l_run);
      if (tl.splits > 1) {
        const int64_t at = (int64_t)w.split * qr.rows * qr.H + packed;
        if (has_row) part_l[at] = lse2;
        if (nt > 0) {
#pragma unroll
          for (int c = 0; c < HD; c += 32) {
            uint32_t r[32];
            tmem_ld32x32b_x32(tO + c, r);
            if (has_row && !none) {
              float4* d = reinterpret_cast<float4*>(part_o + at * HD + c);
#pragma unroll
              for (int v = 0; v < 8; ++v)
                d[v] = make_float4(__uint_as_float(r[4 * v]) * inv, __uint_as_float(r[4 * v + 1]) * inv,
                                   __uint_as_float(r[4 * v + 2]) * inv, __uint_as_float(r[4 * v + 3]) * inv);
            }
          }
        }
      } else {
        if (has_row && qr.lse) qr.lse[packed] = lse2 * 0.6931471805599453f;
        const int64_t orow = ky.cross ? w.b * qr.o_str[0] + i * qr.o_str[1] : (int64_t)(w.sp.first + i) * qr.o_str[1];
        uint4* d = reinterpret_cast<uint4*>(qr.o + (has_row ? orow + h * qr.o_str[2] : 0));
#pragma unroll
        for (int c = 0; c < HD; c += 32) {
          uint32_t r[32];
          if (nt > 0) tmem_ld32x32b_x32(tO + c, r);
          if (has_row) {
#pragma unroll
            for (int v = 0; v < 4; ++v) {
              auto two = [&](int k) {
                return none ? 0u : pack_bf16x2(__uint_as_float(r[k]) * inv, __uint_as_float(r[k + 1]) * inv);
              };
              d[c / 8 + v] = make_uint4(two(8 * v), two(8 * v + 2), two(8 * v + 4), two(8 * v + 6));
            }
          }
        }
      }
      // the next tile's arrival on bar_p lets PV overwrite O, which is in registers here
    }
    teardown();
  } else {
    // ------------------------------------------------------ code expansion
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;\n" ::: "memory");
    if constexpr (KV8) {
      uint32_t slot_n = 0;
      bool ok = true;
      Work w;
      for (long long it = blockIdx.x; ok && find_work(w, ky, qr, tl, n_tiles, G, it, lane); it += gridDim.x) {
        for (int n = 2 * (w.t1 - w.t0); ok && n > 0; --n) {
          const uint32_t s = slot_n % NS;
          if (!(ok = warp_wait(&raw[s], slot_n / NS, abort_flag, ST_PAGED_EXPAND))) break;
          expand_rows<DT>(ring + s * SLOT, (warp - 12) * 32, lane);
          fence_proxy_async_smem();
          mbar_arrive(&full[s]);
          ++slot_n;
        }
      }
    }
    teardown();
  }
}

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
  for (int s = 0; s < splits; ++s) m = max3_nan(m, part_l[s * n + at], -INFINITY);
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

// --------------------------------------------------------------------- host
// What the host knows of a call's size.
static int64_t tiles_bound(const Shape& sh) {
  const int step = 2 * (BM / sh.group);
  if (sh.cross) return (int64_t)sh.seqs * ((sh.Lq + step - 1) / step);
  const int64_t seqs = sh.rows < sh.seqs ? sh.rows : sh.seqs;
  return (sh.rows + seqs * (step - 1)) / step;
}
static int64_t key_tiles(const Shape& sh) {
  const int rows = (sh.page_size + 7) & ~7;
  const int64_t pages = (sh.keys + sh.page_size - 1) / sh.page_size;
  return sh.page_size >= BN ? pages * ((sh.page_size + BN - 1) / BN) : (pages + BN / rows - 1) / (BN / rows);
}

// Splits of the keys: the count that gives the least time for the slowest SM,
// one key tile taking about 1.4 us, an item's start and end about two tiles,
// and the join its launch and one f32 row written and read a split.
int tile_splits(const Shape& sh) {
  const int64_t items = tiles_bound(sh) * (sh.H / sh.group), nt = key_tiles(sh);
  int best = 1;
  double best_us = 1e30;
  for (int s = 1; s <= 32 && (s == 1 || 2 * s <= nt); ++s) {
    const double waves = (double)((items * s + SMS - 1) / SMS);
    double us = waves * (double)((nt + s - 1) / s + 2) * 1.4;
    if (s > 1) us += 3.0 + (double)s * sh.rows * sh.H * (2 * HD * 4) * 2e-7;
    if (us < best_us * 0.98) best_us = us, best = s;
  }
  return best;
}

template <int DT>
static int start(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const Keys& ky,
                 const Queries& qr, const Tiling& tl, unsigned grid, float* part_o, float* part_l, cudaStream_t st) {
  using C = Cfg<DT != WF_DTYPE_BF16>;
  static thread_local int configured = -1;
  int dev = 0;
  WFK_CUDA_TRY(cudaGetDevice(&dev));
  if (configured != dev) {
    WFK_CUDA_TRY(cudaFuncSetAttribute(tile_kernel<DT>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
    configured = dev;
  }
  tile_kernel<DT><<<grid, C::THREADS, C::SMEM, st>>>(tq, tk, tv, ky, qr, tl, part_o, part_l);
  WFK_CUDA_TRY(cudaGetLastError());
  return WF_OK;
}

int tile_launch(const Keys& ky, const Queries& qr, const Shape& sh, void* workspace, cudaStream_t st) {
  const int G = qr.H / qr.group, ps = ky.page_size;
  Tiling tl;
  tl.ps = ps;
  tl.tpp = (ps + BN - 1) / BN;
  tl.rows = ps >= BN ? BN : (ps + 7) & ~7;
  tl.ppt = ps >= BN ? 1 : BN / tl.rows;
  tl.tq = BM / qr.group;
  tl.splits = tile_splits(sh);
  const bool kv8 = ky.dtype != WF_DTYPE_BF16;
  CUtensorMap tq, tk, tv;
  int rc;
  {
    const uint64_t dim[4] = {HD, (uint64_t)qr.H, (uint64_t)(ky.cross ? qr.Lq : qr.rows),
                             (uint64_t)(ky.cross ? qr.seqs : 1)};
    const uint64_t str[3] = {(uint64_t)qr.q_str[2] * 2, (uint64_t)qr.q_str[1] * 2,
                             (uint64_t)(ky.cross ? qr.q_str[0] * 2 : 16)};
    const uint32_t box[4] = {64, (uint32_t)qr.group, (uint32_t)tl.tq, 1};
    if ((rc = encode_tiled(&tq, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, qr.q, dim, str, box,
                           CU_TENSOR_MAP_SWIZZLE_128B)) != WF_OK)
      return rc;
  }
  const uint64_t dim[4] = {HD, (uint64_t)ps, (uint64_t)G, (uint64_t)ky.n_pages};
  const uint32_t box[4] = {kv8 ? 128u : 64u, (uint32_t)tl.rows, 1, 1};
  const uint64_t elem = kv8 ? 1 : 2;
  for (int i = 0; i < 2; ++i) {
    const int64_t* s = i ? ky.v_str : ky.k_str;
    const uint64_t str[3] = {(uint64_t)s[2] * elem, (uint64_t)s[1] * elem, (uint64_t)s[0] * elem};
    if ((rc = encode_tiled(i ? &tv : &tk, kv8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
                           i ? ky.v : ky.k, dim, str, box, CU_TENSOR_MAP_SWIZZLE_128B)) != WF_OK)
      return rc;
  }
  const int64_t items = tiles_bound(sh) * G * tl.splits;
  if (items > INT_MAX) return fail(WF_ERR_INVALID_ARG, "attention: too many query tiles (%lld)", (long long)items);
  // Few key tiles to an item: one CTA per SM walks the items, the next one's
  // loads under the last one's end.  Many: a CTA per item, so that the SM that
  // is done first takes the next.
  const unsigned grid = (unsigned)(key_tiles(sh) / tl.splits < 8 && items > SMS ? SMS : items);
  float *part_o = nullptr, *part_l = nullptr;
  if (tl.splits > 1) {
    part_o = static_cast<float*>(workspace);
    part_l = part_o + (int64_t)tl.splits * qr.rows * qr.H * HD;
  }
  rc = ky.dtype == WF_DTYPE_BF16   ? start<WF_DTYPE_BF16>(tq, tk, tv, ky, qr, tl, grid, part_o, part_l, st)
       : ky.dtype == WF_DTYPE_E4M3 ? start<WF_DTYPE_E4M3>(tq, tk, tv, ky, qr, tl, grid, part_o, part_l, st)
                                   : start<WF_DTYPE_S8>(tq, tk, tv, ky, qr, tl, grid, part_o, part_l, st);
  if (rc != WF_OK || tl.splits == 1) return rc;
  join_kernel<<<(unsigned)(((int64_t)qr.rows * qr.H + 7) / 8), 256, 0, st>>>(ky, qr, part_o, part_l, tl.splits);
  WFK_CUDA_TRY(cudaGetLastError());
  return WF_OK;
}

}  // namespace tile
}  // namespace paged
}  // namespace wfk

extern "C" unsigned int wfk_status_take_paged_tile(void) { return wfk::status_take_local(); }
