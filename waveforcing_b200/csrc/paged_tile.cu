// Attention over pages on tcgen05 for calls with many query rows.
//
// Work item = two sub-tiles of 128 query rows of one K/V head (rows of a
// sub-tile: TQ = 128 / group tokens x the group's query heads) against a run
// of 128-key tiles.  K and V tiles are loaded once for both sub-tiles.
//   warp 0       TMA producer (a lane to a box of a tile)
//   warp 1       MMA issue: S_u = Q_u K_j^T (M=N=K=128), O_u += P_u V_j
//   warp 2       marks the live keys of each tile; bf16: zeroes the V rows of
//                the others (their P is 0, but 0 * NaN is not), and what is not
//                finite in tiles that some rows see and others do not (the rows
//                that do get it back at their end); 8 bits: fetches scales, a
//                tile ahead of the codes
//   warp 3       finds the CTA's items ahead of the other roles
//   warps 4-11   softmax; warpgroup u owns sub-tile u, a thread a row
//   warps 12-15  (8-bit pages) expand codes to f16
// TMEM columns: S_0 [0,128) S_1 [128,256) O_0 [256,384) O_1 [384,512); P_u
// (16 bits) overwrites the first half of S_u, which its warpgroup holds in
// registers by then.  The tensor pipe runs in issue order, PV_0(j) QK_0(j+1)
// PV_1(j) QK_1(j+1) ..., so QK_u(j+1) overwrites P_u(j) only after PV_u(j) has
// read it, and S_u(j+1) complete means that PV_u(j) is: O_u may be rescaled.
// While one sub-tile's products run, the other's exponentials do.
//
// 8-bit pages: both contractions run on f16 operands, whose 11 bits hold
// code * scale to 2^-11 where bf16 would round to 2^-8, with the range taken
// care of by powers of two: Q rows are scaled to at most 1, each K tile by its
// largest row scale, V by the largest so far (O is rescaled when that grows);
// the powers return in the softmax scale and in the last factor of O.  A
// scale per key applied to S and P instead costs two shared-memory reads of
// 512 bytes a row and tile: 525 against 398 us without at 9472 x 16384 x 4
// heads, where the rows' reads and the operands' share shared memory.
//
// Measured at that size, through the torch wrapper as all figures here: bf16 247
// us, 1288 TFLOP/s (0.77 of the cuBLAS burst rate), e4m3 315 to 346 us; 4680 x
// 37440 x 12 heads: bf16 912 us over 128-row pages and 1049 over 1560-row ones
// masked by blocks, e4m3 1242 to 1314 us; 6 x 4680 rows over 512 states and 12
// heads 119 us.  A tile takes about 3600 clocks
// where its products take 2048: a warp's chain from S to P (load, maximum,
// exponentials, store) is as long as the other sub-tile's products cover.  8-bit
// pages: the expansion, with twice the instructions (197 against 104 million at
// that size, issue slots 59 % busy against 42 %) and its shared-memory traffic.
#include <cuda_fp16.h>

#include <cmath>
#include <type_traits>

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
// O is rescaled only when a row's maximum grows by more than 2^SLACK (4680 x 14040 x 12
// heads over e4m3, scores of deviation 1: 550 us; with 4, which would leave P over 8-bit
// pages more of f16's range, 601).
constexpr float SLACK = 8.f;

constexpr int WORK_BYTES = 96, WORKS = 4;  // items found ahead
template <bool KV8>
struct Cfg {
  static constexpr int NS = KV8 ? 4 : 5;  // ring slots
  static constexpr int THREADS = KV8 ? 512 : 384;
  static constexpr int READERS = KV8 ? 15 : 11;  // warps that an item goes to
  static constexpr int NBARS = (3 * NS + 14 + 2 * META + 2 * WORKS + 1 + 1) & ~1;  // even: what follows is 16-byte aligned
  static constexpr int META_BYTES = META * (16 + (KV8 ? 2 * BN * 4 : 0) + 16) + (KV8 ? 4 * BM * 4 : 0);
  static constexpr int SMEM = 1024 + 2 * SLOT + NS * SLOT + NBARS * 8 + META_BYTES + 16 + WORKS * WORK_BYTES;
  static_assert(SMEM <= 232448, "shared memory of one CTA");
};

struct Work : Range {
  int b, hk, split;  // b < 0: no more items
  int i0, nsub;      // first token, sub-tiles with rows
  Span sp;
  int t0, t1;        // this item's share of the tile list
  int slot;          // its partial rows' place in the workspace, -1: none (see Deal)
};
static_assert(sizeof(Work) + 4 <= WORK_BYTES, "room for an item");

// Page (of the sequence) and row of key r of a tile; false: a hole.
template <int N>
__device__ __forceinline__ bool place(const Tiling& tl, const TileAt& a, int r, int& page, int& row) {
  page = a.page;
  row = a.row + r;
  if (tl.dense) {
    if (row >= tl.ps) {
      const int j = page_of(tl, row);
      page += j;
      row -= j * tl.ps;
    }
  } else if (tl.ps < N) {
    const int j = r / tl.rows;
    page += j;
    row = r - j * tl.rows;
    if (j >= tl.boxes) return false;
  }
  return row < tl.ps;
}

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

// Run p of s of n tiles starts here.
__device__ __forceinline__ int run_start(int n, int p, int s) { return n / s * p + n % s * p / s; }

// The item of query tile `tile` of sequence w.b (w.sp) and head w.hk, with all of its key tiles.
__device__ __forceinline__ void fill_work(Work& w, const Queries& qr, const Tiling& tl, int tile) {
  w.i0 = tile * 2 * tl.tq;
  const int i1 = min(w.i0 + 2 * tl.tq, w.sp.n) - 1;  // last token
  w.nsub = i1 >= w.i0 + tl.tq ? 2 : 1;
  static_cast<Range&>(w) = range_of<BN>(qr, w.sp, tl, w.i0, i1);
  w.t0 = 0;
  w.t1 = w.n;
  w.slot = -1;
}

// Item `it` of a launch whose items are taken from the longest to the shortest,
// all K/V heads of a query tile in turn (one warp, at most 32 sequences and MANY
// query tiles): a lane finds the lengths of up to MANY / 32 query tiles, and
// the one that it / G others are longer than is taken.
constexpr int MANY = 128;
__device__ __forceinline__ bool nth_longest(Work& w, const Keys& ky, const Queries& qr, const Tiling& tl, int n_tiles,
                                            int G, unsigned it, int lane) {
  if (it >= (unsigned)n_tiles * G) return false;
  Span mine{};
  if (lane < qr.seqs) mine = span_of(ky, qr, lane);
  const int nq = (mine.n + 2 * tl.tq - 1) / (2 * tl.tq);
  int before = nq;  // query tiles of the sequences before this lane's
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, before, o);
    if (lane >= o) before += x;
  }
  before -= nq;
  int key[MANY / 32], longer[MANY / 32];
#pragma unroll
  for (int k = 0; k < MANY / 32; ++k) {
    key[k] = -1;
    longer[k] = 0;
    if (k * 32 >= n_tiles) continue;
    const int q = k * 32 + lane;
    int b = 0;
#pragma unroll 1
    for (int x = 1; x < qr.seqs; ++x) b = __shfl_sync(0xffffffffu, before, x) <= q ? x : b;
    w.sp.first = __shfl_sync(0xffffffffu, mine.first, b);
    w.sp.n = __shfl_sync(0xffffffffu, mine.n, b);
    w.sp.len = __shfl_sync(0xffffffffu, mine.len, b);
    w.sp.pos0 = __shfl_sync(0xffffffffu, mine.pos0, b);
    const int tile = q - __shfl_sync(0xffffffffu, before, b);
    if (q >= n_tiles) continue;
    fill_work(w, qr, tl, tile);
    key[k] = min(w.n, 1 << 23) * MANY + MANY - 1 - q;  // no two alike
  }
#pragma unroll
  for (int k = 0; k < MANY / 32; ++k) {
    if (k * 32 >= n_tiles) continue;
#pragma unroll 1
    for (int x = 0; x < 32; ++x) {
      const int other = __shfl_sync(0xffffffffu, key[k], x);
#pragma unroll
      for (int y = 0; y < MANY / 32; ++y) longer[y] += other > key[y];
    }
  }
  int q = 0;
#pragma unroll
  for (int k = 0; k < MANY / 32; ++k) {
    const uint32_t here = __ballot_sync(0xffffffffu, key[k] >= 0 && longer[k] == (int)(it / (unsigned)G));
    if (here) q = k * 32 + __ffs(here) - 1;
  }
  w.b = 31 - __clz(__ballot_sync(0xffffffffu, lane < qr.seqs && before <= q));
  w.hk = it % (unsigned)G;
  w.sp = span_of(ky, qr, w.b);
  fill_work(w, qr, tl, q - __shfl_sync(0xffffffffu, before, w.b));
  return true;
}

// Item `it` of the launch (one warp, same result in every lane).
__device__ __forceinline__ bool find_work(Work& w, const Keys& ky, const Queries& qr, const Tiling& tl, int n_tiles,
                                          int G, unsigned it, int lane) {
  if (n_tiles == 0 || it >= (unsigned)n_tiles * G * tl.splits) return false;
  int tile = it % (unsigned)n_tiles;
  const int rest = it / (unsigned)n_tiles;
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
  w.sp = span_of(ky, qr, w.b);
  fill_work(w, qr, tl, nq - 1 - tile);  // a causal sequence's longest rows first
  if (tl.splits > 1) {  // at most 32 of them
    w.t0 = run_start(w.n, w.split, tl.splits);
    w.t1 = run_start(w.n, w.split + 1, tl.splits);
  }
  return true;
}

// One sequence whose rows all see the same keys: its items take the same time,
// n tiles each.  Whole rounds of them go to the CTAs in turn; the `left` others
// are cut into `parts` runs of keys and those dealt in turn, run by run, so that
// the CTAs of a moment share K and V through L2 (with one contiguous stretch of
// tiles to a CTA instead, the loads of 12 heads came from HBM: 833 against 605
// us).  4680 rows and 12 heads are 228 items: 148, then 80 in parts.
struct Deal {
  bool even;
  int n, full, left, parts;  // tiles of an item; items dealt whole, the others, their parts
};
constexpr int MAX_SLOTS = 4 * SMS;  // parts that the workspace holds
// The number of parts with the least estimated time, in hundredths of a tile's:
// four tiles for a part's start and end, then the join's launch and traffic.
__host__ __device__ inline int parts_of(int left, int n, int ctas) {
  int best = 1;
  long long least = 0;
  for (int s = 1; s <= 32 && (s == 1 || (2 * s <= n && left * s <= MAX_SLOTS)); ++s) {
    const long long cost = (left * s + ctas - 1) / ctas * ((n + s - 1) / s + 4) * 100ll + (s > 1 ? 200 + left * s : 0);
    if (s == 1 || cost < least) least = cost, best = s;
  }
  return best;
}
__device__ __forceinline__ Deal deal_of(const Keys& ky, const Queries& qr, const Tiling& tl, int n_tiles, int G,
                                        int ctas) {
  Deal d{false, 0, 0, 0, 1};
  if (!tl.even || n_tiles == 0) return d;
  const Span sp = span_of(ky, qr, 0);
  const Sees a = sees(qr, sp, 0), z = sees(qr, sp, sp.n - 1);
  if (sp.pos0 < 0 || a.hi != z.hi || a.lo != z.lo || a.hi == 0) return d;
  d.even = true;
  d.n = range_of<BN>(qr, sp, tl, 0, sp.n - 1).n;
  d.full = n_tiles * G / ctas * ctas;
  d.left = n_tiles * G - d.full;
  if (d.left > 0) d.parts = parts_of(d.left, d.n, ctas);
  return d;
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

// c * (hi + lo) for a pair of codes: the row's scale in 22 bits, so that its
// rounding does not shift all of a key's products the same way.
__device__ __forceinline__ uint32_t scaled_f16x2(uint32_t c, uint32_t hi, uint32_t lo) {
  uint32_t r;
  asm("{\n\t.reg .b32 t;\n\t"
      "mul.rn.f16x2 t, %1, %3;\n\t"
      "fma.rn.f16x2 %0, %1, %2, t;\n\t}"
      : "=r"(r)
      : "r"(c), "r"(hi), "r"(lo));
  return r;
}
__device__ __forceinline__ uint32_t hi_lo_f16(float x) {  // x as the sum of two f16, the larger in the low half
  const float hi = __half2float(__float2half_rn(x));
  return f16x2(hi, x - hi);
}
// Four codes -> four f16 products with the row's scale.
template <int DT>
__device__ __forceinline__ void expand4(uint32_t w, uint32_t s_hi, uint32_t s_lo, uint32_t& lo, uint32_t& hi) {
  if constexpr (DT == WF_DTYPE_E4M3) {
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(lo) : "h"(static_cast<uint16_t>(w)));
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(hi) : "h"(static_cast<uint16_t>(w >> 16)));
  } else {  // 1024 + (c + 128) by its bits, minus 1152: exact
    const uint32_t x = w ^ 0x80808080u;
    const uint32_t a = __byte_perm(x, 0x64646464u, 0x4140), b = __byte_perm(x, 0x64646464u, 0x4342);
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(lo) : "r"(a), "r"(0x64806480u));
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(hi) : "r"(b), "r"(0x64806480u));
  }
  lo = scaled_f16x2(lo, s_hi, s_lo);
  hi = scaled_f16x2(hi, s_hi, s_lo);
}

// Expands the 32 rows of one converter warp of a code tile (128 bytes a row,
// swizzled, in the slot's upper half) in place to two halves of f16 rows.  A
// code row shares its line with the upper f16 row: the eight lanes of a row
// read all of it before any of them writes.  Lanes 4-7 of a row write their
// odd chunk first, so that a row's eight stores meet eight bank groups.
template <int DT>
__device__ __forceinline__ void expand_rows(uint8_t* slot, int row0, int lane, const uint32_t* scale) {
  const int c = lane & 7, hi = c >> 2;
#pragma unroll 1
  for (int i = 0; i < 32; i += 8) {
    uint32_t h[2][8];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int r = row0 + i + 4 * t + (lane >> 3);
      const uint32_t sc = scale[r], s_hi = __byte_perm(sc, 0, 0x1010), s_lo = __byte_perm(sc, 0, 0x3232);
      uint4 raw = *reinterpret_cast<const uint4*>(slot + HALF + r * 128 + ((c ^ (r & 7)) << 4));
      if (sc == 0) raw = make_uint4(0, 0, 0, 0);  // a row that no query sees may hold NaN codes
      const uint32_t w[4] = {hi ? raw.z : raw.x, hi ? raw.w : raw.y, hi ? raw.x : raw.z, hi ? raw.y : raw.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) expand4<DT>(w[k], s_hi, s_lo, h[t][2 * k], h[t][2 * k + 1]);
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

// Q rows of one converter warp (32 of a sub-tile, swizzled bf16) to f16 in
// place, each divided by the power of two above its largest value; the powers
// go to qpow.  Half a warp to a row, 16 bytes a lane.
__device__ __forceinline__ void expand_q(uint8_t* sub, int row0, int lane, float* qpow) {
#pragma unroll 1
  for (int i = 0; i < 32; i += 2) {
    const int r = row0 + i + (lane >> 4);
    uint4* at = reinterpret_cast<uint4*>(sub + ((lane >> 3) & 1) * HALF + r * 128 + (lane & 7) * 16);
    const uint4 v = *at;
    uint32_t w[4] = {v.x, v.y, v.z, v.w};
    float m = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      m = fmaxf(m, fmaxf(fabsf(__uint_as_float(w[k] << 16)), fabsf(__uint_as_float(w[k] & 0xFFFF0000u))));
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float p = pow2_above(fminf(m, 0x1p122f)), inv = 1.f / p;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      w[k] = f16x2(__uint_as_float(w[k] << 16) * inv, __uint_as_float(w[k] & 0xFFFF0000u) * inv);
    *at = make_uint4(w[0], w[1], w[2], w[3]);
    if ((lane & 15) == 0) qpow[r] = p;
  }
}

// 32 bytes: a whole sector in one store where the address allows it (a lane
// writes its own row, so that two halves would be two passes over 32 sectors).
__device__ __forceinline__ void store32(void* to, const uint32_t* r, bool wide) {
  if (wide) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(r[0]), "r"(r[1]), "r"(r[2]),
                 "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
  } else {
    uint4* d = static_cast<uint4*>(to);
    d[0] = make_uint4(r[0], r[1], r[2], r[3]);
    d[1] = make_uint4(r[4], r[5], r[6], r[7]);
  }
}

// Makes the bf16 V tile at v finite; whether it was not (a warp).  Not inlined: in the
// marks' loop it slowed calls without mixed tiles too (4680 x 37440 x 12 heads: 1010 us, 907
// so, 896 without).
__device__ __noinline__ bool make_finite(uint8_t* v, int lane) {
  v += (lane >> 4) * 128 + ((lane >> 3) & 1) * HALF + (lane & 7) * 16;  // half a warp to a row, 16 bytes a lane
  uint32_t odd[4] = {0, 0, 0, 0};  // sums of 0 * x: 0 or NaN
#pragma unroll 4
  for (int r = 0; r < BN; r += 2) {
    const uint4 x = *reinterpret_cast<const uint4*>(v + r * 128);
    odd[0] = fma_bf16x2(x.x, 0u, odd[0]), odd[1] = fma_bf16x2(x.y, 0u, odd[1]);
    odd[2] = fma_bf16x2(x.z, 0u, odd[2]), odd[3] = fma_bf16x2(x.w, 0u, odd[3]);
  }
  if (!__any_sync(0xffffffffu, ((odd[0] | odd[1] | odd[2] | odd[3]) & 0x7FFF7FFFu) != 0)) return false;
#pragma unroll 1
  for (int r = 0; r < BN; r += 2) {
    uint4* at = reinterpret_cast<uint4*>(v + r * 128);
    const uint4 x = *at;
    *at = make_uint4(finite2(x.x), finite2(x.y), finite2(x.z), finite2(x.w));
  }
  fence_proxy_async_smem();
  __syncwarp();
  return true;
}

// MIXED: bf16 pages of rows that may see different keys (a mask by blocks; without one
// and in cross attention a row sees what every other does, or nothing).
template <int DT, bool SORTED, bool MIXED>
__global__ void __launch_bounds__(Cfg<DT != WF_DTYPE_BF16>::THREADS, 1)
    tile_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ PageMaps tm,
                const __grid_constant__ Keys ky,
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
  uint64_t* bar_p = bar_s + 2;       // [2][2] P_u written, by halves of the keys
  uint64_t* o_full = bar_p + 4;      // [2] the item's last PV_u has completed
  uint64_t* bar_fin = o_full + 2;
  uint64_t* q_raw = bar_fin + 1;     // [2] 8-bit pages: Q_u landed (q_full: as f16)
  uint64_t* marked = q_raw + 2;      // [META] 8-bit pages: a tile's scales are there
  uint64_t* unmarked = marked + META;  // [META] and have been used: P V of the tile is done
  uint64_t* work_full = unmarked + META;  // [WORKS] an item is there
  uint64_t* work_empty = work_full + WORKS;
  uint32_t* live = reinterpret_cast<uint32_t*>(raw + Cfg<KV8>::NBARS);  // [META][4] live keys of a tile
  int* whole = reinterpret_cast<int*>(live + META * 4);                 // [META] every row sees all of it
  float* kpow = reinterpret_cast<float*>(whole + META);                 // [META] power of two of the K tile
  float* vpow = kpow + META;                                            // [META] and of V up to this tile
  uint32_t* scales = reinterpret_cast<uint32_t*>(vpow + 2 * META);      // [META][2][BN] hi_lo_f16
  float* qpow = reinterpret_cast<float*>(scales + META * 2 * BN);       // [2][2][BM], by turns of the sub-tile's items
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(reinterpret_cast<uint8_t*>(live) + Cfg<KV8>::META_BYTES);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  Work* works = reinterpret_cast<Work*>(reinterpret_cast<uint8_t*>(tmem_slot) + 16);  // [WORKS]
  volatile int* odd_v = reinterpret_cast<volatile int*>(works + WORKS);  // [WORKS] V of a mixed tile of the item is not finite

  // Values that steer the roles are broadcast from lane 0, by which the compiler
  // knows them to be the same in a warp: the MMA warp's operands then stay in
  // uniform registers (issue at 115 clocks an instruction otherwise).
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int G = qr.H / qr.group;

  if (threadIdx.x == 0) {
    for (int s = 0; s < NS; ++s) {
      mbar_init(&raw[s], 1);
      mbar_init(&full[s], KV8 ? 128 : 1);
      mbar_init(&empty[s], 1);
    }
    for (int u = 0; u < 2; ++u) {
      mbar_init(&q_full[u], KV8 ? 128 : 1);
      mbar_init(&q_raw[u], 1);
      mbar_init(&q_empty[u], 1);
      mbar_init(&bar_s[u], 1);
      mbar_init(&bar_p[2 * u], 128);
      mbar_init(&bar_p[2 * u + 1], 128);
      mbar_init(&o_full[u], 1);
    }
    for (int m = 0; m < META; ++m) {
      mbar_init(&marked[m], 1);
      mbar_init(&unmarked[m], 1);
    }
    for (int k = 0; k < WORKS; ++k) {
      mbar_init(&work_full[k], 1);
      mbar_init(&work_empty[k], Cfg<KV8>::READERS);
    }
    mbar_init(bar_fin, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  // Rows of Q behind the sub-tiles' tokens (groups that do not divide 128) are never
  // loaded.  Zeros: a NaN left there by an earlier kernel would have its warp rescale O
  // at every tile (3108 x 16384 x 12 heads on 4 over e4m3: 595 us for 314).
  const int q_rows = tl.tq * qr.group;
  for (int i = threadIdx.x; i < (BM - q_rows) * 32; i += Cfg<KV8>::THREADS) {
    const int r = q_rows + (i >> 5), c = i & 31;  // 16 bytes of a row of a half of a sub-tile
    *reinterpret_cast<uint4*>(sQ + (c >> 3) * HALF + r * 128 + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
  }
  fence_proxy_async_smem();
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tbase = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  // Items, as warp 3 found them: `take` copies the next one and frees its place;
  // `next_work` leaves it there until `done_with`.
  uint32_t work_n = 0;
  auto next_work = [&]() -> bool {
    const uint32_t k = work_n % WORKS;
    if (!warp_wait(&work_full[k], work_n / WORKS, abort_flag, ST_PAGED_WORK)) return false;
    ++work_n;
    return works[k].b >= 0;
  };
  auto done_with = [&]() {
    __syncwarp();
    if (lane == 0) mbar_arrive(&work_empty[(work_n - 1) % WORKS]);
  };
  auto take = [&](Work& w) -> bool {
    if (!next_work()) return false;
    w = works[(work_n - 1) % WORKS];
    done_with();
    return true;
  };

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
      // The next tile's page ids as the table has them (INT_MIN: not needed),
      // looked up under the last tile's loads: one, or a lane to a box.
      int nx_id = INT_MIN, nx_row = 0;
      bool nx_one = false;
      auto look = [&](const TileAt& a) {
        nx_one = one_box<BN>(tl, a);
        if (nx_one) {
          nx_row = a.row;
          nx_id = page_id(ky, w.sp, w.b, a.page);
        } else {
          const Box x = box_at<BN>(tl, a, lane);
          nx_row = x.row;
          nx_id = lane < tl.boxes && needed(w, x.pos, min(tl.rows, tl.ps - x.row)) ? page_id(ky, w.sp, w.b, x.page) : INT_MIN;
        }
      };
      auto load = [&](const CUtensorMap* one, const CUtensorMap* box, int id, int row, bool whole) -> bool {
        const uint32_t s = slot_n % NS, n = slot_n / NS;
        if (n > 0 && !warp_wait(&empty[s], n - 1, abort_flag, ST_PAGED_PRODUCER)) return false;
        uint8_t* dst = ring + s * SLOT + (KV8 ? HALF : 0);
        if (whole) {  // one page: operands in uniform registers
          const int uid = __shfl_sync(0xffffffffu, id, 0), urow = __shfl_sync(0xffffffffu, row, 0);
          if (elect_one()) {
            mbar_arrive_expect_tx(&raw[s], uid < 0 ? 0 : KV8 ? HALF : SLOT);
            if (uid >= 0) {
              tma_load_4d(dst, one, &raw[s], 0, urow, w.hk, uid);
              if constexpr (!KV8) tma_load_4d(dst + HALF, one, &raw[s], 64, urow, w.hk, uid);
            }
          }
        } else {
          const uint32_t bytes = (uint32_t)tl.rows * 128;
          const uint32_t some = __popc(__ballot_sync(0xffffffffu, id >= 0));
          if (lane == 0) mbar_arrive_expect_tx(&raw[s], some * bytes * (KV8 ? 1 : 2));
          __syncwarp();
          if (id >= 0) {
            tma_load_4d(dst + lane * bytes, box, &raw[s], 0, row, w.hk, id);
            if constexpr (!KV8) tma_load_4d(dst + HALF + lane * bytes, box, &raw[s], 64, row, w.hk, id);
          }
        }
        __syncwarp();
        ++slot_n;
        return true;
      };
      for (; ok && take(w); ) {
        if (w.t1 <= w.t0) continue;
        for (int u = 0; ok && u < w.nsub; ++u) {
          if (qn[u] > 0 && !(ok = warp_wait(&q_empty[u], qn[u] - 1, abort_flag, ST_PAGED_PRODUCER))) break;
          if (lane == 0) {
            uint64_t* bar = KV8 ? &q_raw[u] : &q_full[u];
            mbar_arrive_expect_tx(bar, 2 * tl.tq * qr.group * 128);
            const int i = w.i0 + u * tl.tq, row = ky.cross ? i : w.sp.first + i, entry = ky.cross ? w.b : 0;
            tma_load_4d(sQ + u * SLOT, &tmQ, bar, 0, w.hk * qr.group, row, entry);
            tma_load_4d(sQ + u * SLOT + HALF, &tmQ, bar, 64, w.hk * qr.group, row, entry);
          }
          ++qn[u];
        }
        Walk<BN> walk(w, tl, w.t0);
        look(walk.a);
        for (int i = w.t0; ok && i < w.t1; ++i) {
          const bool whole = nx_one;
          const int row = nx_row, id = nx_id >= 0 && nx_id < ky.n_pages ? nx_id : -1;
          if (!(ok = load(&tm.k_tile, &tm.k, id, row, whole) && load(&tm.v_tile, &tm.v, id, row, whole))) break;
          if (i + 1 < w.t1) {
            walk.next();
            look(walk.a);
          }
        }
      }
      if (*abort_flag && lane == 0) {
        // let the copies in flight land before the CTA exits
        for (int u = 0; u < 2; ++u)
          if (qn[u] > 0) drain(KV8 ? &q_raw[u] : &q_full[u], qn[u] - 1, 200000000ull);
        for (uint32_t n = slot_n > NS ? slot_n - NS : 0; n < slot_n; ++n) drain(&raw[n % NS], n / NS, 200000000ull);
      }
    } else if (warp == 1) {
      // ----------------------------------------------------------------- MMA
      constexpr uint32_t FMT = KV8 ? FMT_F16 : FMT_BF16;
      constexpr uint32_t idesc_qk = make_idesc(1, FMT, FMT, 0, BM, BN);
      constexpr uint32_t idesc_pv = make_idesc(1, FMT, FMT, 1, BM, HD);
      uint32_t slot_n = 0, items[2] = {0, 0}, pn[2] = {0, 0}, tiles = 0;
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
      auto pv = [&](int u, uint32_t slot, int half, bool add) {
        const uint64_t dV = desc_sw128(smem_u32(ring + (slot % NS) * SLOT), HALF, 1024);
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < BN / 32; ++k) {
            const int kk = half * (BN / 32) + k;
            umma_f16_ts(tbase + COL_O + u * HD, tbase + COL_S + u * BN + kk * 8, dV + kk * 128, idesc_pv,
                        (add || k > 0) ? 1u : 0u);
          }
        }
        __syncwarp();
      };
      for (; ok && take(w); ) {
        const int nt = __shfl_sync(0xffffffffu, w.t1 - w.t0, 0);
        if (nt <= 0) continue;
        const int nsub = __shfl_sync(0xffffffffu, w.nsub, 0), last_u = nsub - 1;
        if (!wait(&full[slot_n % NS], slot_n / NS)) break;
        for (int u = 0; u < nsub; ++u) {
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
          for (int u = 0; u < nsub; ++u) {
            // P_u of an item's first tile also says that the last item's O_u has been read
            if (!wait(&bar_p[2 * u], pn[u])) break;
            tc_fence_after();
            pv(u, sv, 0, j > 0);
            if (!wait(&bar_p[2 * u + 1], pn[u])) break;
            tc_fence_after();
            pv(u, sv, 1, true);
            ++pn[u];
            if (elect_one()) {
              if (u == last_u) umma_commit(&empty[sv % NS]);
              if (KV8 && u == last_u) umma_commit(&unmarked[tiles % META]);
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
          ++tiles;
        }
        for (int u = 0; u < nsub; ++u) ++items[u];
      }
      // nothing of ours may still be running when TMEM is released
      if (elect_one()) {
        umma_commit(bar_fin);
        drain(bar_fin, 0, 200000000ull);
      }
    } else if (warp == 2 && !KV8) {
      // --------------------------------------------------------------- marks
      // Page ids are fetched two tiles ahead and a tile marked one ahead, so that
      // no latency lies between the waits.
      uint32_t slot_n = 0, tiles = 0;
      bool ok = true;
      TileAt nx_at{};
      int ids[4];  // pages of keys c * 32 + lane of the tile to fetch next (a one-box tile: all the same)
      // Pages that divide a tile begin with it: a key's page and row there are fixed.
      const bool even = tl.dense && BN % tl.ps == 0;
      int sub[4], sub_row[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        sub[c] = even ? (c * 32 + lane) / tl.ps : 0;
        sub_row[c] = c * 32 + lane - sub[c] * tl.ps;
      }
      // Key r of a tile: page and row, and whether some row of the item sees it.
      auto key = [&](const TileAt& a, int r, int& page, int& row) -> bool {
        return place<BN>(tl, a, r, page, row) && seen(w, page * tl.ps + row);
      };
      auto look = [&](const TileAt& a) {
        nx_at = a;
        if (one_box<BN>(tl, a)) {
          ids[0] = page_id(ky, w.sp, w.b, a.page);
        } else if (even && inside<BN>(w, a)) {
#pragma unroll
          for (int c = 0; c < 4; ++c) ids[c] = page_id(ky, w.sp, w.b, a.page + sub[c]);
        } else {
          int page, row;
#pragma unroll
          for (int c = 0; c < 4; ++c) ids[c] = key(a, c * 32 + lane, page, row) ? page_id(ky, w.sp, w.b, page) : INT_MIN;
        }
      };
      // The tile's live keys.
      auto fetch = [&](uint32_t (&words)[4]) {
        const TileAt a = nx_at;
        const bool one = one_box<BN>(tl, a);
        if (one && ids[0] >= 0 && ids[0] < ky.n_pages && inside<BN>(w, a) && a.row + BN <= tl.ps && !ky.mask) {
#pragma unroll
          for (int c = 0; c < 4; ++c) words[c] = 0xFFFFFFFFu;
        } else if (even && !one && inside<BN>(w, a)) {  // (cross attention, which has masks, is one page)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const bool in = ids[c] >= 0 && ids[c] < ky.n_pages;
            if (!in) status_raise(ST_PAGE_ID);
            words[c] = __ballot_sync(0xffffffffu, in);
          }
        } else {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            int page, row;
            bool in = key(a, c * 32 + lane, page, row);
            const int id = one ? ids[0] : ids[c];
            if (in && (id < 0 || id >= ky.n_pages)) {
              status_raise(ST_PAGE_ID);
              in = false;
            }
            if (ky.mask && in) in = __ldg(ky.mask + id * ky.mask_stride + row) != 0;
            words[c] = __ballot_sync(0xffffffffu, in);
          }
        }
      };
      for (; ok && take(w); ) {
        uint32_t next[4] = {0, 0, 0, 0};
        if (w.t0 >= w.t1) continue;
        Walk<BN> walk(w, tl, w.t0);
        look(walk.a);
        TileAt a = walk.a, a_next = a;
        fetch(next);
        if (w.t0 + 1 < w.t1) {
          walk.next();
          look(a_next = walk.a);
        }
        for (int i = w.t0; ok && i < w.t1; ++i, ++tiles, a = a_next, a_next = walk.a) {
          uint32_t words[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) words[c] = next[c];
          if (i + 1 < w.t1) fetch(next);
          if (i + 2 < w.t1) {
            walk.next();
            look(walk.a);
          }
          // The marks of tile n - META are dead: its V slot (and with it its
          // P, which was formed with them) has been released before this
          // tile's K could land.
          uint32_t s = slot_n % NS;
          if (!(ok = warp_wait(&raw[s], slot_n / NS, abort_flag, ST_PAGED_MARK))) break;
          const uint32_t m = tiles % META;
          // 128 live keys lie at consecutive positions, whatever the page size.
          const bool all = (words[0] & words[1] & words[2] & words[3]) == 0xFFFFFFFFu && a.base + BN <= w.hi_min &&
                           (a.base >= w.lo_max || a.base + BN <= w.sink_min);
          if (lane < 4) live[m * 4 + lane] = lane < 2 ? (lane ? words[1] : words[0]) : (lane & 1 ? words[3] : words[2]);
          if (lane == 4) whole[m] = all;
          __syncwarp();
          if (lane == 0) mbar_arrive(&full[s]);
          slot_n += 2;
          s = (slot_n - 1) % NS;
          if (!(ok = warp_wait(&raw[s], (slot_n - 1) / NS, abort_flag, ST_PAGED_MARK))) break;
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
          if (MIXED && __builtin_expect(mixed<BN>(w, a), 0) && make_finite(ring + s * SLOT, lane) && lane == 0)
            odd_v[(work_n - 1) % WORKS] = 1;  // (the softmax holds the item until its end)
          if (lane == 0) mbar_arrive(&full[s]);
        }
      }
    } else if (warp == 2) {
      // ---------------------------------------------- marks and scales, 8 bits
      // A tile is marked as soon as the marks of tile n - META are done with, so
      // that its expansion waits for its codes alone; its scales are loaded before
      // that wait and its page ids a tile earlier.
      uint32_t tiles = 0;
      bool ok = true;
      int ids[4], box[4], at_row[4];  // of keys c * 32 + lane: page id, box, row of the box
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        box[c] = tl.ps < BN ? (c * 32 + lane) / tl.rows : 0;
        at_row[c] = c * 32 + lane - box[c] * tl.rows;
      }
      auto key = [&](const TileAt& a, int c, int& page, int& row) -> bool {  // seen by some row of the item?
        page = a.page + box[c];
        row = a.row + at_row[c];
        return box[c] < tl.boxes && row < tl.ps && seen(w, page * tl.ps + row);
      };
      auto look = [&](const TileAt& a) {
        int page, row;
#pragma unroll
        for (int c = 0; c < 4; ++c) ids[c] = key(a, c, page, row) ? page_id(ky, w.sp, w.b, page) : INT_MIN;
      };
      for (; ok && take(w); ) {
        float v_top = 0.f;  // power of two of V so far
        if (w.t0 >= w.t1) continue;
        Walk<BN> walk(w, tl, w.t0);
        look(walk.a);
        for (int i = w.t0; ok && i < w.t1; ++i, ++tiles) {
          const TileAt a = walk.a;
          bool in[4];
          float sk[4], sv[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            in[c] = ids[c] >= 0 && ids[c] < ky.n_pages;
            if (!in[c] && ids[c] != INT_MIN) status_raise(ST_PAGE_ID);
            sk[c] = sv[c] = 0.f;
            if (in[c]) {
              const int row = a.row + at_row[c];
              sk[c] = __ldg(ky.ks + ids[c] * ky.ks_str[0] + w.hk * ky.ks_str[1] + row);
              sv[c] = __ldg(ky.vs + ids[c] * ky.vs_str[0] + w.hk * ky.vs_str[1] + row);
            }
          }
          if (i + 1 < w.t1) {
            walk.next();
            look(walk.a);
          }
          // (a barrier of the ring could pass this phase and the next before the
          // warp looks; unmarked[m] goes no further than the tile that waits)
          if (tiles >= META && !(ok = warp_wait(&unmarked[tiles % META], tiles / META - 1, abort_flag, ST_PAGED_MARK))) break;
          const uint32_t m = tiles % META;
          uint32_t words[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) words[c] = __ballot_sync(0xffffffffu, in[c]);
          // 128 live keys lie at consecutive positions, whatever the page size.
          const bool all = (words[0] & words[1] & words[2] & words[3]) == 0xFFFFFFFFu && a.base + BN <= w.hi_min &&
                           (a.base >= w.lo_max || a.base + BN <= w.sink_min);
          if (lane < 4) live[m * 4 + lane] = lane < 2 ? (lane ? words[1] : words[0]) : (lane & 1 ? words[3] : words[2]);
          if (lane == 4) whole[m] = all;
          // Largest finite scales (non-negative floats order as integers).
          // A row whose V is not finite makes its key's score NaN instead:
          // the queries that see it become NaN, the others never meet it.
          float tk = 0.f, tv = 0.f;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            if (!(fabsf(sv[c]) < INFINITY)) sk[c] = __uint_as_float(0x7FC00000u), sv[c] = 0.f;
            tv = fmaxf(tv, fabsf(sv[c]));
            tk = fmaxf(tk, fabsf(sk[c]) < INFINITY ? fabsf(sk[c]) : 0.f);
          }
          tk = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(tk)));
          tv = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(tv)));
          const float kp = pow2_above(tk);
          if (v_top == 0.f || tv > v_top) v_top = pow2_above(tv) * 8.f;  // room: it should grow rarely
          const float ik = 1.f / kp, iv = 1.f / v_top;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            scales[m * 2 * BN + c * 32 + lane] = hi_lo_f16(sk[c] * ik);
            scales[m * 2 * BN + BN + c * 32 + lane] = hi_lo_f16(sv[c] * iv);
          }
          if (lane == 5) kpow[m] = kp;
          if (lane == 6) vpow[m] = v_top;
          __syncwarp();
          if (lane == 0) mbar_arrive(&marked[m]);
        }
      }
    }
    if (warp == 3) {
      // --------------------------------------------------------------- items
      const int n_tiles = count_tiles(ky, qr, tl, lane), ctas = gridDim.x, c = blockIdx.x;
      const Deal d = deal_of(ky, qr, tl, n_tiles, G, ctas);
      bool ok = true;
      auto give = [&]() {
        const uint32_t k = work_n % WORKS;
        ok = ok && (work_n < WORKS || warp_wait(&work_empty[k], work_n / WORKS - 1, abort_flag, ST_PAGED_WORK));
        if (ok && lane == 0) {
          works[k] = w;
          if (MIXED) odd_v[k] = 0;
          mbar_arrive(&work_full[k]);
        }
        __syncwarp();
        ++work_n;
      };
      const unsigned whole = d.even ? d.full : 0xFFFFFFFFu;
      for (unsigned it = c; ok && it < whole && (SORTED ? nth_longest(w, ky, qr, tl, n_tiles, G, it, lane) : find_work(w, ky, qr, tl, n_tiles, G, it, lane)); it += ctas)
        give();
      for (int v = c; ok && d.even && v < d.left * d.parts; v += ctas) {
        const int p = v / d.left, r = v - p * d.left;
        find_work(w, ky, qr, tl, n_tiles, G, d.full + r, lane);
        if (d.parts > 1) {
          w.t0 = run_start(d.n, p, d.parts);
          w.t1 = run_start(d.n, p + 1, d.parts);
          w.slot = v;
        }
        give();
      }
      w.b = -1;
      give();
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
    // The item stays in shared memory: the loop over its tiles has no registers to spare.
    for (;; done_with()) {
      if (!ok || !next_work()) break;
      const Work& w = works[(work_n - 1) % WORKS];
      const int nt = w.t1 - w.t0;
      if (u >= w.nsub) {
        tiles += nt;
        continue;
      }
      const int i = w.i0 + u * tl.tq + row / qr.group, h = w.hk * qr.group + row % qr.group;
      const bool has_row = row < tl.tq * qr.group && i < w.sp.n;
      const Sees se = sees(qr, w.sp, min(i, w.sp.n - 1));
      // The maximum in use, -inf while nothing has been seen, and what P's exponents
      // are taken from (0 then).
      float m_run = -INFINITY, m_use = 0.f;
      float l_run = 0.f, v_run = 1.f, q_scale = 0.f;
      for (int j = 0; j < nt; ++j, ++sn, ++tiles) {
        ok = warp_wait(&bar_s[u], sn, abort_flag, ST_PAGED_SOFTMAX);
        if (!ok) break;
        tc_fence_after();
        if (KV8 && j == 0) q_scale = qr.scale_log2 * qpow[((items & 1) * 2 + u) * BM + row];
        const uint32_t m = tiles % META;
        const bool masked = whole[m] == 0;
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
        // Which of the tile's keys this row sees.
        uint32_t keep[4];
        if (masked) {
          const TileAt at = tile_at<BN>(tl, nth_tile(w, w.t0 + j));
          const int b_hi = rows_below<BN>(tl, at, se.hi), b_lo = rows_below<BN>(tl, at, se.lo);
          const int b_sink = rows_below<BN>(tl, at, se.sink);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            keep[c] = live[m * 4 + c] & (bit_range(b_lo, b_hi, c * 32) | bit_range(0, b_sink, c * 32));
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
        // (rows of zeros have powers whose product is 0 in f32, huge ones infinity: times
        // -inf and times a score of 0 that would be NaN)
        const float scale = KV8 ? fminf(fmaxf(q_scale * kpow[m], 0x1p-126f), 3.402823466e38f) : qr.scale_log2;
        const float mx2 = mx * scale;
        // l and O use the same stale maximum, so the quotient does not change.  A
        // NaN or +inf score makes the row NaN from here on.
        const bool grow = !(mx2 <= m_run + SLACK);
        const float v_new = KV8 ? vpow[m] : 1.f;
        if (__any_sync(0xffffffffu, grow) || (KV8 && v_new != v_run)) {
          float alpha = 1.f;
          if (grow) {
            const float m_new = mx2 < INFINITY ? mx2 : __uint_as_float(0x7FC00000u);
            const float m_old = m_run == -INFINITY ? -INFINITY : m_use;
            m_run = m_new;
            m_use = KV8 ? p_base(m_new, 15.f - SLACK) : m_new;
            alpha = ex2_approx(m_old - m_use);
            l_run *= alpha;
          }
          if (KV8) alpha *= v_run / v_new;
          v_run = v_new;
          if (j > 0) {
            // (written for the registers that S leaves: unrolled, the wide form's
            // pieces spill S for 8-bit pages, rolled it costs bf16 4 % of cross attention)
            if constexpr (KV8) {
#pragma unroll 1
              for (int c = 0; c < HD; c += 32) {
                uint32_t r[32];
                tmem_ld32x32b_x32(tO + c, r);
#pragma unroll
                for (int k = 0; k < 32; ++k) r[k] = __float_as_uint(__uint_as_float(r[k]) * alpha);
                tmem_st32x32b_x32(tO + c, r);
              }
            } else {
#pragma unroll
              for (int c = 0; c < HD; c += 16) {
                uint32_t r[16];
                tmem_ld32x32b_x16(tO + c, r);
#pragma unroll
                for (int k = 0; k < 16; ++k) r[k] = __float_as_uint(__uint_as_float(r[k]) * alpha);
                tmem_st32x32b_x16(tO + c, r);
              }
            }
          }
        }
        const float2 sc2 = make_float2(scale, scale);
        const float2 nm2 = make_float2(-m_use, -m_use);
        float2 sum[4] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        // P = 2^(s * scale - m), 2 of 8 pairs on the FMA pipe's polynomial, the
        // rest on MUFU (9472 x 16384 x 4 heads, bf16 / e4m3 pages, us: 1 of 8 255 /
        // 371, 2 of 8 257 / 366, 3 of 8 286 / 387, 4 of 8 288 / 390); l sums P
        // before its rounding to 16 bits.  PV starts on the
        // first half of the keys while the second is formed.
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint32_t pk[BN / 4];
#pragma unroll
          for (int kk = 0; kk < BN / 4; ++kk) {
            const int k = half * (BN / 4) + kk;
            const float2 x = ffma2(make_float2(s[2 * k], s[2 * k + 1]), sc2, nm2);
            float2 p;
            if ((k & 7) < 2) {
              p = exp2_poly2(x);
            } else {
              p.x = ex2_approx(x.x);
              p.y = ex2_approx(x.y);
            }
            sum[k & 3] = fadd2(sum[k & 3], p);
            pk[kk] = KV8 ? f16x2(p.x, p.y) : pack_bf16x2(p.x, p.y);
          }
          if (masked) {  // the polynomial's smallest value must not count
#pragma unroll
            for (int kk = 0; kk < BN / 4; ++kk) {
              const int k = half * (BN / 4) + kk;
              const uint32_t two = keep[k >> 4] >> ((2 * k) & 31) & 3;
              pk[kk] &= ((two & 1) ? 0xFFFFu : 0u) | ((two & 2) ? 0xFFFF0000u : 0u);
            }
          }
          tmem_st32x32b_x32(tS + half * (BN / 4), pk);
          tmem_st_wait();
          tc_fence_before();
          mbar_arrive(&bar_p[2 * u + half]);
        }
        const float2 s2 = fadd2(fadd2(sum[0], sum[1]), fadd2(sum[2], sum[3]));
        l_run += s2.x + s2.y;
      }
      if (!ok) break;
      if (nt > 0) {
        ok = warp_wait(&o_full[u], items, abort_flag, ST_PAGED_SOFTMAX);
        if (!ok) break;
        ++items;
        tc_fence_after();
      }
      const bool none = m_run == -INFINITY;
      const float inv = none ? 0.f : m_run != m_run ? m_run : v_run / l_run;
      const int64_t packed = (int64_t)(w.sp.first + i) * qr.H + h;
      const float lse2 = none ? -INFINITY : m_use + log2f(l_run);
      // What the marks took out of V, from the pages, for the keys that this row sees.
      auto add_odd = [&](auto* to) {
#pragma unroll 1
        for (int j = w.t0; j < w.t1; ++j) {
          const TileAt a = tile_at<BN>(tl, nth_tile(w, j));
          if (!mixed<BN>(w, a)) continue;
#pragma unroll 1
          for (int r = 0; r < BN; ++r) {
            int page, at;
            if (!place<BN>(tl, a, r, page, at)) continue;
            const int pos = page * tl.ps + at;
            if (!((pos >= se.lo && pos < se.hi) || pos < se.sink)) continue;
            const int id = page_id(ky, w.sp, w.b, page);
            if (id < 0 || id >= ky.n_pages) continue;
            const __nv_bfloat16* v =
                static_cast<const __nv_bfloat16*>(ky.v) + id * ky.v_str[0] + w.hk * ky.v_str[1] + at * ky.v_str[2];
#pragma unroll 1
            for (int d = 0; d < HD; d += 2) {
              const uint32_t x = *reinterpret_cast<const uint32_t*>(v + d), bad = x & ~finite2(x);
              if (bad) {
                to[d] = static_cast<float>(to[d]) + __uint_as_float(bad << 16);
                to[d + 1] = static_cast<float>(to[d + 1]) + __uint_as_float(bad & 0xFFFF0000u);
              }
            }
          }
        }
      };
      if (tl.splits > 1 || w.slot >= 0) {
        const int64_t at = w.slot >= 0 ? (int64_t)w.slot * (2 * BM) + u * BM + row
                                       : (int64_t)w.split * qr.rows * qr.H + packed;
        if (has_row) part_l[at] = lse2;
        if (nt > 0) {
#pragma unroll
          for (int c = 0; c < HD; c += 32) {
            uint32_t r[32];
            tmem_ld32x32b_x32(tO + c, r);
            if (has_row && !none) {
#pragma unroll
              for (int v = 0; v < 32; ++v) r[v] = __float_as_uint(__uint_as_float(r[v]) * inv);
#pragma unroll
              for (int v = 0; v < 32; v += 8) store32(part_o + at * HD + c + v, r + v, tl.wide);
            }
          }
          if constexpr (MIXED)
            if (odd_v[(work_n - 1) % WORKS] && has_row && !none) add_odd(part_o + at * HD);
        }
      } else {
        if (has_row && qr.lse) qr.lse[packed] = lse2 * 0.6931471805599453f;
        const int64_t orow = ky.cross ? w.b * qr.o_str[0] + i * qr.o_str[1] : (int64_t)(w.sp.first + i) * qr.o_str[1];
        __nv_bfloat16* d = qr.o + (has_row ? orow + h * qr.o_str[2] : 0);
#pragma unroll
        for (int c = 0; c < HD; c += 32) {
          uint32_t r[32];
          if (nt > 0) tmem_ld32x32b_x32(tO + c, r);
          if (has_row) {
            uint32_t o[16];
#pragma unroll
            for (int k = 0; k < 16; ++k)
              o[k] = none ? 0u : pack_bf16x2(__uint_as_float(r[2 * k]) * inv, __uint_as_float(r[2 * k + 1]) * inv);
            store32(d + c, o, tl.wide);
            store32(d + c + 16, o + 8, tl.wide);
          }
        }
        if constexpr (MIXED)
          if (odd_v[(work_n - 1) % WORKS] && has_row && !none) add_odd(d);
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
      uint32_t qn[2] = {0, 0}, tiles = 0;
      const int row0 = (warp - 12) * 32;
      for (; ok && take(w); ) {
        if (w.t1 <= w.t0) continue;
        for (int u = 0; ok && u < w.nsub; ++u) {
          if (!(ok = warp_wait(&q_raw[u], qn[u], abort_flag, ST_PAGED_EXPAND))) break;
          expand_q(sQ + u * SLOT, row0, lane, qpow + ((qn[u]++ & 1) * 2 + u) * BM);
          fence_proxy_async_smem();
          mbar_arrive(&q_full[u]);
        }
        for (int i = w.t0; ok && i < w.t1; ++i, ++tiles) {
          const uint32_t m = tiles % META;
          if (!(ok = warp_wait(&marked[m], tiles / META, abort_flag, ST_PAGED_EXPAND))) break;
#pragma unroll 1
          for (int kv = 0; kv < 2; ++kv, ++slot_n) {
            const uint32_t s = slot_n % NS;
            if (!(ok = warp_wait(&raw[s], slot_n / NS, abort_flag, ST_PAGED_EXPAND))) break;
            expand_rows<DT>(ring + s * SLOT, row0, lane, scales + m * 2 * BN + kv * BN);
            fence_proxy_async_smem();
            mbar_arrive(&full[s]);
          }
        }
      }
    }
    teardown();
  }
}

// Joins the parts of items that were dealt out in parts: blocks (item, run
// of rows), a warp to a row at a time.
__global__ void __launch_bounds__(256) join_dealt_kernel(const __grid_constant__ Keys ky,
                                                         const __grid_constant__ Queries qr,
                                                         const __grid_constant__ Tiling tl,
                                                         const float* __restrict__ part_o,
                                                         const float* __restrict__ part_l, int ctas) {
  const int lane = threadIdx.x & 31;
  const int G = qr.H / qr.group, n_tiles = count_tiles(ky, qr, tl, lane);
  const Deal d = deal_of(ky, qr, tl, n_tiles, G, ctas);
  for (int r = blockIdx.x; d.even && d.parts > 1 && r < d.left; r += gridDim.x) {
    Work w;
    find_work(w, ky, qr, tl, n_tiles, G, d.full + r, lane);
    for (int row = blockIdx.y * 8 + (threadIdx.x >> 5); row < 2 * BM; row += gridDim.y * 8) {
      const int u = row / BM, rr = row % BM, i = w.i0 + u * tl.tq + rr / qr.group, h = w.hk * qr.group + rr % qr.group;
      if (rr >= tl.tq * qr.group || i >= w.sp.n) continue;
      float m = -INFINITY;
      for (int p = 0; p < d.parts; ++p) m = max_nan(m, part_l[(int64_t)(p * d.left + r) * (2 * BM) + row]);
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
      float l = 0.f;
      for (int p = 0; p < d.parts && m != -INFINITY; ++p) {
        const int64_t at = (int64_t)(p * d.left + r) * (2 * BM) + row;
        const float ls = part_l[at];
        if (ls == -INFINITY) continue;
        const float x = exp2f(ls - m);
        const float4 v = __ldcs(reinterpret_cast<const float4*>(part_o + at * HD) + lane);
        o.x += x * v.x, o.y += x * v.y, o.z += x * v.z, o.w += x * v.w;
        l += x;
      }
      const float inv = m == -INFINITY ? 0.f : 1.f / l;
      const int64_t packed = (int64_t)(w.sp.first + i) * qr.H + h;
      const int64_t orow = ky.cross ? w.b * qr.o_str[0] + i * qr.o_str[1] : (int64_t)(w.sp.first + i) * qr.o_str[1];
      *reinterpret_cast<uint2*>(qr.o + orow + h * qr.o_str[2] + lane * 4) =
          make_uint2(pack_bf16x2(o.x * inv, o.y * inv), pack_bf16x2(o.z * inv, o.w * inv));
      if (qr.lse && lane == 0) qr.lse[packed] = m == -INFINITY ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
    }
  }
}

// --------------------------------------------------------------------- host
// What the host knows of a call's size.
static int64_t tiles_bound(const Shape& sh) {
  const int step = 2 * (BM / sh.group);
  if (sh.cross) return (int64_t)sh.seqs * ((sh.Lq + step - 1) / step);
  const int64_t seqs = sh.rows < sh.seqs ? sh.rows : sh.seqs;
  return (sh.rows + seqs * (step - 1)) / step;
}
static int64_t key_tiles(const Shape& sh) { return tiles_of_keys(sh, BN, !sh.kv8); }

// Whether the launch is one sequence on a CTA per SM, dealt out as Deal says
// (should its rows see different keys after all, whole items in turn); worth it
// where the key tiles are many beside a part's start, end and join.
static bool dealt(const Shape& sh) { return sh.seqs == 1 && key_tiles(sh) >= 16; }

// Splits of the keys otherwise: the count that gives the least time for the
// slowest SM, one key tile counted as 1.4 us (whole items measure 1.9 over bf16
// and 2.7 over 8-bit pages), an item's start and end about two tiles, and the join
// its launch and one f32 row written and read a split.
static int splits(const Shape& sh) {
  if (dealt(sh)) return 1;
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
// Whether items are taken from the longest to the shortest (see nth_longest): more
// of them than run at once, of sequences of different lengths, whose K and V stay
// in L2 whatever the order.
static bool sorted(const Shape& sh) {
  const int64_t G = sh.H / sh.group, tiles = tiles_bound(sh);
  return !sh.cross && sh.seqs > 1 && sh.seqs <= 32 && tiles <= MANY && tiles * G > SMS && key_tiles(sh) >= 8 &&
         splits(sh) == 1 && sh.seqs * sh.keys * G * (sh.kv8 ? 2 * (HD + 4) : 4 * HD) <= (64 << 20);
}
int64_t parts(const Shape& sh) {
  if (dealt(sh)) {  // rows that turn out fewer leave other items
    const int64_t items = tiles_bound(sh) * (sh.H / sh.group);
    return (items < SMS ? (items * 32 < MAX_SLOTS ? items * 32 : MAX_SLOTS) : MAX_SLOTS) * 2 * BM;
  }
  const int s = splits(sh);
  return s > 1 ? (int64_t)s * sh.rows * sh.H : 0;
}

template <int DT, bool SORTED, bool MIXED>
static int start(const CUtensorMap& tq, const PageMaps& tm, const Keys& ky,
                 const Queries& qr, const Tiling& tl, unsigned grid, float* part_o, float* part_l, cudaStream_t st) {
  using C = Cfg<DT != WF_DTYPE_BF16>;
  static thread_local int configured = -1;
  int dev = 0;
  WFK_CUDA_TRY(cudaGetDevice(&dev));
  if (configured != dev) {
    WFK_CUDA_TRY(cudaFuncSetAttribute(tile_kernel<DT, SORTED, MIXED>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
    configured = dev;
  }
  tile_kernel<DT, SORTED, MIXED><<<grid, C::THREADS, C::SMEM, st>>>(tq, tm, ky, qr, tl, part_o, part_l);
  WFK_CUDA_TRY(cudaGetLastError());
  return WF_OK;
}

int launch(const Keys& ky, const Queries& qr, const Shape& sh, void* workspace, cudaStream_t st) {
  const int G = qr.H / qr.group, ps = ky.page_size;
  Tiling tl = tiling_of(ps, BN, !sh.kv8);
  tl.tq = BM / qr.group;
  tl.splits = splits(sh);
  tl.even = dealt(sh);
  tl.wide = ((reinterpret_cast<uintptr_t>(qr.o) | reinterpret_cast<uintptr_t>(workspace)) & 31) == 0 &&
            (qr.o_str[0] | qr.o_str[1] | qr.o_str[2]) % 16 == 0;
  CUtensorMap tq;
  PageMaps tm;
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
  if ((rc = page_maps(&tm, ky, G, tl, BN)) != WF_OK) return rc;
  const int64_t items = tiles_bound(sh) * G * tl.splits;
  if (items > INT_MAX / 4) return fail(WF_ERR_INVALID_ARG, "attention: too many query tiles (%lld)", (long long)items);
  // Few key tiles to an item: one CTA per SM walks the items, the next one's
  // loads under the last one's end.  Many: a CTA per item, so that the SM that
  // is done first takes the next.
  const unsigned grid = (unsigned)(tl.even || (key_tiles(sh) / tl.splits < 8 && items > SMS) ? SMS : items);
  const int64_t n_parts = parts(sh);
  float* part_o = static_cast<float*>(workspace);
  float* part_l = part_o + n_parts * HD;
  // (a kernel without the mixed tiles' care: six stages' cross attention 131 us for 135)
  const bool differ = !ky.cross && qr.block > 0;
  auto pick = [&](auto x) {
    constexpr bool S = decltype(x)::value;
    auto run = [&](auto kernel) { return kernel(tq, tm, ky, qr, tl, grid, part_o, part_l, st); };
    return ky.dtype == WF_DTYPE_E4M3 ? run(start<WF_DTYPE_E4M3, S, false>)
           : ky.dtype == WF_DTYPE_S8 ? run(start<WF_DTYPE_S8, S, false>)
           : differ                  ? run(start<WF_DTYPE_BF16, S, true>)
                                     : run(start<WF_DTYPE_BF16, S, false>);
  };
  rc = sorted(sh) ? pick(std::true_type{}) : pick(std::false_type{});
  if (rc != WF_OK || n_parts == 0) return rc;
  if (tl.even) {
    const int64_t left = items % SMS;  // with rows behind the sequence the device may have others
    join_dealt_kernel<<<dim3((unsigned)(left ? left : 1), 8), 256, 0, st>>>(ky, qr, tl, part_o, part_l, SMS);
    WFK_CUDA_TRY(cudaGetLastError());
    return WF_OK;
  }
  return join(ky, qr, part_o, part_l, tl.splits, st);
}

}  // namespace tile
}  // namespace paged
}  // namespace wfk

extern "C" unsigned int wfk_status_take_paged_tile(void) { return wfk::status_take_local(); }
