// Attention over pages for few query rows to a K/V head (single tokens, short
// runs of them): bound by reading K and V once from HBM.
//
// Rows of one K/V head (tokens x the query heads that share it) come in tiles
// of up to 16, the height of mma.sync's A operand, which here only has to keep
// up with the loads: 32 instructions to 8 KB of K and V.  An item of work is one
// tile of rows against its key tiles.  All items' key tiles lie in a line, cut
// into an equal stretch for each of two CTAs an SM, so that ragged lengths
// leave no SM idle; the parts of an item that lies in several stretches (each
// CTA has at most two) are joined by a second launch, whose blocks are in place
// before the first one ends.  Where whole items fill the SMs evenly they are not
// cut.  Warp 4 walks the stretch and loads tiles by TMA into a ring of two or
// three (64 KB in flight), on into the next item while the last one ends; warps
// 0-3 take a quarter of a tile's keys each, multiply them straight from shared
// memory and keep sums of their own, joined through shared memory at an item's
// end.  (With every warp loading its own chunks, issuing four TMA copies cost
// 600 of 1700 clocks a chunk.  With a cluster of CTAs to an item, joined through
// distributed shared memory, the ragged batch below took 94 us and the masked
// cross attention 53.)
//
// Measured: 32 ragged sequences of up to 8192 tokens, 40 heads on 8, e4m3: 78 us,
// 0.53 of the HBM copy rate; 8 x 8192 tokens, 32 heads on 8, bf16: 58 us, 4.6
// TB/s; 32768 tokens, 12 heads, bf16: 47 us, 4.3 TB/s; 24 x 40 single rows over
// 257 masked keys: 44 us.  Bound by the start (12,000 clocks to the first data:
// lengths, page table and pages are loads that wait for each other) and, over
// 8-bit pages, by each warp's chain of load, expansion and product: 3300 clocks a
// tile of 128 keys against 1350 for 64 keys of bf16.
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

#include <algorithm>
#include <cmath>

#include "paged_attn.cuh"

namespace wfk {
namespace paged {
namespace rows {

constexpr int WARPS = 4, THREADS = (WARPS + 1) * 32;
constexpr int STAGE = 32768;               // a tile's K and V rows
constexpr int MAX_BN = 128;
constexpr int META = 2 * MAX_BN * 4 + 32;  // scales of K and V, live keys, whether every row sees all, the tile
constexpr int O_PITCH = 132;               // floats of a row of partial sums, off the banks of the next
constexpr int HEAD = 4096;                 // barriers, items and META of up to three stages
constexpr int smem_of(int stages, int height) {
  return 1024 + HEAD + stages * STAGE + WARPS * height * (O_PITCH + 2) * 4;
}
constexpr int SMEM = 115712;  // two CTAs to an SM
static_assert(smem_of(3, 5) <= SMEM && smem_of(2, 16) <= SMEM);

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
// How the work is shared: all tiles of all items (a sequence's K/V head and
// `height` of its rows) lie in a line, of which each CTA takes an equal stretch;
// with `whole` a CTA takes whole items.
struct Cut {
  Tiling tl;
  int ctas, height, whole, stages;
};
struct Item {
  int b, hk, rt, n;  // sequence, K/V head, tile of rows; items of the sequence
  int t, i0, i1;     // its tiles in the line; this CTA's
  Span sp;
  Range rg;
};

template <int BN>
__device__ __forceinline__ void open_sequence(Item& it, const Keys& ky, const Queries& qr, const Cut& cut, int b) {
  it.b = b;
  it.sp = span_of(ky, qr, b);
  it.n = it.sp.n > 0 ? (it.sp.n * qr.group + cut.height - 1) / cut.height * (qr.H / qr.group) : 0;
  if (it.n == 0) return;
  it.rg = range_of<BN>(qr, it.sp, cut.tl, 0, it.sp.n - 1);
  it.t = cut.whole ? 1 : max(it.rg.n, 1);  // an item without keys still writes its rows
}

// First place of CTA c's stretch.
__device__ __forceinline__ long long stretch(long long len, int c, int ctas) { return len * c / ctas; }
// Where a stretch begins: the line's length, the first place, its sequence and
// that one's first place; found by each warp for itself.
struct Spot {
  long long len, pos, first;
  int b;
};
template <int BN>
__device__ __forceinline__ Spot find_spot(const Keys& ky, const Queries& qr, const Cut& cut, int cta) {
  const int lane = threadIdx.x & 31, per = (qr.seqs + 31) / 32, b0 = lane * per, b1 = min(b0 + per, qr.seqs);
  auto length = [&](int b) -> long long {
    Item it;
    open_sequence<BN>(it, ky, qr, cut, b);
    return it.n > 0 ? (long long)it.t * it.n : 0;
  };
  long long mine = 0;
  for (int b = b0; b < b1; ++b) mine += length(b);
  long long after = mine;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const long long x = __shfl_up_sync(0xffffffffu, after, o);
    if (lane >= o) after += x;
  }
  Spot s;
  s.len = __shfl_sync(0xffffffffu, after, 31);
  s.pos = stretch(s.len, cta, cut.ctas);
  s.first = after - mine;
  s.b = b0;
  const bool here = s.pos >= s.first && s.pos < after;
  if (here && per > 1)
    for (long long n; s.pos >= s.first + (n = length(s.b)); ++s.b) s.first += n;
  const int from = __ffs(__ballot_sync(0xffffffffu, here)) - 1;  // (-1: the line is empty)
  s.first = __shfl_sync(0xffffffffu, s.first, max(from, 0));
  s.b = __shfl_sync(0xffffffffu, s.b, max(from, 0));
  return s;
}

// What the join has to know of an item whose first part is a CTA's last one.
struct Split {
  int b, hk, rt, parts;  // 0 parts: the CTA has none
};

// Row r of an item's rows (tokens x the heads that share the K/V head), one dim.
__device__ __forceinline__ void store_row(const Keys& ky, const Queries& qr, int b, int first, int hk, int r, int dim,
                                          float x, float lse2) {
  const int i = r / qr.group, h = hk * qr.group + r - i * qr.group;
  const int64_t orow = ky.cross ? b * qr.o_str[0] + i * qr.o_str[1] : (int64_t)(first + i) * qr.o_str[1];
  qr.o[orow + h * qr.o_str[2] + dim] = __float2bfloat16_rn(x);
  if (qr.lse && dim == 0) qr.lse[(int64_t)(first + i) * qr.H + h] = lse2 * 0.6931471805599453f;
}

template <int DT>
__global__ void __launch_bounds__(THREADS, 2)
    rows_kernel(const __grid_constant__ PageMaps tm,
                const __grid_constant__ Keys ky, const __grid_constant__ Queries qr, const __grid_constant__ Cut cut,
                float* part_o, float* part_l, Split* split) {
  constexpr bool KV8 = DT != WF_DTYPE_BF16;
  constexpr int BN = KV8 ? 128 : 64;       // keys of a tile
  constexpr int KC = BN / WARPS;           // keys of a warp
  constexpr int ROWB = KV8 ? 128 : 256;    // bytes of a row
  constexpr int NT = KC / 8;               // score tiles of a warp
  // Sums are rescaled when a row's maximum grows by more than 2^SLACK, or V's largest
  // scale beyond the power of two in use, taken with a factor of ROOM.  Both limit P, which
  // f16 holds as 2^(s - m + 15 - SLACK) * (scale / V's power <= 1): the less they leave, the
  // smaller the weights that count (4 and 2, 8 and 8 measured the same: 61 us for 32
  // single tokens).
  constexpr float SLACK = KV8 ? 2.f : 8.f, ROOM = 2.f;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const Tiling& tl = cut.tl;
  const int ps = tl.ps, G = qr.H / qr.group;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem);
  uint64_t* empty = full + 3;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(empty + 3);
  Item& it = reinterpret_cast<Item*>(smem + 64)[warp];  // the warp's; registers are short
  static_assert(64 + (WARPS + 1) * sizeof(Item) <= HEAD - 3 * META);
  uint8_t* meta = smem + HEAD - 3 * META;
  uint8_t* ring = smem + HEAD;
  float* sums = reinterpret_cast<float*>(ring + cut.stages * STAGE);  // [WARPS] of O [height][O_PITCH], m [height], l [height]
  if (threadIdx.x == 0) {
    for (int k = 0; k < cut.stages; ++k) {
      mbar_init(&full[k], KV8 ? 33 : 1);
      mbar_init(&empty[k], WARPS);
    }
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tm.k_tile);
    tma_prefetch_desc(&tm.v_tile);
  }
  const int cta = blockIdx.x;
  const Spot spot = find_spot<BN>(ky, qr, cut, cta);
  const long long len = spot.len;
  long long left = stretch(len, cta + 1, cut.ctas) - stretch(len, cta, cut.ctas);
  __syncthreads();
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");  // the join may take its place (it waits for the end)
  if (left == 0) {  // (the whole CTA)
    if (!cut.whole && threadIdx.x < 16) part_l[cta * 32 + threadIdx.x] = -INFINITY;
    if (!cut.whole && threadIdx.x == 0) split[cta].parts = 0;
    return;
  }
  int st = 0;             // the ring's stage, and how often it has come round
  uint32_t turn = 0;
  auto next_stage = [&]() {
    if (++st == cut.stages) st = 0, ++turn;
  };
  // The CTA's items in turn, each with the tiles that it has to do.  A warp's
  // lanes share `it`: lane 0 writes it, after all of them have read what it held.
  int item, i;
  auto open_from = [&](int b) {  // the first sequence with items from b on
    Item x;
    do open_sequence<BN>(x, ky, qr, cut, b++);
    while (x.n == 0);
    __syncwarp();
    if (lane == 0) it = x;
    __syncwarp();
  };
  {
    open_from(spot.b);
    const long long off = spot.pos - spot.first;
    item = (int)(off / it.t);
    i = (int)(off - (long long)item * it.t);
  }
  auto open_item = [&]() {
    const int rt = item / G, n = (int)min((long long)(it.t - i), left);
    left -= n;
    __syncwarp();
    if (lane == 0) it.rt = rt, it.hk = item - rt * G, it.i0 = i, it.i1 = i + n;
    __syncwarp();
  };
  auto next_item = [&]() -> bool {
    if (left == 0) return false;
    i = 0;
    if (++item == it.n) {
      item = 0;
      open_from(it.b + 1);
    }
    return true;
  };
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
    bool ok = true;
    do {
      open_item();
      const Item w = it;
      const int p0 = cut.whole ? 0 : w.i0, p1 = cut.whole ? w.rg.n : min(w.i1, w.rg.n);
      if (p0 >= p1) continue;
      Box nx{};             // the next tile, or this lane's box of it
      int nx_id = INT_MIN;  // and its page, as the table has it (INT_MIN: not needed)
      auto look = [&](const TileAt& a) {
        const bool one = one_box<BN>(tl, a);
        nx = one ? Box{a.page, a.row, a.base} : box_at<BN>(tl, a, lane);
        nx_id = one || (lane < tl.boxes && needed(w.rg, nx.pos, min(tl.rows, ps - nx.row))) ? page_id(ky, w.sp, w.b, nx.page)
                                                                                          : INT_MIN;
      };
      Walk<BN> walk(w.rg, tl, p0);
      look(walk.a);
      for (int i = p0; ok && i < p1; ++i) {
        const TileAt a = walk.a;
        const bool bad = nx_id != INT_MIN && (nx_id < 0 || nx_id >= ky.n_pages), one = one_box<BN>(tl, a);
        if (bad) status_raise(ST_PAGE_ID);
        const int box = bad || nx_id == INT_MIN ? -1 : nx_id;
        const Box x = nx;
        if (i + 1 < p1) {
          walk.next();
          look(walk.a);
        }
        if (turn > 0 && !(ok = warp_wait(&empty[st], turn - 1, abort_flag, ST_PAGED_ROWS))) break;
        uint8_t *at = ring + st * STAGE, *mt = meta + st * META;
        const uint32_t to = smem_u32(mt) + lane * 4;
        uint32_t all = 0xFFFFFFFFu;
        const int64_t ko = KV8 ? box * ky.ks_str[0] + w.hk * ky.ks_str[1] + x.row : 0;
        const int64_t vo = KV8 ? box * ky.vs_str[0] + w.hk * ky.vs_str[1] + x.row : 0;
        const bool easy = __all_sync(0xffffffffu, (one || lane < tl.boxes) ? box >= 0 : true) && inside<BN>(w.rg, a) &&
                          !ky.mask && (tl.dense || (one && x.row + BN <= ps));  // every key of the tile
#pragma unroll
        for (int c = 0; c < KL; ++c) {
          const int src = one ? 0 : sub[c] & 31, ar = one ? c * 32 + lane : at_row[c];
          bool in = true;
          if (!easy) {
            const int id = __shfl_sync(0xffffffffu, box, src);
            const int off = __shfl_sync(0xffffffffu, x.row, src) + ar;
            const int pos = __shfl_sync(0xffffffffu, x.pos, src) + ar;
            in = id >= 0 && (one || sub[c] < tl.boxes) && off < ps && seen(w.rg, pos);
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
        const bool whole = all == 0xFFFFFFFFu && a.base + BN <= w.rg.hi_min &&
                           (a.base >= w.rg.lo_max || a.base + BN <= w.rg.sink_min);
        if (lane == 4) *reinterpret_cast<uint2*>(mt + 2 * MAX_BN * 4 + 16) = make_uint2(whole, nth_tile(w.rg, i));
        __syncwarp();
        auto copy = [&](const CUtensorMap* mk, const CUtensorMap* mv, uint8_t* k, int row, int id) {
          tma_load_4d(k, mk, &full[st], 0, row, w.hk, id);
          if constexpr (!KV8) tma_load_4d(k + STAGE / 4, mk, &full[st], 64, row, w.hk, id);
          tma_load_4d(k + STAGE / 2, mv, &full[st], 0, row, w.hk, id);
          if constexpr (!KV8) tma_load_4d(k + 3 * STAGE / 4, mv, &full[st], 64, row, w.hk, id);
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
        next_stage();
      }
    } while (ok && next_item());
    if (*abort_flag && lane == 0) {  // let the loads in flight land before the CTA exits
      const uint64_t t0 = globaltimer_ns();
      for (int k = 0; k < cut.stages; ++k) {  // stage k's last load: its turn, or the one before
        const int64_t n = (int64_t)turn - (k >= st);
        while (n >= 0 && !mbar_try_wait(&full[k], n & 1) && globaltimer_ns() - t0 < 200000000ull) {
        }
      }
    }
    __syncwarp();
    return;
  }
  // ------------------------------------------------------------ consumers
  do {
    open_item();
    const int p0 = cut.whole ? 0 : it.i0, p1 = cut.whole ? it.rg.n : min(it.i1, it.rg.n);
    const int n_rows = min(cut.height, it.sp.n * qr.group - it.rt * cut.height);
    // This thread's two rows, g and g + 8.
    int tok[2], head[2];
    bool has[2];
    Sees se[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = it.rt * cut.height + min(g + e * 8, cut.height);
      tok[e] = r / qr.group;
      head[e] = it.hk * qr.group + r - tok[e] * qr.group;
      has[e] = g + e * 8 < cut.height && tok[e] < it.sp.n;
      if (!has[e]) tok[e] = it.sp.n - 1;
      se[e] = sees(qr, it.sp, tok[e]);
    }
    // Q fragments, dims in the order in which K is read.
    uint32_t a[8][4];
    float q_pow[2] = {1.f, 1.f};
    {
      uint2 v[8][2];
      float top[2] = {0.f, 0.f};
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int64_t at = ky.cross ? it.b * qr.q_str[0] + tok[e] * qr.q_str[1] : (int64_t)(it.sp.first + tok[e]) * qr.q_str[1];
        const __nv_bfloat16* q = qr.q + at + (has[e] ? head[e] : it.hk * qr.group) * qr.q_str[2];
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

    const bool differ = !KV8 && rows_differ(it.rg);
    for (int i = p0; i < p1; ++i) {
      if (!warp_wait(&full[st], turn, abort_flag, ST_PAGED_ROWS)) break;
      uint8_t* K = ring + st * STAGE + warp * KC * 128;
      uint8_t* V = K + STAGE / 2;
      const uint8_t* mt = meta + st * META;
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
      // Scores in log2 units, -inf where the row does not see the key.  One factor
      // at a time: the product of both may pass f32's range, and then make NaN of a
      // score of 0.  The maximum is subtracted from rounded scores: in one
      // multiply-add the largest of a row of scores above 2^28 would not become 0.
      float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int k = nt * 8 + key_of(2 * t + (e & 1));
          s[nt][e] = KV8 ? s[nt][e] * scale[k] * q_scale[e >> 1] : s[nt][e] * qr.scale_log2;
          if (!whole && !(keep[e >> 1] >> k & 1)) s[nt][e] = -INFINITY;
          mx[e >> 1] = max_nan(mx[e >> 1], s[nt][e]);
        }
      }
      bool grow = false;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        mx[e] = max_nan(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 1));
        mx[e] = max_nan(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 2));
        grow |= !(mx[e] <= m_run[e] + SLACK);
      }
      float v_new = v_top;
      if constexpr (KV8) {
        float top = fabsf(scale[MAX_BN + lane]);  // 0 where a key is not seen at all
        if (!(top < INFINITY)) top = 0.f;
        top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));
        if (v_top == 0.f || top > v_top) v_new = pow2_above(top) * ROOM;
      }
      // A NaN or +inf score makes its row NaN.
      if (__any_sync(0xffffffffu, grow) || v_new != v_top) {
        float al[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          al[e] = 1.f;
          if (!(mx[e] <= m_run[e] + SLACK)) {
            const float m_new = mx[e] < INFINITY ? mx[e] : __uint_as_float(0x7FC00000u);
            const float m_old = m_run[e] == -INFINITY ? -INFINITY : m_use[e];
            m_run[e] = m_new;
            m_use[e] = KV8 ? p_base(m_new, 15.f - SLACK) : m_new;
            al[e] = exp2f(m_old - m_use[e]);
            l_run[e] *= al[e];
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
      if constexpr (!KV8) {
        if (!whole && differ) {
          uint32_t odd = 0;  // rows of V that are not finite: half a warp to a row
#pragma unroll
          for (int r = lane >> 4; r < KC; r += 2) {
            const uint4 x = *reinterpret_cast<const uint4*>(V + ((lane >> 3) & 1) * (STAGE / 4) + r * 128 + (lane & 7) * 16);
            if (not_finite2(x.x) | not_finite2(x.y) | not_finite2(x.z) | not_finite2(x.w)) odd |= 1u << r;
          }
          for (odd = __reduce_or_sync(0xffffffffu, odd); odd; odd &= odd - 1) {
            const int r = __ffs(odd) - 1;
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              uint32_t* at = reinterpret_cast<uint32_t*>(V + (k >> 3) * (STAGE / 4) + r * 128 + (((k & 7) ^ (r & 7)) << 4)) + t;
              const uint32_t w = *at, bad = w & ~finite2(w);
#pragma unroll
              for (int e = 0; e < 2; ++e)
                if (bad && (keep[e] >> r & 1)) {
                  o[k][2 * e] += __uint_as_float(bad << 16);
                  o[k][2 * e + 1] += __uint_as_float(bad & 0xFFFF0000u);
                }
              __syncwarp();
              if (g == 0) *at = finite2(w);
            }
          }
          fence_proxy_async_smem();
          __syncwarp();
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
          for (int k = 0; k < 16; k += 2) {  // bytes k, k + 1 of each key: the columns' codes of two output tiles
            auto word = [&](const uint4& x) { return k < 4 ? x.x : k < 8 ? x.y : k < 12 ? x.z : x.w; };
            const uint32_t sel = k & 2 ? 0x7362 : 0x5140;
            const uint32_t lo = __byte_perm(word(w[0]), word(w[1]), sel), hi = __byte_perm(word(w[2]), word(w[3]), sel);
            mma_f16(o[k], p[k16], codes_f16<DT>(lo & 0xFFFFu), codes_f16<DT>(hi & 0xFFFFu));
            mma_f16(o[k + 1], p[k16], codes_f16<DT>(lo >> 16), codes_f16<DT>(hi >> 16));
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
      next_stage();
    }
    // The warps' sums, and from them the item's (or this CTA's part of them), a
    // thread to a dim.
    float* mine = sums + warp * cut.height * (O_PITCH + 2);
    constexpr float P_TOP = KV8 ? 0x1p15f : 1.f;  // taken out of O here: l * V may pass f32's range
    const float v_back = KV8 ? (v_top == 0.f ? 1.f : v_top / P_TOP) : 1.f;
    named_bar_sync(1, WARPS * 32);  // the last item's have been read
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      l_run[e] += __shfl_xor_sync(0xffffffffu, l_run[e], 1);
      l_run[e] += __shfl_xor_sync(0xffffffffu, l_run[e], 2);
      const int r = g + e * 8;
      if (r >= n_rows) continue;
      if (t == 0) {
        mine[cut.height * O_PITCH + r] = m_run[e] == -INFINITY ? -INFINITY : m_use[e];
        mine[cut.height * (O_PITCH + 1) + r] = l_run[e];
      }
#pragma unroll
      for (int k = 0; k < 16; ++k)
#pragma unroll
        for (int f = 0; f < 2; ++f) {
          const int d = KV8 ? (2 * t + f) * 16 + k : k * 8 + 2 * t + f;
          mine[r * O_PITCH + d] = o[k][2 * e + f] * v_back;
        }
    }
    named_bar_sync(1, WARPS * 32);
    const int dim = threadIdx.x;
    const bool complete = it.i1 - it.i0 == it.t;
    const int64_t slot = 2 * cta + (it.i0 == 0);  // of a part: the stretch's first or last
#pragma unroll 2
    for (int r = 0; r < n_rows; ++r) {
      const float* at = sums + cut.height * O_PITCH + r;
      const int pitch = cut.height * (O_PITCH + 2);
      float m = -INFINITY, l = 0.f, x = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) m = max_nan(m, at[w * pitch]);
      const float mu = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        const float wt = exp2f(at[w * pitch] - mu);
        l += wt * at[w * pitch + cut.height];
        x += wt * sums[w * pitch + r * O_PITCH + dim];
      }
      const bool none = m == -INFINITY;
      const float inv = none ? 0.f : m != m ? m : P_TOP / l;
      const float lse2 = none ? -INFINITY : m + log2f(l);
      if (complete) {
        store_row(ky, qr, it.b, it.sp.first, it.hk, r + it.rt * cut.height, dim, none ? 0.f : x * inv, lse2);
      } else {
        part_o[(slot * 16 + r) * HD + dim] = x * inv;
        if (dim == 0) part_l[slot * 16 + r] = lse2;
      }
    }
  } while (next_item());
  if (!cut.whole && threadIdx.x == 0) {
    // CTA j's stretch begins before the item's end if j * len < end * ctas
    const long long end = stretch(len, cta + 1, cut.ctas) - it.i1 + it.t;
    const bool tail = it.i0 == 0 && it.i1 < it.t;
    split[cta] = Split{it.b, it.hk, it.rt, tail ? (int)((end * cut.ctas + len - 1) / len) - cta : 0};
  }
}

// Joins items that CTAs hold in parts: block (c, r) row r of the one whose first
// part is CTA c's last.
__global__ void __launch_bounds__(HD) join_line_kernel(const __grid_constant__ Keys ky, const __grid_constant__ Queries qr,
                                                       const __grid_constant__ Cut cut, const float* part_o,
                                                       const float* part_l, const Split* split) {
  __shared__ float weight[2 * SMS], tops[HD / 32];
  const int c = blockIdx.x, r = blockIdx.y, dim = threadIdx.x;
  asm volatile("griddepcontrol.wait;\n" ::: "memory");
  const Split it = split[c];
  if (it.parts == 0) return;
  const Span sp = span_of(ky, qr, it.b);
  if (it.rt * cut.height + r >= sp.n * qr.group) return;
  auto at = [&](int j) { return (int64_t)(2 * (c + j) + (j == 0)) * 16 + r; };
  float m = -INFINITY;
  for (int j = dim; j < it.parts; j += HD) m = max_nan(m, weight[j] = part_l[at(j)]);
#pragma unroll
  for (int o = 16; o > 0; o /= 2) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (dim % 32 == 0) tops[dim / 32] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < HD / 32; ++w) m = max_nan(m, tops[w]);
  for (int j = dim; j < it.parts; j += HD) weight[j] = weight[j] == -INFINITY ? 0.f : exp2f(weight[j] - m);
  __syncthreads();
  float l = 0.f, x = 0.f;
#pragma unroll 8
  for (int j = 0; j < it.parts; ++j) {
    const float w = weight[j], v = part_o[at(j) * HD + dim];
    l += w;
    x += w == 0.f ? 0.f : w * v;  // (what a part without keys holds does not matter)
  }
  store_row(ky, qr, it.b, sp.first, it.hk, r + it.rt * cut.height, dim, m == -INFINITY ? 0.f : x / l,
            m == -INFINITY ? m : m + log2f(l));
}

// --------------------------------------------------------------------- host
// Whole items where that costs no more tiles of a CTA's time than equal
// stretches and their join, about eight tiles.
static Cut cut_of(const Shape& sh) {
  const int bn = sh.kv8 ? 128 : 64;
  Cut c{tiling_of(sh.page_size, bn), 1, (int)std::min<int64_t>(std::max<int64_t>(sh.max_new * sh.group, 1), 16), 1, 2};
  const int64_t seqs = std::min<int64_t>(sh.seqs, sh.rows);
  const int64_t items = seqs * (sh.H / sh.group) * ((sh.max_new * sh.group + c.height - 1) / c.height);
  const int64_t n = std::max<int64_t>(tiles_of_keys(sh, bn), 1);
  const double places = 2 * SMS;
  c.whole = std::ceil((double)items / places) * (double)n <= items * n / places + 8;
  c.ctas = (int)std::max<int64_t>(std::min<int64_t>(2 * SMS, c.whole ? items : items * n), 1);
  c.stages = c.height <= 5 ? 3 : 2;
  return c;
}

int64_t parts(const Shape& sh) {
  const Cut c = cut_of(sh);
  return c.whole ? 0 : (2 * 16 + 1) * c.ctas;  // 16 rows of two parts, and the splits
}

template <int DT>
static int start(const PageMaps& tm, const Keys& ky, const Queries& qr, const Cut& cut, float* part_o, float* part_l,
                 cudaStream_t st) {
  static thread_local int configured = -1;
  int dev = 0;
  WFK_CUDA_TRY(cudaGetDevice(&dev));
  if (configured != dev) {
    WFK_CUDA_TRY(cudaFuncSetAttribute(rows_kernel<DT>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM));
    configured = dev;
  }
  Split* split = reinterpret_cast<Split*>(part_l + 32 * cut.ctas);
  rows_kernel<DT><<<(unsigned)cut.ctas, THREADS, smem_of(cut.stages, cut.height), st>>>(tm, ky, qr, cut, part_o, part_l, split);
  WFK_CUDA_TRY(cudaGetLastError());
  if (cut.whole) return WF_OK;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)cut.ctas, (unsigned)cut.height);
  cfg.blockDim = dim3(HD);
  cfg.stream = st;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  WFK_CUDA_TRY(cudaLaunchKernelEx(&cfg, join_line_kernel, ky, qr, cut, (const float*)part_o, (const float*)part_l,
                                  (const Split*)split));
  return WF_OK;
}

int launch(const Keys& ky, const Queries& qr, const Shape& sh, void* workspace, cudaStream_t st) {
  const Cut cut = cut_of(sh);
  float* part_o = static_cast<float*>(workspace);
  float* part_l = part_o + 32 * cut.ctas * HD;
  PageMaps tm;
  int rc;
  if ((rc = page_maps(&tm, ky, qr.H / qr.group, cut.tl, sh.kv8 ? 128 : 64)) != WF_OK) return rc;
  return ky.dtype == WF_DTYPE_BF16   ? start<WF_DTYPE_BF16>(tm, ky, qr, cut, part_o, part_l, st)
         : ky.dtype == WF_DTYPE_E4M3 ? start<WF_DTYPE_E4M3>(tm, ky, qr, cut, part_o, part_l, st)
                                     : start<WF_DTYPE_S8>(tm, ky, qr, cut, part_o, part_l, st);
}

}  // namespace rows
}  // namespace paged
}  // namespace wfk

extern "C" unsigned int wfk_status_take_paged_rows(void) { return wfk::status_take_local(); }
