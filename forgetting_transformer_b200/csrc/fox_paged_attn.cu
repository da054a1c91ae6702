// Forgetting attention of one new token per request against a paged cache (pages, slots and block tables: fox_paged.cu).
//
//   u_j = (q . k_j) sm_scale + sum_{t > j} g_t,  j < length;   out = sum_j softmax(u)_j v_j;   L = log sum_j exp(u_j)
//
// The paged counterpart of fox_decode.cu, for requests of any lengths: those are on the device, so the split is made there.
// Bound by reading every key, value and gate once.
//
// Work is counted in tiles of 16 keys of one unit (a request and a key head, with up to 8 of the query heads that share it).
// All tiles of all units stand in one row, with kPagStart places more in front of each unit for what its start costs; the row is
// cut into equal ranges for the CTAs of a grid that fills the GPU once, and each of these into equal ranges for its warps: the
// longest request and the shortest cost what their tiles cost.  Every CTA sums up the lengths by itself before its first load and
// finds its range there.  A unit of a few hundred keys is not cut between CTAs (its range is moved to the unit's end).  A unit
// that lies in one warp's range is written at once; of one that is cut, each part's (o, m, l, sum of gates) goes to shared memory.
// The CTA joins its warps' parts at its end (from a workspace in global memory, 2 us later, with HBM busy), and a second kernel
// the CTAs' parts, from a workspace.
//
// The bias of a key is the sum of the gates behind it.  A warp goes through its part of a unit from the right, so that this
// is a running sum (exact where the bias is small, which is where it matters; a prefix sum over the whole request would lose
// what the cache's length costs), and the parts' sums shift their maxima when they are joined.
//
// One lane of a warp asks for a tile (TMA, 128-byte swizzle; the gates each lane by 16 bytes for itself) into a ring of
// kStages tiles (of small ones, pairs) that is the warp's own: no warp waits for another.  (Each lane copying by cp.async what it feeds to the matrix
// instructions itself needed no barrier, but its 300 instructions a tile queued for shared memory: 3.6 TB/s.)
// mma.sync m16n8k16 (the two products are 8 query rows at most; the kernel is bound by memory, with a tensor pipe mostly idle):
//   S (16 x 8 keys) = Q K^T, twice, rows 0-7 the unit's query heads.  Lane (x = lane / 4, c = lane % 4) gives 16-byte pieces
//     2 c and 2 c + 1 of a key's row (of each 64 channels; of 32, piece c; of 16, half a piece); which channels stand at which k of an instruction does not matter as long as Q stands the
//     same way.  The two key columns that a lane gets of each S are keys 4 c .. 4 c + 3 of the tile.
//   O (16 x D) += P V.  The registers of S are those of P.  P is rounded to 16 bits, and what the rounding leaves stands in
//     rows 8-15, which would be idle: the sum of the two halves of O has P to 2^-16 (fp16: 2^-21).
// Head dims 16 and 32, whose tiles are small, are bound by a tile's chain of instructions: a warp takes two tiles together, through
// boxes as wide as they are (16 requests of 1000 to 9000 keys x 16 heads of 32, 126 MB: one tile, filled up to 64 columns, 38 us; two 32).
//
// Tiles never leave a page (pages are 16 keys at least).  Rows behind the last key may hold anything: their logits are
// replaced, their values set to zero.  A table entry outside the pool is not read: its keys take no part.
#include "fox_common.cuh"
#include "fox_host.h"

#include <atomic>

namespace fox {

constexpr int kPagGrid = kSms;
// Warps of a CTA, each with two tiles asked for: some 110 and 140 KB in flight on an SM.  More is slower, since SMs then get more
// uneven shares of the bandwidth (24 x 65536 keys of 64: 12 warps x 2 tiles 70.5 us, 16 x 3 76; 32 x 2048 x 16 heads of 128: 8 x 2
// 91, 8 x 3 98, 10 x 2 94), fewer warps too (8 x 4 88).  Head dims 16 and 32 are bound by what a tile takes a warp, not by its
// bytes: 16 warps (16 requests of 1000 to 9000 keys x 16 heads of 32: 12 warps 35 us, 16 32).
__host__ __device__ constexpr int pag_warps(int64_t D) { return D == 128 ? 8 : D == 64 ? 12 : 16; }
constexpr int kPagTile = 16;
constexpr int kPagRows = 8;          // query heads of a unit
constexpr int kPagStart = 1;         // what the start of a unit costs, in tiles
constexpr int kPagLeast = 3;         // places of a warp
// Units of up to so many places are one CTA's: some 280 KB of keys and values, which one SM reads in the time that parts of several
// CTAs take to be joined.
__host__ __device__ constexpr int pag_whole(int64_t D) { return (D == 128 ? 32 : 64) + kPagStart; }
constexpr int kPagSite = 95;           // of a wait that ran out
constexpr float kPagLog2e = 1.4426950408889634f, kPagLn2 = 0.6931471805599453f;

struct PagedParams {
  const uint16_t* q;
  int64_t q_sr, q_sh, g_sp, g_sh, o_sr, o_sh;
  const float* gates;
  const int32_t *table, *lengths;
  int64_t table_ld;
  uint16_t* o;
  float* L;                            // (R, H) or nullptr
  float* part;                         // (CTAs, 2, rows, D + 4)
  int R, H, group, rows, tiles_of_group, units, n_pages, page_log2;   // rows: of a unit; units: of a request
  int32_t* status;
  Divisor by_units, by_tiles_of_group;
  int64_t most;                        // keys that a table row has entries for
  float qk_scale;                      // sm_scale * log2(e)
};

__device__ __forceinline__ int pag_length(const PagedParams& p, int r) {
  const int64_t n = p.lengths[r];
  return static_cast<int>(n < 0 ? 0 : n < p.most ? n : p.most);
}
__device__ __forceinline__ int pag_per_cta(int places) { return (places + kPagGrid - 1) / kPagGrid; }
// t / d (an integer division is forty instructions): the product is off by less than 2 for quotients below 2^22
__device__ __forceinline__ int pag_div(int t, int d) {
  int q = static_cast<int>(static_cast<float>(t) * __frcp_rn(static_cast<float>(d)));
  int left = static_cast<int>(static_cast<uint32_t>(t) - static_cast<uint32_t>(q) * static_cast<uint32_t>(d));
  while (left < 0) {
    left += d;
    --q;
  }
  while (left >= d) {
    left -= d;
    ++q;
  }
  return q;
}
// a request's length in the row of tiles, for one unit
__device__ __forceinline__ int pag_places(int length) { return length ? (length + kPagTile - 1) / kPagTile + kPagStart : 0; }

// Asks L1 for what will be loaded from here in a while.
__device__ __forceinline__ void touch(const void* p) {
  uint16_t unused;
  asm volatile("ld.global.u16 %0, [%1];" : "=h"(unused) : "l"(p) : "memory");
}

template <bool kBf16>
__device__ __forceinline__ void mma_16816(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (kBf16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kLeft>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory"); }
// a tile of 64-column halves: (64, rows, halves, heads, pages), innermost first
__device__ __forceinline__ void tma_load_5d(uint32_t dst, const CUtensorMap* tm, uint64_t* bar, int row, int head, int page) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %3, %5, %6}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(tm)), "r"(smem_u32(bar)), "r"(0), "r"(row), "r"(head), "r"(page)
      : "memory");
}
// four 8 x 8 matrices of 16-bit values, each transposed, one row's address from every lane
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint4 lds_v4(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}

__device__ __forceinline__ uint2 lds_v2(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
  return v;
}

template <int D>
struct PagedTile {
  static constexpr int kHalves = D == 128 ? 2 : 1;            // boxes of 16 keys x 64 columns, or of all columns
  static constexpr int kRow = D < 64 ? D * 2 : 128;           // bytes of a row in a box, over which the copy's swizzle goes
  static constexpr int kBox = kPagTile * kRow;
  static constexpr int kTile = 2 * kHalves * kBox;            // keys, values
  static constexpr int kSub = D < 64 ? 2 : 1;                 // tiles that a warp takes together
  static constexpr int kStage = kSub * kTile;
  static constexpr int kGates = kSub * kPagRows * kPagTile * 4;
  static constexpr int kCols = D / 8;                         // n of the second product
  static constexpr int kStages = 2;
  static constexpr int kWarps = pag_warps(D), kThreads = kWarps * 32;
  static constexpr int kParts = kWarps * kStages * (kStage + kGates);   // where the warps' parts begin: (warps, 2, rows, D + 4)
  static constexpr int kSmem = kParts + kWarps * 2 * kPagRows * (D + 4) * 4 + 1024;   // (boxes begin at multiples of 1024 bytes)
  // where the swizzle has put 16-byte piece `piece` of a key's row
  static __device__ __forceinline__ uint32_t at(uint32_t key, uint32_t piece) {
    return key * kRow + (piece ^ (D < 32 ? (key >> 2) & 1 : D < 64 ? (key >> 1) & 3 : key & 7)) * 16;
  }
};

// What a stage's tiles are: written by lane 0, read by the warp.
struct PagedItem {
  int r, h0, valid, flags;   // first query head; keys of the tiles that count, 8 bits for each; kItemFirst ... below, and the heads from bit 8 on
};
enum { kItemFirst = 1, kItemLast = 2, kItemWhole = 4, kItemSecond = 8 };   // of its part; a unit's only part; workspace place 1

struct PagedUnit {
  int r, unit, at, places, length;   // at: its first place in the row
};

template <bool kBf16, int D>
__global__ void __launch_bounds__(PagedTile<D>::kThreads, 1)
fox_paged_attn_kernel(const PagedParams p, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v) {
  using Tile = PagedTile<D>;
  constexpr int kStages = Tile::kStages, kThreads = Tile::kThreads, kWarps = Tile::kWarps, kSub = Tile::kSub;
  extern __shared__ __align__(1024) char pag_smem[];
  __shared__ uint64_t s_full[kWarps][kStages];
  __shared__ int s_abort;
  __shared__ int s_before[kThreads + 1];
  __shared__ int s_length[kThreads];
  __shared__ PagedUnit s_unit[kWarps + 1];   // that the warps' ranges begin in; that the CTA's ends in
  __shared__ int s_range[3];
  __shared__ int s_warp[kWarps];
  __shared__ PagedItem s_item[kWarps][kStages];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (lane == 0) {
    for (int s = 0; s < kStages; ++s) mbar_init(&s_full[warp][s], 1);
    mbar_fence_init();
    if (warp == 0) {
      s_abort = 0;
      tma_prefetch_desc(&map_k);
      tma_prefetch_desc(&map_v);
    }
  }
  wait_for_kernel_in_front();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");   // (the joining kernel, which waits for this one's end)

  // ---- where every thread's share of the requests begins in the row of places
  const int share = (p.R + kThreads - 1) / kThreads;
  const int r_first = min(tid * share, p.R), r_end = min(r_first + share, p.R);
  int mine = 0;
  for (int r = r_first; r < r_end; ++r) {
    const int n = pag_length(p, r);
    s_length[tid] = n;   // (used where a share is one request)
    if (share == 1 && n) touch(p.table + r * p.table_ld + ((n - 1) >> p.page_log2));   // (where its pages will be looked up first)
    mine += pag_places(n);
  }
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += y;
  }
  if (lane == 31) s_warp[warp] = incl;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWarps; ++w)
    if (w < warp) incl += s_warp[w];
  s_before[tid + 1] = incl;
  if (tid == 0) s_before[0] = 0;
  __syncthreads();
  // ---- requests without a key
  for (int r = blockIdx.x; r < p.R; r += gridDim.x) {
    if (share == 1 ? s_length[r] : pag_length(p, r)) continue;
    for (int i = tid; i < p.H * D; i += kThreads) p.o[r * p.o_sr + (i / D) * p.o_sh + i % D] = 0;
    if (p.L)
      for (int h = tid; h < p.H; h += kThreads) p.L[static_cast<int64_t>(r) * p.H + h] = -INFINITY;
  }
  const int total = s_before[kThreads] * p.units, per_cta = pag_per_cta(total), raw = min(static_cast<int>(blockIdx.x) * per_cta, total);   // (148 * per_cta is below 2^30 + 148)

  // ---- this CTA's range, moved to the ends of units that are not cut, and in it those of its warps: by one warp, a place to a lane
  if (warp == 0 && total > 0) {
    const int raw_end = min(raw + per_cta, total);
    auto share_of = [&](int t) {   // the last share that begins at or before place t (the same t for all lanes)
      const int q = div_by(p.by_units, t);
      constexpr int kStep = kThreads / 32;
      const int hi = (__popc(__ballot_sync(0xffffffffu, s_before[lane * kStep] <= q)) - 1) * kStep;
      return hi + __popc(__ballot_sync(0xffffffffu, lane < kStep && s_before[hi + lane] <= q)) - 1;
    };
    const int share_lo = share_of(min(raw, total - 1)), share_hi = share_of(min(raw_end, total - 1));
    auto find = [&](int t) {   // the unit that place t (< total, in these shares) of the row belongs to
      const int q = div_by(p.by_units, t);
      int lo = share_lo, hi = share_hi;
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (s_before[mid] <= q) lo = mid;
        else hi = mid - 1;
      }
      int before = s_before[lo];
      PagedUnit f;
      f.r = lo * share;
      f.length = share == 1 ? s_length[lo] : pag_length(p, f.r);
      f.places = pag_places(f.length);
      while (before + f.places <= q) {
        before += f.places;
        f.length = pag_length(p, ++f.r);
        f.places = pag_places(f.length);
      }
      const int off = t - before * p.units;
      f.unit = pag_div(off, f.places);
      f.at = before * p.units + f.unit * f.places;
      return f;
    };
    int edge = lane ? raw_end : raw;   // lane 0: where the range begins; the others: where it ends
    if (edge < total) {
      const PagedUnit f = find(edge);
      if (f.at < edge && f.places <= pag_whole(D)) edge = f.at + f.places;
    }
    const int c_begin = __shfl_sync(0xffffffffu, edge, 0), c_end = __shfl_sync(0xffffffffu, edge, 1);
    const int per = max((c_end - c_begin + kWarps - 1) / kWarps, kPagLeast);
    const int t = lane < kWarps ? c_begin + lane * per : c_end - 1;   // (the last: the unit that the range ends in)
    if (lane <= kWarps && t < c_end && c_begin < c_end) s_unit[lane] = find(t);
    if (lane == 0) {
      s_range[0] = c_begin;
      s_range[1] = c_end;
      s_range[2] = per;
    }
  }
  __syncthreads();
  if (total == 0) return;
  const int c_begin = s_range[0], c_end = s_range[1], per = s_range[2];
  if (c_begin >= c_end) return;
  const int t_begin = min(c_begin + warp * per, c_end);
  int r = 0, unit = 0, n_tiles = 0, place = 0, at = -1, part_lo = 0, length = 0, flags = 0, kh = 0, h0 = 0, heads = 0;   // the part asked for: tiles part_lo .. at
  int left = min(per, c_end - t_begin);   // places not yet gone through
  if (left > 0) {
    const PagedUnit f = s_unit[warp];
    r = f.r;
    unit = f.unit;
    place = t_begin - f.at;
    length = f.length;
    n_tiles = f.places - kPagStart;
  }
  // the unit's part from `place` on, as far as the range goes; none (at < part_lo) where it ends inside the unit's start
  auto begin_part = [&](int second) {
    const int take = min(n_tiles + kPagStart - place, left);
    kh = div_by(p.by_tiles_of_group, unit);
    const int in_group = (unit - kh * p.tiles_of_group) * kPagRows;
    h0 = kh * p.group + in_group;
    heads = min(p.group - in_group, kPagRows);
    part_lo = max(place - kPagStart, 0);
    at = max(place + take - kPagStart, 0) - 1;
    left -= take;
    flags = kItemFirst | second | (part_lo == 0 && at == n_tiles - 1 ? kItemWhole : 0) | heads << 8;
  };
  if (left > 0) begin_part(0);

  const uint32_t smem0 = (smem_u32(pag_smem) + 1023) & ~1023u;
  char* const base = pag_smem + (smem0 - smem_u32(pag_smem));
  char* const ring = base + warp * kStages * Tile::kStage;
  float* const ring_g = reinterpret_cast<float*>(base + kWarps * kStages * Tile::kStage + warp * kStages * Tile::kGates);
  float* const parts = reinterpret_cast<float*>(base + Tile::kParts);
  const int x = lane >> 2, c = lane & 3;
  // (rows of gates that no head fills: finite)
#pragma unroll
  for (int s = 0; s < kStages * kSub; ++s) *reinterpret_cast<float4*>(ring_g + s * (kPagRows * kPagTile) + lane * 4) = make_float4(0.f, 0.f, 0.f, 0.f);
  const uint32_t ring_u32 = smem_u32(ring), gates_u32 = smem_u32(ring_g) + lane * 16;
  int page_r = -1, page_base = 0, page_ids = -1;   // 32 entries of a request's table row, one to a lane

  int ask_stage = 0;
  int pending = 0;   // tiles asked for and not yet used
  auto ask = [&]() {   // the next kSub tiles
    if (at < part_lo) {
      cp_async_commit();
      return;
    }
    int id[kSub], row0[kSub], valid = 0, loads = 0;
#pragma unroll
    for (int s = kSub - 1; s >= 0; --s) {   // (the walk goes to the left)
      id[s] = -1;
      row0[s] = 0;
      if (at < part_lo) continue;
      const int key0 = at * kPagTile, j = key0 >> p.page_log2;
      row0[s] = key0 & ((1 << p.page_log2) - 1);
      if (r != page_r || j < page_base || j >= page_base + 32) {
        page_r = r;
        page_base = j < 31 ? 0 : j - 31;
        const int e = page_base + lane;
        page_ids = static_cast<int64_t>(e) << p.page_log2 < length ? p.table[r * p.table_ld + e] : -1;
      }
      const int page = __shfl_sync(0xffffffffu, page_ids, j - page_base);
      if (page >= 0 && page < p.n_pages) {
        id[s] = page;
        valid |= min(length - key0, kPagTile) << (8 * s);
        ++loads;
      }
      --at;
    }
    const bool last = at < part_lo;
    uint64_t* const bar = &s_full[warp][ask_stage];
    if (lane == 0) {
      s_item[warp][ask_stage] = {r, h0, valid, flags | (last ? kItemLast : 0)};
      if (loads) {
        mbar_expect_tx(bar, loads * Tile::kTile);
#pragma unroll
        for (int s = 0; s < kSub; ++s) {
          const uint32_t to = ring_u32 + ask_stage * Tile::kStage + s * Tile::kTile;
          if (id[s] < 0) continue;
          tma_load_5d(to, &map_k, bar, row0[s], kh, id[s]);
          tma_load_5d(to + Tile::kTile / 2, &map_v, bar, row0[s], kh, id[s]);
        }
      } else {
        mbar_arrive(bar);
      }
    }
#pragma unroll
    for (int s = 0; s < kSub; ++s)
      if (id[s] >= 0 && x < heads)
        cp_async_16(gates_u32 + ask_stage * Tile::kGates + s * (kPagRows * kPagTile * 4), p.gates + id[s] * p.g_sp + (h0 + x) * p.g_sh + row0[s] + 4 * c);
    cp_async_commit();
    if ((flags & kItemFirst) && x < heads) touch(p.q + r * p.q_sr + (h0 + x) * p.q_sh + (D < 32 ? c * 4 : D < 64 ? c * 8 : c * 16));
    flags &= ~kItemFirst;
    ++pending;
    if (last && left > 0) {   // the next unit
      place = 0;
      if (++unit == p.units) {
        unit = 0;
        do {
          length = pag_length(p, ++r);
        } while (length == 0);   // (places are left, so there is a request with keys)
        n_tiles = (length + kPagTile - 1) / kPagTile;
      }
      begin_part(kItemSecond);
    }
    ask_stage = ask_stage == kStages - 1 ? 0 : ask_stage + 1;
  };

#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) ask();

  constexpr float kShift = kBf16 ? 0.f : 12.f;   // fp16: weights up to 2^12, so that small ones keep their bits
  // a lane's pieces of keys 4 (x / 2) + x % 2 and 2 on in a box: from 64 columns on, 2 c and (^ 16) 2 c + 1; of 32 columns, c; of 16,
  // half of one
  const uint32_t key_a = 4 * (x >> 1) + (x & 1), piece = D < 32 ? c >> 1 : D < 64 ? c : 2 * c;
  const uint32_t k_off = Tile::at(key_a, piece) + (D < 32 ? (c & 1) * 8 : 0), k_off2 = Tile::at(key_a + 2, piece) + (D < 32 ? (c & 1) * 8 : 0);
  // the row of the values whose address a lane gives: keys 4 (j / 2) + j % 2, in matrices 1 and 3 2 on; in 2 and 3 the next 8 columns
  const uint32_t key_v = 4 * ((lane & 7) >> 1) + (lane & 1) + 2 * ((lane >> 3) & 1), v_off = Tile::at(key_v, static_cast<uint32_t>(lane) >> 4);
  constexpr int kPieces = D < 64 ? 1 : 2 * Tile::kHalves;
  uint4 qf[kPieces];   // the channels of a lane's pieces
  float o[Tile::kCols][4], m = -INFINITY, l = 0.f, carry = 0.f;
  int stage = 0;
  uint32_t parity = 0;
  for (;;) {
    ask();
    if (pending == 0) break;
    if (!mbar_wait_warp(&s_full[warp][stage], parity, &s_abort, p.status, kPagSite, pending)) break;
    --pending;
    cp_async_wait<kStages - 1>();   // (each lane's own gates)
    __syncwarp();
    const PagedItem item = s_item[warp][stage];
    const uint32_t tile = ring_u32 + stage * Tile::kStage;
    const bool row = x < item.flags >> 8;   // a row of the unit
    if (item.flags & kItemFirst) {
      constexpr int kOwn = D < 32 ? 4 : D < 64 ? 8 : 16;   // channels of a lane in 64, or in all
      const uint16_t* qp = p.q + item.r * p.q_sr + (item.h0 + x) * p.q_sh + c * kOwn;
#pragma unroll
      for (int s = 0; s < kPieces; ++s) {
        qf[s] = make_uint4(0u, 0u, 0u, 0u);
        if constexpr (D < 32) {
          const uint2 v = row ? *reinterpret_cast<const uint2*>(qp) : make_uint2(0u, 0u);
          qf[s].x = v.x;
          qf[s].y = v.y;
        } else if (row) {
          qf[s] = *reinterpret_cast<const uint4*>(qp + (s >> 1) * 64 + (s & 1) * 8);
        }
      }
#pragma unroll
      for (int j = 0; j < Tile::kCols; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[j][i] = 0.f;
      m = -INFINITY;
      l = carry = 0.f;
    }
    int valid[kSub];
#pragma unroll
    for (int s = 0; s < kSub; ++s) valid[s] = kSub == 1 ? item.valid : item.valid >> (8 * s) & 255;
    // ---- gates: sums behind each of the lane's four keys, inside the part
    float bias[kSub][4];
    {
      float own[kSub][3], behind[kSub], y[kSub];   // behind: of this lane and those to its right
#pragma unroll
      for (int s = 0; s < kSub; ++s) {
        const float4 gv = *reinterpret_cast<const float4*>(ring_g + (stage * kSub + s) * (kPagRows * kPagTile) + lane * 4);
        float g[4] = {gv.x, gv.y, gv.z, gv.w};
        if (valid[s] < kPagTile) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (4 * c + i >= valid[s]) g[i] = 0.f;
        }
        own[s][2] = g[3];
        own[s][1] = g[3] + g[2];
        own[s][0] = own[s][1] + g[1];
        behind[s] = own[s][0] + g[0];
      }
#pragma unroll
      for (int s = 0; s < kSub; ++s) y[s] = __shfl_down_sync(0xffffffffu, behind[s], 1, 4);
#pragma unroll
      for (int s = 0; s < kSub; ++s) behind[s] += c < 3 ? y[s] : 0.f;
#pragma unroll
      for (int s = 0; s < kSub; ++s) y[s] = __shfl_down_sync(0xffffffffu, behind[s], 2, 4);
#pragma unroll
      for (int s = 0; s < kSub; ++s) behind[s] += c < 2 ? y[s] : 0.f;
#pragma unroll
      for (int s = 0; s < kSub; ++s) y[s] = __shfl_down_sync(0xffffffffu, behind[s], 1, 4);   // (not behind - sum: a gate of minus
                                                                                             // infinity cannot be taken off again)
#pragma unroll
      for (int s = kSub - 1; s >= 0; --s) {
        const float right = c < 3 ? carry + y[s] : carry;
#pragma unroll
        for (int i = 0; i < 3; ++i) bias[s][i] = (right + own[s][i]) * kPagLog2e;
        bias[s][3] = right * kPagLog2e;
        carry += __shfl_sync(0xffffffffu, behind[s], 0, 4);
      }
    }
    // ---- S
    float u[kSub][4];
#pragma unroll
    for (int s = 0; s < kSub; ++s) {
      float s0[4] = {0.f, 0.f, 0.f, 0.f}, s1[4] = {0.f, 0.f, 0.f, 0.f};
      const uint32_t tile_k = tile + s * Tile::kTile;
      if constexpr (D < 32) {
        const uint2 ka = lds_v2(tile_k + k_off), kb = lds_v2(tile_k + k_off2);
        mma_16816<kBf16>(s0, qf[0].x, 0u, qf[0].y, 0u, ka.x, ka.y);
        mma_16816<kBf16>(s1, qf[0].x, 0u, qf[0].y, 0u, kb.x, kb.y);
      } else {
#pragma unroll
        for (int e = 0; e < kPieces; ++e) {
          const uint32_t at_k = tile_k + (e >> 1) * Tile::kBox;
          const uint4 ka = lds_v4(at_k + (k_off ^ ((e & 1) * 16))), kb = lds_v4(at_k + (k_off2 ^ ((e & 1) * 16)));
          mma_16816<kBf16>(s0, qf[e].x, 0u, qf[e].y, 0u, ka.x, ka.y);
          mma_16816<kBf16>(s1, qf[e].x, 0u, qf[e].y, 0u, kb.x, kb.y);
          mma_16816<kBf16>(s0, qf[e].z, 0u, qf[e].w, 0u, ka.z, ka.w);
          mma_16816<kBf16>(s1, qf[e].z, 0u, qf[e].w, 0u, kb.z, kb.w);
        }
      }
      u[s][0] = fmaf(s0[0], p.qk_scale, bias[s][0]);
      u[s][1] = fmaf(s0[1], p.qk_scale, bias[s][1]);
      u[s][2] = fmaf(s1[0], p.qk_scale, bias[s][2]);
      u[s][3] = fmaf(s1[1], p.qk_scale, bias[s][3]);
      if (valid[s] < kPagTile) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (4 * c + i >= valid[s]) u[s][i] = -INFINITY;
      }
    }
    float mx = m;
#pragma unroll
    for (int s = 0; s < kSub; ++s) mx = fmaxf(fmax3(u[s][0], u[s][1], u[s][2]), fmaxf(u[s][3], mx));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
    if (__any_sync(0xffffffffu, mx > m)) {   // (NaN logits: no new maximum, and NaN weights)
      const float alpha = m == -INFINITY ? 0.f : fast_exp2(m - mx);
      l *= alpha;
#pragma unroll
      for (int j = 0; j < Tile::kCols; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[j][i] *= alpha;
      m = mx;
    }
    const float ref = m == -INFINITY ? 0.f : m - kShift;
#pragma unroll
    for (int s = 0; s < kSub; ++s) {
      // ---- P, its 16-bit values and what they leave
      float w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = fast_exp2(u[s][i] - ref);
      l += (w[0] + w[1]) + (w[2] + w[3]);
      const uint32_t hi0 = pack2<kBf16>(w[0], w[1]), hi1 = pack2<kBf16>(w[2], w[3]);
      const float2 r0 = unpack2<kBf16>(hi0), r1 = unpack2<kBf16>(hi1);
      const uint32_t lo0 = pack2<kBf16>(w[0] - r0.x, w[1] - r0.y), lo1 = pack2<kBf16>(w[2] - r1.x, w[3] - r1.y);
      // ---- O
      const uint32_t tile_v = tile + s * Tile::kTile + Tile::kHalves * Tile::kBox;
      const bool whole = valid[s] == kPagTile;
      uint32_t keep0 = 0xffffffffu, keep1 = 0xffffffffu;   // of keys 4 c, 4 c + 1; of the next two
      if (!whole) {
        const int n = valid[s] - 4 * c;
        keep0 = n >= 2 ? 0xffffffffu : n == 1 ? 0xffffu : 0u;
        keep1 = n >= 4 ? 0xffffffffu : n == 3 ? 0xffffu : 0u;
      }
#pragma unroll
      for (int j = 0; j < Tile::kCols; j += 2) {
        uint32_t v[4];
        ldmatrix_x4_trans(tile_v + (j >> 3) * Tile::kBox + (v_off ^ ((j & 7) * 16)), v);
        if (!whole) {   // (a row behind the last key may hold anything, and zero times NaN is NaN)
          v[0] &= keep0;
          v[1] &= keep1;
          v[2] &= keep0;
          v[3] &= keep1;
        }
        mma_16816<kBf16>(o[j], hi0, lo0, hi1, lo1, v[0], v[1]);
        mma_16816<kBf16>(o[j + 1], hi0, lo0, hi1, lo1, v[2], v[3]);
      }
    }
    if (item.flags & kItemLast) {
      float ls = l + __shfl_xor_sync(0xffffffffu, l, 1);
      ls += __shfl_xor_sync(0xffffffffu, ls, 2);
      const float m_ref = ls != ls ? ls : m == -INFINITY ? -INFINITY : m - kShift;   // (NaN stays visible when parts are joined)
      if (row) {
        const int h = item.h0 + x;
        if (item.flags & kItemWhole) {
          const float inv = ls != 0.f ? 1.f / ls : 0.f;   // (a NaN sum stays one)
          uint16_t* to = p.o + item.r * p.o_sr + h * p.o_sh;
#pragma unroll
          for (int j = 0; j < Tile::kCols; ++j)
            *reinterpret_cast<uint32_t*>(to + j * 8 + 2 * c) = pack2<kBf16>((o[j][0] + o[j][2]) * inv, (o[j][1] + o[j][3]) * inv);
          if (p.L && c == 0) p.L[static_cast<int64_t>(item.r) * p.H + h] = ls != 0.f ? m_ref * kPagLn2 + __logf(ls) : -INFINITY;
        } else {
          float* to = parts + ((warp * 2 + (item.flags & kItemSecond ? 1 : 0)) * p.rows + x) * (D + 4);
#pragma unroll
          for (int j = 0; j < Tile::kCols; ++j)
            *reinterpret_cast<float2*>(to + j * 8 + 2 * c) = make_float2(o[j][0] + o[j][2], o[j][1] + o[j][3]);
          if (c == 0) {
            to[D] = m_ref;
            to[D + 1] = ls;
            to[D + 2] = carry * kPagLog2e;
          }
        }
      }
    }
    __syncwarp();   // (the tile and its item have been read before their place is written again)
    if (++stage == kStages) {
      stage = 0;
      parity ^= 1;
    }
  }
  if (pending > 0) {   // gave up: the copies that are still in flight end before their memory does
    volatile int none = 0;
    for (; pending > 0; --pending) {
      mbar_wait_warp(&s_full[warp][stage], parity, &none, p.status, kPagSite, -1);
      none = 0;
      if (++stage == kStages) {
        stage = 0;
        parity ^= 1;
      }
    }
  }
  cp_async_wait<0>();
  // ---- the parts of this CTA's warps joined: those of the unit that a warp's range begins in, where it ends in that range or the
  // CTA's range ends there, and those of the unit that the CTA's range ends in.  A unit that other CTAs have a part of becomes one
  // part of this CTA's.  The query heads of these units go around the warps.
  __syncthreads();
  for (int i = warp; i < (kWarps + 1) * p.rows; i += kWarps) {
    const int row_j = i / (kWarps + 1), of = i - row_j * (kWarps + 1);
    const int b = of < kWarps ? c_begin + of * per : c_end - 1, e = min(b + per, c_end);
    if (b >= c_end) continue;
    const PagedUnit f = s_unit[of];
    if (of < kWarps ? f.at + f.places > e && e != c_end : f.at <= c_begin + pag_div(c_end - 1 - c_begin, per) * per) continue;   // (the first unit of
                                                                                                       // the last range has its turn as that)
    const int first = max(f.at + kPagStart, c_begin), last = min(f.at + f.places, c_end) - 1;   // of its places with tiles here
    if (first > last) continue;
    const int wa = pag_div(first - c_begin, per), n = pag_div(last - c_begin, per) - wa + 1;
    const bool here = f.at + kPagStart >= c_begin && f.at + f.places <= c_end;   // all of its tiles
    if (here && n == 1) continue;   // (written where it was computed)
    const int kh_j = div_by(p.by_tiles_of_group, f.unit), in_group = (f.unit - kh_j * p.tiles_of_group) * kPagRows;
    const int h_j = kh_j * p.group + in_group + row_j;
    if (row_j >= p.group - in_group) continue;
    const int rows_ld = p.rows * (D + 4);
    const float* from = parts + wa * 2 * rows_ld + row_j * (D + 4);
    const bool second = c_begin + wa * per < f.at;   // the first part's place: its warp has begun in another unit
    auto part = [&](int s) { return from + 2 * s * rows_ld + (s == 0 && second ? rows_ld : 0); };
    // lane s: part s
    float4 st = make_float4(-INFINITY, 0.f, 0.f, 0.f);
    if (lane < n) st = *reinterpret_cast<const float4*>(part(lane) + D);
    constexpr int kPer = D / 32 > 0 ? D / 32 : 1;   // channels of a lane
    float v[kWarps][kPer];
#pragma unroll
    for (int s = 0; s < kWarps; ++s) {
      const float* at_v = part(s) + lane * kPer;
      const bool in = s < n && lane * kPer < D;
      if constexpr (kPer == 4) {
        const float4 x4 = in ? *reinterpret_cast<const float4*>(at_v) : make_float4(0.f, 0.f, 0.f, 0.f);
        v[s][0] = x4.x; v[s][1] = x4.y; v[s][2] = x4.z; v[s][3] = x4.w;
      } else if constexpr (kPer == 2) {
        const float2 x2 = in ? *reinterpret_cast<const float2*>(at_v) : make_float2(0.f, 0.f);
        v[s][0] = x2.x; v[s][1] = x2.y;
      } else {
        v[s][0] = in ? *at_v : 0.f;
      }
    }
    constexpr int kUp = kWarps > 8 ? 16 : 8;   // lanes that the shuffles below go over
    float behind = st.z, y;   // gates of the parts from this one on
#pragma unroll
    for (int o = 1; o < kUp; o <<= 1) {
      y = __shfl_down_sync(0xffffffffu, behind, o);
      if (lane + o < kUp) behind += y;
    }
    const float all = __shfl_sync(0xffffffffu, behind, 0);
    y = __shfl_down_sync(0xffffffffu, behind, 1);
    const float mm = lane < n ? st.x + (lane + 1 < kUp ? y : 0.f) : -INFINITY;
    float top = mm;
#pragma unroll
    for (int o = kUp / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float w = mm == -INFINITY ? 0.f : fast_exp2(mm - top);   // (NaN stays)
    float sum = st.y * w;
#pragma unroll
    for (int o = kUp / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    float acc[kPer];
#pragma unroll
    for (int c_i = 0; c_i < kPer; ++c_i) acc[c_i] = 0.f;
#pragma unroll
    for (int s = 0; s < kWarps; ++s) {
      const float ws = __shfl_sync(0xffffffffu, w, s);
#pragma unroll
      for (int c_i = 0; c_i < kPer; ++c_i)
        if (s < n) acc[c_i] = fmaf(v[s][c_i], ws, acc[c_i]);   // (a weight of zero too: a NaN value counts)
    }
    sum = __shfl_sync(0xffffffffu, sum, 0);
    top = __shfl_sync(0xffffffffu, top, 0);
    if (here) {
      const float inv = sum != 0.f ? 1.f / sum : 0.f;
      uint16_t* to = p.o + f.r * p.o_sr + h_j * p.o_sh + lane * kPer;
      if (lane * kPer < D) {
        if constexpr (kPer == 1) {
          *to = static_cast<uint16_t>(pack2<kBf16>(acc[0] * inv, 0.f) & 0xffffu);
        } else {
#pragma unroll
          for (int c_i = 0; c_i < kPer; c_i += 2) *reinterpret_cast<uint32_t*>(to + c_i) = pack2<kBf16>(acc[c_i] * inv, acc[c_i + 1] * inv);
        }
      }
      if (p.L && lane == 0) p.L[static_cast<int64_t>(f.r) * p.H + h_j] = sum != 0.f ? top * kPagLn2 + __logf(sum) : -INFINITY;
    } else {
      float* to = p.part + (static_cast<int64_t>(blockIdx.x) * 2 + (raw < f.at ? 1 : 0)) * rows_ld + row_j * (D + 4);
      if (lane * kPer < D)
#pragma unroll
        for (int c_i = 0; c_i < kPer; ++c_i) to[lane * kPer + c_i] = acc[c_i];
      if (lane == 0) *reinterpret_cast<float4*>(to + D) = make_float4(sum != sum ? sum : top, sum, all, 0.f);
    }
  }
}

// Joins the CTAs' parts of units that several CTAs have a part of.  A CTA here takes (request, query head) pairs.  A unit's parts
// stand from the left: their gate sums are added from the right by one warp, 32 parts at a time.  kLanes lanes share a part's
// channels, the kGroups groups of threads each take every kGroups-th part; the first kAhead of these are asked for before the weights
// are known.
constexpr int kJoinThreads = 128;
template <bool kBf16, int D>
__global__ void __launch_bounds__(kJoinThreads) fox_paged_join_kernel(const PagedParams p) {
  constexpr int kLanes = D / 4, kGroups = kJoinThreads / kLanes, kAhead = 8;
  __shared__ float s_w[kPagGrid], s_l[kPagGrid], s_g[kPagGrid], s_sum, s_top;
  __shared__ float4 s_o[kJoinThreads];
  __shared__ int s_sum_before[kJoinThreads / 32], s_sum_all[kJoinThreads / 32];
  const int tid = threadIdx.x, sub = tid % kLanes, g0 = tid / kLanes;
  // Lengths may be read before the first kernel has ended: it has waited for what wrote them.
  bool waited = false;
  const int64_t items = static_cast<int64_t>(p.R) * p.H;
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int r = static_cast<int>(item < (int64_t{1} << 31) ? static_cast<uint32_t>(item) / static_cast<uint32_t>(p.H) : item / p.H);
    const int h = static_cast<int>(item - static_cast<int64_t>(r) * p.H);
    const int places = pag_places(pag_length(p, r));
    if (places <= pag_whole(D)) continue;
    int before = 0, all = 0;
    for (int i = tid; i < p.R; i += kJoinThreads) {
      const int n = pag_places(pag_length(p, i));
      all += n;
      if (i < r) before += n;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      before += __shfl_xor_sync(0xffffffffu, before, o);
      all += __shfl_xor_sync(0xffffffffu, all, o);
    }
    if ((tid & 31) == 0) {
      s_sum_before[tid >> 5] = before;
      s_sum_all[tid >> 5] = all;
    }
    __syncthreads();
    before = all = 0;
#pragma unroll
    for (int i = 0; i < kJoinThreads / 32; ++i) {
      before += s_sum_before[i];
      all += s_sum_all[i];
    }
    const int per = pag_per_cta(all * p.units);
    const int kh = h / p.group, row = h - kh * p.group, unit = kh * p.tiles_of_group + row / kPagRows;
    const int u0 = before * p.units + unit * places;
    const int w0 = pag_div(u0 + kPagStart, per), n = pag_div(u0 + places - 1, per) - w0 + 1;
    __syncthreads();   // (the sums have been read)
    if (n == 1) continue;
    const int64_t ld = static_cast<int64_t>(p.rows) * (D + 4);
    const float* base = p.part + (static_cast<int64_t>(w0) * 2 * p.rows + row % kPagRows) * (D + 4);
    const int second = w0 * per < u0;   // the first part's place: its CTA's range has begun in another unit
    auto at = [&](int s) { return base + (2 * s + (s == 0 ? second : 0)) * ld; };
    if (!waited) {
      wait_for_kernel_in_front();
      waited = true;
      asm volatile("griddepcontrol.launch_dependents;" ::: "memory");   // (what comes behind is launched meanwhile: 0.7 us)
    }
    float4 ahead[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int s = g0 + i * kGroups;
      ahead[i] = s < n ? *reinterpret_cast<const float4*>(at(s) + sub * 4) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    for (int s = tid; s < n; s += kJoinThreads) {
      const float4 v = *reinterpret_cast<const float4*>(at(s) + D);
      s_w[s] = v.x;
      s_l[s] = v.y;
      s_g[s] = v.z;
    }
    __syncthreads();
    if (tid < 32) {
      float after = 0.f, top = -INFINITY;
      for (int e = n; e > 0; e -= 32) {   // parts e - 1 - lane
        const int s = e - 1 - tid;
        float incl = s >= 0 ? s_g[s] : 0.f;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const float y = __shfl_up_sync(0xffffffffu, incl, o);
          if (tid >= o) incl += y;
        }
        const float right = __shfl_up_sync(0xffffffffu, incl, 1);   // (not incl less its own: that may be minus infinity)
        if (s >= 0) {
          const float mm = s_w[s] + (tid ? after + right : after);
          s_w[s] = mm;
          top = fmaxf(top, mm);
        }
        after += __shfl_sync(0xffffffffu, incl, 31);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      float sum = 0.f;
      for (int s = n - 1 - tid; s >= 0; s -= 32) {   // (each lane those that it wrote)
        const float mm = s_w[s], w = mm == -INFINITY ? 0.f : fast_exp2(mm - top);
        s_w[s] = w;
        sum = fmaf(s_l[s], w, sum);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (tid == 0) {
        s_sum = sum;
        s_top = top;
      }
    }
    __syncthreads();
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](const float4& v, float w) {   // (a weight of zero too: a NaN value counts)
      a.x = fmaf(v.x, w, a.x);
      a.y = fmaf(v.y, w, a.y);
      a.z = fmaf(v.z, w, a.z);
      a.w = fmaf(v.w, w, a.w);
    };
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int s = g0 + i * kGroups;
      if (s < n) add(ahead[i], s_w[s]);
    }
#pragma unroll 4
    for (int s = g0 + kAhead * kGroups; s < n; s += kGroups) add(*reinterpret_cast<const float4*>(at(s) + sub * 4), s_w[s]);
    s_o[tid] = a;
    __syncthreads();
    if (tid < kLanes) {
#pragma unroll
      for (int g = 1; g < kGroups; ++g) add(s_o[g * kLanes + tid], 1.f);
      const float inv = s_sum != 0.f ? 1.f / s_sum : 0.f;
      *reinterpret_cast<uint2*>(p.o + r * p.o_sr + h * p.o_sh + tid * 4) =
          make_uint2(pack2<kBf16>(a.x * inv, a.y * inv), pack2<kBf16>(a.z * inv, a.w * inv));
    }
    if (tid == 0 && p.L) p.L[item] = s_sum != 0.f ? s_top * kPagLn2 + __logf(s_sum) : -INFINITY;
    __syncthreads();   // (what is shared: the next pair's)
  }
  if (!waited) wait_for_kernel_in_front();   // (this grid's end has to mean the first kernel's)
}

// (64 columns or all, rows of a page, halves, heads, pages)
static int make_paged_tmap(CUtensorMap* out, const fox_tensor4* t, bool bf16, int64_t P, int64_t heads, int64_t page, int64_t D) {
  EncodeTiledFn fn = get_encode_tiled();
  if (!fn) return FOX_ERR_DRIVER;
  const cuuint64_t dims[5] = {(cuuint64_t)(D < 64 ? D : 64), (cuuint64_t)page, (cuuint64_t)(D == 128 ? 2 : 1), (cuuint64_t)heads, (cuuint64_t)P};
  const cuuint64_t strides[4] = {(cuuint64_t)t->st * 2, 128, (cuuint64_t)t->sh * 2, (cuuint64_t)t->sb * 2};
  const cuuint32_t box[5] = {(cuuint32_t)(D < 64 ? D : 64), kPagTile, (cuuint32_t)(D == 128 ? 2 : 1), 1, 1}, ones[5] = {1, 1, 1, 1, 1};
  const CUtensorMapSwizzle swizzle = D < 32 ? CU_TENSOR_MAP_SWIZZLE_32B : D < 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B;
  return fn(out, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 5, t->ptr, dims, strides, box, ones,
            CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
             ? FOX_OK
             : FOX_ERR_TENSORMAP;
}

template <bool kBf16, int D>
static int launch_paged(const PagedParams& p, const CUtensorMap& map_k, const CUtensorMap& map_v, cudaStream_t st) {
  static std::atomic<uint64_t> done{0};   // devices whose limit has been raised
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return FOX_ERR_DEVICE;
  const uint64_t bit = uint64_t{1} << (dev & 63);
  if (!(done.load(std::memory_order_relaxed) & bit)) {
    if (cudaFuncSetAttribute(fox_paged_attn_kernel<kBf16, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, PagedTile<D>::kSmem) !=
        cudaSuccess)
      return FOX_ERR_LAUNCH;
    // (the split of shared memory and L1 as the first kernel has it: changing it needs an SM without CTAs)
    if (cudaFuncSetAttribute(fox_paged_join_kernel<kBf16, D>, cudaFuncAttributePreferredSharedMemoryCarveout, 100) != cudaSuccess)
      return FOX_ERR_LAUNCH;
    done.fetch_or(bit, std::memory_order_relaxed);
  }
  if (int rc = launch_behind(fox_paged_attn_kernel<kBf16, D>, dim3(kPagGrid), PagedTile<D>::kThreads, PagedTile<D>::kSmem, st, p, map_k,
                             map_v))
    return rc;
  if (p.most <= (pag_whole(D) - kPagStart) * kPagTile) return FOX_OK;   // no unit is ever cut between CTAs
  const int64_t pairs = static_cast<int64_t>(p.R) * p.H;
  return launch_behind(fox_paged_join_kernel<kBf16, D>, dim3((unsigned)(pairs < kSms * 8 ? pairs : kSms * 8)), kJoinThreads, 0, st, p);
}

}  // namespace fox

using namespace fox;

static int64_t paged_rows(int64_t H, int64_t Hk) { return H / Hk < kPagRows ? H / Hk : kPagRows; }

extern "C" int64_t fox_paged_attn_workspace_floats(int64_t R, int64_t H, int64_t Hk, int64_t D) {
  if (R <= 0 || H <= 0 || Hk <= 0 || D <= 0) return 1;
  return kPagGrid * 2 * paged_rows(H, Hk) * (D + 4);
}

extern "C" int fox_paged_attn(int device, void* stream, int dtype, int64_t R, int64_t H, int64_t Hk, int64_t D, int64_t n_pages,
                              int64_t page, int64_t width, const void* q, int64_t q_sr, int64_t q_sh, const fox_tensor4* k_pages,
                              const fox_tensor4* v_pages, const float* gate_pages, int64_t gp_sp, int64_t gp_sh,
                              const int32_t* block_table, int64_t table_ld, const int32_t* lengths, float sm_scale, void* o,
                              int64_t o_sr, int64_t o_sh, float* L, float* workspace, int32_t* status) {
  if (!q || !k_pages || !v_pages || !k_pages->ptr || !v_pages->ptr || !gate_pages || !block_table || !lengths || !o || !workspace || !status)
    return FOX_ERR_BAD_ARG;
  if (R <= 0 || H <= 0 || Hk <= 0 || H % Hk || n_pages <= 0 || width <= 0 || table_ld < width || page < 16 || page > 65536 ||
      (page & (page - 1)))
    return FOX_ERR_BAD_ARG;
  if (dtype != FOX_DTYPE_BF16 && dtype != FOX_DTYPE_FP16) return FOX_ERR_BAD_ARG;
  if (D != 16 && D != 32 && D != 64 && D != 128) return FOX_ERR_HEAD_DIM;
  if (R > (1 << 24) || H > 65535 || n_pages > 2147483647LL / page || width > (1 << 30)) return FOX_ERR_TOO_LARGE;
  auto off = [](const void* x, int64_t a, int64_t b, int64_t c, int64_t whole) {
    return reinterpret_cast<uintptr_t>(x) % 16 || a % whole || b % whole || c % whole;
  };
  if (off(q, q_sr, q_sh, 0, 8) || off(k_pages->ptr, k_pages->sb, k_pages->sh, k_pages->st, 8) ||
      off(v_pages->ptr, v_pages->sb, v_pages->sh, v_pages->st, 8) || off(gate_pages, gp_sp, gp_sh, 0, 4) ||
      off(o, o_sr, o_sh, 0, 8) || reinterpret_cast<uintptr_t>(workspace) % 16)
    return FOX_ERR_ALIGNMENT;
  // places are counted with 30 bits: so many requests at a time, going by what their table rows could hold
  const int64_t tiles_of_group = (H / Hk + kPagRows - 1) / kPagRows, most = width * page < 2147483647LL - 64 ? width * page : 2147483647LL - 64;
  const int64_t at_once = (int64_t{1} << 30) / (Hk * tiles_of_group * ((most + kPagTile - 1) / kPagTile + kPagStart));
  if (at_once < 1) return FOX_ERR_TOO_LARGE;
  if (cudaSetDevice(device) != cudaSuccess) return FOX_ERR_DEVICE;
  PagedParams p{};
  p.q = (const uint16_t*)q;
  p.q_sr = q_sr; p.q_sh = q_sh;
  p.status = status;
  p.gates = gate_pages; p.g_sp = gp_sp; p.g_sh = gp_sh;
  p.table = block_table; p.table_ld = table_ld; p.lengths = lengths;
  p.o = (uint16_t*)o; p.o_sr = o_sr; p.o_sh = o_sh; p.L = L;
  p.part = workspace;
  p.R = (int)R; p.H = (int)H; p.group = (int)(H / Hk); p.rows = (int)paged_rows(H, Hk);
  p.tiles_of_group = (int)tiles_of_group;
  p.units = (int)Hk * p.tiles_of_group;
  p.by_units = divisor(p.units);
  p.by_tiles_of_group = divisor(p.tiles_of_group);
  p.n_pages = (int)n_pages;
  for (p.page_log2 = 4; (int64_t{1} << p.page_log2) < page;) ++p.page_log2;
  p.most = most;
  p.qk_scale = sm_scale * kPagLog2e;
  cudaStream_t st = (cudaStream_t)stream;
  const bool bf = dtype == FOX_DTYPE_BF16;
  CUtensorMap mk, mv;
  auto bad = [](const fox_tensor4* x) { return x->sb <= 0 || x->sh <= 0 || x->st <= 0; };
  if (bad(k_pages) || bad(v_pages)) return FOX_ERR_ALIGNMENT;
  if (int rc = make_paged_tmap(&mk, k_pages, bf, n_pages, Hk, page, D)) return rc;
  if (int rc = make_paged_tmap(&mv, v_pages, bf, n_pages, Hk, page, D)) return rc;
  auto launch_one = [&] {
    switch (D) {
      case 16: return bf ? launch_paged<true, 16>(p, mk, mv, st) : launch_paged<false, 16>(p, mk, mv, st);
      case 32: return bf ? launch_paged<true, 32>(p, mk, mv, st) : launch_paged<false, 32>(p, mk, mv, st);
      case 64: return bf ? launch_paged<true, 64>(p, mk, mv, st) : launch_paged<false, 64>(p, mk, mv, st);
      default: return bf ? launch_paged<true, 128>(p, mk, mv, st) : launch_paged<false, 128>(p, mk, mv, st);
    }
  };
  for (int64_t r0 = 0; r0 < R; r0 += at_once) {
    p.R = static_cast<int>(R - r0 < at_once ? R - r0 : at_once);
    if (int rc = launch_one()) return rc;
    p.q += p.R * q_sr;
    p.o += p.R * o_sr;
    p.table += p.R * table_ld;
    p.lengths += p.R;
    if (p.L) p.L += p.R * H;
  }
  return FOX_OK;
}
