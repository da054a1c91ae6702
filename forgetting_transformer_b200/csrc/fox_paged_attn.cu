// Forgetting attention of one new token per request against a paged cache (pages, slots and block tables: fox_paged.cu).
//
//   u_j = (q . k_j) sm_scale + sum_{t > j} g_t,  j < length;   out = sum_j softmax(u)_j v_j;   L = log sum_j exp(u_j)
//
// The paged counterpart of fox_decode.cu, for requests of any lengths: those are on the device, so the split is made there.
// Bound by reading every key, value and gate once.
//
// Work is counted in tiles of 16 keys of one unit (a request and a key head, with up to 8 of the query heads that share it).
// All tiles of all units stand in one row, which is cut into equal ranges, one for each warp of a grid that fills the GPU
// once: the longest request and the shortest cost what their tiles cost.  Every warp sums up the lengths by itself (its CTA
// does, before the first load) and finds its range there.  A unit that lies in one warp's range is written at once; a unit
// cut by ranges leaves (o, m, l, sum of gates) of every part in a workspace, which a second kernel joins.
//
// The bias of a key is the sum of the gates behind it.  A warp goes through its part of a unit from the right, so that this
// is a running sum (exact where the bias is small, which is where it matters; a prefix sum over the whole request would lose
// what the cache's length costs), and the parts' sums shift their maxima when they are joined.
//
// No lane waits for another's data: each lane copies (cp.async) what it will itself feed to the matrix instructions, into
// a ring of kStages tiles of its own.  mma.sync m16n8k16 (the two products are 8 query rows at most; the kernel is bound by
// memory, with a tensor pipe mostly idle):
//   S (16 x 8 keys) = Q K^T, twice, rows 0-7 the unit's query heads.  Lane (x = lane / 4, c = lane % 4) gives 16-byte pieces
//     of a key's row; which channels stand at which k of an instruction does not matter as long as Q stands the same way.
//     The two key columns that a lane gets of each S are keys 4 c .. 4 c + 3 of the tile.
//   O (16 x D) += P V.  The registers of S are those of P.  P is rounded to 16 bits, and what the rounding leaves stands in
//     rows 8-15, which would be idle: the sum of the two halves of O has P to 2^-16 (fp16: 2^-21).
//
// Tiles never leave a page (pages are 16 keys at least).  Rows behind the last key may hold anything: their logits are
// replaced, their values set to zero.  A table entry outside the pool is not read: its keys take no part.
#include "fox_common.cuh"
#include "fox_host.h"

#include <atomic>

namespace fox {

constexpr int kPagWarps = 8, kPagThreads = kPagWarps * 32;
constexpr int kPagGrid = kSms, kPagRanges = kPagGrid * kPagWarps;
constexpr int kPagTile = 16;
constexpr int kPagRows = 8;          // query heads of a unit
constexpr int kPagLeastTiles = 2;    // of a range
constexpr float kPagLog2e = 1.4426950408889634f, kPagLn2 = 0.6931471805599453f;

struct PagedParams {
  const uint16_t *q, *k, *v;
  int64_t q_sr, q_sh, k_sp, k_sk, k_sr, v_sp, v_sk, v_sr, g_sp, g_sh, o_sr, o_sh;
  const float* gates;
  const int32_t *table, *lengths;
  int64_t table_ld;
  uint16_t* o;
  float* L;                            // (R, H) or nullptr
  float* part;                         // (ranges, 2, rows, D + 4)
  int64_t* tiles_before;               // (R + 1)
  int R, H, group, rows, tiles_of_group, units, n_pages, page_log2;   // rows: of a unit; units: of a request
  int64_t most;                        // keys that a table row has entries for
  float qk_scale;                      // sm_scale * log2(e)
};

__device__ __forceinline__ int pag_length(const PagedParams& p, int r) {
  const int64_t n = p.lengths[r];
  return static_cast<int>(n < 0 ? 0 : n < p.most ? n : p.most);
}
__device__ __forceinline__ int64_t pag_per_range(int64_t tiles) {
  const int64_t per = (tiles + kPagRanges - 1) / kPagRanges;
  return per < kPagLeastTiles ? kPagLeastTiles : per;
}

template <int kBytes>
__device__ __forceinline__ void cp_async(uint32_t dst, const void* src) {
  if constexpr (kBytes == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(kBytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kLeft>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory"); }

template <bool kBf16>
__device__ __forceinline__ void mma_16816(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (kBf16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// n words of a lane from the ring: pieces of kBytes, `piece` the first
template <int kBytes>
__device__ __forceinline__ void pag_take(uint32_t* w, const char* stage, int at, int lane) {
  const char* s = stage + at + lane * kBytes;
  if constexpr (kBytes == 16) {
    const uint4 v = *reinterpret_cast<const uint4*>(s);
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
  } else if constexpr (kBytes == 8) {
    const uint2 v = *reinterpret_cast<const uint2*>(s);
    w[0] = v.x; w[1] = v.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t*>(s);
  }
}

// How a lane's pieces of a tile lie in a stage of the ring.
template <int D>
struct PagedTile {
  static constexpr int kKBytes = D >= 32 ? 16 : 8, kKPieces = D >= 32 ? D / 32 : 1;                 // of a row; a lane has 2 rows
  static constexpr int kVBytes = D >= 64 ? 16 : D / 4, kVPieces = D >= 64 ? D / 64 : 1;             // of a row; a lane has 4 rows
  static constexpr int kKWords = kKBytes / 4, kVWords = kVBytes / 4;
  static constexpr int kK = 0, kV = kK + 2 * kKPieces * kKBytes * 32, kG = kV + 4 * kVPieces * kVBytes * 32, kQ = kG + 16 * 32,
                       kStage = kQ + kKPieces * kKBytes * 32;
  static constexpr int kSteps = D / 16;       // k of the first product
  static constexpr int kCols = D / 8;         // n of the second
  static constexpr int kStages = D == 128 ? 2 : 4;
  static constexpr int kRing = kStage * kStages;
  static constexpr int kSmem = kRing * kPagWarps;
};

// What a stage's tile is: written by lane 0, read by the warp.
struct PagedItem {
  int r, unit, valid, flags;   // keys of the tile that count; kFirst ... below
};
enum { kItemFirst = 1, kItemLast = 2, kItemWhole = 4, kItemSecond = 8 };   // of its part; a unit's only part; workspace place 1

template <bool kBf16, int D>
__global__ void __launch_bounds__(kPagThreads, 1) fox_paged_attn_kernel(const PagedParams p) {
  using Tile = PagedTile<D>;
  constexpr int kStages = Tile::kStages;
  extern __shared__ __align__(16) char pag_smem[];
  __shared__ int64_t s_before[kPagThreads + 1];
  __shared__ int64_t s_warp[kPagWarps];
  __shared__ PagedItem s_item[kPagWarps][kStages];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  wait_for_kernel_in_front();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");   // (the joining kernel, which waits for this one's end)

  // ---- where every thread's share of the requests begins in the row of tiles
  const int share = (p.R + kPagThreads - 1) / kPagThreads;
  const int r_first = min(tid * share, p.R), r_end = min(r_first + share, p.R);
  int64_t mine = 0;
  for (int r = r_first; r < r_end; ++r) mine += (pag_length(p, r) + kPagTile - 1) / kPagTile;
  int64_t incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += y;
  }
  if (lane == 31) s_warp[warp] = incl;
  __syncthreads();
  for (int w = 0; w < warp; ++w) incl += s_warp[w];
  s_before[tid + 1] = incl;
  if (tid == 0) s_before[0] = 0;
  __syncthreads();
  const int64_t total = s_before[kPagThreads] * p.units, per = pag_per_range(total);
  if (blockIdx.x == 0) {
    int64_t at = incl - mine;
    for (int r = r_first; r < r_end; ++r) {
      p.tiles_before[r] = at;
      at += (pag_length(p, r) + kPagTile - 1) / kPagTile;
    }
    if (tid == 0) p.tiles_before[p.R] = s_before[kPagThreads];
  }
  // ---- requests without a key
  for (int r = blockIdx.x; r < p.R; r += gridDim.x) {
    if (pag_length(p, r)) continue;
    for (int i = tid; i < p.H * D; i += kPagThreads) p.o[r * p.o_sr + (i / D) * p.o_sh + i % D] = 0;
    if (p.L)
      for (int h = tid; h < p.H; h += kPagThreads) p.L[static_cast<int64_t>(r) * p.H + h] = -INFINITY;
  }

  // ---- this warp's range (neighbours in the row on different SMs, so that little work is on many)
  const int range = warp * gridDim.x + blockIdx.x;
  const int64_t t_begin = range * per, t_end = min(t_begin + per, total);
  if (t_begin >= t_end) return;
  int64_t left = t_end - t_begin;   // tiles to ask for
  int n_left = static_cast<int>(left < 2147483647LL ? left : 2147483647LL);   // tiles to use (a range is far below that)
  int r, unit, n_tiles, part_lo, at;   // the part being asked for: tiles [part_lo, ..] of a unit, next `at`
  int length, flags;
  {
    int lo = 0, hi = kPagThreads;      // the last share that begins at or before the range
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (s_before[mid] * p.units <= t_begin) lo = mid;
      else hi = mid;
    }
    int64_t before = s_before[lo];
    r = lo * share;
    for (;; ++r) {
      length = pag_length(p, r);
      n_tiles = (length + kPagTile - 1) / kPagTile;
      if ((before + n_tiles) * p.units > t_begin) break;
      before += n_tiles;
    }
    const int64_t off = t_begin - before * p.units;
    unit = static_cast<int>(off / n_tiles);
    part_lo = static_cast<int>(off - static_cast<int64_t>(unit) * n_tiles);
  }
  auto begin_part = [&](bool first) {   // from part_lo on, as far as the range goes
    const int hi = static_cast<int>(min(static_cast<int64_t>(n_tiles), part_lo + left));
    flags = (part_lo == 0 && hi == n_tiles ? kItemWhole : 0) | (first ? 0 : kItemSecond);
    at = hi - 1;
    flags |= kItemFirst;
  };
  begin_part(true);

  char* ring = pag_smem + warp * Tile::kRing;
  const uint32_t ring_u32 = smem_u32(ring);
  const int x = lane >> 2, c = lane & 3;
  const int key_a = 4 * (x >> 1) + (x & 1);   // of the first S; the second: + 2
  int page_r = -1, page_base = 0, page_ids = -1;   // 32 entries of a request's table row, one to a lane
  const uint32_t page_rows = 1u << p.page_log2;

  auto ask = [&](int stage) {   // the next tile's pieces
    if (left > 0) {
      const int key0 = at * kPagTile, j = key0 >> p.page_log2;
      if (r != page_r || j < page_base || j >= page_base + 32) {
        page_r = r;
        page_base = j < 31 ? 0 : j - 31;   // (the walk goes to the left)
        const int e = page_base + lane;
        page_ids = static_cast<int64_t>(e) << p.page_log2 < length ? p.table[r * p.table_ld + e] : -1;
      }
      const int id = __shfl_sync(0xffffffffu, page_ids, j - page_base);
      const bool there = id >= 0 && id < p.n_pages;
      const int kh = unit / p.tiles_of_group, h0 = kh * p.group + (unit - kh * p.tiles_of_group) * kPagRows;
      const uint32_t dst = ring_u32 + stage * Tile::kStage + lane * 16, row0 = key0 & (page_rows - 1);
      const int heads = min(p.group - (unit - kh * p.tiles_of_group) * kPagRows, kPagRows);
      if (there) {
        const uint16_t* kp = p.k + id * p.k_sp + kh * p.k_sk + c * (Tile::kKBytes / 2);
        const uint16_t* vp = p.v + id * p.v_sp + kh * p.v_sk + x * (Tile::kVBytes / 2);
        const uint32_t dk = ring_u32 + stage * Tile::kStage + Tile::kK + lane * Tile::kKBytes;
        const uint32_t dv = ring_u32 + stage * Tile::kStage + Tile::kV + lane * Tile::kVBytes;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int s = 0; s < Tile::kKPieces; ++s)
            cp_async<Tile::kKBytes>(dk + (i * Tile::kKPieces + s) * 32 * Tile::kKBytes, kp + (row0 + key_a + 2 * i) * p.k_sr + s * 32);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int s = 0; s < Tile::kVPieces; ++s)
            cp_async<Tile::kVBytes>(dv + (i * Tile::kVPieces + s) * 32 * Tile::kVBytes, vp + (row0 + 4 * c + i) * p.v_sr + s * 64);
        if (x < heads) cp_async<16>(dst + Tile::kG, p.gates + id * p.g_sp + (h0 + x) * p.g_sh + row0 + 4 * c);
      }
      if ((flags & kItemFirst) && x < heads) {
        const uint16_t* qp = p.q + r * p.q_sr + (h0 + x) * p.q_sh + c * (Tile::kKBytes / 2);
        const uint32_t dq = ring_u32 + stage * Tile::kStage + Tile::kQ + lane * Tile::kKBytes;
#pragma unroll
        for (int s = 0; s < Tile::kKPieces; ++s) cp_async<Tile::kKBytes>(dq + s * 32 * Tile::kKBytes, qp + s * 32);
      }
      const bool last = at == part_lo;
      if (lane == 0) s_item[warp][stage] = {r, unit, there ? min(length - key0, kPagTile) : 0, flags | (last ? kItemLast : 0)};
      flags &= ~kItemFirst;
      --at;
      --left;
      if (last && left > 0) {   // the next unit
        part_lo = 0;
        if (++unit == p.units) {
          unit = 0;
          do {
            length = pag_length(p, ++r);
          } while (length == 0);   // (tiles are left, so there is a request with keys)
          n_tiles = (length + kPagTile - 1) / kPagTile;
        }
        begin_part(false);
      }
    }
    cp_async_commit();
  };

#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) ask(s);

  constexpr float kShift = kBf16 ? 0.f : 12.f;   // fp16: weights up to 2^12, so that small ones keep their bits
  uint32_t qf[Tile::kSteps][2];
  float o[Tile::kCols][4], m = -INFINITY, l = 0.f, carry = 0.f;
  int stage = 0;
  for (; n_left > 0; --n_left) {
    ask(stage == 0 ? kStages - 1 : stage - 1);
    cp_async_wait<kStages - 1>();
    __syncwarp();
    const PagedItem item = s_item[warp][stage];
    const char* tile = ring + stage * Tile::kStage;
    const int kh = item.unit / p.tiles_of_group, h0 = kh * p.group + (item.unit - kh * p.tiles_of_group) * kPagRows;
    const int heads = min(p.group - (item.unit - kh * p.tiles_of_group) * kPagRows, kPagRows);
    if (item.flags & kItemFirst) {
#pragma unroll
      for (int s = 0; s < Tile::kKPieces; ++s) {
        uint32_t w[4];
        pag_take<Tile::kKBytes>(w, tile, Tile::kQ + s * 32 * Tile::kKBytes, lane);
#pragma unroll
        for (int i = 0; i < Tile::kKWords; ++i) qf[s * (Tile::kKWords / 2) + i / 2][i & 1] = x < heads ? w[i] : 0u;
      }
#pragma unroll
      for (int j = 0; j < Tile::kCols; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[j][i] = 0.f;
      m = -INFINITY;
      l = carry = 0.f;
    }
    // ---- gates: sums behind each of the lane's four keys, inside the part
    float bias[4];
    {
      const float4 gv = *reinterpret_cast<const float4*>(tile + Tile::kG + lane * 16);
      const float g[4] = {gv.x, gv.y, gv.z, gv.w};
      float own[4], sum = 0.f;
#pragma unroll
      for (int i = 3; i >= 0; --i) {
        own[i] = sum;
        sum += x < heads && 4 * c + i < item.valid ? g[i] : 0.f;
      }
      float behind = sum;   // of this lane and those to its right
      float y = __shfl_down_sync(0xffffffffu, behind, 1, 4);
      if (c < 3) behind += y;
      y = __shfl_down_sync(0xffffffffu, behind, 2, 4);
      if (c < 2) behind += y;
      y = __shfl_down_sync(0xffffffffu, behind, 1, 4);   // (not behind - sum: a gate of minus infinity cannot be taken off again)
      const float right = carry + (c < 3 ? y : 0.f);
#pragma unroll
      for (int i = 0; i < 4; ++i) bias[i] = (right + own[i]) * kPagLog2e;
      carry += __shfl_sync(0xffffffffu, behind, lane & ~3);
    }
    // ---- S
    float s0[4] = {0.f, 0.f, 0.f, 0.f}, s1[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < Tile::kKPieces; ++s) {
      uint32_t ka[4], kb[4];
      pag_take<Tile::kKBytes>(ka, tile, Tile::kK + s * 32 * Tile::kKBytes, lane);
      pag_take<Tile::kKBytes>(kb, tile, Tile::kK + (Tile::kKPieces + s) * 32 * Tile::kKBytes, lane);
#pragma unroll
      for (int i = 0; i < Tile::kKWords / 2; ++i) {
        const uint32_t* qw = qf[s * (Tile::kKWords / 2) + i];
        mma_16816<kBf16>(s0, qw[0], 0u, qw[1], 0u, ka[2 * i], ka[2 * i + 1]);
        mma_16816<kBf16>(s1, qw[0], 0u, qw[1], 0u, kb[2 * i], kb[2 * i + 1]);
      }
    }
    const float u4[4] = {s0[0], s0[1], s1[0], s1[1]};
    float u[4], mx = m;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      u[i] = 4 * c + i < item.valid ? fmaf(u4[i], p.qk_scale, bias[i]) : -INFINITY;
      mx = fmaxf(mx, u[i]);
    }
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
    const float ref = mx == -INFINITY ? 0.f : mx - kShift;
    if (__any_sync(0xffffffffu, mx > m)) {   // (NaN logits: no new maximum, and NaN weights)
      const float alpha = m == -INFINITY ? 0.f : fast_exp2(m - mx);
      l *= alpha;
#pragma unroll
      for (int j = 0; j < Tile::kCols; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[j][i] *= alpha;
      m = mx;
    }
    // ---- P, its 16-bit values and what they leave
    float w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = fast_exp2(u[i] - ref);
      l += w[i];
    }
    const uint32_t hi0 = pack2<kBf16>(w[0], w[1]), hi1 = pack2<kBf16>(w[2], w[3]);
    const float2 r0 = unpack2<kBf16>(hi0), r1 = unpack2<kBf16>(hi1);
    const uint32_t lo0 = pack2<kBf16>(w[0] - r0.x, w[1] - r0.y), lo1 = pack2<kBf16>(w[2] - r1.x, w[3] - r1.y);
    // ---- O
#pragma unroll
    for (int s = 0; s < Tile::kVPieces; ++s) {
      uint32_t vw[4][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        pag_take<Tile::kVBytes>(vw[i], tile, Tile::kV + (i * Tile::kVPieces + s) * 32 * Tile::kVBytes, lane);
        if (item.valid < kPagTile && 4 * c + i >= item.valid)
#pragma unroll
          for (int j = 0; j < Tile::kVWords; ++j) vw[i][j] = 0u;
      }
#pragma unroll
      for (int j = 0; j < Tile::kVWords; ++j) {
        mma_16816<kBf16>(o[s * 8 + 2 * j], hi0, lo0, hi1, lo1, __byte_perm(vw[0][j], vw[1][j], 0x5410),
                         __byte_perm(vw[2][j], vw[3][j], 0x5410));
        mma_16816<kBf16>(o[s * 8 + 2 * j + 1], hi0, lo0, hi1, lo1, __byte_perm(vw[0][j], vw[1][j], 0x7632),
                         __byte_perm(vw[2][j], vw[3][j], 0x7632));
      }
    }
    if (item.flags & kItemLast) {
      float ls = l + __shfl_xor_sync(0xffffffffu, l, 1);
      ls += __shfl_xor_sync(0xffffffffu, ls, 2);
      const float m_ref = ls != ls ? ls : m == -INFINITY ? -INFINITY : m - kShift;   // (NaN stays visible when parts are joined)
      // lane (x, c), column pair (2 c, 2 c + 1) of block j: channels n kVWords 2 + j, n = 2 c and 2 c + 1, of each piece
      constexpr int kRun = Tile::kVWords * 2;   // channels behind one another
      if (x < heads) {
        const int h = h0 + x;
        if (item.flags & kItemWhole) {
          const float inv = ls != 0.f ? 1.f / ls : 0.f;   // (a NaN sum stays one)
          uint16_t* to = p.o + item.r * p.o_sr + h * p.o_sh;
#pragma unroll
          for (int s = 0; s < Tile::kVPieces; ++s)
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
              for (int j = 0; j < kRun; j += 2)
                *reinterpret_cast<uint32_t*>(to + s * 64 + (2 * c + n) * kRun + j) =
                    pack2<kBf16>((o[s * 8 + j][n] + o[s * 8 + j][n + 2]) * inv, (o[s * 8 + j + 1][n] + o[s * 8 + j + 1][n + 2]) * inv);
          if (p.L && c == 0) p.L[static_cast<int64_t>(item.r) * p.H + h] = ls != 0.f ? m_ref * kPagLn2 + __logf(ls) : -INFINITY;
        } else {
          float* to = p.part + ((static_cast<int64_t>(range) * 2 + (item.flags & kItemSecond ? 1 : 0)) * p.rows + x) * (D + 4);
#pragma unroll
          for (int s = 0; s < Tile::kVPieces; ++s)
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
              for (int j = 0; j < kRun; j += 2)
                *reinterpret_cast<float2*>(to + s * 64 + (2 * c + n) * kRun + j) =
                    make_float2(o[s * 8 + j][n] + o[s * 8 + j][n + 2], o[s * 8 + j + 1][n] + o[s * 8 + j + 1][n + 2]);
          if (c == 0) {
            to[D] = m_ref;
            to[D + 1] = ls;
            to[D + 2] = carry * kPagLog2e;
          }
        }
      }
    }
    __syncwarp();   // (the item has been read before its place is written again)
    stage = stage == kStages - 1 ? 0 : stage + 1;
  }
  cp_async_wait<0>();
}

// Joins the parts of units that were cut.  A CTA takes (request, query head) pairs; a unit's parts stand from the left, so
// their gate sums are added from the right, 32 parts at a time by one warp; then 256 / D groups of threads each sum every
// (256 / D)-th part.
template <bool kBf16, int D>
__global__ void __launch_bounds__(256) fox_paged_join_kernel(const PagedParams p) {
  __shared__ float s_w[kPagRanges], s_o[256], s_top, s_sum;
  constexpr int kGroups = 256 / D;
  const int tid = threadIdx.x;
  wait_for_kernel_in_front();
  const int64_t per = pag_per_range(p.tiles_before[p.R] * p.units);
  for (int64_t item = blockIdx.x; item < static_cast<int64_t>(p.R) * p.H; item += gridDim.x) {
    const int r = static_cast<int>(item / p.H), h = static_cast<int>(item - static_cast<int64_t>(r) * p.H);
    const int kh = h / p.group, row = h - kh * p.group, unit = kh * p.tiles_of_group + row / kPagRows;
    const int64_t before = p.tiles_before[r], n_tiles = p.tiles_before[r + 1] - before;
    const int64_t u0 = before * p.units + unit * n_tiles, u1 = u0 + n_tiles;
    if (n_tiles == 0) continue;
    const int w0 = static_cast<int>(u0 / per), n = static_cast<int>((u1 - 1) / per) - w0 + 1;   // (at most kPagRanges)
    if (n == 1) continue;
    const int64_t ld = static_cast<int64_t>(p.rows) * (D + 4);
    const float* base = p.part + (static_cast<int64_t>(w0) * 2 * p.rows + row % kPagRows) * (D + 4);
    const int second = u0 != w0 * per;   // the first part's place
    auto at = [&](int s) { return base + (2 * s + (s == 0 ? second : 0)) * ld; };
    if (tid < 32) {
      float after = 0.f, top = -INFINITY;
      for (int e = n; e > 0; e -= 32) {   // parts e - 1 - lane
        const int s = e - 1 - tid;
        const float g = s >= 0 ? at(s)[D + 2] : 0.f;
        float incl = g;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const float y = __shfl_up_sync(0xffffffffu, incl, o);
          if (tid >= o) incl += y;
        }
        const float right = __shfl_up_sync(0xffffffffu, incl, 1);
        if (s >= 0) {
          const float mm = at(s)[D] + after + (tid ? right : 0.f);
          s_w[s] = mm;
          top = fmaxf(top, mm);
        }
        after += __shfl_sync(0xffffffffu, incl, 31);
      }
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      float sum = 0.f;
      for (int s = n - 1 - tid; s >= 0; s -= 32) {   // (each lane those that it wrote)
        const float mm = s_w[s], w = mm == -INFINITY ? 0.f : fast_exp2(mm - top), ls = at(s)[D + 1];
        s_w[s] = w;
        sum = fmaf(ls, w, sum);
      }
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (tid == 0) {
        s_top = top;
        s_sum = sum;
      }
    }
    __syncthreads();
    const int d = tid % D, g0 = tid / D;
    float a = 0.f;
#pragma unroll 4
    for (int s = g0; s < n; s += kGroups) a = fmaf(at(s)[d], s_w[s], a);   // (a weight of zero too: a NaN value counts)
    s_o[tid] = a;
    __syncthreads();
    if (tid < D) {
#pragma unroll
      for (int g = 1; g < kGroups; ++g) a += s_o[g * D + tid];
      const uint32_t pk = pack2<kBf16>(s_sum != 0.f ? a / s_sum : 0.f, 0.f);
      p.o[r * p.o_sr + h * p.o_sh + tid] = static_cast<uint16_t>(pk & 0xffffu);
    }
    if (tid == 0 && p.L) p.L[item] = s_sum != 0.f ? s_top * kPagLn2 + __logf(s_sum) : -INFINITY;
    __syncthreads();   // (s_w, s_o: the next pair's)
  }
}

template <bool kBf16, int D>
static int launch_paged(const PagedParams& p, cudaStream_t st) {
  static std::atomic<uint64_t> done{0};   // devices whose limit has been raised
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return FOX_ERR_DEVICE;
  const uint64_t bit = uint64_t{1} << (dev & 63);
  if (!(done.load(std::memory_order_relaxed) & bit)) {
    if (cudaFuncSetAttribute(fox_paged_attn_kernel<kBf16, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, PagedTile<D>::kSmem) !=
        cudaSuccess)
      return FOX_ERR_LAUNCH;
    done.fetch_or(bit, std::memory_order_relaxed);
  }
  if (int rc = launch_behind(fox_paged_attn_kernel<kBf16, D>, dim3(kPagGrid), kPagThreads, PagedTile<D>::kSmem, st, p)) return rc;
  const int64_t pairs = static_cast<int64_t>(p.R) * p.H;
  return launch_behind(fox_paged_join_kernel<kBf16, D>, dim3((unsigned)(pairs < kSms * 4 ? pairs : kSms * 4)), 256, 0, st, p);
}

}  // namespace fox

using namespace fox;

static int64_t paged_rows(int64_t H, int64_t Hk) { return H / Hk < kPagRows ? H / Hk : kPagRows; }

extern "C" int64_t fox_paged_attn_workspace_floats(int64_t R, int64_t H, int64_t Hk, int64_t D) {
  if (R <= 0 || H <= 0 || Hk <= 0 || D <= 0) return 1;
  return 2 * (R + 1) + 4 + kPagRanges * 2 * paged_rows(H, Hk) * (D + 4);
}

extern "C" int fox_paged_attn(int device, void* stream, int dtype, int64_t R, int64_t H, int64_t Hk, int64_t D, int64_t n_pages,
                              int64_t page, int64_t width, const void* q, int64_t q_sr, int64_t q_sh, const fox_tensor4* k_pages,
                              const fox_tensor4* v_pages, const float* gate_pages, int64_t gp_sp, int64_t gp_sh,
                              const int32_t* block_table, int64_t table_ld, const int32_t* lengths, float sm_scale, void* o,
                              int64_t o_sr, int64_t o_sh, float* L, float* workspace) {
  if (!q || !k_pages || !v_pages || !k_pages->ptr || !v_pages->ptr || !gate_pages || !block_table || !lengths || !o || !workspace)
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
  if (cudaSetDevice(device) != cudaSuccess) return FOX_ERR_DEVICE;
  PagedParams p{};
  p.q = (const uint16_t*)q; p.k = (const uint16_t*)k_pages->ptr; p.v = (const uint16_t*)v_pages->ptr;
  p.q_sr = q_sr; p.q_sh = q_sh;
  p.k_sp = k_pages->sb; p.k_sk = k_pages->sh; p.k_sr = k_pages->st;
  p.v_sp = v_pages->sb; p.v_sk = v_pages->sh; p.v_sr = v_pages->st;
  p.gates = gate_pages; p.g_sp = gp_sp; p.g_sh = gp_sh;
  p.table = block_table; p.table_ld = table_ld; p.lengths = lengths;
  p.o = (uint16_t*)o; p.o_sr = o_sr; p.o_sh = o_sh; p.L = L;
  p.tiles_before = reinterpret_cast<int64_t*>(workspace);
  p.part = workspace + (2 * (R + 1) + 3) / 4 * 4;
  p.R = (int)R; p.H = (int)H; p.group = (int)(H / Hk); p.rows = (int)paged_rows(H, Hk);
  p.tiles_of_group = (p.group + kPagRows - 1) / kPagRows;
  p.units = (int)Hk * p.tiles_of_group;
  p.n_pages = (int)n_pages;
  for (p.page_log2 = 4; (int64_t{1} << p.page_log2) < page;) ++p.page_log2;
  p.most = width * page < 2147483647LL - 64 ? width * page : 2147483647LL - 64;
  p.qk_scale = sm_scale * kPagLog2e;
  cudaStream_t st = (cudaStream_t)stream;
  const bool bf = dtype == FOX_DTYPE_BF16;
  switch (D) {
    case 16: return bf ? launch_paged<true, 16>(p, st) : launch_paged<false, 16>(p, st);
    case 32: return bf ? launch_paged<true, 32>(p, st) : launch_paged<false, 32>(p, st);
    case 64: return bf ? launch_paged<true, 64>(p, st) : launch_paged<false, 64>(p, st);
    default: return bf ? launch_paged<true, 128>(p, st) : launch_paged<false, 128>(p, st);
  }
}
