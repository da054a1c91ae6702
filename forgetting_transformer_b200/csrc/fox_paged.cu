// The bookkeeping and the writing side of a paged generation cache: which pages the requests of a batch own, where a new
// token's row goes, and the rows themselves.
//
// A pool of P pages holds, for every page, `page` consecutive tokens of one request: keys and values (P, heads, page, D) and
// fp32 log gates (P, heads, page).  Request r has lengths[r] tokens; the page of its token t is block_table[r][t / page] and
// the token's slot is that page times `page` plus t mod page.  Pages nobody owns are a stack: free_pages[0 .. num_free).
// (Upstream keeps one growing tensor per layer for a batch of one length, fgate_cache.py:77-116.)
#include "fox_common.cuh"
#include "fox_host.h"

namespace fox {

constexpr int kTabThreads = 1024, kTabWarps = kTabThreads / 32;
constexpr int64_t kTabOneCta = 8192;   // tokens up to which the scanning CTA places them itself

// inclusive sum over the block's threads, and the total
__device__ __forceinline__ int64_t block_scan(int64_t x, int64_t& total, int64_t* s_warp) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();   // (the last scan's sums have been read)
  if (lane == 31) s_warp[warp] = x;
  __syncthreads();
  int64_t w = lane < kTabWarps ? s_warp[lane] : 0;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, w, o);
    if (lane >= o) w += y;
  }
  total = __shfl_sync(0xffffffffu, w, kTabWarps - 1);
  const int64_t before = __shfl_sync(0xffffffffu, w, warp ? warp - 1 : 0);
  return warp ? x + before : x;
}

struct TableParams {
  const int32_t *lengths, *new_tokens;
  int32_t* table;
  int64_t table_ld;
  const int32_t *free_pages, *num_free;
  int32_t *lengths_out, *num_free_out, *starts, *granted, *requests, *positions, *slots;
  int32_t* work;      // (R + 1): pages taken by the requests in front, and the pages that were free
  int R, width, n_free_max, page_log2, max_tokens;
};

__device__ __forceinline__ int clamp31(int64_t x) { return x > 2147483647LL ? 2147483647 : static_cast<int>(x); }

// What a token is placed by, for every request: first token of the packed batch, tokens granted, old length, pages taken by the
// requests in front.  (starts has one more; free_before: pages that were free.)
struct Placing {
  const int32_t *starts, *granted, *lengths, *taken;   // lengths: with what was granted
  int free_before;
};

// Token t's request, position and slot.  A page that the call has given out is known from the stack, without the table; the
// token at its first place writes the table's entry (there is one: a fresh page begins at or behind the old length).
__device__ __forceinline__ void place_token(const TableParams& p, const Placing& a, int t) {
  int lo = 0, hi = p.R;   // the last request that starts at or before t, so that t < starts[lo + 1] where there is one
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.starts[mid] <= t) lo = mid;
    else hi = mid;
  }
  int request = -1, pos = 0, slot = -1;
  if (t < a.starts[p.R]) {
    request = lo;
    const int n = a.granted[lo], old = a.lengths[lo] - n;
    const int64_t at = static_cast<int64_t>(old) + t - a.starts[lo];
    pos = clamp31(at);
    if (n > 0) {
      const int j = pos >> p.page_log2, have = static_cast<int>((static_cast<int64_t>(old) + (1 << p.page_log2) - 1) >> p.page_log2);
      int32_t* entry = p.table + lo * p.table_ld + j;
      int id;
      if (j >= have) {
        id = p.free_pages[a.free_before - 1 - (a.taken[lo] + j - have)];
        if ((pos & ((1 << p.page_log2) - 1)) == 0) *entry = id;
      } else {
        id = *entry;
      }
      const int64_t s = (static_cast<int64_t>(id) << p.page_log2) + (pos & ((1 << p.page_log2) - 1));
      slot = id >= 0 && s <= 2147483647LL ? static_cast<int>(s) : -1;
    }
  }
  p.requests[t] = request;
  p.positions[t] = pos;
  p.slots[t] = slot;
}

// One CTA.  Requests are served in order while pages last; one whose tokens do not fit (its table row, the packed batch or
// the free pages) gets nothing and keeps its length.
__global__ void __launch_bounds__(kTabThreads) fox_page_tables_kernel(const TableParams p, const bool place) {
  __shared__ int64_t s_warp[kTabWarps];
  __shared__ int32_t s_starts[kTabThreads + 1], s_granted[kTabThreads], s_lengths[kTabThreads], s_taken[kTabThreads];
  __shared__ int s_served;
  if (threadIdx.x == 0) s_served = s_starts[0] = 0;
  wait_for_kernel_in_front();
  if (!place) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");   // (the placing kernel, which waits for this one's end)
  const int free_before = max(0, min(*p.num_free, p.n_free_max));
  const int64_t page_less_1 = (1 << p.page_log2) - 1;
  const bool staged = p.R <= kTabThreads;   // all requests in shared memory
  int64_t tokens = 0, taken = 0;
  for (int base = 0; base < p.R; base += kTabThreads) {
    const int r = base + threadIdx.x;
    const bool in = r < p.R;
    const int64_t old = in ? max(p.lengths[r], 0) : 0, fresh = in ? max(p.new_tokens[r], 0) : 0;
    int64_t sum;
    const int64_t end = tokens + block_scan(fresh, sum, s_warp);
    tokens += sum;
    const int64_t have = (old + page_less_1) >> p.page_log2, want = (old + fresh + page_less_1) >> p.page_log2;
    const bool fits = want <= p.width && end <= p.max_tokens && old + fresh <= 2147483647LL;
    const int64_t need = fits ? want - have : 0;
    const int64_t upto = taken + block_scan(need, sum, s_warp);
    taken += sum;
    const bool ok = fits && (need == 0 || upto <= free_before);
    if (ok && need) atomicMax(&s_served, static_cast<int>(upto));   // (those that get pages are the first ones that need any)
    if (in) {
      const int start = clamp31(end), given = ok ? static_cast<int>(fresh) : 0, length = static_cast<int>(old) + given,
                front = clamp31(upto - need);
      p.starts[r + 1] = start;
      if (r == 0) p.starts[0] = 0;
      p.granted[r] = given;
      p.lengths_out[r] = length;
      if (staged) {
        s_starts[r + 1] = start;
        s_granted[r] = given;
        s_lengths[r] = length;
        s_taken[r] = front;
      }
      p.work[r] = front;
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    p.work[p.R] = free_before;
    *p.num_free_out = free_before - s_served;
  }
  if (!place) return;
  const Placing a = staged ? Placing{s_starts, s_granted, s_lengths, s_taken, free_before}
                           : Placing{p.starts, p.granted, p.lengths_out, p.work, free_before};
  for (int t = threadIdx.x; t < p.max_tokens; t += kTabThreads) place_token(p, a, t);
}
constexpr int kPlaceStaged = 4096;   // requests whose starts a block keeps
__global__ void __launch_bounds__(256) fox_page_slots_kernel(const TableParams p) {
  __shared__ int32_t s_starts[kPlaceStaged + 1];
  wait_for_kernel_in_front();
  const bool staged = p.R <= kPlaceStaged;
  if (staged)
    for (int i = threadIdx.x; i <= p.R; i += 256) s_starts[i] = p.starts[i];
  __syncthreads();
  const Placing a{staged ? s_starts : p.starts, p.granted, p.lengths_out, p.work, p.work[p.R]};
  const int64_t t = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (t < p.max_tokens) place_token(p, a, static_cast<int>(t));
}

// One CTA.  The pages behind keep[r] tokens go back on the stack, in the order of requests and of their tables' entries.
struct ReleaseParams {
  int32_t* lengths;
  const int32_t* keep;
  int32_t* table;
  int64_t table_ld;
  int32_t *free_pages, *num_free;
  int R, width, n_free_max, page_log2;
};
__global__ void __launch_bounds__(kTabThreads) fox_release_pages_kernel(const ReleaseParams p) {
  __shared__ int64_t s_warp[kTabWarps];
  wait_for_kernel_in_front();
  int64_t top = max(0, min(*p.num_free, p.n_free_max));
  const int64_t page_less_1 = (1 << p.page_log2) - 1;
  const int lane = threadIdx.x & 31;
  for (int base = 0; base < p.R; base += kTabThreads) {
    const int r = base + threadIdx.x;
    const bool in = r < p.R;
    const int64_t old = in ? max(p.lengths[r], 0) : 0, kept = in ? min(static_cast<int64_t>(max(p.keep[r], 0)), old) : 0;
    // (a row beyond the table's width has no entries)
    const int from = static_cast<int>(min((kept + page_less_1) >> p.page_log2, static_cast<int64_t>(p.width)));
    const int to = static_cast<int>(min((old + page_less_1) >> p.page_log2, static_cast<int64_t>(p.width)));
    int64_t sum;
    const int64_t at = top + block_scan(to - from, sum, s_warp) - (to - from);
    // a warp takes its requests' pages one request after the other, 32 pages at a time
    uint32_t todo = __ballot_sync(0xffffffffu, to > from);
    while (todo) {
      const int l = __ffs(todo) - 1;
      todo &= todo - 1;
      const int f = __shfl_sync(0xffffffffu, from, l), n = __shfl_sync(0xffffffffu, to, l) - f;
      const int64_t a = __shfl_sync(0xffffffffu, at, l);
      int32_t* entry = p.table + (base + static_cast<int>(threadIdx.x & ~31u) + l) * p.table_ld + f;
      for (int j = lane; j < n; j += 32) {
        if (a + j < p.n_free_max) p.free_pages[a + j] = entry[j];
        entry[j] = -1;
      }
    }
    if (in) p.lengths[r] = static_cast<int>(kept);
    top += sum;
  }
  if (threadIdx.x == 0) *p.num_free = static_cast<int>(min(top, static_cast<int64_t>(p.n_free_max)));
}

// ------------------------------------------------------------------- rows
// Bound by HBM: each row is read once and written once.  A CTA takes a tile of tokens; a thread holds one 16-byte piece of a
// token's keys or values and goes through the tile with it, kAhead tokens' loads in front of their stores (8 where an
// SM has 16 tiles or more: 30000 tokens x 24 heads of 64 59.9 -> 57.5 us; else 4, which take fewer registers: 5000 tokens x 16 heads of
// 128 16.0 -> 15.4, 2000 7.9 -> 6.0).  The gates of a
// tile go with one token to a lane, so that tokens behind one another in a page are written side by side.
// (30000 tokens x 24 heads of 64, tiles of 32 / 16 / 8 tokens with 4 ahead: 64, 61, 60 us; 16 heads of 128: 81, 77, 74.)
constexpr int kUpdThreads = 256, kUpdTile = 8;   // threads: at most

struct UpdateParams {
  const uint16_t *k, *v;
  int64_t k_st, k_sh, v_st, v_sh;
  const void* gates;
  int64_t g_st, g_sh;
  int gate_kind;                       // FOX_GATE_LOG, or the dtype of logits
  uint16_t *k_pages, *v_pages;
  int64_t k_sp, k_sk, k_sr, v_sp, v_sk, v_sr;   // strides of pages, heads, rows
  float* gate_pages;
  int64_t g_sp, g_sk;
  const void* slots;
  int slots_64;
  int64_t T, n_slots;
  int H, Hk, lanes, tile, page_log2;
};

__device__ __forceinline__ float upd_gate(const UpdateParams& p, int64_t i) {
  if (p.gate_kind == FOX_GATE_LOG) return static_cast<const float*>(p.gates)[i];
  float x;
  if (p.gate_kind == FOX_DTYPE_FP32) x = static_cast<const float*>(p.gates)[i];
  else {
    const uint32_t u = static_cast<const uint16_t*>(p.gates)[i];
    x = p.gate_kind == FOX_DTYPE_BF16 ? unpack2<true>(u).x : unpack2<false>(u).x;
  }
  return fminf(x, 0.f) - log1pf(expf(-fabsf(x)));
}

template <int kAhead>
__global__ void __launch_bounds__(kUpdThreads) fox_paged_update_kernel(const UpdateParams p) {
  __shared__ int64_t s_page[kUpdTile];
  __shared__ int s_row[kUpdTile];
  wait_for_kernel_in_front();
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * p.tile;
  const int n = static_cast<int>(min(static_cast<int64_t>(p.tile), p.T - t0));
  if (threadIdx.x < n) {
    const int64_t t = t0 + threadIdx.x;
    const int64_t s = p.slots_64 ? static_cast<const int64_t*>(p.slots)[t] : static_cast<const int32_t*>(p.slots)[t];
    s_page[threadIdx.x] = s >= 0 && s < p.n_slots ? s >> p.page_log2 : -1;   // (a token without a place is left out)
    s_row[threadIdx.x] = static_cast<int>(s & ((1 << p.page_log2) - 1));
  }
  __syncthreads();
  const int pieces = p.Hk * p.lanes;
  for (int c = threadIdx.x; c < 2 * pieces; c += blockDim.x) {
    const bool is_v = c >= pieces;
    const int i = is_v ? c - pieces : c, h = i / p.lanes, sub = i - h * p.lanes;
    const uint16_t* from = (is_v ? p.v + h * p.v_sh + t0 * p.v_st : p.k + h * p.k_sh + t0 * p.k_st) + sub * 8;
    uint16_t* to = (is_v ? p.v_pages + h * p.v_sk : p.k_pages + h * p.k_sk) + sub * 8;
    const int64_t st = is_v ? p.v_st : p.k_st, sp = is_v ? p.v_sp : p.k_sp, sr = is_v ? p.v_sr : p.k_sr;
    for (int u0 = 0; u0 < n; u0 += kAhead) {
      uint4 x[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (u0 + u < n) x[u] = ld_v4_here(reinterpret_cast<const uint4*>(from + (u0 + u) * st));
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (u0 + u < n && s_page[u0 + u] >= 0) *reinterpret_cast<uint4*>(to + s_page[u0 + u] * sp + s_row[u0 + u] * sr) = x[u];
    }
  }
  for (int i = threadIdx.x; i < p.H * kUpdTile; i += blockDim.x) {
    const int u = i & (kUpdTile - 1), h = i / kUpdTile;
    if (u < n && s_page[u] >= 0) p.gate_pages[s_page[u] * p.g_sp + h * p.g_sk + s_row[u]] = upd_gate(p, (t0 + u) * p.g_st + h * p.g_sh);
  }
}

static bool page_size_ok(int64_t page) { return page >= 16 && page <= 65536 && !(page & (page - 1)); }
static int log2_of(int64_t x) {
  int n = 0;
  while ((int64_t{1} << n) < x) ++n;
  return n;
}

}  // namespace fox

using namespace fox;

extern "C" int fox_page_tables(int device, void* stream, int64_t R, int64_t width, int64_t page, int64_t max_tokens,
                               const int32_t* lengths, const int32_t* new_tokens, int32_t* block_table, int64_t table_ld,
                               const int32_t* free_pages, int64_t n_pages, const int32_t* num_free, int32_t* lengths_out,
                               int32_t* num_free_out, int32_t* starts, int32_t* granted, int32_t* requests, int32_t* positions,
                               int32_t* slots, int32_t* workspace) {
  if (!lengths || !new_tokens || !block_table || !free_pages || !num_free || !lengths_out || !num_free_out || !starts || !granted ||
      !workspace || (max_tokens > 0 && (!requests || !positions || !slots)))
    return FOX_ERR_BAD_ARG;
  if (R <= 0 || width <= 0 || max_tokens < 0 || n_pages <= 0 || table_ld < width || !page_size_ok(page)) return FOX_ERR_BAD_ARG;
  if (R > (1 << 24) || width > (1 << 30) || max_tokens > (1 << 30) || n_pages > 2147483647LL) return FOX_ERR_TOO_LARGE;
  if (cudaSetDevice(device) != cudaSuccess) return FOX_ERR_DEVICE;
  const TableParams p{lengths, new_tokens, block_table, table_ld, free_pages, num_free, lengths_out, num_free_out, starts, granted,
                      requests, positions, slots, workspace, (int)R, (int)width, (int)n_pages, log2_of(page), (int)max_tokens};
  const bool one = max_tokens <= kTabOneCta;
  cudaStream_t st = (cudaStream_t)stream;
  if (int rc = launch_behind(fox_page_tables_kernel, dim3(1), kTabThreads, 0, st, p, one)) return rc;
  return one ? FOX_OK : launch_behind(fox_page_slots_kernel, dim3((unsigned)((max_tokens + 255) / 256)), 256, 0, st, p);
}

extern "C" int fox_release_pages(int device, void* stream, int64_t R, int64_t width, int64_t page, int32_t* lengths,
                                 const int32_t* keep, int32_t* block_table, int64_t table_ld, int32_t* free_pages, int64_t n_pages,
                                 int32_t* num_free) {
  if (!lengths || !keep || !block_table || !free_pages || !num_free) return FOX_ERR_BAD_ARG;
  if (R <= 0 || width <= 0 || n_pages <= 0 || table_ld < width || !page_size_ok(page)) return FOX_ERR_BAD_ARG;
  if (R > (1 << 24) || width > (1 << 30) || n_pages > 2147483647LL) return FOX_ERR_TOO_LARGE;
  if (cudaSetDevice(device) != cudaSuccess) return FOX_ERR_DEVICE;
  const ReleaseParams p{lengths, keep, block_table, table_ld, free_pages, num_free, (int)R, (int)width, (int)n_pages, log2_of(page)};
  return launch_behind(fox_release_pages_kernel, dim3(1), kTabThreads, 0, (cudaStream_t)stream, p);
}

extern "C" int fox_paged_update(int device, void* stream, int64_t T, int64_t H, int64_t Hk, int64_t D, int64_t n_pages, int64_t page,
                                const void* k, int64_t k_st, int64_t k_sh, const void* v, int64_t v_st, int64_t v_sh, int gate_kind,
                                const void* gates, int64_t g_st, int64_t g_sh, const fox_tensor4* k_pages, const fox_tensor4* v_pages,
                                float* gate_pages, int64_t gp_sp, int64_t gp_sh, const void* slots, int slots_64) {
  if (!k || !v || !gates || !k_pages || !v_pages || !k_pages->ptr || !v_pages->ptr || !gate_pages || !slots) return FOX_ERR_BAD_ARG;
  if (T <= 0 || H <= 0 || Hk <= 0 || n_pages <= 0 || !page_size_ok(page)) return FOX_ERR_BAD_ARG;
  if (gate_kind != FOX_GATE_LOG && gate_kind != FOX_DTYPE_FP16 && gate_kind != FOX_DTYPE_BF16 && gate_kind != FOX_DTYPE_FP32)
    return FOX_ERR_BAD_ARG;
  if (D != 16 && D != 32 && D != 64 && D != 128) return FOX_ERR_HEAD_DIM;
  if (H > 65535 || Hk > 65535 || T > (int64_t{1} << 31) - 1 || n_pages > 2147483647LL / page) return FOX_ERR_TOO_LARGE;
  auto off = [](const void* q, std::initializer_list<int64_t> strides) {
    bool bad = reinterpret_cast<uintptr_t>(q) % 16;
    for (int64_t s : strides) bad |= s % 8 != 0;
    return bad;
  };
  if (off(k, {k_st, k_sh}) || off(v, {v_st, v_sh}) || off(k_pages->ptr, {k_pages->sb, k_pages->sh, k_pages->st}) ||
      off(v_pages->ptr, {v_pages->sb, v_pages->sh, v_pages->st}))
    return FOX_ERR_ALIGNMENT;
  if (cudaSetDevice(device) != cudaSuccess) return FOX_ERR_DEVICE;
  // a tile of 8 tokens, fewer where those are fewer than four CTAs to an SM
  const int64_t fit = (T + kSms * 4 - 1) / (kSms * 4), tile = fit < kUpdTile ? fit : kUpdTile;
  // threads: a token's pieces over as few turns as 256 take, evenly; 128 at least
  const int64_t pieces = 2 * Hk * (D / 8), turns = (pieces + kUpdThreads - 1) / kUpdThreads, even = ((pieces + turns - 1) / turns + 31) / 32 * 32;
  const unsigned threads = even < 128 ? 128 : (unsigned)even;
  const UpdateParams p{(const uint16_t*)k, (const uint16_t*)v, k_st, k_sh, v_st, v_sh, gates, g_st, g_sh, gate_kind,
                       (uint16_t*)k_pages->ptr, (uint16_t*)v_pages->ptr, k_pages->sb, k_pages->sh, k_pages->st, v_pages->sb,
                       v_pages->sh, v_pages->st, gate_pages, gp_sp, gp_sh, slots, slots_64, T, n_pages * page, (int)H, (int)Hk,
                       (int)(D / 8), (int)tile, log2_of(page)};
  const dim3 grid((unsigned)((T + tile - 1) / tile));
  if (grid.x >= 16 * kSms) return launch_behind(fox_paged_update_kernel<kUpdTile>, grid, threads, 0, (cudaStream_t)stream, p);
  return launch_behind(fox_paged_update_kernel<kUpdTile / 2>, grid, threads, 0, (cudaStream_t)stream, p);
}
