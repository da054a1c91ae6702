// Rotary positions, alone or with the per-head RMSNorm of queries and keys in the same pass, forward and backward.
// HBM-bound: every element is read once and written once.
//
//   n = x rstd w,  rstd = (mean_d x^2 + eps)^-1/2              (n = x without the norm)
//   a = position * inv_freq_i;  c = scale cos a, s = scale sin a
//   y_p = n_p c - n_p' s,  y_p' = n_p' c + n_p s               pairs (p, p') = (i, i + half) or (2i, 2i + 1), i < half
//   y_d = n_d                                                  channels from 2 half on
//   backward: dn = the rotation by -a of dy;  dw_h += dn xhat (xhat = x rstd);  dx = rstd (dn w - xhat mean_d(dn w xhat))
//
// Upstream norms q and k in one kernel (layernorm.py:183-245 as modeling_forgetting_transformer.py:264-265, 314-316 builds
// it) and rotates them in another (rotary.py:22-153, from a table of cosines and sines in the tensors' type); here the
// normed values are never rounded or written in between, and one launch takes both tensors.
//
// There is no table of all positions: a CTA forms the angles of its own tile of tokens, once for all of its heads.  The
// product of position and frequency and its reduction by turns are in 64 bits (at position 10^6 a 32-bit product is off by
// 0.03 rad), sine and cosine of what is left, at most pi, in 32.
//
// Thread (h, sub) owns the 8 channels [8 sub, 8 sub + 8) of head h (queries' heads, then keys') for every token that its CTA
// visits: 16-byte loads, the row's sum of squares by a shuffle over D/8 neighbouring lanes, weights and dw in registers.
// kMode: where the other channel of a pair is:
//   kNext    in the same lane (neighbouring channels)
//   kLanes   at the same place of the lane half/8 away (half a multiple of 8): packed values by shuffle
//   kAny     halves that are no multiple of 8: read from the row again, channel by channel (L1 has it)
#include "fox_common.cuh"
#include "fox_host.h"

namespace fox {

enum RotaryMode { kNext, kLanes, kAny };

constexpr int kRotThreads = 256;
constexpr int kRotTile = 16;      // tokens whose angles are in shared memory at a time
constexpr int kRotAhead = 4;      // tokens whose rows a thread has asked for
constexpr int64_t kRotTokens = (int64_t{1} << 31) - 65536;   // counted with 32 bits, a tile's more among them
constexpr int kRotFill = kSms * 4; // CTAs below which tiles are made smaller

struct RotaryTensor {
  const uint16_t *x, *dy;
  uint16_t* y;                    // forward: y; backward: dx
  int64_t x_sb, x_sh, x_st, dy_sb, dy_sh, dy_st, y_sb, y_sh, y_st;
  const void* w;
  int w_dtype;
  int64_t w_sh;                   // D, or 0: one weight for all heads
};
struct RotaryParams {
  RotaryTensor t[2];
  const float* inv_freq;
  const void* positions;          // or nullptr: first + t
  int64_t pos_sb, pos_st, first;
  float* dw_partial;              // (grid.x, heads, D)
  float scale, sign, eps;         // sign: of the sine
  int pos_64, half, D, T, tokens, H, heads, heads_here, tile;
};

template <bool kBf16>
__device__ __forceinline__ void rot_unpack(const uint4& v, float* f) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 t = unpack2<kBf16>(w[j]);
    f[2 * j] = t.x;
    f[2 * j + 1] = t.y;
  }
}
template <bool kBf16>
__device__ __forceinline__ uint4 rot_pack(const float* f) {
  return make_uint4(pack2<kBf16>(f[0], f[1]), pack2<kBf16>(f[2], f[3]), pack2<kBf16>(f[4], f[5]), pack2<kBf16>(f[6], f[7]));
}
__device__ __forceinline__ float rot_weight(const void* w, int dtype, int64_t i) {
  if (dtype == FOX_DTYPE_FP32) return static_cast<const float*>(w)[i];
  const uint32_t u = static_cast<const uint16_t*>(w)[i];
  return dtype == FOX_DTYPE_BF16 ? unpack2<true>(u).x : unpack2<false>(u).x;
}

// cosines and sines of `n` tokens from t0 on, (tile, D / 2) each
__device__ __forceinline__ void rot_angles(const RotaryParams& p, int t0, int n, float* s_cos, float* s_sin) {
  const int pairs = p.D >> 1;
  for (int i = threadIdx.x; i < n * p.half; i += blockDim.x) {
    const int u = i / p.half, f = i - u * p.half, token = t0 + u;
    const int b = token / p.T, t = token - b * p.T;
    int64_t pos = p.first + t;
    if (p.positions) {
      const int64_t at = b * p.pos_sb + t * p.pos_st;
      pos = p.pos_64 ? static_cast<const int64_t*>(p.positions)[at] : static_cast<const int32_t*>(p.positions)[at];
    }
    const double a = static_cast<double>(pos) * static_cast<double>(p.inv_freq[f]);
    const double turns = rint(a * 0.15915494309189535);
    // 2 pi in two parts
    const double r = fma(turns, -2.4492935982947064e-16, fma(turns, -6.283185307179586, a));
    float sn, cs;
    sincosf(static_cast<float>(r), &sn, &cs);
    s_cos[u * pairs + f] = cs * p.scale;
    s_sin[u * pairs + f] = sn * p.scale * p.sign;
  }
}

// The rotation of one lane's 8 channels.  n: its values; raw: what they were packed in; other(j): the value of the other
// channel of a pair, for kAny.
template <bool kBf16, int kMode, class Other>
__device__ __forceinline__ void rot_turn(const RotaryParams& p, int ch, const float* c, const float* s, const float* n,
                                         const float* pair, Other&& other, float* out) {
  if constexpr (kMode == kNext) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = (ch >> 1) + j;
      const bool in = i < p.half;
      const float cs = in ? c[i] : 1.f, sn = in ? s[i] : 0.f;
      out[2 * j] = n[2 * j] * cs - n[2 * j + 1] * sn;
      out[2 * j + 1] = n[2 * j + 1] * cs + n[2 * j] * sn;
    }
  } else if constexpr (kMode == kLanes) {
    const bool in = ch < 2 * p.half, low = ch < p.half;
    const int i0 = in ? (low ? ch : ch - p.half) : 0;
    const float4 c0 = *reinterpret_cast<const float4*>(c + i0), c1 = *reinterpret_cast<const float4*>(c + i0 + 4);
    const float4 s0 = *reinterpret_cast<const float4*>(s + i0), s1 = *reinterpret_cast<const float4*>(s + i0 + 4);
    const float cs[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
    const float sn[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
#pragma unroll
    for (int j = 0; j < 8; ++j) out[j] = in ? n[j] * cs[j] + pair[j] * (low ? -sn[j] : sn[j]) : n[j];
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int d = ch + j;
      out[j] = n[j];
      if (d < 2 * p.half) {
        const bool low = d < p.half;
        const int i = low ? d : d - p.half;
        const float m = other(low ? d + p.half : i);
        out[j] = n[j] * c[i] + m * (low ? -s[i] : s[i]);
      }
    }
  }
}

// lane of the other channels of a pair, for kLanes (a lane beyond the rotated part: itself)
__device__ __forceinline__ int rot_partner(const RotaryParams& p, int ch, int lane) {
  return ch < p.half ? lane + (p.half >> 3) : ch < 2 * p.half ? lane - (p.half >> 3) : lane;
}
__device__ __forceinline__ uint4 rot_shuffle(const uint4& v, int from) {
  return make_uint4(__shfl_sync(0xffffffffu, v.x, from), __shfl_sync(0xffffffffu, v.y, from), __shfl_sync(0xffffffffu, v.z, from),
                    __shfl_sync(0xffffffffu, v.w, from));
}

// grid: (tiles of tokens, blocks of heads_here heads); blockDim.x = heads_here * D / 8 up to a whole warp
template <bool kBf16, int kMode, bool kNorm>
__global__ void __launch_bounds__(kRotThreads) fox_rotary_fwd_kernel(const RotaryParams p) {
  extern __shared__ __align__(16) float rot_smem[];
  const int lanes = p.D >> 3, pairs = p.D >> 1;
  float *s_cos = rot_smem, *s_sin = rot_smem + p.tile * pairs;
  const int sub = threadIdx.x % lanes, slot = threadIdx.x / lanes, head = blockIdx.y * p.heads_here + slot;
  const bool active = slot < p.heads_here && head < p.heads;
  const bool is_k = active && head >= p.H;
  const RotaryTensor& x = p.t[is_k];
  const int h = active ? (is_k ? head - p.H : head) : 0, ch = sub * 8;
  const int lane = threadIdx.x & 31, from = rot_partner(p, ch, lane);
  wait_for_kernel_in_front();
  const int t0 = blockIdx.x * p.tile, n = min(p.tile, p.tokens - t0);
  const uint16_t* row = x.x + h * x.x_sh + ch;
  auto load = [&](int u) {
    uint4 v = make_uint4(0, 0, 0, 0);
    if (active && u < n) {
      const int token = t0 + u, b = token / p.T;
      v = ld_v4_here(reinterpret_cast<const uint4*>(row + b * x.x_sb + (token - b * p.T) * x.x_st));
    }
    return v;
  };
  uint4 ahead[kRotAhead];
#pragma unroll
  for (int u = 0; u < kRotAhead; ++u) ahead[u] = load(u);
  float w[8], wp[8];
  if constexpr (kNorm) {
    const int chp = ch + (from - lane) * 8;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      w[j] = active ? rot_weight(x.w, x.w_dtype, h * x.w_sh + ch + j) : 0.f;
      wp[j] = active && kMode == kLanes ? rot_weight(x.w, x.w_dtype, h * x.w_sh + chp + j) : 0.f;
    }
  }
  const float inv_d = 1.f / static_cast<float>(p.D);
  rot_angles(p, t0, n, s_cos, s_sin);
  __syncthreads();
  for (int u0 = 0; u0 < n; u0 += kRotAhead) {
    uint4 raw[kRotAhead];
#pragma unroll
    for (int u = 0; u < kRotAhead; ++u) {
      raw[u] = ahead[u];
      ahead[u] = load(u0 + kRotAhead + u);
    }
#pragma unroll
    for (int u = 0; u < kRotAhead; ++u) {
      if (u0 + u >= n) break;   // (the same for all threads)
      float v[8], pair[8], out[8], r = 1.f;
      rot_unpack<kBf16>(raw[u], v);
      if constexpr (kNorm) {
        float ss = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) ss = fmaf(v[j], v[j], ss);
        for (int o = lanes >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        r = rsqrtf(ss * inv_d + p.eps);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] *= r * w[j];
      }
      if constexpr (kMode == kLanes) {
        rot_unpack<kBf16>(rot_shuffle(raw[u], from), pair);
        if constexpr (kNorm) {
#pragma unroll
          for (int j = 0; j < 8; ++j) pair[j] *= r * wp[j];
        }
      }
      const int token = t0 + u0 + u, b = token / p.T, t = token - b * p.T;
      auto other = [&](int d) {
        const float m = active ? rot_weight(row - ch + b * x.x_sb + t * x.x_st, kBf16 ? FOX_DTYPE_BF16 : FOX_DTYPE_FP16, d) : 0.f;
        return kNorm ? m * (r * (active ? rot_weight(x.w, x.w_dtype, h * x.w_sh + d) : 0.f)) : m;
      };
      rot_turn<kBf16, kMode>(p, ch, s_cos + (u0 + u) * pairs, s_sin + (u0 + u) * pairs, v, pair, other, out);
      if (active) *reinterpret_cast<uint4*>(x.y + b * x.y_sb + h * x.y_sh + t * x.y_st + ch) = rot_pack<kBf16>(out);
    }
  }
}

// The norm's backward with the rotation in front.  A CTA takes every grid.x-th tile, so that its share of dw stays in
// registers; fox_rotary_dw_kernel adds the shares in a fixed order.
template <bool kBf16, int kMode>
__global__ void __launch_bounds__(kRotThreads) fox_rotary_bwd_kernel(const RotaryParams p) {
  constexpr int kAhead = 2;
  extern __shared__ __align__(16) float rot_smem[];
  const int lanes = p.D >> 3, pairs = p.D >> 1;
  float *s_cos = rot_smem, *s_sin = rot_smem + p.tile * pairs;
  const int sub = threadIdx.x % lanes, slot = threadIdx.x / lanes, head = blockIdx.y * p.heads_here + slot;
  const bool active = slot < p.heads_here && head < p.heads;
  const bool is_k = active && head >= p.H;
  const RotaryTensor& x = p.t[is_k];
  const int h = active ? (is_k ? head - p.H : head) : 0, ch = sub * 8;
  const int lane = threadIdx.x & 31, from = rot_partner(p, ch, lane);
  wait_for_kernel_in_front();
  float w[8], dw[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    w[j] = active ? rot_weight(x.w, x.w_dtype, h * x.w_sh + ch + j) : 0.f;
    dw[j] = 0.f;
  }
  const float inv_d = 1.f / static_cast<float>(p.D);
  for (int64_t t64 = static_cast<int64_t>(blockIdx.x) * p.tile; t64 < p.tokens; t64 += static_cast<int64_t>(gridDim.x) * p.tile) {
    const int t0 = static_cast<int>(t64), n = min(p.tile, p.tokens - t0);
    uint4 ahead_x[kAhead], ahead_g[kAhead];
    auto load = [&](int u, uint4& vx, uint4& vg) {
      vx = vg = make_uint4(0, 0, 0, 0);
      if (active && u < n) {
        const int token = t0 + u, b = token / p.T, t = token - b * p.T;
        vx = ld_v4_here(reinterpret_cast<const uint4*>(x.x + b * x.x_sb + h * x.x_sh + t * x.x_st + ch));
        vg = ld_v4_here(reinterpret_cast<const uint4*>(x.dy + b * x.dy_sb + h * x.dy_sh + t * x.dy_st + ch));
      }
    };
#pragma unroll
    for (int u = 0; u < kAhead; ++u) load(u, ahead_x[u], ahead_g[u]);
    __syncthreads();
    rot_angles(p, t0, n, s_cos, s_sin);
    __syncthreads();
    for (int u0 = 0; u0 < n; u0 += kAhead) {
      uint4 raw_x[kAhead], raw_g[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        raw_x[u] = ahead_x[u];
        raw_g[u] = ahead_g[u];
        load(u0 + kAhead + u, ahead_x[u], ahead_g[u]);
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if (u0 + u >= n) break;
        float v[8], g[8], pair[8], dn[8], out[8];
        rot_unpack<kBf16>(raw_x[u], v);
        rot_unpack<kBf16>(raw_g[u], g);
        if constexpr (kMode == kLanes) rot_unpack<kBf16>(rot_shuffle(raw_g[u], from), pair);
        const int token = t0 + u0 + u, b = token / p.T, t = token - b * p.T;
        auto other = [&](int d) {
          return active ? rot_weight(x.dy + b * x.dy_sb + h * x.dy_sh + t * x.dy_st, kBf16 ? FOX_DTYPE_BF16 : FOX_DTYPE_FP16, d) : 0.f;
        };
        rot_turn<kBf16, kMode>(p, ch, s_cos + (u0 + u) * pairs, s_sin + (u0 + u) * pairs, g, pair, other, dn);
        float ss = 0.f, dot = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          ss = fmaf(v[j], v[j], ss);
          dot = fmaf(dn[j] * w[j], v[j], dot);
        }
        for (int o = lanes >> 1; o > 0; o >>= 1) {
          ss += __shfl_xor_sync(0xffffffffu, ss, o);
          dot += __shfl_xor_sync(0xffffffffu, dot, o);
        }
        const float r = rsqrtf(ss * inv_d + p.eps), mean = dot * r * inv_d;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float xhat = v[j] * r;
          dw[j] = fmaf(dn[j], xhat, dw[j]);
          out[j] = r * (dn[j] * w[j] - xhat * mean);
        }
        if (active) *reinterpret_cast<uint4*>(x.y + b * x.y_sb + h * x.y_sh + t * x.y_st + ch) = rot_pack<kBf16>(out);
      }
    }
  }
  if (active) {
    float* to = p.dw_partial + (static_cast<int64_t>(blockIdx.x) * p.heads + head) * p.D + ch;
    reinterpret_cast<float4*>(to)[0] = make_float4(dw[0], dw[1], dw[2], dw[3]);
    reinterpret_cast<float4*>(to)[1] = make_float4(dw[4], dw[5], dw[6], dw[7]);
  }
}

// dw of both tensors: 16 columns a CTA, its rows (shares, and heads where the weight is one for all) over 16 groups of threads
struct RotaryDwParams {
  const float* partial;
  void* dw[2];
  int w_dtype[2];
  int shared[2];
  int heads[2];
  int n_partials, D;
};
__global__ void __launch_bounds__(256) fox_rotary_dw_kernel(const RotaryDwParams p) {
  __shared__ float s_sum[16][17];
  wait_for_kernel_in_front();
  const int col = threadIdx.x & 15, grp = threadIdx.x >> 4;
  const int cols0 = p.shared[0] ? p.D : p.heads[0] * p.D;
  const int c_all = blockIdx.x * 16 + col, which = blockIdx.x * 16 >= cols0, c = c_all - (which ? cols0 : 0);
  const int heads_all = p.heads[0] + p.heads[1];
  const int64_t base = (which ? static_cast<int64_t>(p.heads[0]) * p.D : 0) + c, ld = static_cast<int64_t>(heads_all) * p.D;
  float sum = 0.f;
  if (p.shared[which]) {
    for (int h = 0; h < p.heads[which]; ++h)
#pragma unroll 4
      for (int r = grp; r < p.n_partials; r += 16) sum += p.partial[r * ld + base + h * p.D];
  } else {
#pragma unroll 4
    for (int r = grp; r < p.n_partials; r += 16) sum += p.partial[r * ld + base];
  }
  s_sum[grp][col] = sum;
  __syncthreads();
  if (grp == 0) {
#pragma unroll
    for (int g = 1; g < 16; ++g) sum += s_sum[g][col];
    if (p.w_dtype[which] == FOX_DTYPE_FP32) static_cast<float*>(p.dw[which])[c] = sum;
    else
      static_cast<uint16_t*>(p.dw[which])[c] =
          static_cast<uint16_t>((p.w_dtype[which] == FOX_DTYPE_BF16 ? pack2<true>(sum, 0.f) : pack2<false>(sum, 0.f)) & 0xffffu);
  }
}

// ------------------------------------------------------------------- launches
struct RotaryGrid {
  int blocks, heads_here, threads;
};
// heads of a token over as few CTAs of up to 256 threads as hold them, evenly
static RotaryGrid rotary_grid(int64_t heads, int64_t D) {
  const int64_t most = kRotThreads / (D / 8), blocks = (heads + most - 1) / most, here = (heads + blocks - 1) / blocks;
  return {static_cast<int>(blocks), static_cast<int>(here), static_cast<int>((here * (D / 8) + 31) / 32 * 32)};
}
// Tiles of 16 tokens, and smaller ones where those do not fill the GPU.
static int rotary_tile(int64_t tokens, int64_t blocks) {
  const int64_t t = (tokens * blocks + kRotFill - 1) / kRotFill;
  return static_cast<int>(t < 1 ? 1 : t < kRotTile ? t : kRotTile);
}

enum RotaryKind { kTurn, kNormTurn, kNormBack };
template <bool kBf16, int kMode>
static int rotary_launch_at(RotaryKind kind, dim3 grid, unsigned threads, size_t smem, cudaStream_t st, const RotaryParams& p) {
  if (kind == kTurn) return launch_behind(fox_rotary_fwd_kernel<kBf16, kMode, false>, grid, threads, smem, st, p);
  if (kind == kNormTurn) return launch_behind(fox_rotary_fwd_kernel<kBf16, kMode, true>, grid, threads, smem, st, p);
  return launch_behind(fox_rotary_bwd_kernel<kBf16, kMode>, grid, threads, smem, st, p);
}
static int rotary_launch(RotaryKind kind, int dtype, int64_t half, int interleaved, unsigned tiles, const RotaryGrid& g, cudaStream_t st,
                         const RotaryParams& p) {
  const dim3 grid(tiles, g.blocks);
  const size_t smem = static_cast<size_t>(p.tile) * p.D * sizeof(float);
  const bool bf = dtype == FOX_DTYPE_BF16;
  if (interleaved) return bf ? rotary_launch_at<true, kNext>(kind, grid, g.threads, smem, st, p) : rotary_launch_at<false, kNext>(kind, grid, g.threads, smem, st, p);
  if (half % 8) return bf ? rotary_launch_at<true, kAny>(kind, grid, g.threads, smem, st, p) : rotary_launch_at<false, kAny>(kind, grid, g.threads, smem, st, p);
  return bf ? rotary_launch_at<true, kLanes>(kind, grid, g.threads, smem, st, p) : rotary_launch_at<false, kLanes>(kind, grid, g.threads, smem, st, p);
}

static bool rotary_bad_rows(const fox_tensor4* t) {
  return reinterpret_cast<uintptr_t>(t->ptr) % 16 || t->sb % 8 || t->sh % 8 || t->st % 8;
}
static bool rotary_bad_weight(int dtype) { return dtype != FOX_DTYPE_FP16 && dtype != FOX_DTYPE_BF16 && dtype != FOX_DTYPE_FP32; }

static int rotary_check(int dtype, int64_t B, int64_t T, int64_t H, int64_t Hk, int64_t D, const float* inv_freq, int64_t half) {
  if (B <= 0 || T <= 0 || H <= 0 || Hk < 0 || half <= 0 || !inv_freq) return FOX_ERR_BAD_ARG;
  if (dtype != FOX_DTYPE_BF16 && dtype != FOX_DTYPE_FP16) return FOX_ERR_BAD_ARG;
  if (D != 16 && D != 32 && D != 64 && D != 128) return FOX_ERR_HEAD_DIM;
  if (2 * half > D) return FOX_ERR_BAD_ARG;
  if (H > 65535 || Hk > 65535 || T > kRotTokens || B > kRotTokens / T) return FOX_ERR_TOO_LARGE;
  return FOX_OK;
}
static RotaryParams rotary_params(int64_t B, int64_t T, int64_t H, int64_t Hk, int64_t D, const float* inv_freq, int64_t half,
                                  float scale, float eps, const void* positions, int pos_64, int64_t pos_sb, int64_t pos_st,
                                  int64_t first) {
  RotaryParams p{};
  p.inv_freq = inv_freq;
  p.positions = positions;
  p.pos_sb = pos_sb; p.pos_st = pos_st; p.first = first; p.pos_64 = pos_64;
  p.scale = scale; p.sign = 1.f; p.eps = eps;
  p.half = (int)half; p.D = (int)D; p.T = (int)T; p.tokens = (int)(B * T);
  p.H = (int)H; p.heads = (int)(H + Hk);
  return p;
}
static void rotary_in(RotaryTensor& t, const fox_tensor4* x) {
  t.x = (const uint16_t*)x->ptr; t.x_sb = x->sb; t.x_sh = x->sh; t.x_st = x->st;
}
static void rotary_out(RotaryTensor& t, const fox_tensor4* y) {
  t.y = (uint16_t*)y->ptr; t.y_sb = y->sb; t.y_sh = y->sh; t.y_st = y->st;
}

}  // namespace fox

using namespace fox;

extern "C" int fox_rotary(int device, void* stream, int dtype, int64_t B, int64_t T, int64_t H, int64_t D, const fox_tensor4* x,
                          const float* inv_freq, int64_t half, int interleaved, float scale, int inverse, const void* positions,
                          int pos_64, int64_t pos_sb, int64_t pos_st, int64_t first, const fox_tensor4* y) {
  if (!x || !y || !x->ptr || !y->ptr) return FOX_ERR_BAD_ARG;
  if (int rc = rotary_check(dtype, B, T, H, 0, D, inv_freq, half)) return rc;
  if (rotary_bad_rows(x) || rotary_bad_rows(y)) return FOX_ERR_ALIGNMENT;
  if (cudaSetDevice(device) != cudaSuccess) return FOX_ERR_DEVICE;
  RotaryParams p = rotary_params(B, T, H, 0, D, inv_freq, half, scale, 0.f, positions, pos_64, pos_sb, pos_st, first);
  p.sign = inverse ? -1.f : 1.f;
  rotary_in(p.t[0], x);
  rotary_out(p.t[0], y);
  const RotaryGrid g = rotary_grid(H, D);
  p.heads_here = g.heads_here;
  p.tile = rotary_tile(p.tokens, g.blocks);
  return rotary_launch(kTurn, dtype, half, interleaved, (p.tokens + p.tile - 1) / p.tile, g, (cudaStream_t)stream, p);
}

extern "C" int fox_qk_norm_rotary_fwd(int device, void* stream, int dtype, int64_t B, int64_t T, int64_t H, int64_t Hk, int64_t D,
                                      const fox_tensor4* q, const fox_tensor4* k, const void* wq, int wq_dtype, int64_t wq_sh,
                                      const void* wk, int wk_dtype, int64_t wk_sh, float eps, const float* inv_freq, int64_t half,
                                      int interleaved, float scale, const void* positions, int pos_64, int64_t pos_sb,
                                      int64_t pos_st, int64_t first, const fox_tensor4* q_out, const fox_tensor4* k_out) {
  if (!q || !k || !q_out || !k_out || !q->ptr || !k->ptr || !q_out->ptr || !k_out->ptr || !wq || !wk || Hk <= 0) return FOX_ERR_BAD_ARG;
  if (int rc = rotary_check(dtype, B, T, H, Hk, D, inv_freq, half)) return rc;
  if (rotary_bad_weight(wq_dtype) || rotary_bad_weight(wk_dtype)) return FOX_ERR_BAD_ARG;
  if (rotary_bad_rows(q) || rotary_bad_rows(k) || rotary_bad_rows(q_out) || rotary_bad_rows(k_out)) return FOX_ERR_ALIGNMENT;
  if (cudaSetDevice(device) != cudaSuccess) return FOX_ERR_DEVICE;
  RotaryParams p = rotary_params(B, T, H, Hk, D, inv_freq, half, scale, eps, positions, pos_64, pos_sb, pos_st, first);
  rotary_in(p.t[0], q); rotary_in(p.t[1], k);
  rotary_out(p.t[0], q_out); rotary_out(p.t[1], k_out);
  p.t[0].w = wq; p.t[0].w_dtype = wq_dtype; p.t[0].w_sh = wq_sh;
  p.t[1].w = wk; p.t[1].w_dtype = wk_dtype; p.t[1].w_sh = wk_sh;
  const RotaryGrid g = rotary_grid(H + Hk, D);
  p.heads_here = g.heads_here;
  p.tile = rotary_tile(p.tokens, g.blocks);
  return rotary_launch(kNormTurn, dtype, half, interleaved, (p.tokens + p.tile - 1) / p.tile, g, (cudaStream_t)stream, p);
}

extern "C" int64_t fox_qk_norm_rotary_partials(int64_t B, int64_t T, int64_t H, int64_t Hk, int64_t D) {
  if (B <= 0 || T <= 0 || H <= 0 || Hk <= 0 || (D != 16 && D != 32 && D != 64 && D != 128)) return 1;
  const RotaryGrid g = rotary_grid(H + Hk, D);
  const int64_t tile = rotary_tile(B * T, g.blocks), tiles = (B * T + tile - 1) / tile, most = (kRotFill + g.blocks - 1) / g.blocks;
  return tiles < most ? tiles : most;
}

extern "C" int fox_qk_norm_rotary_bwd(int device, void* stream, int dtype, int64_t B, int64_t T, int64_t H, int64_t Hk, int64_t D,
                                      const fox_tensor4* q, const fox_tensor4* k, const void* wq, int wq_dtype, int64_t wq_sh,
                                      const void* wk, int wk_dtype, int64_t wk_sh, float eps, const float* inv_freq, int64_t half,
                                      int interleaved, float scale, const void* positions, int pos_64, int64_t pos_sb,
                                      int64_t pos_st, int64_t first, const fox_tensor4* dq_out, const fox_tensor4* dk_out,
                                      const fox_tensor4* dq, const fox_tensor4* dk, float* dw_partial, void* dwq, void* dwk) {
  if (!q || !k || !dq_out || !dk_out || !dq || !dk || !q->ptr || !k->ptr || !dq_out->ptr || !dk_out->ptr || !dq->ptr || !dk->ptr ||
      !wq || !wk || !dw_partial || !dwq || !dwk || Hk <= 0)
    return FOX_ERR_BAD_ARG;
  if (int rc = rotary_check(dtype, B, T, H, Hk, D, inv_freq, half)) return rc;
  if (rotary_bad_weight(wq_dtype) || rotary_bad_weight(wk_dtype)) return FOX_ERR_BAD_ARG;
  for (const fox_tensor4* t : {q, k, dq_out, dk_out, dq, dk})
    if (rotary_bad_rows(t)) return FOX_ERR_ALIGNMENT;
  if (reinterpret_cast<uintptr_t>(dw_partial) % 16) return FOX_ERR_ALIGNMENT;
  if (cudaSetDevice(device) != cudaSuccess) return FOX_ERR_DEVICE;
  RotaryParams p = rotary_params(B, T, H, Hk, D, inv_freq, half, scale, eps, positions, pos_64, pos_sb, pos_st, first);
  p.sign = -1.f;
  const fox_tensor4 *xs[2] = {q, k}, *gs[2] = {dq_out, dk_out}, *ds[2] = {dq, dk};
  for (int i = 0; i < 2; ++i) {
    rotary_in(p.t[i], xs[i]);
    rotary_out(p.t[i], ds[i]);
    p.t[i].dy = (const uint16_t*)gs[i]->ptr;
    p.t[i].dy_sb = gs[i]->sb; p.t[i].dy_sh = gs[i]->sh; p.t[i].dy_st = gs[i]->st;
  }
  p.t[0].w = wq; p.t[0].w_dtype = wq_dtype; p.t[0].w_sh = wq_sh;
  p.t[1].w = wk; p.t[1].w_dtype = wk_dtype; p.t[1].w_sh = wk_sh;
  p.dw_partial = dw_partial;
  const RotaryGrid g = rotary_grid(H + Hk, D);
  const int64_t n = fox_qk_norm_rotary_partials(B, T, H, Hk, D);
  p.heads_here = g.heads_here;
  p.tile = rotary_tile(p.tokens, g.blocks);
  cudaStream_t st = (cudaStream_t)stream;
  if (int rc = rotary_launch(kNormBack, dtype, half, interleaved, (unsigned)n, g, st, p)) return rc;
  const RotaryDwParams d{dw_partial, {dwq, dwk}, {wq_dtype, wk_dtype}, {wq_sh == 0, wk_sh == 0}, {(int)H, (int)Hk}, (int)n, (int)D};
  const int64_t cols = (wq_sh ? H * D : D) + (wk_sh ? Hk * D : D);
  return launch_behind(fox_rotary_dw_kernel, dim3((unsigned)(cols / 16)), 256, 0, st, d);
}
