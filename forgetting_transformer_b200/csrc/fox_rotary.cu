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
constexpr int kRotFill = kSms * 4;    // CTAs below which tiles are made smaller
constexpr int kRotShares = kSms * 4;  // CTAs of a backward, each with a share of dw

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
  const void* positions;          // or nullptr: first + t step
  int64_t pos_sb, pos_st, first, step;
  float* dw_partial;              // (shares, heads, D)
  float scale, sign, eps;         // sign: of the sine
  Divisor by_half;
  int pos_64, half, D, B, T, H, heads, heads_here, tile;
};

template <bool kBf16>
__device__ __forceinline__ void rot_unpack(const uint4& v, float2* f) {
  f[0] = unpack2<kBf16>(v.x);
  f[1] = unpack2<kBf16>(v.y);
  f[2] = unpack2<kBf16>(v.z);
  f[3] = unpack2<kBf16>(v.w);
}
template <bool kBf16>
__device__ __forceinline__ uint4 rot_pack(const float2* f) {
  return make_uint4(pack2<kBf16>(f[0].x, f[0].y), pack2<kBf16>(f[1].x, f[1].y), pack2<kBf16>(f[2].x, f[2].y), pack2<kBf16>(f[3].x, f[3].y));
}
__device__ __forceinline__ float rot_weight(const void* w, int dtype, int64_t i) {
  if (dtype == FOX_DTYPE_FP32) return static_cast<const float*>(w)[i];
  const uint32_t u = static_cast<const uint16_t*>(w)[i];
  return dtype == FOX_DTYPE_BF16 ? unpack2<true>(u).x : unpack2<false>(u).x;
}
// eight weights from element i on, a multiple of 8 (16-byte aligned)
__device__ __forceinline__ void rot_weights(const void* w, int dtype, int64_t i, float2* f) {
  if (dtype == FOX_DTYPE_FP32) {
    const float4 *v = reinterpret_cast<const float4*>(static_cast<const float*>(w) + i), a = v[0], b = v[1];
    f[0] = make_float2(a.x, a.y);
    f[1] = make_float2(a.z, a.w);
    f[2] = make_float2(b.x, b.y);
    f[3] = make_float2(b.z, b.w);
  } else {
    const uint4 v = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(w) + i);
    if (dtype == FOX_DTYPE_BF16) rot_unpack<true>(v, f);
    else rot_unpack<false>(v, f);
  }
}
__device__ __forceinline__ float2 rot_mul(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float2 rot_fma(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }
__device__ __forceinline__ float2 rot_both(float a) { return make_float2(a, a); }

// cosines and sines of tokens t0 .. t0 + n of sequence b, (tile, D / 2) each; s_pos: (tile).  A barrier is inside and one behind.
__device__ __forceinline__ void rot_angles(const RotaryParams& p, int b, int t0, int n, double* s_pos, float* s_cos, float* s_sin) {
  const int pairs = p.D >> 1;
  for (int u = threadIdx.x; u < n; u += blockDim.x) {
    const int t = t0 + u;
    int64_t pos = p.first + t * p.step;
    if (p.positions) {
      const int64_t at = b * p.pos_sb + t * p.pos_st;
      pos = p.pos_64 ? static_cast<const int64_t*>(p.positions)[at] : static_cast<const int32_t*>(p.positions)[at];
    }
    s_pos[u] = static_cast<double>(pos);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n * p.half; i += blockDim.x) {
    const int u = div_by(p.by_half, i), f = i - u * p.half;
    const double a = s_pos[u] * static_cast<double>(p.inv_freq[f]);
    const double turns = rint(a * 0.15915494309189535);
    // less whole turns, 2 pi in two parts; in units of pi
    const double r = fma(turns, -2.4492935982947064e-16, fma(turns, -6.283185307179586, a)) * 0.3183098861837907;
    float sn, cs;
    sincospif(static_cast<float>(r), &sn, &cs);
    s_cos[u * pairs + f] = cs * p.scale;
    s_sin[u * pairs + f] = sn * p.scale * p.sign;
  }
  __syncthreads();
}

// The rotation of one lane's 8 channels n.  pair: the values half the rotated part away, turned in sign where those are the
// second ones (kLanes); other(d): the value of channel d (kAny).
template <int kMode, class Other>
__device__ __forceinline__ void rot_turn(const RotaryParams& p, int ch, const float* c, const float* s, const float2* n,
                                         const float2* pair, Other&& other, float2* out) {
  if constexpr (kMode == kNext) {
    if (ch + 8 <= 2 * p.half) {
      const float4 cs = *reinterpret_cast<const float4*>(c + (ch >> 1)), sn = *reinterpret_cast<const float4*>(s + (ch >> 1));
      const float cv[4] = {cs.x, cs.y, cs.z, cs.w}, sv[4] = {sn.x, sn.y, sn.z, sn.w};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        out[j] = rot_fma(n[j], rot_both(cv[j]), rot_mul(make_float2(n[j].y, n[j].x), make_float2(-sv[j], sv[j])));
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = (ch >> 1) + j;
        const float cv = i < p.half ? c[i] : 1.f, sv = i < p.half ? s[i] : 0.f;
        out[j] = make_float2(n[j].x * cv - n[j].y * sv, n[j].y * cv + n[j].x * sv);
      }
    }
  } else if constexpr (kMode == kLanes) {
    if (ch < 2 * p.half) {
      const int i0 = ch < p.half ? ch : ch - p.half;
      const float4 c0 = *reinterpret_cast<const float4*>(c + i0), c1 = *reinterpret_cast<const float4*>(c + i0 + 4);
      const float4 s0 = *reinterpret_cast<const float4*>(s + i0), s1 = *reinterpret_cast<const float4*>(s + i0 + 4);
      out[0] = rot_fma(n[0], make_float2(c0.x, c0.y), rot_mul(pair[0], make_float2(s0.x, s0.y)));
      out[1] = rot_fma(n[1], make_float2(c0.z, c0.w), rot_mul(pair[1], make_float2(s0.z, s0.w)));
      out[2] = rot_fma(n[2], make_float2(c1.x, c1.y), rot_mul(pair[2], make_float2(s1.x, s1.y)));
      out[3] = rot_fma(n[3], make_float2(c1.z, c1.w), rot_mul(pair[3], make_float2(s1.z, s1.w)));
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) out[j] = n[j];
    }
  } else {
    auto one = [&](int d, float v) {
      if (d >= 2 * p.half) return v;
      const bool low = d < p.half;
      const int i = low ? d : d - p.half;
      const float m = other(low ? d + p.half : i);
      return v * c[i] + m * (low ? -s[i] : s[i]);
    };
#pragma unroll
    for (int j = 0; j < 4; ++j) out[j] = make_float2(one(ch + 2 * j, n[j].x), one(ch + 2 * j + 1, n[j].y));
  }
}

// lane of the other channels of a pair, for kLanes (a lane beyond the rotated part: itself)
__device__ __forceinline__ int rot_partner(const RotaryParams& p, int ch, int lane) {
  return ch < p.half ? lane + (p.half >> 3) : ch < 2 * p.half ? lane - (p.half >> 3) : lane;
}
// the packed values of another lane, `flip` (both sign bits, or none) turned
__device__ __forceinline__ uint4 rot_shuffle(const uint4& v, int from, uint32_t flip) {
  return make_uint4(__shfl_sync(0xffffffffu, v.x, from) ^ flip, __shfl_sync(0xffffffffu, v.y, from) ^ flip,
                    __shfl_sync(0xffffffffu, v.z, from) ^ flip, __shfl_sync(0xffffffffu, v.w, from) ^ flip);
}

// grid: (tiles of a sequence's tokens, blocks of heads_here heads, every which sequence); blockDim.x = heads_here * D / 8 up to a
// whole warp.  Positions that all sequences share: their angles are formed once for all sequences of a CTA.
template <bool kBf16, int kMode, bool kNorm>
__global__ void __launch_bounds__(kRotThreads) fox_rotary_fwd_kernel(const RotaryParams p) {
  extern __shared__ __align__(16) float rot_smem[];
  const int lanes = p.D >> 3, pairs = p.D >> 1;
  double* s_pos = reinterpret_cast<double*>(rot_smem);
  float *s_cos = rot_smem + 2 * kRotTile, *s_sin = s_cos + p.tile * pairs;
  const int sub = threadIdx.x % lanes, slot = threadIdx.x / lanes, head = blockIdx.y * p.heads_here + slot;
  const bool active = slot < p.heads_here && head < p.heads;
  const bool is_k = active && head >= p.H;
  const RotaryTensor& x = p.t[is_k];
  const int h = active ? (is_k ? head - p.H : head) : 0, ch = sub * 8;
  const int lane = threadIdx.x & 31, from = rot_partner(p, ch, lane);
  const uint32_t flip = ch < p.half ? 0x80008000u : 0u;
  const int t0 = blockIdx.x * p.tile, n = min(p.tile, p.T - t0);
  wait_for_kernel_in_front();
  float2 w[4], wp[4];
  const float inv_d = 1.f / static_cast<float>(p.D);
  for (int b = blockIdx.z; b < p.B; b += gridDim.z) {
    const uint16_t* row = x.x + b * x.x_sb + h * x.x_sh + t0 * x.x_st + ch;
    uint16_t* to = x.y + b * x.y_sb + h * x.y_sh + t0 * x.y_st + ch;
    auto load = [&](int u) { return active && u < n ? ld_v4_here(reinterpret_cast<const uint4*>(row + u * x.x_st)) : make_uint4(0, 0, 0, 0); };
    uint4 ahead[kRotAhead];
#pragma unroll
    for (int u = 0; u < kRotAhead; ++u) ahead[u] = load(u);
    if (b == static_cast<int>(blockIdx.z) || p.pos_sb) {
      if constexpr (kNorm) {
        if (b == static_cast<int>(blockIdx.z)) {
          rot_weights(x.w, x.w_dtype, h * x.w_sh + ch, w);
          if constexpr (kMode == kLanes) rot_weights(x.w, x.w_dtype, h * x.w_sh + ch + (from - lane) * 8, wp);
        }
      }
      if (b != static_cast<int>(blockIdx.z)) __syncthreads();   // (the last sequence's angles have been used)
      rot_angles(p, b, t0, n, s_pos, s_cos, s_sin);
    }
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
        float2 v[4], pair[4], out[4];
        float r = 1.f;
        rot_unpack<kBf16>(raw[u], v);
        if constexpr (kMode == kLanes) rot_unpack<kBf16>(rot_shuffle(raw[u], from, flip), pair);
        if constexpr (kNorm) {
          float2 sq = rot_mul(v[0], v[0]);
#pragma unroll
          for (int j = 1; j < 4; ++j) sq = rot_fma(v[j], v[j], sq);
          float ss = sq.x + sq.y;
          for (int o = lanes >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
          r = rsqrtf(fmaf(ss, inv_d, p.eps));
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            v[j] = rot_mul(v[j], w[j]);
            if constexpr (kMode == kLanes) pair[j] = rot_mul(pair[j], wp[j]);
          }
        }
        auto other = [&](int d) {
          const float m = active ? rot_weight(row + (u0 + u) * x.x_st - ch, kBf16 ? FOX_DTYPE_BF16 : FOX_DTYPE_FP16, d) : 0.f;
          return kNorm ? m * rot_weight(x.w, x.w_dtype, h * x.w_sh + d) : m;
        };
        rot_turn<kMode>(p, ch, s_cos + (u0 + u) * pairs, s_sin + (u0 + u) * pairs, v, pair, other, out);
        if constexpr (kNorm) {   // (1 / rms last: it is the same for both channels of a pair)
#pragma unroll
          for (int j = 0; j < 4; ++j) out[j] = rot_mul(out[j], rot_both(r));
        }
        if (active) *reinterpret_cast<uint4*>(to + (u0 + u) * x.y_st) = rot_pack<kBf16>(out);
      }
    }
  }
}

// The norm's backward with the rotation in front.  A CTA takes every grid.x-th tile of every grid.z-th sequence, so that its share
// of dw stays in registers; fox_rotary_dw_kernel adds the shares in a fixed order.
template <bool kBf16, int kMode>
__global__ void __launch_bounds__(kRotThreads) fox_rotary_bwd_kernel(const RotaryParams p) {
  constexpr int kAhead = 2;
  extern __shared__ __align__(16) float rot_smem[];
  const int lanes = p.D >> 3, pairs = p.D >> 1;
  double* s_pos = reinterpret_cast<double*>(rot_smem);
  float *s_cos = rot_smem + 2 * kRotTile, *s_sin = s_cos + p.tile * pairs;
  const int sub = threadIdx.x % lanes, slot = threadIdx.x / lanes, head = blockIdx.y * p.heads_here + slot;
  const bool active = slot < p.heads_here && head < p.heads;
  const bool is_k = active && head >= p.H;
  const RotaryTensor& x = p.t[is_k];
  const int h = active ? (is_k ? head - p.H : head) : 0, ch = sub * 8;
  const int lane = threadIdx.x & 31, from = rot_partner(p, ch, lane);
  const uint32_t flip = ch < p.half ? 0x80008000u : 0u;
  wait_for_kernel_in_front();
  float2 w[4], dw[4];
  rot_weights(x.w, x.w_dtype, h * x.w_sh + ch, w);
#pragma unroll
  for (int j = 0; j < 4; ++j) dw[j] = rot_both(0.f);
  const float inv_d = 1.f / static_cast<float>(p.D);
  for (int64_t t64 = static_cast<int64_t>(blockIdx.x) * p.tile; t64 < p.T; t64 += static_cast<int64_t>(gridDim.x) * p.tile) {
    const int t0 = static_cast<int>(t64), n = min(p.tile, p.T - t0);
    for (int b = blockIdx.z; b < p.B; b += gridDim.z) {
      const uint16_t *row = x.x + b * x.x_sb + h * x.x_sh + t0 * x.x_st + ch, *row_g = x.dy + b * x.dy_sb + h * x.dy_sh + t0 * x.dy_st + ch;
      uint16_t* to = x.y + b * x.y_sb + h * x.y_sh + t0 * x.y_st + ch;
      uint4 ahead_x[kAhead], ahead_g[kAhead];
      auto load = [&](int u, uint4& vx, uint4& vg) {
        vx = vg = make_uint4(0, 0, 0, 0);
        if (active && u < n) {
          vx = ld_v4_here(reinterpret_cast<const uint4*>(row + u * x.x_st));
          vg = ld_v4_here(reinterpret_cast<const uint4*>(row_g + u * x.dy_st));
        }
      };
#pragma unroll
      for (int u = 0; u < kAhead; ++u) load(u, ahead_x[u], ahead_g[u]);
      if (b == static_cast<int>(blockIdx.z) || p.pos_sb) {
        __syncthreads();
        rot_angles(p, b, t0, n, s_pos, s_cos, s_sin);
      }
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
          float2 v[4], g[4], pair[4], dn[4], gw[4], out[4];
          rot_unpack<kBf16>(raw_x[u], v);
          rot_unpack<kBf16>(raw_g[u], g);
          if constexpr (kMode == kLanes) rot_unpack<kBf16>(rot_shuffle(raw_g[u], from, flip), pair);
          auto other = [&](int d) {
            return active ? rot_weight(row_g + (u0 + u) * x.dy_st - ch, kBf16 ? FOX_DTYPE_BF16 : FOX_DTYPE_FP16, d) : 0.f;
          };
          rot_turn<kMode>(p, ch, s_cos + (u0 + u) * pairs, s_sin + (u0 + u) * pairs, g, pair, other, dn);
          float2 sq = rot_both(0.f), dot2 = rot_both(0.f);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            gw[j] = rot_mul(dn[j], w[j]);
            sq = rot_fma(v[j], v[j], sq);
            dot2 = rot_fma(gw[j], v[j], dot2);
          }
          float ss = sq.x + sq.y, dot = dot2.x + dot2.y;
          for (int o = lanes >> 1; o > 0; o >>= 1) {
            ss += __shfl_xor_sync(0xffffffffu, ss, o);
            dot += __shfl_xor_sync(0xffffffffu, dot, o);
          }
          const float r = rsqrtf(fmaf(ss, inv_d, p.eps));
          const float2 r2 = rot_both(r), back = rot_both(-dot * r * inv_d * r);   // dx = r gw - xhat mean r
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 xhat = rot_mul(v[j], r2);
            dw[j] = rot_fma(dn[j], xhat, dw[j]);
            out[j] = rot_fma(xhat, back, rot_mul(gw[j], r2));
          }
          if (active) *reinterpret_cast<uint4*>(to + (u0 + u) * x.y_st) = rot_pack<kBf16>(out);
        }
      }
    }
  }
  if (active) {
    const int64_t share = static_cast<int64_t>(blockIdx.z) * gridDim.x + blockIdx.x;
    float* to = p.dw_partial + (share * p.heads + head) * p.D + ch;
    reinterpret_cast<float4*>(to)[0] = make_float4(dw[0].x, dw[0].y, dw[1].x, dw[1].y);
    reinterpret_cast<float4*>(to)[1] = make_float4(dw[2].x, dw[2].y, dw[3].x, dw[3].y);
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
  int blocks, heads_here, threads, tile, tiles, slices;   // slices: of the sequences
};
// Heads of a token over as few CTAs of up to 256 threads as hold them, evenly.  Tiles of 16 tokens, and smaller ones where those of
// all sequences do not fill the GPU; as few slices of the sequences as do, so that angles are formed once for several.
static RotaryGrid rotary_grid(int64_t heads, int64_t D, int64_t B, int64_t T) {
  const int64_t most = kRotThreads / (D / 8), blocks = (heads + most - 1) / most, here = (heads + blocks - 1) / blocks;
  const int64_t fit = (T * B * blocks + kRotFill - 1) / kRotFill, tile = fit < 1 ? 1 : fit < kRotTile ? fit : kRotTile;
  const int64_t tiles = (T + tile - 1) / tile, want = (2 * kRotFill + tiles * blocks - 1) / (tiles * blocks);
  const int64_t slices = want < B ? want : B;
  return {static_cast<int>(blocks), static_cast<int>(here), static_cast<int>((here * (D / 8) + 31) / 32 * 32), static_cast<int>(tile),
          static_cast<int>(tiles), static_cast<int>(slices < 65535 ? slices : 65535)};
}
// A backward's CTAs to a block of heads: (tiles, slices), with some kRotShares CTAs in all.
static RotaryGrid rotary_grid_bwd(int64_t heads, int64_t D, int64_t B, int64_t T) {
  RotaryGrid g = rotary_grid(heads, D, B, T);
  const int most = (kRotShares + g.blocks - 1) / g.blocks;
  if (g.tiles > most) g.tiles = most;
  const int want = most / g.tiles;
  g.slices = static_cast<int>(want < B ? want : B);
  return g;
}

enum RotaryKind { kTurn, kNormTurn, kNormBack };
template <bool kBf16, int kMode>
static int rotary_launch_at(RotaryKind kind, dim3 grid, unsigned threads, size_t smem, cudaStream_t st, const RotaryParams& p) {
  if (kind == kTurn) return launch_behind(fox_rotary_fwd_kernel<kBf16, kMode, false>, grid, threads, smem, st, p);
  if (kind == kNormTurn) return launch_behind(fox_rotary_fwd_kernel<kBf16, kMode, true>, grid, threads, smem, st, p);
  return launch_behind(fox_rotary_bwd_kernel<kBf16, kMode>, grid, threads, smem, st, p);
}
static int rotary_launch(RotaryKind kind, int dtype, int64_t half, int interleaved, const RotaryGrid& g, cudaStream_t st, RotaryParams p) {
  p.heads_here = g.heads_here;
  p.tile = g.tile;
  const dim3 grid(g.tiles, g.blocks, g.slices);
  const size_t smem = kRotTile * sizeof(double) + static_cast<size_t>(p.tile) * p.D * sizeof(float);
  const bool bf = dtype == FOX_DTYPE_BF16;
  if (interleaved) return bf ? rotary_launch_at<true, kNext>(kind, grid, g.threads, smem, st, p) : rotary_launch_at<false, kNext>(kind, grid, g.threads, smem, st, p);
  if (half % 8) return bf ? rotary_launch_at<true, kAny>(kind, grid, g.threads, smem, st, p) : rotary_launch_at<false, kAny>(kind, grid, g.threads, smem, st, p);
  return bf ? rotary_launch_at<true, kLanes>(kind, grid, g.threads, smem, st, p) : rotary_launch_at<false, kLanes>(kind, grid, g.threads, smem, st, p);
}

static bool rotary_bad_rows(const fox_tensor4* t) {
  return reinterpret_cast<uintptr_t>(t->ptr) % 16 || t->sb % 8 || t->sh % 8 || t->st % 8;
}
static bool rotary_bad_weight(int dtype) { return dtype != FOX_DTYPE_FP16 && dtype != FOX_DTYPE_BF16 && dtype != FOX_DTYPE_FP32; }
static bool rotary_bad_weights(const void* w, int64_t sh, int64_t D) { return reinterpret_cast<uintptr_t>(w) % 16 || (sh != 0 && sh != D); }

static int rotary_check(int dtype, int64_t B, int64_t T, int64_t H, int64_t Hk, int64_t D, const float* inv_freq, int64_t half) {
  if (B <= 0 || T <= 0 || H <= 0 || Hk < 0 || half <= 0 || !inv_freq) return FOX_ERR_BAD_ARG;
  if (dtype != FOX_DTYPE_BF16 && dtype != FOX_DTYPE_FP16) return FOX_ERR_BAD_ARG;
  if (D != 16 && D != 32 && D != 64 && D != 128) return FOX_ERR_HEAD_DIM;
  if (2 * half > D) return FOX_ERR_BAD_ARG;
  if (H > 65535 || Hk > 65535 || T > kRotTokens || B > kRotTokens / T) return FOX_ERR_TOO_LARGE;
  return FOX_OK;
}
// One token of each of many sequences is one sequence of many tokens.
static bool rotary_fold(int64_t& B, int64_t& T) {
  if (T > 1 || B == 1) return false;
  T = B;
  B = 1;
  return true;
}
static fox_tensor4 rotary_view(const fox_tensor4* t, bool folded) { return folded ? fox_tensor4{t->ptr, 0, t->sh, t->sb} : *t; }
static RotaryParams rotary_params(int64_t B, int64_t T, int64_t H, int64_t Hk, int64_t D, const float* inv_freq, int64_t half,
                                  float scale, float eps, const void* positions, int pos_64, int64_t pos_sb, int64_t pos_st,
                                  int64_t first, bool folded) {
  RotaryParams p{};
  p.inv_freq = inv_freq;
  p.positions = positions;
  p.pos_sb = folded || B == 1 ? 0 : positions ? pos_sb : 0;
  p.pos_st = folded ? pos_sb : pos_st;
  p.first = first; p.step = folded ? 0 : 1; p.pos_64 = pos_64;
  p.scale = scale; p.sign = 1.f; p.eps = eps;
  p.by_half = divisor(half);
  p.half = (int)half; p.D = (int)D; p.B = (int)B; p.T = (int)T;
  p.H = (int)H; p.heads = (int)(H + Hk);
  return p;
}
static void rotary_in(RotaryTensor& t, const fox_tensor4& x) {
  t.x = (const uint16_t*)x.ptr; t.x_sb = x.sb; t.x_sh = x.sh; t.x_st = x.st;
}
static void rotary_out(RotaryTensor& t, const fox_tensor4& y) {
  t.y = (uint16_t*)y.ptr; t.y_sb = y.sb; t.y_sh = y.sh; t.y_st = y.st;
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
  const bool folded = rotary_fold(B, T);
  RotaryParams p = rotary_params(B, T, H, 0, D, inv_freq, half, scale, 0.f, positions, pos_64, pos_sb, pos_st, first, folded);
  p.sign = inverse ? -1.f : 1.f;
  rotary_in(p.t[0], rotary_view(x, folded));
  rotary_out(p.t[0], rotary_view(y, folded));
  return rotary_launch(kTurn, dtype, half, interleaved, rotary_grid(H, D, B, T), (cudaStream_t)stream, p);
}

extern "C" int fox_qk_norm_rotary_fwd(int device, void* stream, int dtype, int64_t B, int64_t T, int64_t H, int64_t Hk, int64_t D,
                                      const fox_tensor4* q, const fox_tensor4* k, const void* wq, int wq_dtype, int64_t wq_sh,
                                      const void* wk, int wk_dtype, int64_t wk_sh, float eps, const float* inv_freq, int64_t half,
                                      int interleaved, float scale, const void* positions, int pos_64, int64_t pos_sb,
                                      int64_t pos_st, int64_t first, const fox_tensor4* q_out, const fox_tensor4* k_out) {
  if (!q || !k || !q_out || !k_out || !q->ptr || !k->ptr || !q_out->ptr || !k_out->ptr || !wq || !wk || Hk <= 0) return FOX_ERR_BAD_ARG;
  if (int rc = rotary_check(dtype, B, T, H, Hk, D, inv_freq, half)) return rc;
  if (rotary_bad_weight(wq_dtype) || rotary_bad_weight(wk_dtype)) return FOX_ERR_BAD_ARG;
  if (rotary_bad_weights(wq, wq_sh, D) || rotary_bad_weights(wk, wk_sh, D)) return FOX_ERR_ALIGNMENT;
  if (rotary_bad_rows(q) || rotary_bad_rows(k) || rotary_bad_rows(q_out) || rotary_bad_rows(k_out)) return FOX_ERR_ALIGNMENT;
  if (cudaSetDevice(device) != cudaSuccess) return FOX_ERR_DEVICE;
  const bool folded = rotary_fold(B, T);
  RotaryParams p = rotary_params(B, T, H, Hk, D, inv_freq, half, scale, eps, positions, pos_64, pos_sb, pos_st, first, folded);
  rotary_in(p.t[0], rotary_view(q, folded)); rotary_in(p.t[1], rotary_view(k, folded));
  rotary_out(p.t[0], rotary_view(q_out, folded)); rotary_out(p.t[1], rotary_view(k_out, folded));
  p.t[0].w = wq; p.t[0].w_dtype = wq_dtype; p.t[0].w_sh = wq_sh;
  p.t[1].w = wk; p.t[1].w_dtype = wk_dtype; p.t[1].w_sh = wk_sh;
  return rotary_launch(kNormTurn, dtype, half, interleaved, rotary_grid(H + Hk, D, B, T), (cudaStream_t)stream, p);
}

extern "C" int64_t fox_qk_norm_rotary_partials(int64_t B, int64_t T, int64_t H, int64_t Hk, int64_t D) {
  if (B <= 0 || T <= 0 || H <= 0 || Hk <= 0 || (D != 16 && D != 32 && D != 64 && D != 128)) return 1;
  rotary_fold(B, T);
  const RotaryGrid g = rotary_grid_bwd(H + Hk, D, B, T);
  return static_cast<int64_t>(g.tiles) * g.slices;
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
  if (rotary_bad_weights(wq, wq_sh, D) || rotary_bad_weights(wk, wk_sh, D)) return FOX_ERR_ALIGNMENT;
  for (const fox_tensor4* t : {q, k, dq_out, dk_out, dq, dk})
    if (rotary_bad_rows(t)) return FOX_ERR_ALIGNMENT;
  if (reinterpret_cast<uintptr_t>(dw_partial) % 16) return FOX_ERR_ALIGNMENT;
  if (cudaSetDevice(device) != cudaSuccess) return FOX_ERR_DEVICE;
  const bool folded = rotary_fold(B, T);
  RotaryParams p = rotary_params(B, T, H, Hk, D, inv_freq, half, scale, eps, positions, pos_64, pos_sb, pos_st, first, folded);
  p.sign = -1.f;
  const fox_tensor4 *xs[2] = {q, k}, *gs[2] = {dq_out, dk_out}, *ds[2] = {dq, dk};
  for (int i = 0; i < 2; ++i) {
    rotary_in(p.t[i], rotary_view(xs[i], folded));
    rotary_out(p.t[i], rotary_view(ds[i], folded));
    const fox_tensor4 g = rotary_view(gs[i], folded);
    p.t[i].dy = (const uint16_t*)g.ptr;
    p.t[i].dy_sb = g.sb; p.t[i].dy_sh = g.sh; p.t[i].dy_st = g.st;
  }
  p.t[0].w = wq; p.t[0].w_dtype = wq_dtype; p.t[0].w_sh = wq_sh;
  p.t[1].w = wk; p.t[1].w_dtype = wk_dtype; p.t[1].w_sh = wk_sh;
  p.dw_partial = dw_partial;
  const RotaryGrid g = rotary_grid_bwd(H + Hk, D, B, T);
  const int64_t n = static_cast<int64_t>(g.tiles) * g.slices;
  cudaStream_t st = (cudaStream_t)stream;
  if (int rc = rotary_launch(kNormBack, dtype, half, interleaved, g, st, p)) return rc;
  const RotaryDwParams d{dw_partial, {dwq, dwk}, {wq_dtype, wk_dtype}, {wq_sh == 0, wk_sh == 0}, {(int)H, (int)Hk}, (int)n, (int)D};
  const int64_t cols = (wq_sh ? H * D : D) + (wk_sh ? Hk * D : D);
  return launch_behind(fox_rotary_dw_kernel, dim3((unsigned)(cols / 16)), 256, 0, st, d);
}
