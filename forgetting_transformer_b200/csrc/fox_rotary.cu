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
// it) and rotates them in another (rotary.py:22-153, from tables of cosines and sines); here the
// normed values are never rounded or written in between, and one launch takes both tensors.
//
// There is no table of all positions: a CTA forms the angles of its own tile of tokens, once for all of its heads.  The
// product of position and frequency and its reduction by turns are in 64 bits (at position 10^6 a 32-bit product is off by
// 0.03 rad), sine and cosine of what is left, at most pi, by the fast functions in 32.
//
// Thread (h, sub) owns 8 channels of head h (queries' heads, then keys') for every token that its CTA visits; the row's sum of
// squares is a shuffle over D/8 neighbouring lanes, weights and dw stay in registers.  kMode: which 8 channels, two runs of 4:
//   kHalves  halves that are a multiple of 4: 4 sub .. of the first half and the same of the second, so that a pair is one
//            thread's and needs a cosine and a sine once; behind the rotated part 8 channels as they stand.  (With 8 neighbouring
//            channels a thread and the other ones by shuffle, the kernels were bound by shared memory and shuffles: 66 us
//            for what takes 48.)
//   kNext    neighbouring channels paired: 8 neighbouring channels
//   kAny     halves that are no multiple of 4: 8 neighbouring channels, the others of the pairs by way of shared memory, where the
//            angles stand once for each channel (read from L1 again one by one: 214 us for what takes 83 so)
#include "fox_common.cuh"
#include "fox_host.h"

namespace fox {

enum RotaryMode { kHalves, kNext, kAny };

constexpr int kRotThreads = 256;
constexpr int kRotTile = 32;      // tokens whose angles are in shared memory at a time
constexpr int kRotAhead = 4;      // tokens whose rows a thread has asked for
constexpr int64_t kRotTokens = (int64_t{1} << 31) - 65536;   // counted with 32 bits, a tile's more among them
__host__ __device__ constexpr int rot_fwd_per_sm(int mode) { return mode == kAny ? 3 : 4; }   // CTAs, by registers
constexpr int kRotBwdPerSm = 2;

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
  int fold;                       // dw: both weights are one for all heads
  int pos_64, half, D, T, tokens, H, heads, heads_here, per_cta, tile;   // per_cta: tokens
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
// four weights from element i on, a multiple of 4 (16-byte aligned in fp32, 8-byte in 16 bits)
__device__ __forceinline__ void rot_weights(const void* w, int dtype, int64_t i, float2* f) {
  if (dtype == FOX_DTYPE_FP32) {
    const float4 a = *reinterpret_cast<const float4*>(static_cast<const float*>(w) + i);
    f[0] = make_float2(a.x, a.y);
    f[1] = make_float2(a.z, a.w);
  } else {
    const uint2 v = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(w) + i);
    f[0] = dtype == FOX_DTYPE_BF16 ? unpack2<true>(v.x) : unpack2<false>(v.x);
    f[1] = dtype == FOX_DTYPE_BF16 ? unpack2<true>(v.y) : unpack2<false>(v.y);
  }
}
__device__ __forceinline__ uint2 ld_v2_here(const uint16_t* p) {   // (as ld_v4_here)
  uint2 v;
  asm volatile("ld.global.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p) : "memory");
  return v;
}

// Where a thread's two runs of 4 channels begin; `turned`: of a rotated part (kHalves).
struct RotaryRuns {
  int a, b;
  bool turned;
};
template <int kMode>
__device__ __forceinline__ RotaryRuns rot_runs(const RotaryParams& p, int sub) {
  const int quarter = p.half >> 2;   // threads with pairs
  if (kMode != kHalves || sub >= quarter) {
    const int ch = kMode != kHalves ? sub * 8 : 2 * p.half + (sub - quarter) * 8;
    return {ch, ch + 4, kMode != kHalves};
  }
  return {4 * sub, p.half + 4 * sub, true};
}
template <int kMode>
__device__ __forceinline__ uint4 rot_load(const uint16_t* row, const RotaryRuns& c) {   // row: of 8 (kHalves: 4) aligned channels
  if constexpr (kMode == kHalves) {
    const uint2 a = ld_v2_here(row + c.a), b = ld_v2_here(row + c.b);
    return make_uint4(a.x, a.y, b.x, b.y);
  } else {
    return ld_v4_here(reinterpret_cast<const uint4*>(row + c.a));
  }
}
template <int kMode>
__device__ __forceinline__ void rot_store(uint16_t* row, const RotaryRuns& c, const uint4& v) {
  if constexpr (kMode == kHalves) {
    *reinterpret_cast<uint2*>(row + c.a) = make_uint2(v.x, v.y);
    *reinterpret_cast<uint2*>(row + c.b) = make_uint2(v.z, v.w);
  } else {
    *reinterpret_cast<uint4*>(row + c.a) = v;
  }
}
__device__ __forceinline__ float2 rot_mul(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float2 rot_fma(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }
__device__ __forceinline__ float2 rot_both(float a) { return make_float2(a, a); }

// cosines and sines of tokens t0 .. t0 + n of sequence b, (tile, D / 2) each, kAny: (tile, D), a sine with the sign of its channel;
// s_pos: (tile).  A barrier is inside and one behind.
template <int kMode>
__device__ __forceinline__ void rot_angles(const RotaryParams& p, int b, int t0, int n, double* s_pos, float* s_cos, float* s_sin) {
  const int ld = kMode == kAny ? p.D : p.D >> 1;
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
  // a thread stays with one frequency (with fewer threads than frequencies, a few)
  const int across = min(p.half, static_cast<int>(blockDim.x)), groups = div_by(p.by_half, blockDim.x);
  const int u0 = groups ? div_by(p.by_half, threadIdx.x) : 0, f0 = threadIdx.x - u0 * across;
  for (int f = u0 < max(groups, 1) ? f0 : p.half; f < p.half; f += across) {
    const double freq = p.inv_freq[f];
    for (int u = u0; u < n; u += max(groups, 1)) {
      const double a = s_pos[u] * freq;
      const double turns = a * 0.15915494309189535 + 6755399441055744.0 - 6755399441055744.0;   // rounded to whole ones
      // less whole turns, 2 pi in two parts
      const float r = static_cast<float>(fma(turns, -2.4492935982947064e-16, fma(turns, -6.283185307179586, a)));
      // (the fast functions: off by 2^-21 at most from minus pi to pi, far below half a step of 16 bits)
      const float cs = __cosf(r) * p.scale, sn = __sinf(r) * (p.scale * p.sign);
      s_cos[u * ld + f] = cs;
      s_sin[u * ld + f] = kMode == kAny ? -sn : sn;
      if constexpr (kMode == kAny) {
        s_cos[u * ld + p.half + f] = cs;
        s_sin[u * ld + p.half + f] = sn;
      }
    }
  }
  __syncthreads();
}

// The rotation of a thread's 8 channels n; pair: the other channels of their pairs (kAny).
template <int kMode>
__device__ __forceinline__ void rot_turn(const RotaryParams& p, const RotaryRuns& at, const float* c, const float* s, const float2* n,
                                         const float* pair, float2* out) {
  if constexpr (kMode == kHalves) {
    if (at.turned) {
      const float4 cv = *reinterpret_cast<const float4*>(c + at.a), sv = *reinterpret_cast<const float4*>(s + at.a);
      const float2 c0 = make_float2(cv.x, cv.y), c1 = make_float2(cv.z, cv.w), s0 = make_float2(sv.x, sv.y), s1 = make_float2(sv.z, sv.w);
      const float2 m0 = make_float2(-s0.x, -s0.y), m1 = make_float2(-s1.x, -s1.y);
      out[0] = rot_fma(n[0], c0, rot_mul(n[2], m0));
      out[1] = rot_fma(n[1], c1, rot_mul(n[3], m1));
      out[2] = rot_fma(n[2], c0, rot_mul(n[0], s0));
      out[3] = rot_fma(n[3], c1, rot_mul(n[1], s1));
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) out[j] = n[j];
    }
  } else if constexpr (kMode == kNext) {
    if (at.a + 8 <= 2 * p.half) {
      const float4 cs = *reinterpret_cast<const float4*>(c + (at.a >> 1)), sn = *reinterpret_cast<const float4*>(s + (at.a >> 1));
      const float cv[4] = {cs.x, cs.y, cs.z, cs.w}, sv[4] = {sn.x, sn.y, sn.z, sn.w};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        out[j] = rot_fma(n[j], rot_both(cv[j]), rot_mul(make_float2(n[j].y, n[j].x), make_float2(-sv[j], sv[j])));
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = (at.a >> 1) + j;
        const float cv = i < p.half ? c[i] : 1.f, sv = i < p.half ? s[i] : 0.f;
        out[j] = make_float2(n[j].x * cv - n[j].y * sv, n[j].y * cv + n[j].x * sv);
      }
    }
  } else {
    float cv[8], sv[8];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      *reinterpret_cast<float4*>(cv + 4 * i) = *reinterpret_cast<const float4*>(c + at.a + 4 * i);
      *reinterpret_cast<float4*>(sv + 4 * i) = *reinterpret_cast<const float4*>(s + at.a + 4 * i);
    }
    auto one = [&](int j, float v) { return at.a + j < 2 * p.half ? v * cv[j] + pair[j] * sv[j] : v; };
#pragma unroll
    for (int j = 0; j < 4; ++j) out[j] = make_float2(one(2 * j, n[j].x), one(2 * j + 1, n[j].y));
  }
}

// kAny: a warp's packed values go to `slot` (512 bytes), and each thread takes the other channels of its pairs from there.
__device__ __forceinline__ int rot_other(const RotaryParams& p, int d) {
  return d < p.half ? d + p.half : d < 2 * p.half ? d - p.half : d;
}
template <bool kBf16>
__device__ __forceinline__ void rot_exchange(const RotaryParams& p, uint16_t* slot, int lanes, int ch, const uint4& v, float* pair) {
  const int lane = threadIdx.x & 31;
  *reinterpret_cast<uint4*>(slot + lane * 8) = v;
  __syncwarp();
  const uint16_t* row = slot + (lane & ~(lanes - 1)) * 8;
  if (p.half & 1) {
#pragma unroll
    for (int j = 0; j < 8; ++j) pair[j] = unpack2<kBf16>(row[rot_other(p, ch + j)]).x;
  } else {   // (two neighbours' others are neighbours: norms of 16384 tokens x 32 heads of 128, half 22, 70 us, half 21 84)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = unpack2<kBf16>(*reinterpret_cast<const uint32_t*>(row + rot_other(p, ch + 2 * j)));
      pair[2 * j] = f.x;
      pair[2 * j + 1] = f.y;
    }
  }
}

// grid: (ranges of per_cta tokens, blocks of heads_here heads); blockDim.x = heads_here * D / 8 up to a whole warp.  Equal
// ranges (rotary_grid), each in tiles of one sequence's tokens.
template <bool kBf16, int kMode, bool kNorm, int kD>
__global__ void __launch_bounds__(kRotThreads, rot_fwd_per_sm(kMode)) fox_rotary_fwd_kernel(const RotaryParams p) {
  constexpr int kAhead = kMode == kAny ? 2 : kRotAhead;
  extern __shared__ __align__(16) float rot_smem[];
  const int D = kD ? kD : p.D, lanes = D >> 3, pairs = kMode == kAny ? D : D >> 1;
  double* s_pos = reinterpret_cast<double*>(rot_smem);
  float *s_cos = rot_smem + 2 * kRotTile, *s_sin = s_cos + p.tile * pairs;
  uint16_t* s_rows = reinterpret_cast<uint16_t*>(s_sin + p.tile * pairs) + (threadIdx.x >> 5) * (kAhead * 256);   // kAny: of this warp
  const int sub = threadIdx.x % lanes, slot = threadIdx.x / lanes, head = blockIdx.y * p.heads_here + slot;
  const bool active = slot < p.heads_here && head < p.heads;
  const bool is_k = active && head >= p.H;
  const RotaryTensor& x = p.t[is_k];
  const int h = active ? (is_k ? head - p.H : head) : 0;
  const RotaryRuns ch = rot_runs<kMode>(p, sub);
  wait_for_kernel_in_front();
  const int begin = static_cast<int>(blockIdx.x) * p.per_cta, end = begin + min(p.per_cta, p.tokens - begin);
  float2 w[4];
  float wp[8];   // kAny: of the other channels
  const int64_t x_st = x.x_st, y_st = x.y_st;
  const float inv_d = 1.f / static_cast<float>(D);
  for (int at = begin, n; at < end; at += n) {
    const int b = at / p.T, t0 = at - b * p.T;
    n = min(min(p.tile, end - at), p.T - t0);
    const uint16_t* row = x.x + b * x.x_sb + h * x.x_sh + t0 * x.x_st;
    uint16_t* to = x.y + b * x.y_sb + h * x.y_sh + t0 * x.y_st;
    int to_ask = active ? n : 0;
    uint4 ahead[kAhead];
    auto ask = [&] {
#pragma unroll
      for (int u = 0; u < kAhead; ++u) ahead[u] = u < to_ask ? rot_load<kMode>(row + u * x_st, ch) : make_uint4(0, 0, 0, 0);
      row += kAhead * x_st;
      to_ask -= kAhead;
    };
    ask();
    if constexpr (kNorm) {
      if (at == begin) {
        rot_weights(x.w, x.w_dtype, h * x.w_sh + ch.a, w);
        rot_weights(x.w, x.w_dtype, h * x.w_sh + ch.b, w + 2);
        if constexpr (kMode == kAny)
#pragma unroll
          for (int j = 0; j < 8; ++j) wp[j] = rot_weight(x.w, x.w_dtype, h * x.w_sh + rot_other(p, ch.a + j));
      }
    }
    if (at != begin) __syncthreads();   // (the last tile's angles have been used)
    rot_angles<kMode>(p, b, t0, n, s_pos, s_cos, s_sin);
    const float *c = s_cos, *s = s_sin;
    for (int left = n; left > 0; left -= kAhead) {
      uint4 raw[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) raw[u] = ahead[u];
      ask();
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if (u >= left) break;   // (the same for all threads)
        float2 v[4], out[4];
        float r = 1.f, pair[8];
        rot_unpack<kBf16>(raw[u], v);
        if constexpr (kMode == kAny) {
          rot_exchange<kBf16>(p, s_rows + u * 256, lanes, ch.a, raw[u], pair);
          if constexpr (kNorm) {
#pragma unroll
            for (int j = 0; j < 8; ++j) pair[j] *= wp[j];
          }
        }
        if constexpr (kNorm) {
          float2 sq = rot_mul(v[0], v[0]);
#pragma unroll
          for (int j = 1; j < 4; ++j) sq = rot_fma(v[j], v[j], sq);
          float ss = sq.x + sq.y;
#pragma unroll
          for (int o = lanes >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
          r = rsqrtf(fmaf(ss, inv_d, p.eps));
#pragma unroll
          for (int j = 0; j < 4; ++j) v[j] = rot_mul(v[j], w[j]);
        }
        rot_turn<kMode>(p, ch, c + u * pairs, s + u * pairs, v, pair, out);
        if constexpr (kNorm) {   // (1 / rms last: it is the same for both channels of a pair)
#pragma unroll
          for (int j = 0; j < 4; ++j) out[j] = rot_mul(out[j], rot_both(r));
        }
        if (active) rot_store<kMode>(to + u * y_st, ch, rot_pack<kBf16>(out));
      }
      if constexpr (kMode == kAny) __syncwarp();   // (the rows have been read before the next ones are written)
      to += kAhead * y_st;
      c += kAhead * pairs;
      s += kAhead * pairs;
    }
  }
}

// The norm's backward with the rotation in front.  A CTA's share of dw stays in registers; fox_rotary_dw_kernel adds the
// shares in a fixed order.
template <bool kBf16, int kMode, int kD>
__global__ void __launch_bounds__(kRotThreads, kRotBwdPerSm) fox_rotary_bwd_kernel(const RotaryParams p) {
  constexpr int kAhead = kMode == kAny ? 2 : kRotAhead;
  extern __shared__ __align__(16) float rot_smem[];
  const int D = kD ? kD : p.D, lanes = D >> 3, pairs = kMode == kAny ? D : D >> 1;
  double* s_pos = reinterpret_cast<double*>(rot_smem);
  float *s_cos = rot_smem + 2 * kRotTile, *s_sin = s_cos + p.tile * pairs;
  uint16_t* s_rows = reinterpret_cast<uint16_t*>(s_sin + p.tile * pairs) + (threadIdx.x >> 5) * (kAhead * 256);   // kAny: of this warp
  const int sub = threadIdx.x % lanes, slot = threadIdx.x / lanes, head = blockIdx.y * p.heads_here + slot;
  const bool active = slot < p.heads_here && head < p.heads;
  const bool is_k = active && head >= p.H;
  const RotaryTensor& x = p.t[is_k];
  const int h = active ? (is_k ? head - p.H : head) : 0;
  const RotaryRuns ch = rot_runs<kMode>(p, sub);
  wait_for_kernel_in_front();
  float2 w[4], dw[4];
  rot_weights(x.w, x.w_dtype, h * x.w_sh + ch.a, w);
  rot_weights(x.w, x.w_dtype, h * x.w_sh + ch.b, w + 2);
#pragma unroll
  for (int j = 0; j < 4; ++j) dw[j] = rot_both(0.f);
  const int64_t x_st = x.x_st, dy_st = x.dy_st, y_st = x.y_st;
  const float inv_d = 1.f / static_cast<float>(D);
  const int begin = static_cast<int>(blockIdx.x) * p.per_cta, end = begin + min(p.per_cta, p.tokens - begin);
  for (int at = begin, n; at < end; at += n) {
    const int b = at / p.T, t0 = at - b * p.T;
    n = min(min(p.tile, end - at), p.T - t0);
    {
      const uint16_t *row = x.x + b * x.x_sb + h * x.x_sh + t0 * x.x_st, *row_g = x.dy + b * x.dy_sb + h * x.dy_sh + t0 * x.dy_st;
      uint16_t* to = x.y + b * x.y_sb + h * x.y_sh + t0 * x.y_st;
      uint4 ahead_x[kAhead], ahead_g[kAhead];
      int to_ask = active ? n : 0;
      auto ask = [&] {
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          ahead_x[u] = u < to_ask ? rot_load<kMode>(row + u * x_st, ch) : make_uint4(0, 0, 0, 0);
          ahead_g[u] = u < to_ask ? rot_load<kMode>(row_g + u * dy_st, ch) : make_uint4(0, 0, 0, 0);
        }
        row += kAhead * x_st;
        row_g += kAhead * dy_st;
        to_ask -= kAhead;
      };
      ask();
      if (at != begin) __syncthreads();   // (the last tile's angles have been used)
      rot_angles<kMode>(p, b, t0, n, s_pos, s_cos, s_sin);
      const float *c = s_cos, *s = s_sin;
      for (int left = n; left > 0; left -= kAhead) {
        uint4 raw_x[kAhead], raw_g[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          raw_x[u] = ahead_x[u];
          raw_g[u] = ahead_g[u];
        }
        ask();
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          if (u >= left) break;
          float2 v[4], g[4], dn[4], gw[4], out[4];
          rot_unpack<kBf16>(raw_x[u], v);
          rot_unpack<kBf16>(raw_g[u], g);
          float pair[8];
          if constexpr (kMode == kAny) rot_exchange<kBf16>(p, s_rows + u * 256, lanes, ch.a, raw_g[u], pair);
          rot_turn<kMode>(p, ch, c + u * pairs, s + u * pairs, g, pair, dn);
          float2 sq = rot_both(0.f), dot2 = rot_both(0.f);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            gw[j] = rot_mul(dn[j], w[j]);
            sq = rot_fma(v[j], v[j], sq);
            dot2 = rot_fma(gw[j], v[j], dot2);
          }
          float ss = sq.x + sq.y, dot = dot2.x + dot2.y;
#pragma unroll
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
          if (active) rot_store<kMode>(to + u * y_st, ch, rot_pack<kBf16>(out));
        }
        if constexpr (kMode == kAny) __syncwarp();   // (the rows have been read before the next ones are written)
        to += kAhead * y_st;
        c += kAhead * pairs;
        s += kAhead * pairs;
      }
    }
  }
  if (p.fold) {   // weights that all heads share: the heads of this CTA added up first, (ranges, blocks, 2, D)
    __syncthreads();
    float* s_dw = rot_smem;
    if (active) {
      *reinterpret_cast<float4*>(s_dw + slot * D + ch.a) = make_float4(dw[0].x, dw[0].y, dw[1].x, dw[1].y);
      *reinterpret_cast<float4*>(s_dw + slot * D + ch.b) = make_float4(dw[2].x, dw[2].y, dw[3].x, dw[3].y);
    }
    __syncthreads();
    const int first = blockIdx.y * p.heads_here, slots = min(p.heads_here, p.heads - first), of_q = min(max(p.H - first, 0), slots);
    for (int i = threadIdx.x; i < 2 * D; i += blockDim.x) {
      const int which = i >= D, d = i - which * D;
      float sum = 0.f;
      for (int j = which ? of_q : 0; j < (which ? slots : of_q); ++j) sum += s_dw[j * D + d];
      p.dw_partial[((static_cast<int64_t>(blockIdx.x) * gridDim.y + blockIdx.y) * 2 + which) * D + d] = sum;
    }
  } else if (active) {
    float* to = p.dw_partial + (static_cast<int64_t>(blockIdx.x) * p.heads + head) * D;
    *reinterpret_cast<float4*>(to + ch.a) = make_float4(dw[0].x, dw[0].y, dw[1].x, dw[1].y);
    *reinterpret_cast<float4*>(to + ch.b) = make_float4(dw[2].x, dw[2].y, dw[3].x, dw[3].y);
  }
}

// dw of both tensors: 16 columns a CTA, its rows (shares, and heads where one weight is one for all) over 32 groups of threads
struct RotaryDwParams {
  const float* partial;
  void* dw[2];
  int w_dtype[2];
  int shared[2];
  int heads[2];
  int n_partials, D;
};
__global__ void __launch_bounds__(512) fox_rotary_dw_kernel(const RotaryDwParams p) {
  __shared__ float s_sum[32][17];
  wait_for_kernel_in_front();
  const int col = threadIdx.x & 15, grp = threadIdx.x >> 4;
  const int cols0 = p.shared[0] ? p.D : p.heads[0] * p.D;
  const int c_all = blockIdx.x * 16 + col, which = blockIdx.x * 16 >= cols0, c = c_all - (which ? cols0 : 0);
  const int64_t ld = static_cast<int64_t>(p.heads[0] + p.heads[1]) * p.D;
  const float* from = p.partial + (which ? static_cast<int64_t>(p.heads[0]) * p.D : 0) + c;
  float sum = 0.f;
  for (int h = 0; h < (p.shared[which] ? p.heads[which] : 1); ++h)
#pragma unroll 8
    for (int r = grp; r < p.n_partials; r += 32) sum += from[r * ld + h * p.D];
  s_sum[grp][col] = sum;
  __syncthreads();
  if (grp == 0) {
#pragma unroll
    for (int g = 1; g < 32; ++g) sum += s_sum[g][col];
    if (p.w_dtype[which] == FOX_DTYPE_FP32) static_cast<float*>(p.dw[which])[c] = sum;
    else
      static_cast<uint16_t*>(p.dw[which])[c] =
          static_cast<uint16_t>((p.w_dtype[which] == FOX_DTYPE_BF16 ? pack2<true>(sum, 0.f) : pack2<false>(sum, 0.f)) & 0xffffu);
  }
}

// ------------------------------------------------------------------- launches
static RotaryMode rotary_mode(int64_t half, int interleaved) { return interleaved ? kNext : half % 4 ? kAny : kHalves; }
struct RotaryGrid {
  int blocks, heads_here, threads, ranges, per_cta, tile;
};
enum RotaryKind { kTurn, kNormTurn, kNormBack };
// Heads of a token over as few CTAs of up to 256 threads as hold them, evenly; tokens over as many ranges as make one wave.  Forward,
// up to four waves while ranges keep 8 tokens: SMs get uneven shares of the bandwidth, and one that is ahead takes the next range
// (norms of 2 x 8192 tokens x 32 heads of 128: 1 wave 48.5 us, 3 45.4; 32768 tokens x 24 heads of 64 rotated only: 36.5, 4 waves 34.9).
// Not where the angles of a range cost more (kAny: 83 us, 92), nor backward, where every range adds a share of dw (70 us, 2 waves 73).  CTAs of
// fewer threads are more to an SM (36 heads of 64, 160 threads each: 61 -> 57 us, backward 104 -> 88), up to the threads that a kernel is
// fastest with (24 heads of 64 rotated only, 192 threads: 4 CTAs 36.5 us, 5 37.2); where the weights' shares are added up
// afterwards, while ranges keep 16 tokens (3000 tokens x 16 heads of 64: 8.9 us, of 6 tokens 11.2).
static RotaryGrid rotary_grid(RotaryKind kind, bool any, int64_t heads, int64_t D, int64_t tokens) {
  const int64_t most = kRotThreads / (D / 8), blocks = (heads + most - 1) / most, here = (heads + blocks - 1) / blocks;
  const int64_t threads = (here * (D / 8) + 31) / 32 * 32;
  const int64_t smem = kRotTile * (8 + D * 4) + threads / 32 * 1024 + 1024;   // of a CTA at most
  const int64_t least = kind == kNormBack ? kRotBwdPerSm : rot_fwd_per_sm(any ? kAny : kHalves);   // CTAs to an SM
  const int64_t by_threads = (kind == kNormBack ? 512 : kind == kTurn || any ? 768 : 1024) / threads, by_smem = 220 * 1024 / smem;
  const int64_t more = by_threads < by_smem ? by_threads : by_smem;
  auto ranges = [&](int64_t per_sm) { return kSms * per_sm / blocks < 1 ? 1 : kSms * per_sm / blocks; };
  int64_t want = ranges(more > least ? more : least);
  if (kind != kNormBack && !any) {
    const int64_t waves = tokens / (8 * want);
    want *= waves < 1 ? 1 : waves < 4 ? waves : 4;
  } else if (kind == kNormBack && tokens < 16 * want) {
    want = ranges(least) > tokens / 16 ? ranges(least) : tokens / 16;
  }
  const int64_t per = (tokens + want - 1) / want;
  return {static_cast<int>(blocks), static_cast<int>(here), static_cast<int>(threads),
          static_cast<int>((tokens + per - 1) / per), static_cast<int>(per), static_cast<int>(per < kRotTile ? per : kRotTile)};
}

template <bool kBf16, int kMode, int kD>
static int rotary_launch_of(RotaryKind kind, dim3 grid, unsigned threads, size_t smem, cudaStream_t st, const RotaryParams& p) {
  if (kind == kTurn) return launch_behind(fox_rotary_fwd_kernel<kBf16, kMode, false, kD>, grid, threads, smem, st, p);
  if (kind == kNormTurn) return launch_behind(fox_rotary_fwd_kernel<kBf16, kMode, true, kD>, grid, threads, smem, st, p);
  return launch_behind(fox_rotary_bwd_kernel<kBf16, kMode, kD>, grid, threads, smem, st, p);
}
// (the head dims of the layers' own configurations as constants; others, and halves that are no multiple of 4, by the general kernel)
template <bool kBf16, int kMode>
static int rotary_launch_at(RotaryKind kind, dim3 grid, unsigned threads, size_t smem, cudaStream_t st, const RotaryParams& p) {
  if constexpr (kMode != kAny) {
    if (p.D == 64) return rotary_launch_of<kBf16, kMode, 64>(kind, grid, threads, smem, st, p);
    if (p.D == 128) return rotary_launch_of<kBf16, kMode, 128>(kind, grid, threads, smem, st, p);
  }
  return rotary_launch_of<kBf16, kMode, 0>(kind, grid, threads, smem, st, p);
}
static int rotary_launch(RotaryKind kind, int dtype, int64_t half, int interleaved, const RotaryGrid& g, cudaStream_t st, RotaryParams p) {
  p.heads_here = g.heads_here;
  p.tile = rotary_mode(half, interleaved) == kAny && g.tile > 16 ? 16 : g.tile;   // (two angles to a channel)
  p.per_cta = g.per_cta;
  const dim3 grid(g.ranges, g.blocks);
  const bool any = rotary_mode(half, interleaved) == kAny;
  size_t smem = kRotTile * sizeof(double) + static_cast<size_t>(p.tile) * p.D * sizeof(float) * (any ? 2 : 1);
  if (any) smem += g.threads / 32 * 2 * 512;
  if (p.fold && smem < static_cast<size_t>(p.heads_here) * p.D * sizeof(float)) smem = static_cast<size_t>(p.heads_here) * p.D * sizeof(float);
  const bool bf = dtype == FOX_DTYPE_BF16;
  if (interleaved) return bf ? rotary_launch_at<true, kNext>(kind, grid, g.threads, smem, st, p) : rotary_launch_at<false, kNext>(kind, grid, g.threads, smem, st, p);
  if (half % 4) return bf ? rotary_launch_at<true, kAny>(kind, grid, g.threads, smem, st, p) : rotary_launch_at<false, kAny>(kind, grid, g.threads, smem, st, p);
  return bf ? rotary_launch_at<true, kHalves>(kind, grid, g.threads, smem, st, p) : rotary_launch_at<false, kHalves>(kind, grid, g.threads, smem, st, p);
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
  p.half = (int)half; p.D = (int)D; p.T = (int)T; p.tokens = (int)(B * T);
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
  return rotary_launch(kTurn, dtype, half, interleaved, rotary_grid(kTurn, rotary_mode(half, interleaved) == kAny, H, D, B * T), (cudaStream_t)stream, p);
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
  return rotary_launch(kNormTurn, dtype, half, interleaved, rotary_grid(kNormTurn, rotary_mode(half, interleaved) == kAny, H + Hk, D, B * T), (cudaStream_t)stream, p);
}

extern "C" int64_t fox_rotary_range(int kind, int64_t B, int64_t T, int64_t heads, int64_t D, int64_t half, int interleaved) {
  if (kind < kTurn || kind > kNormBack || B <= 0 || T <= 0 || heads <= 0 || (D != 16 && D != 32 && D != 64 && D != 128)) return 1;
  if (heads > 2 * 65535 || T > kRotTokens || B > kRotTokens / T) return 1;
  return rotary_grid(static_cast<RotaryKind>(kind), kind != kNormBack && rotary_mode(half, interleaved) == kAny, heads, D, B * T).per_cta;
}

extern "C" int64_t fox_qk_norm_rotary_partials(int64_t B, int64_t T, int64_t H, int64_t Hk, int64_t D) {
  if (B <= 0 || T <= 0 || H <= 0 || Hk <= 0 || (D != 16 && D != 32 && D != 64 && D != 128)) return 1;
  return rotary_grid(kNormBack, false, H + Hk, D, B * T).ranges;
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
  p.fold = !wq_sh && !wk_sh;
  const RotaryGrid g = rotary_grid(kNormBack, false, H + Hk, D, B * T);
  cudaStream_t st = (cudaStream_t)stream;
  if (int rc = rotary_launch(kNormBack, dtype, half, interleaved, g, st, p)) return rc;
  const RotaryDwParams d = p.fold ? RotaryDwParams{dw_partial, {dwq, dwk}, {wq_dtype, wk_dtype}, {0, 0}, {1, 1}, g.ranges * g.blocks, (int)D}
                                  : RotaryDwParams{dw_partial, {dwq, dwk}, {wq_dtype, wk_dtype}, {wq_sh == 0, wk_sh == 0}, {(int)H, (int)Hk},
                                                   g.ranges, (int)D};
  const int64_t cols = (wq_sh ? H * D : D) + (wk_sh ? Hk * D : D);
  return launch_behind(fox_rotary_dw_kernel, dim3((unsigned)(cols / 16)), 512, 0, st, d);
}
