// Per-head q/k RMSNorm(1 + w) and partial rotate-half RoPE whose positions are
// given: one row of int32 positions for each axis (text: one; images and
// video: time, height, width), each frequency pair reading the axis it
// belongs to.
//
//   y = x * rsqrt(mean(x^2) + eps) * (1 + w)            (w absent: y = x)
//   a = p[axis(i), t] * theta^(-2i/rot),  i < rot/2
//   out[i]       = y[i] cos a - y[i + rot/2] sin a
//   out[i+rot/2] = y[i + rot/2] cos a + y[i] sin a,  out[j] = y[j] for j >= rot
//
// All arithmetic is FP32 with one rounding at the store (clef_op_qk_norm_rope
// also rounds the norm, cos, sin and both products to bf16).  The angle never
// exists as a float: theta^(-2i/rot) / 2pi is held as a 64-bit fraction of a
// turn, and p times it, modulo 2^64, is the exact turn of the product for any
// int32 position (error p * 2^-65 of a turn); a float product would be off by
// 0.06 rad at position 10^6.
#pragma once

#include "common.cuh"

namespace clef {

constexpr int kRopeMaxHalf = 128;  // head_dim <= 256

struct RopeAxesArgs {
  const void* x[2];      // q, k
  void* out[2];
  const void* w[2];      // norm weights, nullptr = no norm
  long long ldx[2], hsx[2], ldo[2], hso[2];  // token and head strides (elements)
  int heads[2];
  const int32_t* pos;    // [axes, ldp]
  long long ldp;
  int tokens, d, half;
  float eps;
  unsigned long long turn[kRopeMaxHalf];  // theta^(-2i/rot) / 2pi as a fraction of 2^64
  unsigned char axis[kRopeMaxHalf];
};

// (cos, sin) of position p at frequency `turn`: the fraction of a turn as a
// signed 32-bit number is the angle in units of pi * 2^-31.
__device__ __forceinline__ float2 rope_cos_sin(int p, unsigned long long turn) {
  const unsigned long long frac = static_cast<unsigned long long>(static_cast<long long>(p)) * turn;
  const float half_turns = static_cast<float>(static_cast<int>(frac >> 32)) * 4.656612873077393e-10f;  // 2^-31
  float2 cs;
  sincospif(half_turns, &cs.y, &cs.x);
  return cs;
}

// Any head size and alignment: one warp per (token, head), the row staged in shared memory.
template <typename T>
__global__ void __launch_bounds__(256) rope_axes_any_kernel(const __grid_constant__ RopeAxesArgs a) {
  extern __shared__ float rope_rows[];  // 8 warps x d
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int heads = a.heads[0] + a.heads[1];
  const long long item = static_cast<long long>(blockIdx.x) * 8 + warp;
  if (item >= static_cast<long long>(a.tokens) * heads) return;
  const int t = static_cast<int>(item / heads);
  int h = static_cast<int>(item % heads);
  const int which = h >= a.heads[0];
  if (which) h -= a.heads[0];
  const T* x = static_cast<const T*>(which ? a.x[1] : a.x[0]) + t * (which ? a.ldx[1] : a.ldx[0]) +
               h * (which ? a.hsx[1] : a.hsx[0]);
  T* out = static_cast<T*>(which ? a.out[1] : a.out[0]) + t * (which ? a.ldo[1] : a.ldo[0]) +
           h * (which ? a.hso[1] : a.hso[0]);
  const T* w = static_cast<const T*>(which ? a.w[1] : a.w[0]);
  float* row = rope_rows + warp * a.d;
  float ss = 0.f;
  for (int i = lane; i < a.d; i += 32) {
    const float v = to_f32(x[i]);
    row[i] = v;
    ss = fmaf(v, v, ss);
  }
  if (w) {
    const float r = rsqrtf(warp_sum(ss) / static_cast<float>(a.d) + a.eps);
    for (int i = lane; i < a.d; i += 32) row[i] *= r * (1.f + to_f32(w[i]));
  }
  __syncwarp();
  for (int i = lane; i < a.half; i += 32) {
    const float2 cs = rope_cos_sin(a.pos[a.axis[i] * a.ldp + t], a.turn[i]);
    const float lo = row[i], hi = row[i + a.half];
    out[i] = from_f32<T>(lo * cs.x - hi * cs.y);
    out[i + a.half] = from_f32<T>(hi * cs.x + lo * cs.y);
  }
  for (int i = 2 * a.half + lane; i < a.d; i += 32) out[i] = from_f32<T>(row[i]);
}

// The elements of a 16-byte vector as floats, and back.
__device__ __forceinline__ void unpack16(const uint4 u, float (&v)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    v[2 * j] = __uint_as_float(w[j] << 16);
    v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
  }
}
__device__ __forceinline__ void unpack16(const uint4 u, float (&v)[4]) {
  v[0] = __uint_as_float(u.x), v[1] = __uint_as_float(u.y), v[2] = __uint_as_float(u.z), v[3] = __uint_as_float(u.w);
}
__device__ __forceinline__ void store16(__nv_bfloat16* p, const float (&v)[8]) {
  *reinterpret_cast<uint4*>(p) =
      make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
}
__device__ __forceinline__ void store16(float* p, const float (&v)[4]) {
  *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
}

template <typename T>
struct RopeShape {
  static constexpr int V = 16 / sizeof(T);  // elements of a 16-byte vector
  static constexpr int DEPTH = 4;           // rows a lane has on the way, the current one among them
  static constexpr size_t ring(int threads) { return static_cast<size_t>(DEPTH) * 2 * threads * sizeof(uint4); }
};

// 16-byte aligned rows, d and rot multiples of two vectors: LANES lanes hold a
// head row, each a 16-byte vector and the one its rotation pairs it with (or two
// behind the rotated part, as far apart as keeps neighbours adjacent), so that a
// row is read and written once by whole sectors and its norm is one reduction
// over the lanes.  A lane keeps its head
// and walks the block's `span` tokens, so the weights stay in registers and a
// row costs no index arithmetic (a walk over (token, head) pairs issued 2.6
// times the instructions and was bound by them at 4.8 TB/s).  cos and sin of
// the block's tokens are computed once, while the first rows load.  HBM bound:
// rows come by asynchronous copies, DEPTH on the way, into slots of shared
// memory that only their lane reads, so nothing waits at a barrier.
// 131072 tokens x 48 heads of 128, bf16: 556 us, 5.8 TB/s; 4097 x 24 heads of 256, FP32:
// 36.8 us, 5.5 TB/s.
// grid (token spans, head groups of blockDim / LANES).
template <typename T, int LANES>
__global__ void __launch_bounds__(512) rope_axes_kernel(const __grid_constant__ RopeAxesArgs a, int span) {
  using S = RopeShape<T>;
  constexpr int V = S::V;
  extern __shared__ uint4 rope_ring[];  // [DEPTH][2][threads], then cos, sin [span][half]
  const int threads = blockDim.x, tid = threadIdx.x, j = tid % LANES;
  float2* rope_cs = reinterpret_cast<float2*>(rope_ring + S::DEPTH * 2 * threads);
  const int t0 = blockIdx.x * span, n = min(span, a.tokens - t0);
  int h = blockIdx.y * (threads / LANES) + tid / LANES;
  const bool live = h < a.heads[0] + a.heads[1] && j < a.d / (2 * V);  // lanes behind the heads or the row's end
  const int which = h >= a.heads[0];
  if (which) h -= a.heads[0];
  const bool turns = j < a.half / V;
  const int lo_at = turns ? V * j : a.half + V * j;  // behind the rotated part: 2 half + V (j - half / V)
  const int hi_at = lo_at + (turns ? a.half : a.d / 2 - a.half);
  const long long ldx = which ? a.ldx[1] : a.ldx[0], ldo = which ? a.ldo[1] : a.ldo[0];
  const T* x = static_cast<const T*>(which ? a.x[1] : a.x[0]) + t0 * ldx + h * (which ? a.hsx[1] : a.hsx[0]);
  T* out = static_cast<T*>(which ? a.out[1] : a.out[0]) + t0 * ldo + h * (which ? a.hso[1] : a.hso[0]);
  const T* w = static_cast<const T*>(which ? a.w[1] : a.w[0]);
  int fill = 0;
  auto fetch = [&](int t) {  // the row of token t, into slot `fill`
    if (live && t < n) {
      uint4* dst = rope_ring + fill * 2 * threads + tid;
      cp_async16(dst, x + lo_at, true);
      cp_async16(dst + threads, x + hi_at, true);
      x += ldx;
    }
    cp_async_commit();
    if (++fill == S::DEPTH) fill = 0;
  };
#pragma unroll
  for (int i = 0; i < S::DEPTH - 1; ++i) fetch(i);
  float wl[V], wh[V];  // 1 + w of this lane's vectors
#pragma unroll
  for (int e = 0; e < V; ++e) wl[e] = wh[e] = 1.f;
  if (live && w) {
    unpack16(*reinterpret_cast<const uint4*>(w + lo_at), wl);
    unpack16(*reinterpret_cast<const uint4*>(w + hi_at), wh);
#pragma unroll
    for (int e = 0; e < V; ++e) wl[e] += 1.f, wh[e] += 1.f;
  }
  for (int e = tid; e < n * a.half; e += threads) {
    // a lane reads two pairs at a time: the lanes' two lie side by side
    const int t = e / a.half, i = e % a.half;
    rope_cs[t * a.half + (i % V / 2 * (a.half / V) + i / V) * 2 + (i & 1)] =
        rope_cos_sin(a.pos[a.axis[i] * a.ldp + t0 + t], a.turn[i]);
  }
  __syncthreads();
  const float inv_d = 1.f / static_cast<float>(a.d);
  int take = 0;
  for (int t = 0; t < n; ++t) {
    fetch(t + S::DEPTH - 1);
    cp_async_wait<S::DEPTH - 1>();
    float lo[V], hi[V];
    const uint4* src = rope_ring + take * 2 * threads + tid;
    unpack16(src[0], lo);
    unpack16(src[threads], hi);
    if (++take == S::DEPTH) take = 0;
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < V; ++e) ss = fmaf(lo[e], lo[e], fmaf(hi[e], hi[e], ss));
    if (!live) ss = 0.f;  // nothing was fetched
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const float r = w ? rsqrtf(ss * inv_d + a.eps) : 1.f;
    if (live) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        lo[e] *= r * wl[e];
        hi[e] *= r * wh[e];
      }
      if (turns) {
        const float4* cs = reinterpret_cast<const float4*>(rope_cs + t * a.half) + j;
#pragma unroll
        for (int e = 0; e < V / 2; ++e) {
          const float4 c = cs[e * (a.half / V)];  // cos, sin of two pairs
          const float l0 = lo[2 * e], h0 = hi[2 * e], l1 = lo[2 * e + 1], h1 = hi[2 * e + 1];
          lo[2 * e] = l0 * c.x - h0 * c.y;
          hi[2 * e] = h0 * c.x + l0 * c.y;
          lo[2 * e + 1] = l1 * c.z - h1 * c.w;
          hi[2 * e + 1] = h1 * c.z + l1 * c.w;
        }
      }
      store16(out + lo_at, lo);
      store16(out + hi_at, hi);
      out += ldo;
    }
  }
}

}  // namespace clef
