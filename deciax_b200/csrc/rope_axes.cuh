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

// Eight consecutive elements.
__device__ __forceinline__ void load_vec8(const __nv_bfloat16* p, float (&v)[8]) {
  const uint4 u = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    v[2 * j] = __uint_as_float(w[j] << 16);
    v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
  }
}
__device__ __forceinline__ void load_vec8(const float* p, float (&v)[8]) {
  *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(p);
  *reinterpret_cast<float4*>(v + 4) = *reinterpret_cast<const float4*>(p + 4);
}
__device__ __forceinline__ void store_vec8(__nv_bfloat16* p, const float (&v)[8]) {
  *reinterpret_cast<uint4*>(p) =
      make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
}
__device__ __forceinline__ void store_vec8(float* p, const float (&v)[8]) {
  *reinterpret_cast<float4*>(p) = *reinterpret_cast<const float4*>(v);
  *reinterpret_cast<float4*>(p + 4) = *reinterpret_cast<const float4*>(v + 4);
}

// 16-byte aligned rows, d and rot multiples of 16: a block takes `span` tokens.
// Their cos and sin are computed once, into shared memory, while the first
// rows load; then LANES lanes hold a head row, each an element run of 8 and the
// run its rotation pairs it with (or two runs behind the rotated part), so that
// a row is read and written once by 16-byte accesses and its norm is one
// reduction over the lanes.  HBM bound; the next row of a lane loads while the
// current one is computed.
template <typename T, int LANES>
__global__ void __launch_bounds__(256) rope_axes_kernel(const __grid_constant__ RopeAxesArgs a, int span) {
  extern __shared__ float2 rope_cs[];  // [span][half]
  constexpr int SLOTS = 256 / LANES;   // head rows in flight in the block
  const int tid = threadIdx.x, j = tid % LANES;
  const int t0 = blockIdx.x * span, n = min(span, a.tokens - t0);
  const int heads = a.heads[0] + a.heads[1];
  const bool active = j < a.d / 16;
  const bool turns = j < a.half / 8;
  const int lo_at = turns ? 8 * j : 2 * a.half + 16 * (j - a.half / 8);
  const int hi_at = turns ? lo_at + a.half : lo_at + 8;
  int t = (tid / LANES) / heads, h = (tid / LANES) % heads;
  float lo[8] = {}, hi[8] = {};
  auto load = [&](int t, int h, float (&lo)[8], float (&hi)[8]) {
    if (t < n && active) {
      const int which = h >= a.heads[0];
      const T* x = static_cast<const T*>(which ? a.x[1] : a.x[0]) + (t0 + t) * (which ? a.ldx[1] : a.ldx[0]) +
                   (which ? (h - a.heads[0]) * a.hsx[1] : h * a.hsx[0]);
      load_vec8(x + lo_at, lo);
      load_vec8(x + hi_at, hi);
    }
  };
  load(t, h, lo, hi);
  for (int e = tid; e < n * a.half; e += 256) {
    const int i = e % a.half;
    rope_cs[e] = rope_cos_sin(a.pos[a.axis[i] * a.ldp + t0 + e / a.half], a.turn[i]);
  }
  __syncthreads();
  while (__any_sync(0xffffffffu, t < n)) {
    int t_next = t, h_next = h + SLOTS;
    while (h_next >= heads) {
      h_next -= heads;
      ++t_next;
    }
    float lo_next[8] = {}, hi_next[8] = {};
    load(t_next, h_next, lo_next, hi_next);
    const int which = h >= a.heads[0];
    const T* w = static_cast<const T*>(which ? a.w[1] : a.w[0]);
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = fmaf(lo[e], lo[e], fmaf(hi[e], hi[e], ss));
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (t < n && active) {
      if (w) {
        const float r = rsqrtf(ss / static_cast<float>(a.d) + a.eps);
        float wl[8], wh[8];
        load_vec8(w + lo_at, wl);
        load_vec8(w + hi_at, wh);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          lo[e] *= r * (1.f + wl[e]);
          hi[e] *= r * (1.f + wh[e]);
        }
      }
      if (turns) {
        const float4* cs = reinterpret_cast<const float4*>(rope_cs + t * a.half + 8 * j);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float4 c = cs[e];  // cos, sin of two pairs
          const float l0 = lo[2 * e], h0 = hi[2 * e], l1 = lo[2 * e + 1], h1 = hi[2 * e + 1];
          lo[2 * e] = l0 * c.x - h0 * c.y;
          hi[2 * e] = h0 * c.x + l0 * c.y;
          lo[2 * e + 1] = l1 * c.z - h1 * c.w;
          hi[2 * e + 1] = h1 * c.z + l1 * c.w;
        }
      }
      T* out = static_cast<T*>(which ? a.out[1] : a.out[0]) + (t0 + t) * (which ? a.ldo[1] : a.ldo[0]) +
               (which ? (h - a.heads[0]) * a.hso[1] : h * a.hso[0]);
      store_vec8(out + lo_at, lo);
      store_vec8(out + hi_at, hi);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      lo[e] = lo_next[e];
      hi[e] = hi_next[e];
    }
    t = t_next;
    h = h_next;
  }
}

}  // namespace clef
