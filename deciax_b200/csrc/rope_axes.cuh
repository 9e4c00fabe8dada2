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

}  // namespace clef
