// Causal grouped-head attention over packed sequences: rows cu[s] .. cu[s+1]-1
// of the operands are sequence s, and row i attends to the keys
// max(start of its sequence, i - window + 1) .. i:
//
//   x_ij = cap(q_i . k_j / sqrt d),  cap(x) = softcap tanh(x / softcap) or x
//   o_i  = sum_j exp(x_ij - m_i) v_j / sum_j exp(x_ij - m_i),  times sigmoid(gate_i)
//
// A query tile is 64 (128 on the tensor cores) consecutive rows of the packed
// stream, whatever sequences they belong to: the rows' key ranges differ only
// by their lower ends, which never decrease, so the tile walks one contiguous
// key range and a row masks what is not its own.  Hundreds of short sequences
// then cost no more tiles than one long one.
//
// Masked entries are excluded by selection, so scores of foreign keys may hold
// anything.  Their values enter P.V times zero, which is not zero where a value
// is infinite or NaN; a row whose result holds a NaN (on the tensor cores, where
// a tile's exponentials use the maximum of the tiles before, or an infinity) is
// therefore computed once more from its own keys alone (attn_packed_redo), so
// that what a sequence holds never reaches another.  A row whose own scores
// hold a NaN is NaN whatever else it sees: in BF16, and on the CUDA cores, it is
// left as it came out, and FP32 on the tensor cores, where infinite operands come
// out NaN too, ends the second pass at the first NaN score (4096 rows of NaN, 16
// heads of 128: 650 us against 390 of numbers).  Costly is an infinite value among
// the row's own: one at the start of 4096 rows makes all of them run twice, 12 ms
// at 16 heads of 256 in BF16 against 0.13 (15 ms at 128), 13 ms at 128 in FP32
// against 0.39.
//
// attn_packed_simt_kernel (here): FP32 products on the CUDA cores, any head
// size to 256, any strides and alignment: bf16 rows that TMA cannot read, FP32
// heads above 128 and a few FP32 rows.  64 x 64 score tiles, 4 x 4 a thread;
// queries, keys, values and P in shared memory as FP32, pairs of elements (of
// columns) a multiplication.  Latency bound: 16 warps an SM issue in 42% of the
// cycles between the tile's barriers (2047 rows, 16 heads of 128, window 200,
// capped: 182 us; the tensor cores take 63).
#pragma once

#include "common.cuh"

namespace clef {

template <typename T>
struct AttnPackedArgs {
  const T* q;
  const T* k;
  const T* v;
  const T* gate;  // nullptr = no gate
  T* out;
  long long ldq, hsq, ldk, hsk, ldv, hsv, ldg, hsg, ldo, hso;  // token and head strides (elements)
  const int32_t* cu;  // [n_seqs + 1]
  int n_seqs, tokens, H, Hk, d;
  float softcap;
  int window;
  int* status;
};

// The packed rows that belong to a sequence: [first, total).  Whatever cu
// holds, the bounds lie inside the buffers.
template <typename A>
__device__ __forceinline__ void packed_extent(const A& a, int& first, int& total) {
  total = min(a.cu[a.n_seqs], a.tokens);
  first = max(a.cu[0], 0);
}

// First key of `row`: the start of its sequence (the last s with cu[s] <= row)
// or the window's edge.  Inside [0, row] whatever cu holds.
template <typename A>
__device__ __forceinline__ int packed_first_key(const A& a, int row, int lo_seq, int hi_seq) {
  while (lo_seq < hi_seq) {  // cu[lo_seq] <= row < cu[hi_seq + 1]
    const int mid = (lo_seq + hi_seq + 1) >> 1;
    if (a.cu[mid] <= row)
      lo_seq = mid;
    else
      hi_seq = mid - 1;
  }
  const int start = min(max(a.cu[lo_seq], 0), row);
  return a.window > 0 ? max(start, row - a.window + 1) : start;
}

// 1 / softcap, 0 without one; finite, so that a score of 0 stays 0 under any cap.
__device__ __forceinline__ float inverse_cap(float softcap) { return softcap > 0.f ? fminf(1.f / softcap, 3e38f) : 0.f; }

// A score from a product: scaled, and capped where inv_cap is above 0.
__device__ __forceinline__ float packed_score(float x, float scale, float softcap, float inv_cap) {
  x *= scale;
  return inv_cap > 0.f ? softcap * tanh_flat(x * inv_cap) : x;
}

// One row again from its own keys [lo, row] alone, by a warp: a lane holds eight
// elements of every row it reads.  Four keys' partial products are summed over the
// lanes at once, by halves: after the first two exchanges a lane holds the sum
// of four lanes for one of the keys, `mine` below; after five of 32.  Eight such
// groups give every lane the score of one of 32 keys.  VEC: rows by 16-byte loads.
// With `state` the warp takes every `warps`-th 32 keys from its own on and leaves
// o [256], m and l there, to be joined with the other warps'.
constexpr int kRedoState = 258;
template <typename T, bool VEC>
__device__ __noinline__ void attn_packed_redo_row(const AttnPackedArgs<T>& a, int h, int row, int lo, int warp, int warps,
                                                  float* state) {
  const int lane = threadIdx.x & 31, c = lane * 8, hk = h / (a.H / a.Hk);
  const int mine = (lane >> 4 & 1) * 2 + (lane >> 3 & 1);
  const int step = state ? 32 * warps : 32;  // keys from one turn of this warp to its next
  if (state) lo += 32 * warp;
  T* out = a.out + row * a.ldo + h * a.hso;
  const float scale = rsqrtf(static_cast<float>(a.d)), inv_cap = inverse_cap(a.softcap);
  float q[8], o[8] = {};
  load8<T, VEC>(a.q + row * a.ldq + h * a.hsq, c, a.d, true, q);
  float m = -INFINITY, l = 0.f;
  for (; lo <= row; lo += step) {
    const int left = row + 1 - lo;
    const T* k = a.k + hk * a.hsk + lo * a.ldk;
    const T* v = a.v + hk * a.hsv + lo * a.ldv;
    const int groups = min(8, (left + 3) / 4);
    float x = 0.f;
#pragma unroll 1
    for (int g = 0; g < groups; ++g) {
      float s[4];
#pragma unroll
      for (int j = 0; j < 4; ++j, k += a.ldk) {
        float e[8];
        load8<T, VEC>(k, c, a.d, 4 * g + j < left, e);
        s[j] = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) s[j] = fmaf(q[i], e[i], s[j]);
      }
#pragma unroll
      for (int half = 2; half > 0; half /= 2) {
        const bool upper = lane & 8 * half;
#pragma unroll
        for (int j = 0; j < half; ++j) {
          const float other = __shfl_xor_sync(0xffffffffu, upper ? s[j] : s[j + half], 8 * half);
          s[j] = (upper ? s[j + half] : s[j]) + other;
        }
      }
#pragma unroll
      for (int w = 4; w > 0; w /= 2) s[0] += __shfl_xor_sync(0xffffffffu, s[0], w);
      if ((lane & 7) == g) x = s[0];
    }
    x = 4 * (lane & 7) + mine < left ? packed_score(x, scale, a.softcap, inv_cap) : -INFINITY;
    if (__any_sync(0xffffffffu, x != x)) {  // a NaN score: the row is NaN
      if (state) {
        l = __int_as_float(0x7fffffff);
        break;
      }
      for (int i = lane; i < a.d; i += 32) out[i] = from_f32<T>(__int_as_float(0x7fffffff));
      return;
    }
    const float mn = fmaxf(m, warp_max(x));
    const float corr = m == mn ? 1.f : expf(m - mn);
    m = mn;
    const float p = x == -INFINITY ? 0.f : expf(x - mn);  // also where no score so far is above -inf
    l = l * corr + warp_sum(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] *= corr;
#pragma unroll 1
    for (int g = 0; g < groups; ++g)
#pragma unroll
      for (int j = 0; j < 4; ++j, v += a.ldv) {
        float e[8];
        load8<T, VEC>(v, c, a.d, 4 * g + j < left, e);
        const float pj = __shfl_sync(0xffffffffu, p, 8 * j + g);  // the lane of key 4 g + j
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = fmaf(pj, e[i], o[i]);
      }
  }
  if (state) {
#pragma unroll
    for (int i = 0; i < 8; ++i) state[c + i] = o[i];
    if (lane == 0) state[256] = m, state[257] = l;
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (c + i < a.d) {
      float y = o[i] / l;
      if (a.gate) y *= sigmoidf_exact(to_f32(a.gate[row * a.ldg + h * a.hsg + c + i]));
      out[c + i] = from_f32<T>(y);
    }
}

// The rows of the tile at q0 whose bit in `bad` (32 rows a word) is set, again: a warp
// a row where there are as many rows as warps, else the warps share each row's
// keys.  smem: warps * kRedoState floats.  Every thread of the block must call it.
template <typename T, bool VEC>
__device__ __noinline__ void attn_packed_redo(const AttnPackedArgs<T>& a, int h, int q0, const uint32_t* bad, int words, float* smem) {
  const int warp = threadIdx.x / 32, warps = blockDim.x / 32;
  int count = 0;
  for (int w = 0; w < words; ++w) count += __popc(bad[w]);
  const bool shared = count < warps;
  uint32_t rows = bad[0];
  for (int turn = 0, w = 0; turn < count; ++turn, rows &= rows - 1) {
    while (!rows) rows = bad[++w];
    if (!shared && turn % warps != warp) continue;
    const int row = q0 + 32 * w + __ffs(static_cast<int>(rows)) - 1;
    attn_packed_redo_row<T, VEC>(a, h, row, packed_first_key(a, row, 0, a.n_seqs - 1), warp, warps,
                                 shared ? smem + warp * kRedoState : nullptr);
    if (!shared) continue;
    __syncthreads();
    const int c = threadIdx.x;
    if (c < a.d) {
      float m = -INFINITY, l = 0.f, o = 0.f;
      for (int w = 0; w < warps; ++w) m = fmaxf(m, smem[w * kRedoState + 256]);
      for (int w = 0; w < warps; ++w) {
        const float* st = smem + w * kRedoState;
        const float weight = st[256] == -INFINITY ? 0.f : expf(st[256] - m);
        l = fmaf(weight, st[257], l);
        o = fmaf(weight, st[c], o);
      }
      float y = o / l;
      if (a.gate) y *= sigmoidf_exact(to_f32(a.gate[row * a.ldg + h * a.hsg + c]));
      a.out[row * a.ldo + h * a.hso + c] = from_f32<T>(y);
    }
    __syncthreads();
  }
}

// Rows of a tile whose kernel gave up on a wait: NaN, whatever the kernel has
// stored there.  Every thread of the block must call it.
template <typename T, int NT>
__device__ __noinline__ void attn_packed_give_up(const AttnPackedArgs<T>& a, int h, int q_first, int q_end) {
  const long long n = static_cast<long long>(q_end - q_first) * a.d;
  for (long long i = threadIdx.x; i < n; i += NT)
    a.out[(q_first + i / a.d) * a.ldo + h * a.hso + i % a.d] = from_f32<T>(__int_as_float(0x7fffffff));
}

template <int DP>
struct AttnPackedSimtShape {
  static constexpr int BQ = 64, BK = 64, LD = DP + 4, LDP = BK + 4;
  static constexpr int CTAS = DP <= 128 ? 2 : 1;  // per SM
  static constexpr size_t SMEM = (2 * 64 * LD + BQ * LDP) * sizeof(float);
};

// A 64-row tile in registers on its way to shared memory: float4 i of a thread is
// float4 tid + 256 i of the tile.  Rows past `end` and elements past d read zero.
template <typename T, int DP>
struct TileOnTheWay {
  float4 v[DP / 16];
  __device__ __forceinline__ void load(const T* base, long long ld, int row0, int end, int d, bool vec) {
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) {
      const int at = static_cast<int>(threadIdx.x) + 256 * i, r = at / (DP / 4), c = at % (DP / 4) * 4;
      const T* p = base + (row0 + r) * ld + c;
      v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (row0 + r < end) {
        if (sizeof(T) == 4 && vec) {
          if (c < d) v[i] = *reinterpret_cast<const float4*>(p);
        } else {
          if (c < d) v[i].x = to_f32(p[0]);
          if (c + 1 < d) v[i].y = to_f32(p[1]);
          if (c + 2 < d) v[i].z = to_f32(p[2]);
          if (c + 3 < d) v[i].w = to_f32(p[3]);
        }
      }
    }
  }
  __device__ __forceinline__ void store(float* tile, int ld) const {
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) {
      const int at = static_cast<int>(threadIdx.x) + 256 * i;
      *reinterpret_cast<float4*>(tile + at / (DP / 4) * ld + at % (DP / 4) * 4) = v[i];
    }
  }
};

template <typename T, int DP>
__global__ void __launch_bounds__(256, AttnPackedSimtShape<DP>::CTAS)
    attn_packed_simt_kernel(const __grid_constant__ AttnPackedArgs<T> a, bool vec) {
  using Sh = AttnPackedSimtShape<DP>;
  constexpr int BQ = Sh::BQ, BK = Sh::BK, LD = Sh::LD, LDP = Sh::LDP, NC = DP / 64;
  constexpr float LOG2E = 1.4426950408889634f;
  extern __shared__ __align__(16) float simt_smem[];
  float* sQ = simt_smem;
  float* sKV = sQ + BQ * LD;  // the key tile, then the value tile
  float* sP = sKV + BK * LD;
  __shared__ int s_lo[BQ];
  __shared__ uint32_t s_nan[2];

  int first, total;
  packed_extent(a, first, total);
  const int q0 = (static_cast<int>(gridDim.x) - 1 - static_cast<int>(blockIdx.x)) * BQ, h = blockIdx.y;
  const int q_end = min(q0 + BQ, total), q_first = max(q0, first);
  if (q_first >= q_end) return;  // no row of this tile belongs to a sequence
  const int hk = h / (a.H / a.Hk);
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  if (tid < BQ) {  // rows outside the sequences see no key
    const int row = q0 + tid;
    s_lo[tid] = row >= q_first && row < q_end ? packed_first_key(a, row, 0, a.n_seqs - 1) : row + 1;
  }
  if (tid < 2) s_nan[tid] = 0u;
  TileOnTheWay<T, DP> way;
  way.load(a.q + h * a.hsq, a.ldq, q0, q_end, a.d, vec);
  way.store(sQ, LD);
  __syncthreads();
  int lo[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) lo[i] = s_lo[ty * 4 + i];
  const int k_begin = s_lo[q_first - q0];
  const float scale = rsqrtf(static_cast<float>(a.d)), inv_cap = inverse_cap(a.softcap);
  float m[4], l[4];
  uint64_t o[4][2 * NC];  // pairs of columns
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int c = 0; c < 2 * NC; ++c) o[i][c] = 0ull;
  }
  // rows of this warp: tiles above the last or below the first one's keys cost it nothing
  const int w_last = q0 + (tid / 32) * 8 + 7, w_lo = s_lo[(tid / 32) * 8];
  way.load(a.k + hk * a.hsk, a.ldk, k_begin, q_end, a.d, vec);
  for (int k0 = k_begin; k0 < q_end; k0 += BK) {
    const bool any = k0 <= w_last && k0 + BK > w_lo;
    __syncthreads();  // the last value tile has been read
    way.store(sKV, LD);
    __syncthreads();
    way.load(a.v + hk * a.hsv, a.ldv, k0, q_end, a.d, vec);
    if (any) {
      uint64_t s2[4][4] = {};  // sums of even and odd elements
#pragma unroll 4
      for (int c = 0; c < DP; c += 4) {
        ulonglong2 qf[4], kf[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) qf[i] = *reinterpret_cast<const ulonglong2*>(&sQ[(ty * 4 + i) * LD + c]);
#pragma unroll
        for (int j = 0; j < 4; ++j) kf[j] = *reinterpret_cast<const ulonglong2*>(&sKV[(tx + 16 * j) * LD + c]);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            s2[i][j] = fma2(qf[i].x, kf[j].x, s2[i][j]);
            s2[i][j] = fma2(qf[i].y, kf[j].y, s2[i][j]);
          }
      }
      float s[4][4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 x = unpair2(s2[i][j]);
          s[i][j] = x.x + x.y;
        }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = q0 + ty * 4 + i;
        float mt = -INFINITY;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int key = k0 + tx + 16 * j;
          s[i][j] = key >= lo[i] && key <= row ? packed_score(s[i][j], scale, a.softcap, inv_cap) * LOG2E : -INFINITY;
          mt = fmaxf(mt, s[i][j]);
        }
#pragma unroll
        for (int w = 8; w > 0; w >>= 1) mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, w));
        const float mn = fmaxf(m[i], mt);
        const float base = mn == -INFINITY ? 0.f : mn;  // no key of this row yet: every p is exp2(-inf) = 0
        const float corr = exp2f(m[i] - base);
        m[i] = mn;
        float ps = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float p = exp2f(s[i][j] - base);
          sP[(ty * 4 + i) * LDP + tx + 16 * j] = p;
          ps += p;
        }
#pragma unroll
        for (int w = 8; w > 0; w >>= 1) ps += __shfl_xor_sync(0xffffffffu, ps, w);
        l[i] = l[i] * corr + ps;
#pragma unroll
        for (int c = 0; c < 2 * NC; ++c) o[i][c] = corr == 0.f ? 0ull : mul2(o[i][c], pair2(corr, corr));
      }
    }
    __syncthreads();  // the key tile has been read
    way.store(sKV, LD);
    __syncthreads();
    if (k0 + BK < q_end) way.load(a.k + hk * a.hsk, a.ldk, k0 + BK, q_end, a.d, vec);
    if (any) {
#pragma unroll 2
      for (int j = 0; j < BK; j += 4) {
        float4 pf[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) pf[i] = *reinterpret_cast<const float4*>(&sP[(ty * 4 + i) * LDP + j]);
#pragma unroll
        for (int jj = 0; jj < 4; ++jj) {
          uint64_t p2[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float p = jj == 0 ? pf[i].x : jj == 1 ? pf[i].y : jj == 2 ? pf[i].z : pf[i].w;
            p2[i] = pair2(p, p);
          }
#pragma unroll
          for (int c = 0; c < NC; ++c) {
            const ulonglong2 vf = *reinterpret_cast<const ulonglong2*>(&sKV[(j + jj) * LD + 64 * c + tx * 4]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              o[i][2 * c] = fma2(p2[i], vf.x, o[i][2 * c]);
              o[i][2 * c + 1] = fma2(p2[i], vf.y, o[i][2 * c + 1]);
            }
          }
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = q0 + ty * 4 + i;
    if (row < q_first || row >= q_end) continue;
    bool bad = false;
#pragma unroll
    for (int c = 0; c < 4 * NC; ++c) {
      const int col = 64 * (c / 4) + tx * 4 + (c & 3);
      if (col >= a.d) continue;
      const float2 oo = unpair2(o[i][c / 2]);
      float y = (c & 1 ? oo.y : oo.x) / l[i];
      bad |= y != y;
      if (a.gate) y *= sigmoidf_exact(to_f32(a.gate[row * a.ldg + h * a.hsg + col]));
      a.out[row * a.ldo + h * a.hso + col] = from_f32<T>(y);
    }
    // a NaN sum has a NaN (or infinite) score of the row's own: the row is NaN, and stays so
    if (bad && l[i] == l[i]) atomicOr(&s_nan[ty / 8], 1u << (ty * 4 + i) % 32);
  }
  __syncthreads();
  if (s_nan[0] | s_nan[1]) attn_packed_redo<T, false>(a, h, q0, s_nan, 2, simt_smem);
}

}  // namespace clef
