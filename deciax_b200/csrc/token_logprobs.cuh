// Log probabilities of given tokens under the language head, with the entropy
// of each row's distribution and its top alternatives:
//
//   x = h W^T,  z = cap(x) = softcap tanh(x / softcap) or x
//   lse = log sum_v exp z_v,   logp(t) = z_t - lse,   H = lse - sum_v p_v z_v
//
// The [rows, vocab] logits never exist: each vocabulary tile's scores go from
// the accumulators straight into a running state per row,
//   m = max z,  s = sum exp(z - m),  t = sum exp(z - m) (z - m)   (log2 units),
// and a sorted list of the largest x with their ids.  The vocabulary is split
// into S runs of tiles, so that few rows still fill the GPU; a run of a row
// tile is one unit of work and leaves its rows' states and lists in scratch.
// token_logprobs_finish_kernel joins the S states and lists of a row and takes the
// given tokens' scores from their own dot products.
//
// With s and t joined at m = max m_i:  H = ln s - ln2 t / s.
//
// Here: the state, the joining kernel, and the CUDA-core form (FP32 operands, or
// rows that are not 16-byte aligned).  token_logprobs_sm100.cuh has the tensor-core form.
#pragma once

#include "common.cuh"

namespace clef {

constexpr int kTopMax = 32;

struct LogprobArgs {
  const void* hidden;
  const void* head;
  long long ldh, ldw;
  int rows, vocab, dim;
  float softcap;
  int top;
  // units of work: num_m row tiles x splits runs of the num_n vocabulary tiles
  int num_m, num_n, splits;
  // scratch: per (split, row) the state, then the list
  float* part_m;
  float* part_s;
  float* part_t;
  float* list_x;    // [splits][rows][top], largest first
  int32_t* list_id;
  int* status;
};

__device__ __forceinline__ int split_begin(int split, int num_n, int splits) {
  return static_cast<int>(static_cast<long long>(num_n) * split / splits);
}

template <bool CAP>
__device__ __forceinline__ float capped(float x, float softcap) {
  return CAP ? softcap * tanhf(x / softcap) : x;
}

// A row's running state.  m, s, t are in log2 units of z; thr is the smallest x of
// its list, which lies in shared memory, entry j of row r at [j * 128 + r].
struct RowState {
  float m = -INFINITY, s = 0.f, t = 0.f, thr = -INFINITY;
};

__device__ __forceinline__ void list_clear(float* lx, int32_t* lid, int top, int r) {
  for (int j = 0; j < top; ++j) {
    lx[j * 128 + r] = -INFINITY;
    lid[j * 128 + r] = -1;
  }
}

// Ids arrive in rising order, so an equal score stays behind the entry it equals.
__device__ __forceinline__ void list_insert(RowState& st, float x, int id, float* lx, int32_t* lid, int top, int r) {
  int j = top - 1;
  for (; j > 0 && lx[(j - 1) * 128 + r] < x; --j) {
    lx[j * 128 + r] = lx[(j - 1) * 128 + r];
    lid[j * 128 + r] = lid[(j - 1) * 128 + r];
  }
  lx[j * 128 + r] = x;
  lid[j * 128 + r] = id;
  st.thr = lx[(top - 1) * 128 + r];
}

// Scores x of columns col .. col + 31, the first `valid` of which exist.
template <bool CAP>
__device__ __forceinline__ void scan32(RowState& st, const float (&x)[32], int col, int valid, float softcap, float* lx,
                                       int32_t* lid, int top, int r) {
  constexpr float LOG2E = 1.4426950408889634f;
  float z[32];
  float px[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int c = 0; c < 32; ++c) {
    const bool in = c < valid;
    if (in) px[c & 3] = fmaxf(px[c & 3], x[c]);
    z[c] = CAP ? (in ? capped<CAP>(x[c], softcap) : -INFINITY) : x[c];
  }
  const float xmax = fmaxf(fmaxf(px[0], px[1]), fmaxf(px[2], px[3]));
  const float zmax = capped<CAP>(xmax, softcap) * LOG2E;
  if (zmax > st.m) {  // the sums move to the new maximum
    const float step = st.m - zmax, f = exp2f(step);
    st.t = st.s == 0.f ? 0.f : f * fmaf(step, st.s, st.t);
    st.s *= f;
    st.m = zmax;
  }
  float ps[4] = {0.f, 0.f, 0.f, 0.f}, pt[4] = {0.f, 0.f, 0.f, 0.f};
  const float neg_m = -st.m;
  if (valid >= 32) {
#pragma unroll
    for (int c = 0; c < 32; ++c) {
      const float d = fmaf(z[c], LOG2E, neg_m);
      const float e = ex2_approx(d);
      ps[c & 3] += e;
      pt[c & 3] = fmaf(d, e, pt[c & 3]);
    }
  } else {
#pragma unroll
    for (int c = 0; c < 32; ++c)
      if (c < valid) {
        const float d = fmaf(z[c], LOG2E, neg_m);
        const float e = ex2_approx(d);
        ps[c & 3] += e;
        pt[c & 3] = fmaf(d, e, pt[c & 3]);
      }
  }
  st.s += (ps[0] + ps[1]) + (ps[2] + ps[3]);
  st.t += (pt[0] + pt[1]) + (pt[2] + pt[3]);
  if (top > 0 && xmax > st.thr) {
#pragma unroll
    for (int c = 0; c < 32; ++c)
      if (c < valid && x[c] > st.thr) list_insert(st, x[c], col + c, lx, lid, top, r);
  }
}

__device__ __forceinline__ void store_state(const LogprobArgs& a, const RowState& st, int split, int row, const float* lx,
                                            const int32_t* lid, int r) {
  const size_t at = static_cast<size_t>(split) * a.rows + row;
  a.part_m[at] = st.m;
  a.part_s[at] = st.s;
  a.part_t[at] = st.t;
  for (int j = 0; j < a.top; ++j) {
    a.list_x[at * a.top + j] = lx[j * 128 + r];
    a.list_id[at * a.top + j] = lid[j * 128 + r];
  }
}

// ---------------------------------------------------------------------------
// CUDA cores: 128 x 128 tiles, 8 x 8 a thread, FP32 products and sums
// ---------------------------------------------------------------------------
// Sixteen values of k at a time through shared memory, the next sixteen in
// registers meanwhile; 6 shared-memory wavefronts for 16 cycles of FMA.  A
// finished tile goes through shared memory once more so that a thread scans a row.

constexpr int kLogprobSimtLdc = 132;
constexpr size_t logprob_simt_smem(int top) {
  return (2 * 16 * 132 + 128 * kLogprobSimtLdc + 2 * 128 * top) * sizeof(float);
}

// Elements k .. k + 7 of a row (zeros past its end); VEC: by 16-byte loads.
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* p, int k, int dim, bool live, float (&v)[8]) {
  if constexpr (VEC && sizeof(T) == 4) {
    const float4 z = make_float4(0.f, 0.f, 0.f, 0.f);
    const float4 a = live && k < dim ? *reinterpret_cast<const float4*>(p + k) : z;
    const float4 b = live && k + 4 < dim ? *reinterpret_cast<const float4*>(p + k + 4) : z;
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else if constexpr (VEC) {
    const uint4 u = live && k < dim ? *reinterpret_cast<const uint4*>(p + k) : make_uint4(0u, 0u, 0u, 0u);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[2 * j] = __uint_as_float(w[j] << 16);
      v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = live && k + j < dim ? to_f32(p[k + j]) : 0.f;
  }
}

template <typename T, bool VEC, bool CAP>
__global__ void __launch_bounds__(256) token_logprobs_simt_kernel(const __grid_constant__ LogprobArgs a) {
  extern __shared__ __align__(16) float lp_smem[];
  float(*sA)[132] = reinterpret_cast<float(*)[132]>(lp_smem);
  float(*sB)[132] = reinterpret_cast<float(*)[132]>(lp_smem + 16 * 132);
  float* sC = lp_smem + 2 * 16 * 132;
  float* lx = sC + 128 * kLogprobSimtLdc;
  int32_t* lid = reinterpret_cast<int32_t*>(lx + 128 * a.top);
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const int lr = tid >> 1, lk = (tid & 1) * 8;  // row and first k this thread loads
  for (int unit = blockIdx.x; unit < a.num_m * a.splits; unit += gridDim.x) {
    const int m0 = unit % a.num_m * 128, split = unit / a.num_m;
    const int n_end = split_begin(split + 1, a.num_n, a.splits);
    RowState st;
    if (tid < 128) list_clear(lx, lid, a.top, tid);
    const T* pa = static_cast<const T*>(a.hidden) + (m0 + lr) * a.ldh;
    const bool la = m0 + lr < a.rows;
    for (int n = split_begin(split, a.num_n, a.splits); n < n_end; ++n) {
      const int n0 = n * 128;
      const T* pb = static_cast<const T*>(a.head) + static_cast<long long>(n0 + lr) * a.ldw;
      const bool lb = n0 + lr < a.vocab;
      float va[8], vb[8], acc[8][8] = {};
      load8<T, VEC>(pa, lk, a.dim, la, va);
      load8<T, VEC>(pb, lk, a.dim, lb, vb);
      for (int k0 = 0; k0 < a.dim; k0 += 16) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          sA[lk + j][lr] = va[j];
          sB[lk + j][lr] = vb[j];
        }
        __syncthreads();
        if (k0 + 16 < a.dim) {
          load8<T, VEC>(pa, k0 + 16 + lk, a.dim, la, va);
          load8<T, VEC>(pb, k0 + 16 + lk, a.dim, lb, vb);
        }
#pragma unroll
        for (int kk = 0; kk < 16; ++kk) {
          float fa[8], fb[8];
          *reinterpret_cast<float4*>(fa) = *reinterpret_cast<const float4*>(&sA[kk][ty * 4]);
          *reinterpret_cast<float4*>(fa + 4) = *reinterpret_cast<const float4*>(&sA[kk][64 + ty * 4]);
          *reinterpret_cast<float4*>(fb) = *reinterpret_cast<const float4*>(&sB[kk][tx * 4]);
          *reinterpret_cast<float4*>(fb + 4) = *reinterpret_cast<const float4*>(&sB[kk][64 + tx * 4]);
#pragma unroll
          for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) acc[i][j] = fmaf(fa[i], fb[j], acc[i][j]);
        }
        __syncthreads();
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float* row = sC + (i / 4 * 64 + ty * 4 + i % 4) * kLogprobSimtLdc;
        *reinterpret_cast<float4*>(row + tx * 4) = make_float4(acc[i][0], acc[i][1], acc[i][2], acc[i][3]);
        *reinterpret_cast<float4*>(row + 64 + tx * 4) = make_float4(acc[i][4], acc[i][5], acc[i][6], acc[i][7]);
      }
      __syncthreads();
      if (tid < 128 && m0 + tid < a.rows) {
#pragma unroll 1
        for (int c = 0; c < 128 && n0 + c < a.vocab; c += 32) {
          float x[32];
#pragma unroll
          for (int j = 0; j < 8; ++j)
            *reinterpret_cast<float4*>(x + 4 * j) = *reinterpret_cast<const float4*>(sC + tid * kLogprobSimtLdc + c + 4 * j);
          scan32<CAP>(st, x, n0 + c, a.vocab - n0 - c, a.softcap, lx, lid, a.top, tid);
        }
      }
      // the next tile writes sC only after its own barriers
    }
    if (tid < 128 && m0 + tid < a.rows) store_state(a, st, split, m0 + tid, lx, lid, tid);
  }
}

// ---------------------------------------------------------------------------
// joining the splits; the given tokens
// ---------------------------------------------------------------------------

struct FinishArgs {
  LogprobArgs l;
  const int32_t* targets;  // [rows, n_targets]
  int n_targets;
  float* logprobs;         // [rows, n_targets]
  float* entropy;          // [rows] or nullptr
  int32_t* top_ids;        // [rows, top]
  float* top_logprobs;
};

// One block a row: warp 0 joins states and lists, then the warps take the
// targets in turn, a dot product each.
template <typename T, bool VEC, bool CAP>
__global__ void __launch_bounds__(128) token_logprobs_finish_kernel(const __grid_constant__ FinishArgs f) {
  constexpr float LN2 = 0.6931471805599453f;
  const LogprobArgs& a = f.l;
  __shared__ float s_lse;
  const int row = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp == 0) {
    float m = -INFINITY;
    for (int i = lane; i < a.splits; i += 32) m = fmaxf(m, a.part_m[static_cast<size_t>(i) * a.rows + row]);
    m = warp_max(m);
    float s = 0.f, t = 0.f;
    for (int i = lane; i < a.splits; i += 32) {
      const size_t at = static_cast<size_t>(i) * a.rows + row;
      const float step = a.part_m[at] - m, w = exp2f(step), si = a.part_s[at];
      s = fmaf(w, si, s);
      if (w != 0.f) t = fmaf(w, fmaf(step, si, a.part_t[at]), t);
    }
    s = warp_sum(s);
    t = warp_sum(t);
    const float lse = (m + log2f(s)) * LN2;
    if (lane == 0) {
      s_lse = lse;
      if (f.entropy) f.entropy[row] = logf(s) - LN2 * (t / s);
    }
    if (a.top > 0) {
      // lane i owns the lists of splits i, i + 32, ..; each round takes the
      // largest of the lanes' heads, the lowest id among equals
      constexpr int kOwn = 8;  // splits <= 256
      int head[kOwn] = {};
      for (int j = 0; j < a.top; ++j) {
        float bx = -INFINITY;
        int bid = INT32_MAX, own = -1;
#pragma unroll
        for (int o = 0; o < kOwn; ++o) {
          const int i = lane + 32 * o;
          if (i < a.splits && head[o] < a.top) {
            const size_t at = (static_cast<size_t>(i) * a.rows + row) * a.top + head[o];
            const int id = a.list_id[at];
            const float x = a.list_x[at];
            if (id >= 0 && (x > bx || (x == bx && id < bid))) bx = x, bid = id, own = o;
          }
        }
        float wx = bx;
        int wid = bid;
#pragma unroll
        for (int w = 16; w > 0; w >>= 1) {
          const float ox = __shfl_xor_sync(0xffffffffu, wx, w);
          const int oid = __shfl_xor_sync(0xffffffffu, wid, w);
          if (ox > wx || (ox == wx && oid < wid)) wx = ox, wid = oid;
        }
        if (own >= 0 && bid == wid) {
#pragma unroll
          for (int o = 0; o < kOwn; ++o)
            if (o == own) ++head[o];
        }
        if (lane == 0) {
          const bool some = wid != INT32_MAX;
          f.top_ids[static_cast<size_t>(row) * a.top + j] = some ? wid : -1;
          f.top_logprobs[static_cast<size_t>(row) * a.top + j] = some ? capped<CAP>(wx, a.softcap) - lse : -INFINITY;
        }
      }
    }
  }
  __syncthreads();
  const float lse = s_lse;
  const T* h = static_cast<const T*>(a.hidden) + row * a.ldh;
  for (int c = warp; c < f.n_targets; c += 4) {
    const size_t at = static_cast<size_t>(row) * f.n_targets + c;
    const int id = f.targets[at];
    float x = 0.f;
    if (id >= 0 && id < a.vocab) {
      const T* w = static_cast<const T*>(a.head) + id * a.ldw;
      float p[8] = {};
      for (int k = lane * 8; k < a.dim; k += 256) {
        float u[8], v[8];
        load8<T, VEC>(h, k, a.dim, true, u);
        load8<T, VEC>(w, k, a.dim, true, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) p[j] = fmaf(u[j], v[j], p[j]);
      }
      x = warp_sum(((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7])));
      x = capped<CAP>(x, a.softcap) - lse;
    } else if (id >= a.vocab) {
      x = __int_as_float(0x7fffffff);  // NaN: no such token
    }
    if (lane == 0) f.logprobs[at] = x;
  }
}

}  // namespace clef
