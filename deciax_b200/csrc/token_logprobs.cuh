// Log probabilities of given tokens under the language head, with the entropy
// of each row's distribution and its top alternatives:
//
//   x = h W^T,  z = cap(x) = softcap tanh(x / softcap) or x
//   lse = log sum_v exp z_v,   logp(t) = z_t - lse,   H = lse - sum_v p_v z_v
//
// The [rows, vocab] logits never exist: each vocabulary tile's scores go from
// the accumulators straight into a running state per row,
//   m = max z,  s = sum exp(z - m),  t = sum exp(z - m) (z - m)   (log2 units),
// and a list of the largest x with their ids.  The vocabulary is split into S
// runs of columns, so that few rows still fill the GPU; a run of a row
// tile is one unit of work and leaves its rows' states and lists in scratch.
// token_logprobs_finish_kernel joins the S states and lists of a row and takes the
// given tokens' scores from their own dot products.
//
// With s and t joined at m = max m_i:  H = ln s - ln2 t / s.
//
// Here: the state, the joining kernel, and the CUDA-core form (rows that are not
// 16-byte aligned).  token_logprobs_sm100.cuh has the tensor-core form.
#pragma once

#include "common.cuh"

namespace clef {

constexpr int kTopMax = 32;
constexpr int kLogprobMaxSplits = 256;

struct LogprobArgs {
  const void* hidden;
  const void* head;
  long long ldh, ldw;
  int rows, vocab, dim;
  float softcap;
  int top;
  // units of work: num_m row tiles x `splits` runs of `run` columns, in tiles of `tile`
  int num_m, splits, run, tile;
  int copies;  // tensor cores, at most 32 (64) rows: the row tile holds them four times (twice)
  // scratch, a row's splits side by side: states {m, s, t, 0} and lists
  float4* part;     // [rows][splits]
  float* list_x;    // [rows][splits][top], largest first
  int32_t* list_id;
  int* status;
};

// First column of a run (one past the last run: the end).
__device__ __forceinline__ int run_begin(const LogprobArgs& a, int split) {
  return static_cast<int>(min(static_cast<long long>(a.vocab), static_cast<long long>(split) * a.run));
}

template <bool CAP>
__device__ __forceinline__ float capped(float x, float softcap) {
  return CAP ? softcap * tanhf(x / softcap) : x;
}

// A row's running sums, in log2 units of z.
struct RowState {
  float m = -INFINITY, s = 0.f, t = 0.f;
};

__device__ __forceinline__ float min_nan(float a, float b) {  // NaN if one is
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// The `top` largest scores of a row, entered by a chunk of 32 columns at a time.
// Ids rise from chunk to chunk, so a score that equals the smallest entry stays
// out.  A free place holds NaN, which no comparison "at most" admits: any score goes
// before it, -inf too (a score of NaN goes nowhere).  Both forms use `area` (shared memory, list_bytes(top) a CTA); r is the
// thread's place in it (0..127).
//
// The list lies in registers, largest first, K = 8 or 32 places.  An insertion is
// K independent comparisons and the moves they choose; a chunk with a candidate is
// laid down in `area` so that a bit mask can walk the candidates.  (Lists in shared memory, and
// the chunk's maximum searched for again for every insertion, took 1100 cycles an
// insertion of a warp: 227 us instead of 104 without a list at 2000 rows x 32000 x 1024.)
template <int K>
struct TopList {
  float v[K];
  int32_t id[K];
  float thr;

  __device__ __forceinline__ void clear(int top) {
#pragma unroll
    for (int j = 0; j < K; ++j) {
      v[j] = __int_as_float(0x7fffffff);
      id[j] = -1;
    }
    thr = top > 0 ? v[0] : INFINITY;
  }
  template <bool ANY_ORDER = false>
  __device__ __forceinline__ void insert(float x, int32_t i, int top) {
    bool before[K];  // x goes before entry j
#pragma unroll
    for (int j = 0; j < K; ++j) before[j] = !(x <= v[j]) || (ANY_ORDER && x == v[j] && i < id[j]);
#pragma unroll
    for (int j = K - 1; j > 0; --j) {
      v[j] = before[j - 1] ? v[j - 1] : before[j] ? x : v[j];
      id[j] = before[j - 1] ? id[j - 1] : before[j] ? i : id[j];
    }
    v[0] = before[0] ? x : v[0];
    id[0] = before[0] ? i : id[0];
    thr = v[0];
#pragma unroll
    for (int j = 1; j < K; ++j) thr = j < top ? min_nan(thr, v[j]) : thr;  // entry top - 1
  }
  // best = the largest of x, of which the first `valid` count
  __device__ __forceinline__ void take(float (&x)[32], float best, int col, int valid, int top, float* area, int r) {
    if (best <= thr) return;
    uint32_t mask[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int c = 0; c < 32; ++c) {
      if (!(x[c] <= thr)) mask[c & 3] |= 1u << c;
      area[c * 128 + r] = x[c];
    }
    const uint32_t exist = valid < 32 ? (1u << valid) - 1 : ~0u;
    for (uint32_t left = ((mask[0] | mask[1]) | (mask[2] | mask[3])) & exist; left; left &= left - 1) {
      const int c = __ffs(static_cast<int>(left)) - 1;
      const float y = area[c * 128 + r];
      if (!(y <= thr) && y == y) insert(y, col + c, top);
    }
  }
  __device__ __forceinline__ void publish(float* area, int r) const {
#pragma unroll
    for (int j = 0; j < K; ++j) {
      area[j * 128 + r] = v[j];
      reinterpret_cast<int32_t*>(area)[(K + j) * 128 + r] = id[j];
    }
  }
  __device__ __forceinline__ void join(int top, float* area, int r, int r2) {
    for (int j = 0; j < top; ++j) {
      const float x = area[j * 128 + r2];
      const int32_t i = reinterpret_cast<const int32_t*>(area)[(K + j) * 128 + r2];
      if (i < 0 || x < thr) break;  // it is sorted
      insert<true>(x, i, top);
    }
  }
  __device__ __forceinline__ void store(int top, float* lx, int32_t* lid) const {
#pragma unroll
    for (int j = 0; j < K; ++j)
      if (j < top) {
        lx[j] = v[j];
        lid[j] = id[j];
      }
  }
};

__device__ __forceinline__ float max32(const float (&x)[32]) {
  float p[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
  for (int c = 4; c < 32; ++c) p[c & 3] = fmaxf(p[c & 3], x[c]);
  return fmaxf(fmaxf(p[0], p[1]), fmaxf(p[2], p[3]));
}

// Shared memory of a CTA's 128 lists.
__host__ __device__ constexpr size_t list_bytes(int top) {
  return top == 0 ? 0 : 128 * (top <= 8 ? 32 : 2 * kTopMax) * sizeof(float);
}

// Scores x of columns col .. col + 31, the first `valid` of which exist.
template <bool CAP, int K>
__device__ __forceinline__ void scan32(RowState& st, TopList<K>& list, float (&x)[32], int col, int valid, float softcap,
                                       int top, float* area, int r) {
  constexpr float LOG2E = 1.4426950408889634f;
  if (valid < 32) {
#pragma unroll
    for (int c = 0; c < 32; ++c)
      if (c >= valid) x[c] = -INFINITY;
  }
  const float best = max32(x);
  const float zmax = capped<CAP>(best, softcap) * LOG2E;
  if (zmax > st.m) {  // the sums move to the new maximum
    const float step = st.m - zmax, f = exp2f(step);
    st.t = st.s == 0.f ? 0.f : f * fmaf(step, st.s, st.t);
    st.s *= f;
    st.m = zmax;
  }
  const float neg_m = st.m == -INFINITY ? 0.f : -st.m;  // no score above -inf yet: exp2(-inf) = 0
  bool done = false;
  if (valid >= 32) {  // two columns at a time
    const uint64_t log2e2 = pair2(LOG2E, LOG2E), neg_m2 = pair2(neg_m, neg_m);
    uint64_t ps[2] = {0ull, 0ull}, pt[2] = {0ull, 0ull};
    auto add = [&](int e, uint64_t z2) {
      const uint64_t d2 = fma2(z2, log2e2, neg_m2);
      const float2 d = unpair2(d2);
      const uint64_t e2 = pair2(ex2_approx(d.x), ex2_approx(d.y));
      ps[e & 1] = add2(ps[e & 1], e2);
      pt[e & 1] = fma2(d2, e2, pt[e & 1]);
    };
    if constexpr (CAP) {
      // tanh by its series where all 32 columns allow it (2e-8 off), else by tanhf
      const float inv = fminf(1.f / softcap, 3e38f);
      const uint64_t inv2 = pair2(inv, inv), cap2 = pair2(softcap, softcap);
      float far = 0.f;
#pragma unroll
      for (int c = 0; c < 32; ++c) far = fmaxf(far, fabsf(x[c]));
      if (far * inv < kTanhSeries) {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const uint64_t y = mul2(pair2(x[2 * e], x[2 * e + 1]), inv2), y2 = mul2(y, y);
          uint64_t p = pair2(kTanh[5], kTanh[5]);
#pragma unroll
          for (int i = 4; i >= 0; --i) p = fma2(p, y2, pair2(kTanh[i], kTanh[i]));
          add(e, mul2(fma2(mul2(y, y2), p, y), cap2));
        }
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) add(e, pair2(capped<CAP>(x[2 * e], softcap), capped<CAP>(x[2 * e + 1], softcap)));
      }
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e) add(e, pair2(x[2 * e], x[2 * e + 1]));
    }
    const float2 s2 = unpair2(add2(ps[0], ps[1])), t2 = unpair2(add2(pt[0], pt[1]));
    const float t = t2.x + t2.y;
    if (t == t) {
      st.s += s2.x + s2.y;
      st.t += t;
      done = true;
    }
  }
  if (!done) {  // few columns, or one of them scores -inf (whose product of 0 and -inf is NaN), +inf or NaN
    float ps = 0.f, pt = 0.f;
#pragma unroll
    for (int c = 0; c < 32; ++c)
      if (c < valid) {
        const float d = fmaf(capped<CAP>(x[c], softcap), LOG2E, neg_m);
        const float e = ex2_approx(d);
        ps += e;
        pt = e == 0.f ? pt : fmaf(d, e, pt);
      }
    st.s += ps;
    st.t += pt;
  }
  list.take(x, best, col, valid, top, area, r);
}

// Joins another state into this one.  A side without columns, or whose columns all score -inf, has m = -inf,
// s = t = 0: it weighs nothing.
__device__ __forceinline__ void join_state(RowState& st, float m, float s, float t) {
  const float mx = fmaxf(st.m, m);
  if (mx == -INFINITY) {  // NaN sums stay
    st.s += s;
    st.t += t;
    return;
  }
  const float d0 = st.m - mx, d1 = m - mx, w0 = exp2f(d0), w1 = exp2f(d1);
  st.t = (w0 == 0.f ? 0.f : w0 * fmaf(d0, st.s, st.t)) + (w1 == 0.f ? 0.f : w1 * fmaf(d1, s, t));
  st.s = w0 * st.s + w1 * s;
  st.m = mx;
}

// Leaves the state, and the list in order, in scratch.
template <int K>
__device__ __forceinline__ void store_state(const LogprobArgs& a, const RowState& st, const TopList<K>& list, int split,
                                            int row) {
  const size_t at = static_cast<size_t>(row) * a.splits + split;
  a.part[at] = make_float4(st.m, st.s, st.t, 0.f);
  list.store(a.top, a.list_x + at * a.top, a.list_id + at * a.top);
}

// In place of a state that a failed wait left out: the row's sums become NaN
// (scratch may hold an earlier call's).
__device__ __forceinline__ void store_no_state(const LogprobArgs& a, int split, int row) {
  const size_t at = static_cast<size_t>(row) * a.splits + split;
  const float nan = __int_as_float(0x7fffffff);
  a.part[at] = make_float4(nan, nan, nan, 0.f);
  for (int j = 0; j < a.top; ++j) a.list_id[at * a.top + j] = -1;
}

// ---------------------------------------------------------------------------
// CUDA cores: 128 x 128 tiles, 8 x 8 a thread, FP32 products and sums
// ---------------------------------------------------------------------------
// Sixteen values of k at a time through shared memory, the next sixteen in
// registers meanwhile; 6 shared-memory wavefronts for 16 cycles of FMA.  A
// finished tile goes through shared memory once more so that a thread scans a row.

constexpr int kLogprobSimtLdc = 132;
constexpr size_t logprob_simt_smem(int top) {
  return (2 * 16 * 132 + 128 * kLogprobSimtLdc) * sizeof(float) + list_bytes(top);
}

template <typename T, bool CAP, int K>
__global__ void __launch_bounds__(256) token_logprobs_simt_kernel(const __grid_constant__ LogprobArgs a) {
  extern __shared__ __align__(16) float lp_smem[];
  float(*sA)[132] = reinterpret_cast<float(*)[132]>(lp_smem);
  float(*sB)[132] = reinterpret_cast<float(*)[132]>(lp_smem + 16 * 132);
  float* sC = lp_smem + 2 * 16 * 132;
  float* area = sC + 128 * kLogprobSimtLdc;
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const int lr = tid >> 1, lk = (tid & 1) * 8;  // row and first k this thread loads
  for (int unit = blockIdx.x; unit < a.num_m * a.splits; unit += gridDim.x) {
    const int m0 = unit % a.num_m * 128, split = unit / a.num_m;
    const int n_end = run_begin(a, split + 1);
    RowState st;
    TopList<K> list;
    list.clear(a.top);
    const T* pa = static_cast<const T*>(a.hidden) + (m0 + lr) * a.ldh;
    const bool la = m0 + lr < a.rows;
    for (int n0 = run_begin(a, split); n0 < n_end; n0 += 128) {
      const T* pb = static_cast<const T*>(a.head) + static_cast<long long>(n0 + lr) * a.ldw;
      const bool lb = n0 + lr < a.vocab;
      float va[8], vb[8], acc[8][8] = {};
      load8<T, false>(pa, lk, a.dim, la, va);
      load8<T, false>(pb, lk, a.dim, lb, vb);
      for (int k0 = 0; k0 < a.dim; k0 += 16) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          sA[lk + j][lr] = va[j];
          sB[lk + j][lr] = vb[j];
        }
        __syncthreads();
        if (k0 + 16 < a.dim) {
          load8<T, false>(pa, k0 + 16 + lk, a.dim, la, va);
          load8<T, false>(pb, k0 + 16 + lk, a.dim, lb, vb);
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
          scan32<CAP>(st, list, x, n0 + c, a.vocab - n0 - c, a.softcap, a.top, area, tid);
        }
      }
      // the next tile writes sC only after its own barriers
    }
    if (tid < 128 && m0 + tid < a.rows) store_state(a, st, list, split, m0 + tid);
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

// x of target c of a row: its own dot product, by a warp.
template <typename T, bool VEC>
__device__ __forceinline__ float target_score(const FinishArgs& f, int row, int c, int lane) {
  const LogprobArgs& a = f.l;
  const int id = f.targets[static_cast<size_t>(row) * f.n_targets + c];
  if (id < 0 || id >= a.vocab) return 0.f;
  const T* h = static_cast<const T*>(a.hidden) + row * a.ldh;
  const T* w = static_cast<const T*>(a.head) + id * a.ldw;
  float p[8] = {};
#pragma unroll 4
  for (int k = lane * 8; k < a.dim; k += 256) {
    float u[8], v[8];
    load8<T, VEC>(h, k, a.dim, true, u);
    load8<T, VEC>(w, k, a.dim, true, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) p[j] = fmaf(u[j], v[j], p[j]);
  }
  return warp_sum(((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7])));
}

// A padded slot (negative id) gives 0, a token that does not exist NaN.
template <bool CAP>
__device__ __forceinline__ void store_logprob(const FinishArgs& f, int row, int c, float x, float lse, int lane) {
  const size_t at = static_cast<size_t>(row) * f.n_targets + c;
  const int id = f.targets[at];
  if (lane == 0)
    f.logprobs[at] = id < 0 ? 0.f : id >= f.l.vocab ? __int_as_float(0x7fffffff) : capped<CAP>(x, f.l.softcap) - lse;
}

// One block a row: each warp takes its targets' dot products, all threads join
// the states and stage the lists, warp 0 joins the lists.
template <typename T, bool VEC, bool CAP>
__global__ void __launch_bounds__(128) token_logprobs_finish_kernel(const __grid_constant__ FinishArgs f) {
  constexpr float LN2 = 0.6931471805599453f;
  constexpr int kOwn = kLogprobMaxSplits / 32;
  const LogprobArgs& a = f.l;
  extern __shared__ float fin_x[];  // [splits * top], then their ids
  int32_t* fin_id = reinterpret_cast<int32_t*>(fin_x + a.splits * a.top);
  __shared__ float s_red[3][4];
  const int row = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  // The targets' products need nothing of the kernel before: they run while it
  // ends.  Each of the first kHeld stays with its warp until lse is known.
  constexpr int kHeld = 2;
  float held[kHeld];
#pragma unroll
  for (int o = 0; o < kHeld; ++o)
    held[o] = warp + 4 * o < f.n_targets ? target_score<T, VEC>(f, row, warp + 4 * o, lane) : 0.f;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  float pm[kLogprobMaxSplits / 128], ps[kLogprobMaxSplits / 128], pt[kLogprobMaxSplits / 128];
  float m = -INFINITY;
#pragma unroll
  for (int o = 0; o < kLogprobMaxSplits / 128; ++o) {
    const int i = tid + 128 * o;
    const float4 p = i < a.splits ? a.part[static_cast<size_t>(row) * a.splits + i] : make_float4(-INFINITY, 0.f, 0.f, 0.f);
    pm[o] = p.x, ps[o] = p.y, pt[o] = p.z;
    m = fmaxf(m, p.x);
  }
  const int entries = a.splits * a.top;
  for (int e = tid; e < entries; e += 128) {
    fin_x[e] = a.list_x[static_cast<size_t>(row) * entries + e];
    fin_id[e] = a.list_id[static_cast<size_t>(row) * entries + e];
  }
  m = warp_max(m);
  if (lane == 0) s_red[0][warp] = m;
  __syncthreads();
  m = fmaxf(fmaxf(s_red[0][0], s_red[0][1]), fmaxf(s_red[0][2], s_red[0][3]));
  float s = 0.f, t = 0.f;
#pragma unroll
  for (int o = 0; o < kLogprobMaxSplits / 128; ++o) {
    const float step = pm[o] - m, w = exp2f(step);
    s = fmaf(w, ps[o], s);
    if (w != 0.f) t = fmaf(w, fmaf(step, ps[o], pt[o]), t);
  }
  s = warp_sum(s);
  t = warp_sum(t);
  if (lane == 0) s_red[1][warp] = s, s_red[2][warp] = t;
  __syncthreads();
  s = (s_red[1][0] + s_red[1][1]) + (s_red[1][2] + s_red[1][3]);
  t = (s_red[2][0] + s_red[2][1]) + (s_red[2][2] + s_red[2][3]);
  const float lse = (m + log2f(s)) * LN2;
  if (tid == 0 && f.entropy) f.entropy[row] = logf(s) - LN2 * (t / s);
  if (warp == 0 && a.top > 0) {
    // lane i owns the lists of splits i, i + 32, ..; each round takes the
    // largest of the lanes' heads, the lowest id among equals
    float hx[kOwn];
    int hid[kOwn], head[kOwn] = {};
    auto load_head = [&](int o) {
      const int i = lane + 32 * o;
      const bool in = i < a.splits && head[o] < a.top;
      const int id = in ? fin_id[i * a.top + head[o]] : -1;
      hx[o] = id >= 0 ? fin_x[i * a.top + head[o]] : -INFINITY;
      hid[o] = id >= 0 ? id : INT32_MAX;
    };
#pragma unroll
    for (int o = 0; o < kOwn; ++o) {
      load_head(o);
    }
    for (int j = 0; j < a.top; ++j) {
      float bx = hx[0];
      int bid = hid[0];
#pragma unroll
      for (int o = 1; o < kOwn; ++o)
        if (hx[o] > bx || (hx[o] == bx && hid[o] < bid)) bx = hx[o], bid = hid[o];
#pragma unroll
      for (int w = 16; w > 0; w >>= 1) {
        const float ox = __shfl_xor_sync(0xffffffffu, bx, w);
        const int oid = __shfl_xor_sync(0xffffffffu, bid, w);
        if (ox > bx || (ox == bx && oid < bid)) bx = ox, bid = oid;
      }
      const bool some = bid != INT32_MAX;
#pragma unroll
      for (int o = 0; o < kOwn; ++o)
        if (some && hid[o] == bid) {  // ids are unique: one lane, one list
          ++head[o];
          load_head(o);
        }
      if (lane == 0) {
        f.top_ids[static_cast<size_t>(row) * a.top + j] = some ? bid : -1;
        f.top_logprobs[static_cast<size_t>(row) * a.top + j] = some ? capped<CAP>(bx, a.softcap) - lse : -INFINITY;
      }
    }
  }
#pragma unroll
  for (int o = 0; o < kHeld; ++o)
    if (warp + 4 * o < f.n_targets) store_logprob<CAP>(f, row, warp + 4 * o, held[o], lse, lane);
  for (int c = warp + 4 * kHeld; c < f.n_targets; c += 4)
    store_logprob<CAP>(f, row, c, target_score<T, VEC>(f, row, c, lane), lse, lane);
}

}  // namespace clef
