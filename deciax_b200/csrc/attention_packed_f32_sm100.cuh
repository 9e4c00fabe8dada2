// Packed causal attention (attention_packed.cuh) in FP32 on the 5th-generation
// tensor cores, heads up to 128 (computed as 64 or 128): every value is the sum
// of three bf16 parts, x = h + m + l to 2^-24, and a product of two values is
// the six products of their parts that matter,
//   h h',  then  l h' + h l' + m m' + m h' + h m'
// in an accumulator of their own: the tensor core cuts a sum off at the last
// place of its largest term, which the five small ones would not survive.
//
// split_heads_kernel writes the parts of Q, K and V to scratch once (a key is
// read by every query tile behind it); the tile kernel is the bf16 one with
// three operand planes, one CTA = 128 rows of one head, 352 threads:
//   warp 0      TMA: Q, then the K and V tiles of 64 keys from the diagonal down
//   warp 1      issues S = Q K^T (48 MMAs a tile at d = 128), warp 2 O += P V (24)
//   warps 3..10 softmax, two warps a row: a row's parts exchange their maxima
//               every tile (exact online softmax), P goes back over its scores
//               as three parts
// Q, one K and one V stage fill 192 KB of shared memory, two S buffers and O
// (two accumulators each) the tensor memory's 512 columns.  Heads above 128 do
// not fit and run on the CUDA cores (365 us for the work below at heads of 256).
//
// 2047 rows in records of 512, 16 heads of 128, window 200, capped: 63 us, 12 of
// them the split (84 MB, HBM bound); one sequence of 2048, no window: 118 us.
// Q from shared memory bounds the scores' MMAs (64 keys a tile: 6 KB read for 16
// cycles of products) and the single stages a tile's loads.
#pragma once

#include "attention_packed.cuh"
#include "attention_packed_sm100.cuh"
#include "attention_sm100.cuh"
#include "common.cuh"

namespace clef {

struct SplitHeadsArgs {
  const float* x[3];  // q, k, v
  long long ld[3], hs[3];
  int heads[3];
  __nv_bfloat16* out[3];  // [3 parts][tokens][heads][d8]
  int tokens, d, d8;      // d8 = d rounded up to 8, zeros behind d
  bool vec;               // rows are 16-byte aligned and d % 4 == 0
};

// Eight elements of a row a thread.
__global__ void __launch_bounds__(256) split_heads_kernel(const __grid_constant__ SplitHeadsArgs a) {
  const int per_row = a.d8 / 8, heads = a.heads[0] + a.heads[1] + a.heads[2];
  const long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= static_cast<long long>(a.tokens) * heads * per_row) return;
  const long long item = i / per_row;
  const int c = static_cast<int>(i - item * per_row) * 8, t = static_cast<int>(item / heads);
  int h = static_cast<int>(item % heads), which = 0;
  while (h >= a.heads[which]) h -= a.heads[which++];
  const float* x = a.x[which] + t * a.ld[which] + h * a.hs[which] + c;
  float v[8];
  if (a.vec) {
    const float4 z = make_float4(0.f, 0.f, 0.f, 0.f);
    const float4 lo = *reinterpret_cast<const float4*>(x), hi = c + 4 < a.d ? *reinterpret_cast<const float4*>(x + 4) : z;
    v[0] = lo.x, v[1] = lo.y, v[2] = lo.z, v[3] = lo.w, v[4] = hi.x, v[5] = hi.y, v[6] = hi.z, v[7] = hi.w;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = c + e < a.d ? x[e] : 0.f;
  }
  uint4 p[3];
  split3(v[0], v[1], p[0].x, p[1].x, p[2].x);
  split3(v[2], v[3], p[0].y, p[1].y, p[2].y);
  split3(v[4], v[5], p[0].z, p[1].z, p[2].z);
  split3(v[6], v[7], p[0].w, p[1].w, p[2].w);
  const long long plane = static_cast<long long>(a.tokens) * a.heads[which] * a.d8;
  __nv_bfloat16* out = a.out[which] + (static_cast<long long>(t) * a.heads[which] + h) * a.d8 + c;
#pragma unroll
  for (int k = 0; k < 3; ++k) *reinterpret_cast<uint4*>(out + k * plane) = p[k];
}

template <int D>
struct AttnPackedF32Shape {
  static constexpr int BQ = 128, BK = 64, ATOMS = D / 64, FIRST = 96, THREADS = FIRST + 256;
  static constexpr uint32_t Q_PART = BQ * D * 2, KV_PART = BK * D * 2;  // ATOMS x [rows x 128 B]
  // columns: two S buffers of 2 x BK (sums of h h', sums of the others), then O twice
  static constexpr uint32_t S_BUF = 2 * BK, O_COL = 2 * S_BUF, TMEM_COLS = 512;
  static constexpr size_t SMEM = 1024 + 3 * Q_PART + 6 * KV_PART + 256 + 6 * 128 * 4;
  static_assert(O_COL + 2 * D <= TMEM_COLS, "tensor memory");
  static_assert(BQ * D * 4 <= 3 * Q_PART, "the result is staged in the Q parts");
  static_assert(SMEM <= 227 * 1024, "shared memory");
};

// Tensor maps of the parts: [d8][head][3 tokens], boxes of 64 x 1 x 64.
struct AttnPackedF32Maps {
  CUtensorMap q, k, v;
};

template <int D, bool CAP>
__global__ void __launch_bounds__(AttnPackedF32Shape<D>::THREADS, 1)
    attn_packed_f32_tc_kernel(const __grid_constant__ AttnPackedF32Maps maps,
                              const __grid_constant__ AttnPackedArgs<float> a, bool vec, bool vec_in) {
  using Sh = AttnPackedF32Shape<D>;
  constexpr int BQ = Sh::BQ, BK = Sh::BK, ATOMS = Sh::ATOMS;
  constexpr uint32_t IDESC_QK = idesc_bf16_f32(BQ, BK);
  constexpr uint32_t IDESC_PV = idesc_bf16_f32(BQ, D) | (1u << 16);  // B (V) is MN-major
  constexpr float LOG2E = 1.4426950408889634f;
  constexpr int A[6] = {0, 2, 0, 1, 1, 0}, B[6] = {0, 0, 2, 1, 0, 1};  // parts of the six products, h h' first

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;                       // three parts each
  uint8_t* sK = sQ + 3 * Sh::Q_PART;
  uint8_t* sV = sK + 3 * Sh::KV_PART;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sV + 3 * Sh::KV_PART);
  uint64_t* qfull = bars;
  uint64_t* kfull = bars + 1;
  uint64_t* kempty = bars + 2;
  uint64_t* vfull = bars + 3;
  uint64_t* vempty = bars + 4;
  uint64_t* sfull = bars + 5;   // [2]
  uint64_t* pfull = bars + 7;   // [2]
  uint64_t* pempty = bars + 9;  // [2]
  uint64_t* ofull = bars + 11;
  uint64_t* ofinal = bars + 12;
  uint64_t* drain = bars + 13;  // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 15);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* s_begin = abort_flag + 1;  // first key of the tile's first row
  uint32_t* s_nan = tmem_slot + 3;         // [4] rows that came out infinite or NaN
  float* xbuf = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(bars) + 256);  // maxima [2][2][128], sums [2][128]

  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const int h = blockIdx.x, q0 = (static_cast<int>(gridDim.y) - 1 - static_cast<int>(blockIdx.y)) * BQ;
  const int hk = h / (a.H / a.Hk);
  const int k_end = q0 + BQ;  // tile t holds keys k_end - (t + 1) BK ..
  // rows behind the last one hold the next part's: no row of a sequence sees them
  auto load_parts = [&](uint8_t* dst, const CUtensorMap* map, uint64_t* bar, int head, int row, int rows) {
    mbar_arrive_expect_tx(bar, 3 * ATOMS * rows * 128);
    for (int p = 0; p < 3; ++p)
      for (int at = 0; at < ATOMS; ++at)
        for (int bx = 0; bx < rows; bx += 64)
          tma_load_3d(dst + ((p * ATOMS + at) * rows + bx) * 128, map, bar, at * 64, head, p * a.tokens + row + bx);
  };
  int first, total, seq_start = 0;
  packed_extent(a, first, total);
  const int q_end = min(q0 + BQ, total), q_first = max(q0, first);
  if (q_first >= q_end) {  // no row of this tile belongs to a sequence
    // what follows this kernel counts on the parts being written, even where no tile reads them
    asm volatile("griddepcontrol.wait;" ::: "memory");
    return;
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < 15; ++i) mbar_init(&bars[i], i == 7 || i == 8 ? 256 : 1);  // pfull: every softmax thread
    *abort_flag = 0;
    s_nan[0] = s_nan[1] = s_nan[2] = s_nan[3] = 0u;
    fence_barrier_init();
    fence_async_smem();
    // launched while the parts are still being written: only these loads wait for them
    asm volatile("griddepcontrol.wait;" ::: "memory");
    load_parts(sQ, &maps.q, qfull, h, q0, BQ);
    load_parts(sK, &maps.k, kfull, hk, k_end - BK, BK);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, Sh::TMEM_COLS);
    tmem_relinquish();
  }
  if (warp == 3) {
    packed_seq_warp(a.cu, a.n_seqs, q0, lane, seq_start);
    if (q_first != q0) seq_start = first;  // the first sequence starts inside the tile
    const int start = min(max(seq_start, 0), q_first);
    if (lane == 0) *s_begin = a.window > 0 ? max(start, q_first - a.window + 1) : start;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int n = (k_end - *s_begin + BK - 1) / BK;  // the lowest tile starts at key 0 or above: BQ is a multiple of BK

  if (warp == 0) {
    if (lane == 0) {
      int nk = 1, nv = 0;  // tiles whose K / V load has been issued
      for (int i = 0; i <= n && !*abort_flag; ++i) {
        if (i > 0 && i < n) {
          if (!mbar_wait(kempty, (i & 1) ^ 1, a.status, kTimeoutAttention)) {
            *abort_flag = 1;
            break;
          }
          load_parts(sK, &maps.k, kfull, hk, k_end - (i + 1) * BK, BK);
          nk = i + 1;
        }
        if (i >= 1) {
          if (!mbar_wait(vempty, ((i - 1) & 1) ^ 1, a.status, kTimeoutAttention)) {
            *abort_flag = 1;
            break;
          }
          load_parts(sV, &maps.v, vfull, hk, k_end - i * BK, BK);
          nv = i;
        }
      }
      // every issued load must land before the CTA may exit
      mbar_wait(qfull, 0, a.status, kTimeoutDrain);
      mbar_wait(kfull, (nk - 1) & 1, a.status, kTimeoutDrain);
      if (nv > 0) mbar_wait(vfull, (nv - 1) & 1, a.status, kTimeoutDrain);
    }
  } else if (warp < 3) {
    const uint64_t q_desc = smem_desc_k128(smem_u32(sQ)), k_desc = smem_desc_k128(smem_u32(sK));
    const uint64_t v_desc = smem_desc_mn128(smem_u32(sV), BK * 128);
    auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
      return __all_sync(0xffffffffu, mbar_wait(bar, parity, a.status, kTimeoutAttention));
    };
    auto issue_qk = [&](int t) -> bool {
      const int s = t & 1;
      if (!wait(kfull, t & 1) || !wait(&pempty[s], ((t >> 1) & 1) ^ 1)) return false;
      tc_fence_after();
      if (elect_one()) {
        const uint32_t sum = tmem + s * Sh::S_BUF;
#pragma unroll 1
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t w = kk & 3, q_at = (kk >> 2) * (BQ * 128) + w * 32, k_at = (kk >> 2) * (BK * 128) + w * 32;
#pragma unroll
          for (int p = 0; p < 6; ++p)
            umma_bf16(p == 0 ? sum : sum + BK, q_desc + ((A[p] * Sh::Q_PART + q_at) >> 4),
                      k_desc + ((B[p] * Sh::KV_PART + k_at) >> 4), IDESC_QK, (kk > 0 || p > 1) ? 1u : 0u);
        }
        umma_commit(kempty);
        umma_commit(&sfull[s]);
      }
      __syncwarp();
      return true;
    };
    auto issue_pv = [&](int u) -> bool {
      const int s = u & 1;
      if (!wait(vfull, u & 1)) return false;
      const int live = total - (k_end - (u + 1) * BK);  // value rows of this tile that belong to a sequence
      if (live < BK) {
        // rows behind the last sequence hold anything: zero times it is not zero
        for (int i = max(live, 0) * 8 + lane; i < BK * 8; i += 32)
          for (int at = 0; at < 3 * ATOMS; ++at)
            *reinterpret_cast<uint4*>(sV + at * (BK * 128) + i * 16) = make_uint4(0u, 0u, 0u, 0u);
        fence_async_smem();
        __syncwarp();
      }
      if (!wait(&pfull[s], (u >> 1) & 1)) return false;
      tc_fence_after();
      if (elect_one()) {
        constexpr uint32_t P[3] = {0, 16, BK};  // where a share's part of P lies, from the start of its scores
#pragma unroll 1
        for (int kk = 0; kk < BK / 16; ++kk) {
          const uint32_t p_at = tmem + s * Sh::S_BUF + (kk >> 1) * 32 + (kk & 1) * 8;  // 16 keys = 8 columns; 32 keys a share
#pragma unroll
          for (int p = 0; p < 6; ++p)
            umma_bf16_ts(tmem + Sh::O_COL + (p == 0 ? 0 : D), p_at + P[A[p]],
                         v_desc + ((B[p] * Sh::KV_PART + kk * (16 * 128)) >> 4), IDESC_PV,
                         (u > 0 || kk > 0 || p > 1) ? 1u : 0u);
        }
        umma_commit(vempty);
        umma_commit(&pempty[s]);
        umma_commit(ofull);
      }
      __syncwarp();
      return true;
    };
    bool ok = warp == 2 || wait(qfull, 0);
    for (int t = 0; ok && t < n; ++t) ok = warp == 1 ? issue_qk(t) : issue_pv(t);
    if (elect_one()) {
      if (!ok) *abort_flag = 1;
      if (warp == 2) umma_commit(ofinal);
      umma_commit(&drain[warp - 1]);
      mbar_wait(&drain[warp - 1], 0, a.status, kTimeoutDrain);
    }
  } else {
    // two warps per TMEM lane quarter: part p of row r takes keys [32 p, 32 p + 32)
    // of every tile and O columns [p D/2, (p + 1) D/2)
    constexpr int NT = 256, DP = D / 2;
    const int q4 = warp & 3, part = (warp - 3) >> 2, c0 = part * 32;
    const int r = q4 * 32 + lane, row = q0 + r;
    const bool live = row >= q_first && row < q_end;
    int lo = row + 1;  // no key for a row outside the sequences
    {
      const int w0 = max(q0 + q4 * 32, q_first), w1 = min(q0 + q4 * 32 + 31, q_end - 1);
      if (w0 <= w1) {
        int start;
        const int s0 = packed_seq_warp(a.cu, a.n_seqs, w0, lane, start), s1 = packed_seq_warp(a.cu, a.n_seqs, w1, lane, start);
        if (live) lo = packed_first_key(a, row, s0, s1);
      }
    }
    const int lo_max = __reduce_max_sync(0xffffffffu, lo), lo_min = __reduce_min_sync(0xffffffffu, lo);
    const int w_first = q0 + q4 * 32, w_last = w_first + 31;
    const uint32_t lanes = static_cast<uint32_t>(q4 * 32) << 16;
    const float scale = rsqrtf(static_cast<float>(a.d)), scale_cap = scale * inverse_cap(a.softcap);
    const float scale_log2 = CAP ? LOG2E : scale * LOG2E;  // a capped score is scaled already
    float m = -INFINITY, l = 0.f;  // the maximum P is taken against (log2 units); this part's sum
    bool fail = false;  // a failed wait: the two warps of a row leave together, by their exchange
    bool ok = true;
    for (int t = 0; t < n; ++t) {
      const int s = t & 1, k0 = k_end - (t + 1) * BK + c0;
      if (!fail) {
        const bool ready = mbar_wait(&sfull[s], (t >> 1) & 1, a.status, kTimeoutAttention);
        __syncwarp();
        fail = !__all_sync(0xffffffffu, ready);
      }
      tc_fence_after();
      const uint32_t at = tmem + lanes + s * Sh::S_BUF + c0;  // this part's scores, then its P
      const bool none = k0 > w_last || k0 + 31 < lo_min;     // keys that every row of the warp masks
      uint32_t z[32];
      float mt = -INFINITY;
      if (!fail && !none) {
        uint32_t small[32];
        tmem_ld32(at, z);
        tmem_ld32(at + BK, small);
        tmem_wait_ld();
#pragma unroll
        for (int c = 0; c < 32; ++c) z[c] = __float_as_uint(__uint_as_float(z[c]) + __uint_as_float(small[c]));
        if constexpr (CAP) cap_scores(z, scale_cap, a.softcap);
        if (k0 + 31 > w_first || k0 < lo_max) {  // some key is masked for some row of the warp
          const int top = row - k0, low = lo - k0;
#pragma unroll
          for (int c = 0; c < 32; ++c) z[c] = c >= low && c <= top ? z[c] : 0xff800000u;  // -inf
        }
        float best[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < 32; c += 2)
          best[c / 2 & 3] = max3(best[c / 2 & 3], __uint_as_float(z[c]), __uint_as_float(z[c + 1]));
        mt = fmaxf(fmaxf(best[0], best[1]), fmaxf(best[2], best[3])) * scale_log2;
      }
      float* mine = xbuf + (t & 1) * 256;
      mine[part * 128 + r] = mt;
      if (bar_red_or(4 + q4, 64, fail)) {
        ok = false;
        break;
      }
      const float mn = fmaxf(m, fmaxf(mt, mine[(part ^ 1) * 128 + r]));
      // the parts of a row see the same m and mn, so they decide alike
      if (__any_sync(0xffffffffu, mn > m + 8.f)) {
        const float corr = mn == -INFINITY ? 1.f : ex2_approx(m - mn);
        if (t > 0) {  // O must hold P_{t-1} V_{t-1} before it is rescaled
          const bool done = mbar_wait(ofull, (t - 1) & 1, a.status, kTimeoutAttention);
          __syncwarp();
          fail = !__all_sync(0xffffffffu, done);
          tc_fence_after();
          if (!fail) {
#pragma unroll 1
            for (int c = 0; c < 2 * DP; c += 16) {
              const uint32_t o_at = tmem + lanes + Sh::O_COL + (c < DP ? part * DP + c : D + part * DP + c - DP);
              uint32_t o[16];
              tmem_ld16(o_at, o);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * corr);
              tmem_st16(o_at, o);
            }
            tmem_wait_st();
          }
        }
        m = mn;
        l *= corr;
      }
      // P = exp2(z scale_log2 - m) in three parts: P_h over the sums of h h' with P_m behind it, P_l over the others
      const float neg_m = m == -INFINITY ? 0.f : -m;  // no key yet: every p is exp2(-inf) = 0
      const uint64_t scale2 = pair2(scale_log2, scale_log2), neg_m2 = pair2(neg_m, neg_m);
      uint64_t ps[2] = {0ull, 0ull};  // sums of even and odd keys
      uint32_t ph[16], pm[16], pl[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        if (none) {
          ph[e] = pm[e] = pl[e] = 0u;
        } else {
          const float2 x = unpair2(fma2(pair2(__uint_as_float(z[2 * e]), __uint_as_float(z[2 * e + 1])), scale2, neg_m2));
          const float p0 = ex2_approx(x.x), p1 = ex2_approx(x.y);
          ps[e & 1] = add2(ps[e & 1], pair2(p0, p1));
          split3(p0, p1, ph[e], pm[e], pl[e]);
        }
      }
      if (!fail) {
        tmem_st16(at, ph);
        tmem_st16(at + 16, pm);
        tmem_st16(at + BK, pl);
        tmem_wait_st();
      }
      tc_fence_before();
      mbar_arrive(&pfull[s]);
      const float2 sum = unpair2(add2(ps[0], ps[1]));
      l += sum.x + sum.y;
    }
    ok = ok && !fail;
    if (!ok) *abort_flag = 1;
    // the row sum: the parts' sums, added in part order
    float* lbuf = xbuf + 512;
    lbuf[part * 128 + r] = l;
    const bool fin = ok && mbar_wait(ofinal, 0, a.status, kTimeoutAttention);
    const bool out_ok = !bar_red_or(1, NT, !fin);  // every softmax warp agrees
    if (!out_ok) *abort_flag = 1;
    if (out_ok) {
      l = lbuf[r] + lbuf[128 + r];
      tc_fence_after();
      // The row goes through the Q parts (free: every MMA has completed), 16-byte
      // chunks swizzled by the row, so that gates and results move by whole lines.
      float* stage = reinterpret_cast<float*>(sQ);
      auto place = [&](int rr, int chunk) { return rr * D + ((chunk ^ (rr & 7)) << 2); };
      const float inv = 1.f / l;
      float odd = 0.f;  // sum of 0 * y: NaN once a y is infinite or NaN
#pragma unroll 1
      for (int c = part * DP; c < (part + 1) * DP; c += 16) {
        uint32_t big[16], small[16];
        tmem_ld16(tmem + lanes + Sh::O_COL + c, big);
        tmem_ld16(tmem + lanes + Sh::O_COL + D + c, small);
        tmem_wait_ld();
#pragma unroll
        for (int v4 = 0; v4 < 4; ++v4) {
          float y[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            y[e] = (__uint_as_float(big[4 * v4 + e]) + __uint_as_float(small[4 * v4 + e])) * inv;
            odd = fmaf(0.f, y[e], odd);
          }
          *reinterpret_cast<float4*>(stage + place(r, c / 4 + v4)) = make_float4(y[0], y[1], y[2], y[3]);
        }
      }
      // infinite values and products have no parts: such a row is computed again, even where its sum is NaN
      const unsigned bad_rows = __ballot_sync(0xffffffffu, odd != 0.f && live);
      if (lane == 0 && bad_rows) atomicOr(&s_nan[q4], bad_rows);
      asm volatile("bar.sync 1, %0;" ::"n"(NT) : "memory");
      const int chunks = (a.d + 3) / 4;
      for (int idx = static_cast<int>(threadIdx.x) - Sh::FIRST; idx < BQ * chunks; idx += NT) {
        const int rr = idx / chunks, ch = idx - rr * chunks;
        const long long to = q0 + rr;
        if (to < q_first || to >= q_end) continue;
        float4 y = *reinterpret_cast<const float4*>(stage + place(rr, ch));
        const float* g = a.gate + to * a.ldg + h * a.hsg + 4 * ch;
        float* out = a.out + to * a.ldo + h * a.hso + 4 * ch;
        if (vec) {
          if (a.gate) {
            const float4 gv = *reinterpret_cast<const float4*>(g);
            y.x *= sigmoidf_exact(gv.x), y.y *= sigmoidf_exact(gv.y), y.z *= sigmoidf_exact(gv.z), y.w *= sigmoidf_exact(gv.w);
          }
          *reinterpret_cast<float4*>(out) = y;
        } else {
          const float yy[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (4 * ch + e < a.d) out[e] = a.gate ? yy[e] * sigmoidf_exact(g[e]) : yy[e];
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, Sh::TMEM_COLS);
  if (*abort_flag) {
    attn_packed_give_up<float, Sh::THREADS>(a, h, q_first, q_end);
    return;
  }
  if (s_nan[0] | s_nan[1] | s_nan[2] | s_nan[3]) {
    if (vec_in)
      attn_packed_redo<float, true>(a, h, q0, s_nan, 4, reinterpret_cast<float*>(sQ));
    else
      attn_packed_redo<float, false>(a, h, q0, s_nan, 4, reinterpret_cast<float*>(sQ));
  }
}

}  // namespace clef
