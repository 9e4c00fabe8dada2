// Packed causal attention (attention_packed.cuh) on the 5th-generation tensor
// cores: bf16 operands with 16-byte aligned rows, head size a multiple of 8 up
// to 256 (computed as 64, 128 or 256: TMA reads zeros past the head's end).
//
// One CTA = 128 consecutive packed rows of one query head, 352 threads:
//   warp 0      TMA producer: the Q tile, then K and V tiles through one ring
//               each, then the gate tile into the K stages.
//   warp 1      issues tcgen05.mma: S_t = Q K_t^T into one of two TMEM buffers.
//   warp 2      issues O += P_t V_t.
//   warps 3..10 softmax, two warps a row (part 0 and 1: half of every key tile
//               and half of O's columns each): mask, running maximum and sum, P
//               as bf16 back over its S buffer, the A operand of P.V; at the end
//               O / l * sigmoid(gate).
// Key tiles are taken from the diagonal down.  The first one then lies beside
// the query tile: it loads with the queries, before the tile knows where its
// first row's sequence starts, and every row meets its own key at once.  Only
// the diagonal and tiles that reach below some row's first key need a mask.
// P is taken against the maximum of the tiles before the last one: the row's
// parts then exchange their maxima while P.V runs instead of before it (bf16
// has FP32's exponents, so a P above 1 loses nothing); only the first tile's is
// exchanged before its P.  The maximum moves, and O is rescaled, only when it
// grows by more than 2^8.  Where scores jump from one tile to the next by so much
// that P, a sum or an O leaves FP32's range (2^128), the row comes out infinite or
// NaN and is computed again like any that came out NaN, and so is a row whose first
// tile holds no score above -inf.  32 keys that every row of a warp masks leave P = 0
// and nothing else.
//
// D = 256: 128-key tiles, one CTA an SM (Q, K and V stages fill shared memory,
// two S buffers and O the tensor memory).  D <= 128: 64-key tiles, two CTAs
// (128-key tiles leave room for one S buffer: the two CTAs then took turns, and
// serving batches ran 10% slower).
//
// 16 heads, gated: one sequence of 16384, d = 256: 1.9 ms under the power cap
// (1142 TFLOP/s), 1.6 ms alone; records of 600, 16384 rows: 350 us, half of a
// tile's time outside its key loop; 32 heads of 128, records of 1 to 64, 16001
// rows: 150 us.  Bound by the tensor pipe on long sequences (61% busy at 8192
// rows), at d = 128 by issue slots as much, by a tile's start and end on short ones.
// A cap costs most beyond its bend: one sequence of 8192, d = 256, 450 us without
// one, 540 with scores within the series of tanh, 820 beyond it.
//
// Differs from attention_sm100.cuh in what bounds a row's keys, and in the
// rounding: the sigmoid gate multiplies in FP32 and the result is rounded once.
#pragma once

#include "attention_packed.cuh"
#include "attention_sm100.cuh"
#include "common.cuh"

namespace clef {

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
          smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}
__device__ __forceinline__ void tma_store_3d(const CUtensorMap* map, const void* src, int x, int y, int z) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(smem_u32(src)), "r"(x), "r"(y), "r"(z)
               : "memory");
}
__device__ __forceinline__ void tma_prefetch_3d(const CUtensorMap* map, int x, int y, int z) {  // into L2
  asm volatile("cp.async.bulk.prefetch.tensor.3d.L2.global.tile [%0, {%1, %2, %3}];" ::"l"(reinterpret_cast<uint64_t>(map)),
               "r"(x), "r"(y), "r"(z)
               : "memory");
}
// Every store of this thread's bulk groups is complete, not only read.
__device__ __forceinline__ void tma_store_wait_all() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

// Tensor maps [d][head][row] with boxes of 64 x 1 x 64.
struct AttnPackedMaps {
  CUtensorMap q, k, v, gate, out;
};

// The last s in [0, n) with cu[s] <= row, by a whole warp, 32 probes a round
// (0 where there is none).  `start` gets cu[s].
__device__ __forceinline__ int packed_seq_warp(const int32_t* cu, int n, int row, int lane, int& start) {
  int lo = 0;
  start = 0;
  do {
    const int step = (n + 31) >> 5;
    const int at = lane * step;
    const int c = at < n ? cu[lo + at] : INT32_MAX;
    const unsigned hit = __ballot_sync(0xffffffffu, c <= row);
    const int j = hit ? 31 - __clz(hit) : 0;
    start = __shfl_sync(0xffffffffu, c, j);
    lo += j * step;
    n = min(step, n - j * step);
  } while (n > 1);
  return lo;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

__device__ __forceinline__ float max3_nan(float a, float b, float c) {  // NaN if one is
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Scores x = softcap tanh(scale_cap x), 32 of a row.  While none of the warp's
// lies beyond the series of tanh_flat (0.45: scores below 0.42 softcap), the
// series alone, two scores at a time; else tanh_flat for each.
__device__ __forceinline__ void cap_scores(uint32_t (&x)[32], float scale_cap, float softcap) {
  const uint64_t sc2 = pair2(scale_cap, scale_cap), cap2 = pair2(softcap, softcap);
  uint64_t y[16];
  float top = 0.f;
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    y[e] = mul2(pair2(__uint_as_float(x[2 * e]), __uint_as_float(x[2 * e + 1])), sc2);
    const float2 u = unpair2(y[e]);
    top = max3(top, fabsf(u.x), fabsf(u.y));
  }
  if (__any_sync(0xffffffffu, top >= kTanhSeries)) {
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const float2 u = unpair2(y[e]);
      x[2 * e] = __float_as_uint(softcap * tanh_flat(u.x));
      x[2 * e + 1] = __float_as_uint(softcap * tanh_flat(u.y));
    }
  } else {
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const uint64_t y2 = mul2(y[e], y[e]);
      uint64_t p = pair2(kTanh[5], kTanh[5]);
#pragma unroll
      for (int i = 4; i >= 0; --i) p = fma2(p, y2, pair2(kTanh[i], kTanh[i]));
      const float2 t = unpair2(mul2(fma2(mul2(y[e], y2), p, y[e]), cap2));
      x[2 * e] = __float_as_uint(t.x);
      x[2 * e + 1] = __float_as_uint(t.y);
    }
  }
}

// Sigmoids of 8 Q gates (bf16).  Two share one reciprocal, 1/a = b / (ab), for
// the special-function unit gives 16 results a cycle and SM (exponentials from
// the FMA pipe instead, for a quarter or half of them, were no faster).
// The product of two sums 1 + e^-g stays finite while -g log2 e <= 63; a row
// with a gate below -43, or NaN, takes a reciprocal for each.
template <int Q>
__device__ __forceinline__ void sigmoids(const uint4 (&gq)[Q], uint64_t (&sg)[4 * Q]) {
  const uint64_t neg_log2e = pair2(-1.4426950408889634f, -1.4426950408889634f);
  float top = -INFINITY;
#pragma unroll
  for (int q = 0; q < Q; ++q) {
    const uint32_t gw[4] = {gq[q].x, gq[q].y, gq[q].z, gq[q].w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      sg[4 * q + e] = mul2(pair2(__uint_as_float(gw[e] << 16), __uint_as_float(gw[e] & 0xffff0000u)), neg_log2e);
      const float2 t = unpair2(sg[4 * q + e]);
      top = max3_nan(top, t.x, t.y);
    }
  }
  const uint64_t one = pair2(1.f, 1.f);
  if (top <= 63.f) {
#pragma unroll
    for (int e = 0; e < 4 * Q; ++e) {
      const float2 t = unpair2(sg[e]);
      const uint64_t ab = add2(one, pair2(ex2_approx(t.x), ex2_approx(t.y)));
      const float2 d = unpair2(ab);
      const float r = rcp_approx(d.x * d.y);
      sg[e] = mul2(pair2(r, r), pair2(d.y, d.x));
    }
  } else {
#pragma unroll
    for (int e = 0; e < 4 * Q; ++e) {
      const float2 t = unpair2(sg[e]);
      sg[e] = pair2(rcp_approx(1.f + ex2_approx(t.x)), rcp_approx(1.f + ex2_approx(t.y)));
    }
  }
}

template <int D>
struct AttnPackedTcShape {
  static constexpr int BQ = 128, BK = D == 256 ? 128 : 64, ATOMS = D / 64;
  static constexpr int KST = D == 256 ? 1 : 2;   // K and V stages each
  static constexpr int NP = 2;                   // softmax warps a row
  static constexpr int CTAS = D == 256 ? 1 : 2;  // per SM
  static constexpr int FIRST = 96;               // first softmax thread
  static constexpr int THREADS = FIRST + 128 * NP;
  static constexpr uint32_t Q_BYTES = BQ * D * 2;   // ATOMS x [128 rows x 128 B]
  static constexpr uint32_t KV_BYTES = BK * D * 2;  // ATOMS x [BK rows x 128 B]
  static constexpr uint32_t TMEM_COLS = D + 2 * BK <= 256 ? 256 : 512;
  static constexpr uint32_t S_COL = 0, O_COL = 2 * BK;  // S buffers at 0 and BK, O after them
  static constexpr uint32_t XCH_BYTES = 3 * NP * 128 * 4;  // row maxima [2][NP][128], sums [NP][128]
  static constexpr size_t SMEM = 1024 + Q_BYTES + 2 * KST * KV_BYTES + 256 + XCH_BYTES;
  static_assert(D + 2 * BK <= 512 && CTAS * TMEM_COLS <= 512, "tensor memory");
  static_assert(Q_BYTES <= KST * KV_BYTES, "the gate tile is loaded into the K stages");
  static_assert(THREADS / 32 * kRedoState * 4 <= Q_BYTES, "rows computed again join in the Q tile");
  static_assert(CTAS * (SMEM + 1024) <= 228 * 1024, "shared memory");
};

template <int D, bool CAP>
__global__ void __launch_bounds__(AttnPackedTcShape<D>::THREADS, AttnPackedTcShape<D>::CTAS)
    attn_packed_tc_kernel(const __grid_constant__ AttnPackedMaps maps,
                          const __grid_constant__ AttnPackedArgs<__nv_bfloat16> a) {
  using Sh = AttnPackedTcShape<D>;
  constexpr int BQ = Sh::BQ, BK = Sh::BK, ATOMS = Sh::ATOMS, KST = Sh::KST, BKP = BK / Sh::NP;
  constexpr uint32_t IDESC_QK = idesc_bf16_f32(BQ, BK);
  constexpr uint32_t IDESC_PV = idesc_bf16_f32(BQ, D) | (1u << 16);  // B (V) is MN-major
  constexpr float LOG2E = 1.4426950408889634f;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sK = sQ + Sh::Q_BYTES;          // KST stages
  uint8_t* sV = sK + KST * Sh::KV_BYTES;   // KST stages
  uint64_t* bars = reinterpret_cast<uint64_t*>(sV + KST * Sh::KV_BYTES);
  uint64_t* qfull = bars;
  uint64_t* kfull = bars + 1;
  uint64_t* kempty = bars + 3;
  uint64_t* vfull = bars + 5;
  uint64_t* vempty = bars + 7;
  uint64_t* sfull = bars + 9;
  uint64_t* pfull = bars + 11;
  uint64_t* pempty = bars + 13;
  uint64_t* ofull = bars + 15;
  uint64_t* ofinal = bars + 16;
  uint64_t* drain = bars + 17;  // [2]
  uint64_t* gfull = bars + 19;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 20);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* s_begin = abort_flag + 1;  // first key of the tile's first row
  uint32_t* s_nan = tmem_slot + 3;         // [4] rows that came out infinite or NaN
  uint32_t* s_lost = s_nan + 4;            // [4] rows whose first key tile holds no score above -inf
  float* xbuf = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(bars) + 256);  // softmax parts' exchange

  // from a shuffle, so that the compiler knows the warp's index, and what follows from it, to be uniform
  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  // grid (heads side by side, tiles, rounds of heads): of a round's heads the
  // last tiles come first, the longest where sequences are long
  const int h = blockIdx.z * gridDim.x + blockIdx.x, q0 = (static_cast<int>(gridDim.y) - 1 - static_cast<int>(blockIdx.y)) * BQ;
  const int hk = h / (a.H / a.Hk);
  // tile t holds keys k_end - (t + 1) BK .., possibly below the buffer (read as zero)
  const int k_end = q0 + BQ;
  auto load_tile = [&](uint8_t* dst, const CUtensorMap* map, uint64_t* bar, int head, int row, int rows) {
    for (int at = 0; at < ATOMS; ++at)
      for (int bx = 0; bx < rows; bx += 64)
        tma_load_3d(dst + at * (rows * 128) + bx * 128, map, bar, at * 64, head, row + bx);
  };
  if (threadIdx.x == 0) {
    for (int i = 0; i < 20; ++i) {
      const bool softmax_arrives = (i >= 11 && i < 13);  // pfull[2]: one arrive per softmax thread
      mbar_init(&bars[i], softmax_arrives ? 128 * Sh::NP : 1);
    }
    *abort_flag = 0;
    s_nan[0] = s_nan[1] = s_nan[2] = s_nan[3] = 0u;
    s_lost[0] = s_lost[1] = s_lost[2] = s_lost[3] = 0u;
    fence_barrier_init();
    fence_async_smem();
    // the queries and the first keys wait for nothing
    mbar_arrive_expect_tx(qfull, Sh::Q_BYTES);
    load_tile(sQ, &maps.q, qfull, h, q0, BQ);
    mbar_arrive_expect_tx(&kfull[0], Sh::KV_BYTES);
    load_tile(sK, &maps.k, &kfull[0], hk, k_end - BK, BK);
  }
  int first, total, seq_start = 0;
  packed_extent(a, first, total);
  const int q_end = min(q0 + BQ, total), q_first = max(q0, first);
  if (q_first >= q_end) {  // no row of this tile belongs to a sequence
    if (threadIdx.x == 0) {
      mbar_wait(qfull, 0, a.status, kTimeoutDrain);
      mbar_wait(&kfull[0], 0, a.status, kTimeoutDrain);
    }
    return;
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
  const int n = (k_end - *s_begin + BK - 1) / BK;

  if (warp == 0) {
    if (lane == 0) {
      // ---------------- TMA producer ----------------
      // The gate tile's place frees late (below): it waits for it in L2.
      if (a.gate)
        for (int at = 0; at < ATOMS; ++at)
          for (int half = 0; half < 2; ++half) tma_prefetch_3d(&maps.gate, at * 64, h, q0 + half * 64);
      // K runs one tile ahead of V: a K stage frees when its QK^T is done,
      // a V stage only after the (later) P.V that reads it.
      int nk = 1, nv = 0;  // tiles whose K / V load has been issued
      for (int i = 0; i <= n && !*abort_flag; ++i) {
        if (i > 0 && i < n) {
          const int s = i % KST;
          if (!mbar_wait(&kempty[s], ((i / KST) & 1) ^ 1, a.status, kTimeoutAttention)) {
            *abort_flag = 1;
            break;
          }
          mbar_arrive_expect_tx(&kfull[s], Sh::KV_BYTES);
          load_tile(sK + s * Sh::KV_BYTES, &maps.k, &kfull[s], hk, k_end - (i + 1) * BK, BK);
          nk = i + 1;
        }
        if (i >= 1) {
          const int u = i - 1, s = u % KST;
          if (!mbar_wait(&vempty[s], ((u / KST) & 1) ^ 1, a.status, kTimeoutAttention)) {
            *abort_flag = 1;
            break;
          }
          mbar_arrive_expect_tx(&vfull[s], Sh::KV_BYTES);
          load_tile(sV + s * Sh::KV_BYTES, &maps.v, &vfull[s], hk, k_end - i * BK, BK);
          nv = u + 1;
        }
      }
      // Gate prefetch: once the last QK^T has consumed every K stage, load
      // this tile's gate rows (128 x D) into them for the epilogue.
      bool gate_issued = false;
      if (a.gate && !*abort_flag && nk == n) {
        bool free_ = true;
        for (int t = max(0, n - KST); t < n; ++t)
          free_ = free_ && mbar_wait(&kempty[t % KST], (t / KST) & 1, a.status, kTimeoutAttention);
        if (free_) {
          mbar_arrive_expect_tx(gfull, Sh::Q_BYTES);
          load_tile(sK, &maps.gate, gfull, h, q0, BQ);
          gate_issued = true;
        } else {
          *abort_flag = 1;
        }
      }
      // Every issued load must land before the CTA may exit.
      mbar_wait(qfull, 0, a.status, kTimeoutDrain);
      if (gate_issued) mbar_wait(gfull, 0, a.status, kTimeoutDrain);
      for (int t = max(0, nk - KST); t < nk; ++t) mbar_wait(&kfull[t % KST], (t / KST) & 1, a.status, kTimeoutDrain);
      for (int t = max(0, nv - KST); t < nv; ++t) mbar_wait(&vfull[t % KST], (t / KST) & 1, a.status, kTimeoutDrain);
    }
  } else if (warp < 3) {
    // ---------------- MMA issuers (one lane; the warp waits together) ----------------
    // Issue is serial work (8 or 16 instructions and four waits a tile cost 2000
    // cycles in one warp): warp 1 issues S_t = Q K_t^T, warp 2 O += P_t V_t.
    // Descriptors of the first stages; others are a constant further.
    const uint64_t q_desc = smem_desc_k128(smem_u32(sQ)), k_desc = smem_desc_k128(smem_u32(sK));
    const uint64_t v_desc = smem_desc_mn128(smem_u32(sV), BK * 128);
    auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
      return __all_sync(0xffffffffu, mbar_wait(bar, parity, a.status, kTimeoutAttention));
    };
    auto issue_qk = [&](int t) -> bool {
      const int s = t & 1, ks = t % KST;  // S buffer, K stage
      // the buffer is free when the P.V that read the P in it is done
      if (!wait(&kfull[ks], (t / KST) & 1) || !wait(&pempty[s], ((t >> 1) & 1) ^ 1)) return false;
      tc_fence_after();
      if (elect_one()) {
        const uint64_t k = k_desc + ks * (Sh::KV_BYTES >> 4);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const int at = kk >> 2, w = kk & 3;
          umma_bf16(tmem + Sh::S_COL + s * BK, q_desc + ((at * (BQ * 128) + w * 32) >> 4),
                    k + ((at * (BK * 128) + w * 32) >> 4), IDESC_QK, kk > 0 ? 1u : 0u);
        }
        umma_commit(&kempty[ks]);
        umma_commit(&sfull[s]);
      }
      __syncwarp();
      return true;
    };
    auto issue_pv = [&](int u) -> bool {
      const int s = u & 1, vs = u % KST;  // S/P buffer, V stage
      if (!wait(&vfull[vs], (u / KST) & 1)) return false;
      const int live = total - (k_end - (u + 1) * BK);  // value rows of this tile that belong to a sequence
      if (live < BK) {
        // rows behind the last sequence hold anything: zero times it is not zero
        for (int i = max(live, 0) * 8 + lane; i < BK * 8; i += 32)
          for (int at = 0; at < ATOMS; ++at)
            *reinterpret_cast<uint4*>(sV + vs * Sh::KV_BYTES + at * (BK * 128) + i * 16) = make_uint4(0u, 0u, 0u, 0u);
        fence_async_smem();
        __syncwarp();
      }
      if (!wait(&pfull[s], (u >> 1) & 1)) return false;
      tc_fence_after();
      if (elect_one()) {
        const uint64_t v = v_desc + vs * (Sh::KV_BYTES >> 4);
#pragma unroll
        for (int kk = 0; kk < BK / 16; ++kk) {
          // 16 keys of P = 8 TMEM columns, each part's from the start of its share of S
          const int p_col = kk * 16 / BKP * BKP + kk * 16 % BKP / 2;
          umma_bf16_ts(tmem + Sh::O_COL, tmem + Sh::S_COL + s * BK + p_col, v + kk * (16 * 128 >> 4), IDESC_PV,
                       (u > 0 || kk > 0) ? 1u : 0u);
        }
        umma_commit(&vempty[vs]);
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
    // ---------------- softmax / epilogue warps ----------------
    // NP warps per TMEM lane quarter: part p of row r takes keys
    // [p BKP, (p + 1) BKP) of every tile and O columns [p D/NP, (p + 1) D/NP).
    // The parts exchange their tile maxima through shared memory (one
    // barrier per tile); their row sums are added once, at the end.
    constexpr int NP = Sh::NP, NWP = BKP / 32, NT = 128 * NP, DP = D / NP;
    const int q4 = warp & 3;  // TMEM lane quarter
    const int part = (warp - 3) >> 2;
    const int c0 = part * BKP;  // this part's first key column within a tile
    const int r = q4 * 32 + lane;
    const int row = q0 + r;
    const bool live = row >= q_first && row < q_end;
    // first key of this row (none for a row outside the sequences), and over the warp's rows
    int lo = row + 1;
    {
      const int w0 = max(q0 + q4 * 32, q_first), w1 = min(q0 + q4 * 32 + 31, q_end - 1);
      if (w0 <= w1) {
        int start;
        const int s0 = packed_seq_warp(a.cu, a.n_seqs, w0, lane, start), s1 = packed_seq_warp(a.cu, a.n_seqs, w1, lane, start);
        if (live) lo = packed_first_key(a, row, s0, s1);
      }
    }
    // over the warp's rows: keys below lo_min or above its last row are masked for all of them
    const int lo_max = __reduce_max_sync(0xffffffffu, lo), lo_min = __reduce_min_sync(0xffffffffu, lo);
    const int w_first = q0 + q4 * 32, w_last = w_first + 31;
    const uint32_t t_lane = static_cast<uint32_t>(q4 * 32) << 16;
    const float scale = rsqrtf(static_cast<float>(a.d)), scale_cap = scale * inverse_cap(a.softcap);
    const float scale_log2 = CAP ? LOG2E : scale * LOG2E;  // a capped score is scaled already
    // m: the maximum P is taken against (log2 units), at most 8 below that of the
    // tiles before the last; l: this part's sum; last: this part's maximum of the last tile
    float m = -INFINITY, l = 0.f, last = -INFINITY;
    const int t_own = (k_end - 1 - w_last) / BK;  // the tile with the warp's own rows' keys: the first it sees
    bool ok = true;
    // A failed wait sets `fail`; the two warps of a row leave together, by their
    // next exchange barrier, and the others by their own waits.
    bool fail = false;
    for (int t = 0; t < n; ++t) {
      const int s = t & 1;
      const int k0 = k_end - (t + 1) * BK + c0;  // first key of this part
      if (!fail) {
        const bool ready = mbar_wait(&sfull[s], (t >> 1) & 1, a.status, kTimeoutAttention);
        __syncwarp();
        fail = !__all_sync(0xffffffffu, ready);
      }
      tc_fence_after();
      const uint32_t s_at = tmem + t_lane + Sh::S_COL + s * BK + c0;  // this part's scores, then its P
      uint32_t sr[NWP][32];
      // 32 keys that every row of the warp masks: short sequences, a window's edge
      auto none = [&](int w) { return k0 + 32 * w > w_last || k0 + 32 * w + 31 < lo_min; };
      float mt = -INFINITY;  // this part's row maximum (log2 units)
      auto row_max = [&] {
        float pm[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int w = 0; w < NWP; ++w)
          if (!none(w)) {
#pragma unroll
            for (int c = 0; c < 32; c += 2)
              pm[c / 2 & 3] = max3(pm[c / 2 & 3], __uint_as_float(sr[w][c]), __uint_as_float(sr[w][c + 1]));
          }
        mt = fmaxf(fmaxf(pm[0], pm[1]), fmaxf(pm[2], pm[3])) * scale_log2;
      };
      if (!fail) {
#pragma unroll
        for (int w = 0; w < NWP; ++w) tmem_ld32(s_at + 32 * w, sr[w]);
        tmem_wait_ld();
#pragma unroll
        for (int w = 0; w < NWP; ++w) {
          if (none(w)) continue;
          const int k = k0 + 32 * w;
          if constexpr (CAP) cap_scores(sr[w], scale_cap, a.softcap);
          if (k + 31 > w_first || k < lo_max) {  // some key is masked for some row of the warp
            const int top = row - k, low = lo - k;
#pragma unroll
            for (int c = 0; c < 32; ++c) sr[w][c] = c >= low && c <= top ? sr[w][c] : 0xff800000u;  // -inf
          }
        }
      }
      if (t == t_own) {
        // the rows' first keys: the parts agree on their maximum at once
        row_max();
        xbuf[((t & 1) * NP + part) * 128 + r] = mt;
        if (bar_red_or(4 + q4, 32 * NP, fail)) {
          ok = false;
          break;
        }
        m = fmaxf(mt, xbuf[((t & 1) * NP + (part ^ 1)) * 128 + r]);
        // nothing to take the next tile's P against: such a row is computed again
        const unsigned lost = __ballot_sync(0xffffffffu, live && m == -INFINITY);
        if (lost && lane == 0) s_lost[q4] = lost;
      } else if (t > t_own + 1) {
        // later the maximum of the tile before: this one's P may be large
        if (bar_red_or(4 + q4, 32 * NP, fail)) {
          ok = false;
          break;
        }
        const float mn = fmaxf(fmaxf(m, last), xbuf[(((t - 1) & 1) * NP + (part ^ 1)) * 128 + r]);
        // the parts of a row see the same m and mn, so they decide alike
        if (__any_sync(0xffffffffu, mn > m + 8.f)) {
          // O must hold P_{t-1} V_{t-1} before it is rescaled.
          const bool done = mbar_wait(ofull, (t - 1) & 1, a.status, kTimeoutAttention);
          __syncwarp();
          if (!__all_sync(0xffffffffu, done)) {
            fail = true;
            continue;
          }
          tc_fence_after();
          // 2^(m - mn) in two steps: P_{t-1} may hold up to 2^128, whose inverse is no normal
          // number.  A P or a sum that overflowed stays infinite or becomes NaN.
          const float root = mn == -INFINITY ? 1.f : ex2_approx(0.5f * (m - mn));
          m = mn;
          l = root == 0.f ? 0.f : l * root * root;  // 0 times a sum that overflowed: only a NaN score makes a NaN sum
#pragma unroll 1
          for (int c = part * DP; c < (part + 1) * DP; c += 16) {
            uint32_t o[16];
            tmem_ld16(tmem + t_lane + Sh::O_COL + c, o);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * root * root);
            tmem_st16(tmem + t_lane + Sh::O_COL + c, o);
          }
          tmem_wait_st();
        }
      }
      // P = exp2(x * scale_log2 - m) as bf16, the operand type of P.V; the row sum keeps the FP32 values
      const float neg_m = m == -INFINITY ? 0.f : -m;  // no key yet: every p is exp2(-inf) = 0
      const uint64_t scale2 = pair2(scale_log2, scale_log2), neg_m2 = pair2(neg_m, neg_m);
      uint64_t ps[2] = {0ull, 0ull};  // sums of even and odd keys
      // packed as bf16 pairs from the start of this part's scores (key j in
      // column j/2), which only this warp reads
#pragma unroll
      for (int w = 0; w < NWP; ++w) {
        uint32_t pw[16];
        if (none(w)) {
#pragma unroll
          for (int e = 0; e < 16; ++e) pw[e] = 0u;
        } else {
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float2 x = unpair2(fma2(pair2(__uint_as_float(sr[w][2 * e]), __uint_as_float(sr[w][2 * e + 1])), scale2, neg_m2));
            const float p0 = ex2_approx(x.x), p1 = ex2_approx(x.y);
            ps[e & 1] = add2(ps[e & 1], pair2(p0, p1));
            pw[e] = pack_bf16x2(p0, p1);
          }
        }
        tmem_st16(s_at + 16 * w, pw);
      }
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(&pfull[s]);
      const float2 sum = unpair2(add2(ps[0], ps[1]));
      l += sum.x + sum.y;
      if (t > t_own) {  // for the next tile, while P.V runs
        row_max();
        last = mt;
        xbuf[((t & 1) * NP + part) * 128 + r] = mt;
      }
    }
    ok = ok && !fail;
    if (!ok) *abort_flag = 1;
    // the row sum: the parts' sums, added in part order
    float* lbuf = xbuf + 2 * NP * 128;
    lbuf[part * 128 + r] = l;
    asm volatile("bar.sync 1, %0;" ::"r"(NT) : "memory");
    l = lbuf[r] + lbuf[128 + r];
    // ---------------- epilogue ----------------
    // Phase 1: thread r forms its row (its part's columns) and writes it into
    // the Q buffer (free: every MMA has completed once ofinal fires) in the
    // TMA layout [atom][128 rows][128 B] with the 128-byte swizzle; the gate
    // rows come from the same layout in the K stages.
    // The first PRE of a thread's chunks have their gates ready before the last
    // P.V is done: half of the gates' time passes in that wait.
    constexpr int EC = D == 256 ? 32 : 16, NC = DP / EC, PRE = D == 256 ? 3 : 2;  // columns a chunk, chunks
    auto place = [&](int c, int v4) {  // 16 bytes of row r, columns c + 8 v4 ..
      return (c >> 6) * (BQ * 128) + r * 128 + (((((c >> 3) + v4) & 7) ^ (r & 7)) << 4);
    };
    auto gates = [&](int c, uint64_t (&sg)[EC / 2]) {
      uint4 gq[EC / 8];
#pragma unroll
      for (int v4 = 0; v4 < EC / 8; ++v4) gq[v4] = *reinterpret_cast<const uint4*>(sK + place(c, v4));
      sigmoids(gq, sg);
    };
    uint64_t early[PRE][EC / 2];
    const bool have_gate = ok && a.gate && mbar_wait(gfull, 0, a.status, kTimeoutAttention);
    if (have_gate) {
#pragma unroll
      for (int i = 0; i < PRE; ++i) gates(part * DP + i * EC, early[i]);
    }
    const bool fin = ok && mbar_wait(ofinal, 0, a.status, kTimeoutAttention);
    // Phase 2: a tile of sequence rows only leaves through TMA bulk stores, each
    // 64-column atom as soon as its rows are staged (D = 64: the parts share the
    // atom); otherwise the rows leave through coalesced 16-byte stores at the
    // end, and rows outside the sequences stay as they were.
    const bool whole = q_first == q0 && q_end == q0 + BQ;
    const bool out_ok = !bar_red_or(1, NT, !(fin && (have_gate || !a.gate)));  // every softmax warp agrees
    if (!out_ok) *abort_flag = 1;
    if (out_ok) {
      tc_fence_after();
      auto store_atom = [&](int at) {
        for (int half = 0; half < 2; ++half)
          tma_store_3d(&maps.out, sQ + at * (BQ * 128) + half * (64 * 128), at * 64, h, q0 + half * 64);
        tma_store_commit();
      };
      const float inv = 1.f / l;
      const uint64_t inv2 = pair2(inv, inv);
      uint64_t odd2 = 0ull;  // sum of 0 * y: NaN once a y is infinite or NaN
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        const int c = part * DP + i * EC;
        uint32_t o[EC];
#pragma unroll
        for (int w = 0; w < EC; w += 16) tmem_ld16(tmem + t_lane + Sh::O_COL + c + w, o + w);
        uint64_t sg[EC / 2];
        if (a.gate) {
          if (i < PRE) {
#pragma unroll
            for (int e = 0; e < EC / 2; ++e) sg[e] = early[i < PRE ? i : 0][e];
          } else {
            gates(c, sg);  // while O is on its way
          }
        }
        tmem_wait_ld();
#pragma unroll
        for (int v4 = 0; v4 < EC / 8; ++v4) {
          uint32_t yw[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int at = v4 * 4 + e;
            uint64_t y = mul2(pair2(__uint_as_float(o[2 * at]), __uint_as_float(o[2 * at + 1])), inv2);
            odd2 = fma2(y, 0ull, odd2);
            if (a.gate) y = mul2(y, sg[at]);
            const float2 yy = unpair2(y);
            yw[e] = pack_bf16x2(yy.x, yy.y);
          }
          *reinterpret_cast<uint4*>(sQ + place(c, v4)) = make_uint4(yw[0], yw[1], yw[2], yw[3]);
        }
        if (D >= 128 && whole && (c + EC) % 64 == 0 && (c & ~63) < a.d) {
          fence_async_smem();  // generic-proxy writes -> visible to the TMA engine
          if (part == 0)  // the four warps of this part
            asm volatile("bar.sync 2, 128;" ::: "memory");
          else
            asm volatile("bar.sync 3, 128;" ::: "memory");
          if (r == 0) store_atom(c >> 6);
        }
      }
      const float2 odd = unpair2(odd2);
      // a NaN sum has a NaN (or infinite) score of the row's own: the row is NaN, and stays so.
      // One that overflowed and was rescaled to 0 left NaN in O.
      const bool bad = l == l && (l == INFINITY || odd.x != 0.f || odd.y != 0.f || (s_lost[q4] >> lane & 1u));
      const unsigned bad_rows = __ballot_sync(0xffffffffu, bad && live);
      if (lane == 0 && bad_rows) atomicOr(&s_nan[q4], bad_rows);
      if (D == 64 && whole) fence_async_smem();
      asm volatile("bar.sync 1, %0;" ::"r"(NT) : "memory");  // every softmax warp
      if (whole) {
        if (r == 0) {
          if (D == 64 && part == 0) store_atom(0);
          // the staging buffer must outlive the copy; a row that is computed again must find it done
          if (s_nan[0] | s_nan[1] | s_nan[2] | s_nan[3])
            tma_store_wait_all();
          else
            tma_store_wait_read();
        }
      } else {
        const int chunks = a.d / 8;
        for (int idx = static_cast<int>(threadIdx.x) - Sh::FIRST; idx < BQ * chunks; idx += NT) {
          const int rr = idx / chunks, ch = idx % chunks;
          if (q0 + rr < q_first || q0 + rr >= q_end) continue;
          *reinterpret_cast<uint4*>(a.out + (q0 + rr) * a.ldo + h * a.hso + ch * 8) =
              *reinterpret_cast<const uint4*>(sQ + (ch >> 3) * (BQ * 128) + rr * 128 + (((ch & 7) ^ (rr & 7)) << 4));
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, Sh::TMEM_COLS);
  if (*abort_flag) {
    tma_store_wait_all();  // of the threads that stored
    __syncthreads();
    attn_packed_give_up<__nv_bfloat16, Sh::THREADS>(a, h, q_first, q_end);
    return;
  }
  if (s_nan[0] | s_nan[1] | s_nan[2] | s_nan[3])
    attn_packed_redo<__nv_bfloat16, true>(a, h, q0, s_nan, 4, reinterpret_cast<float*>(sQ));
}

}  // namespace clef
