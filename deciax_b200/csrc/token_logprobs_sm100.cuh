// Token log probabilities (token_logprobs.cuh) on the 5th-generation tensor
// cores: bf16 operands with 16-byte aligned rows.
//
// The GEMM's shape, with the running state of a row in place of its store:
//   warp 0      TMA producer: 64-deep stages of hidden rows and head rows
//   warp 1      one thread issues tcgen05.mma into one of two TMEM accumulators
//   warps 2..5  thread = row: reads 32 columns at a time and scans them
// PAIR (more than 128 rows): CTA pairs on 256 rows x 256 columns, each CTA
// loading half of both operands; otherwise one CTA on 128 rows x 256 columns,
// where the head's bytes are the bound and a pair would only wait for its peer.
// At most 32 (64) rows lie in the tile four times (twice), and the warps share
// each row's columns instead of leaving them to one.
// A unit is one row tile and one run of columns; units of the same run are
// neighbours, so the row tiles that read it share it in L2.  Every worker gets
// the same number of columns.  Pairs cut a run into tiles of 256 and a narrower
// last one (head rows by 16: their MMAs are the bound); one CTA, bound by the
// head's bytes, cuts it into equal tiles of any multiple of 8 columns, one box
// each (a last tile in boxes of 16 rows made one row 30 us slower).
//
// Vocabulary 256000, dim 3584: 1 row 313 us and 32 rows 324 us, HBM bound (1.835 GB
// at 5.9 and 5.7 TB/s; a stream of the head with nothing else takes 270 us); 2048
// rows 2.80 ms, 1341 TFLOP/s, the tensor pipe under the power cap.  Logits beyond
// the series of tanh (scan32) make 2048 capped rows 3.3 ms, 2.5 within it.
#pragma once

#include "attention_sm100.cuh"
#include "common.cuh"
#include "gemm2_sm100.cuh"
#include "token_logprobs.cuh"

namespace clef {

template <bool PAIR>
struct LogprobShape {
  static constexpr int BM = PAIR ? 256 : 128, BN = 256, BK = 64;
  static constexpr int STAGES = PAIR ? 6 : 4;
  static constexpr uint32_t A_BYTES = 128 * BK * 2;                 // rows a CTA holds
  static constexpr uint32_t B_BYTES = (PAIR ? 128 : 256) * BK * 2;  // head rows a CTA holds
  static constexpr uint32_t TMEM_COLS = 512;
  static constexpr size_t smem(int top) { return 1024 + STAGES * (A_BYTES + B_BYTES) + 256 + list_bytes(top); }
};

// Columns the MMA of the tile at c computes, in the instruction's steps of 32
// for a pair and 16 for one CTA.
template <bool PAIR>
__device__ __forceinline__ int tile_width(const LogprobArgs& a, int c, int c_end) {
  return PAIR ? min(256, (c_end - c + 31) / 32 * 32) : (a.tile + 15) / 16 * 16;
}

// Rows of the box that loads hidden states: a box much taller than the rows
// that exist costs the TMA unit their zeros (one row of 128: 430 us for the
// head's 1.8 GB, against 308 us with 8 of 128).  The tile's other rows hold
// whatever shared memory held; their scores are never read.
__host__ __device__ inline int hidden_box(int rows) { return rows > 64 ? 128 : rows > 32 ? 64 : rows > 8 ? 32 : 8; }

template <bool PAIR, bool CAP, int K>
__global__ void __launch_bounds__(192, 1)
    token_logprobs_tc_kernel(const __grid_constant__ CUtensorMap tma_a, const __grid_constant__ CUtensorMap tma_b,
                             const __grid_constant__ CUtensorMap tma_b16, const __grid_constant__ LogprobArgs args) {
  using S = LogprobShape<PAIR>;
  constexpr int BM = S::BM, BN = S::BN, BK = S::BK, STAGES = S::STAGES;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = smem + STAGES * S::A_BYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(sB + STAGES * S::B_BYTES);
  uint64_t* empty = full + STAGES;
  uint64_t* tfull = empty + STAGES;
  uint64_t* tempty = tfull + 2;
  uint64_t* drain = tempty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float* area = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(full) + 256);  // of the lists
  __shared__ float3 state[PAIR ? 1 : 128];

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = PAIR ? cluster_ctarank() : 0;
  const bool leader = rank == 0;
  const int worker = PAIR ? blockIdx.x >> 1 : blockIdx.x, workers = PAIR ? gridDim.x >> 1 : gridDim.x;
  const int units = args.num_m * args.splits;
  const int num_kb = (args.dim + BK - 1) / BK;

  if (threadIdx.x == 0) {
    prefetch_tmap(&tma_a);
    prefetch_tmap(&tma_b);
    prefetch_tmap(&tma_b16);
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&tfull[i], 1);
      mbar_init(&tempty[i], PAIR ? 8 : 4);  // one arrive per epilogue warp
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    if constexpr (PAIR) {
      tmem_alloc_pair(tmem_slot, S::TMEM_COLS);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(tmem_slot, S::TMEM_COLS);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync_all();  // the peer's barriers exist before anyone signals them
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      const int a_box = hidden_box(args.rows);
      const uint32_t full0 = PAIR ? mapa_shared(smem_u32(full), 0) : 0;
      int stage = 0;
      uint32_t phase = 0;
      long long issued = 0;
      for (int unit = worker; unit < units && !*abort_flag; unit += workers) {
        const int m = unit % args.num_m, split = unit / args.num_m;
        const int c_end = run_begin(args, split + 1);
        for (int c = run_begin(args, split); c < c_end && !*abort_flag; c += args.tile) {
          // head rows of this tile: pairs load half of them each
          const int w = PAIR ? tile_width<PAIR>(args, c, c_end) : args.tile;
          const int rows = PAIR ? w / 2 : w, first = PAIR ? c + static_cast<int>(rank) * rows : c;
          for (int kb = 0; kb < num_kb; ++kb) {
            if (!mbar_wait(&empty[stage], phase ^ 1, args.status, kTimeoutProducer) || *abort_flag) {
              *abort_flag = 1;
              break;
            }
            uint8_t* dst = sB + stage * S::B_BYTES;
            if constexpr (PAIR) {
              if (leader) mbar_arrive_expect_tx(&full[stage], 2 * S::A_BYTES + w * BK * 2);
              const uint32_t bar = full0 + stage * 8;
              tma_load_2d_pair(sA + stage * S::A_BYTES, &tma_a, bar, kb * BK, m * BM + static_cast<int>(rank) * 128);
              if (w == BN)
                tma_load_2d_pair(dst, &tma_b, bar, kb * BK, first);
              else
                for (int i = 0; i < rows; i += 16) tma_load_2d_pair(dst + i * 128, &tma_b16, bar, kb * BK, first + i);
            } else {
              mbar_arrive_expect_tx(&full[stage], args.copies * a_box * BK * 2 + w * BK * 2);
              for (int i = 0; i < args.copies; ++i)
                tma_load_2d(sA + stage * S::A_BYTES + i * (BM / args.copies) * 128, &tma_a, &full[stage], kb * BK, m * BM);
              tma_load_2d(dst, &tma_b, &full[stage], kb * BK, first);
            }
            ++issued;
            if (++stage == STAGES) {
              stage = 0;
              phase ^= 1;
            }
          }
        }
      }
      if constexpr (!PAIR) {
        // Every issued load must land before the CTA may exit.
        for (int i = 0; i < STAGES && i < issued; ++i) {
          if (stage == 0) {
            stage = STAGES - 1;
            phase ^= 1;
          } else {
            --stage;
          }
          mbar_wait(&full[stage], phase, args.status, kTimeoutDrain);
        }
      }
    }
  } else if (warp == 1) {
    if (leader && lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      int local = 0;
      bool ok = true;
      for (int unit = worker; ok && unit < units; unit += workers) {
        const int split = unit / args.num_m;
        const int c_end = run_begin(args, split + 1);
        for (int c = run_begin(args, split); ok && c < c_end; c += args.tile, ++local) {
          const int acc = local & 1;
          const uint32_t idesc = idesc_bf16_f32(BM, tile_width<PAIR>(args, c, c_end));
          ok = mbar_wait(&tempty[acc], ((local >> 1) & 1) ^ 1, args.status, kTimeoutMma) && !*abort_flag;
          tc_fence_after();
          const uint32_t d_tmem = tmem_base + acc * BN;
          for (int kb = 0; ok && kb < num_kb; ++kb) {
            if (!mbar_wait(&full[stage], phase, args.status, kTimeoutMma) || *abort_flag) {
              ok = false;
              break;
            }
            tc_fence_after();
            const uint32_t a_addr = smem_u32(sA + stage * S::A_BYTES);
            const uint32_t b_addr = smem_u32(sB + stage * S::B_BYTES);
#pragma unroll
            for (int k = 0; k < BK / 16; ++k) {
              if constexpr (PAIR)
                umma_bf16_pair(d_tmem, smem_desc_k128(a_addr + k * 32), smem_desc_k128(b_addr + k * 32), idesc,
                               (kb | k) != 0 ? 1u : 0u);
              else
                umma_bf16(d_tmem, smem_desc_k128(a_addr + k * 32), smem_desc_k128(b_addr + k * 32), idesc,
                          (kb | k) != 0 ? 1u : 0u);
            }
            if constexpr (PAIR)
              umma_commit_pair(&empty[stage]);
            else
              umma_commit(&empty[stage]);
            if (++stage == STAGES) {
              stage = 0;
              phase ^= 1;
            }
          }
          if (ok) {
            if constexpr (PAIR)
              umma_commit_pair(&tfull[acc]);
            else
              umma_commit(&tfull[acc]);
          }
        }
      }
      if (!ok) *abort_flag = 1;
      // Wait for this thread's MMAs to finish before the CTA can tear down.
      if constexpr (PAIR)
        umma_commit_pair(drain);
      else
        umma_commit(drain);
      mbar_wait(drain, 0, args.status, kTimeoutDrain);
    }
  } else {
    const int q = warp & 3, r = q * 32 + lane;  // TMEM lane quarter; row within the CTA's 128
    // with copies, this warp's rows are seen by others too: each takes every copies-th 32 columns
    const int copies = PAIR ? 1 : args.copies, rows_seen = 128 / copies;
    const int share = r / rows_seen;
    const uint32_t tempty0 = PAIR ? mapa_shared(smem_u32(tempty), 0) : 0;
    int local = 0, done = worker;  // done: the first unit without a state
    bool ok = true;
    for (int unit = worker; ok && unit < units; unit += workers) {
      const int m = unit % args.num_m, split = unit / args.num_m;
      const int c_end = run_begin(args, split + 1);
      const int row = m * BM + static_cast<int>(rank) * 128 + r - share * rows_seen;
      const bool any = row - lane < args.rows;  // some row of this warp exists
      RowState st;
      TopList<K> list;
      list.clear(args.top);
      for (int c0 = run_begin(args, split); c0 < c_end; c0 += args.tile, ++local) {
        const int acc = local & 1;
        ok = mbar_wait(&tfull[acc], (local >> 1) & 1, args.status, kTimeoutEpilogue);
        __syncwarp();
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) {
          *abort_flag = 1;
          break;
        }
        tc_fence_after();
        const uint32_t taddr = tmem_base + acc * BN + (static_cast<uint32_t>(q * 32) << 16);
        if (any) {
          const int cols = min(args.tile, c_end - c0);
#pragma unroll 1
          for (int c = 32 * share; c < cols; c += 32 * copies) {
            uint32_t v[32];
            tmem_ld32(taddr + c, v);
            tmem_wait_ld();
            float x[32];
#pragma unroll
            for (int j = 0; j < 32; ++j) x[j] = __uint_as_float(v[j]);
            if (row < args.rows) scan32<CAP>(st, list, x, c0 + c, cols - c, args.softcap, args.top, area, r);
            __syncwarp();
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if constexpr (PAIR)
            mbar_arrive_cluster(tempty0 + acc * 8);
          else
            mbar_arrive(&tempty[acc]);
        }
      }
      if constexpr (!PAIR) {
        if (copies > 1) {
          // the shares of a row meet in the first one's thread
          state[r] = make_float3(st.m, st.s, st.t);
          if (args.top > 0) list.publish(area, r);
          ok = !bar_red_or(1, 128, !ok);  // a failed wait ends every warp's loop together
          if (ok && share == 0 && row < args.rows)
            for (int i = 1; i < copies; ++i) {
              const int r2 = r + i * rows_seen;
              const float3 o = state[r2];
              join_state(st, o.x, o.y, o.z);
              list.join(args.top, area, r, r2);
            }
        }
      }
      if (ok && share == 0 && row < args.rows) store_state(args, st, list, split, row);
      if (ok) done += workers;
      if (!PAIR && copies > 1) asm volatile("bar.sync 1, 128;" ::: "memory");  // the lists may be cleared
    }
    for (; done < units; done += workers) {  // a wait failed
      const int row = done % args.num_m * BM + static_cast<int>(rank) * 128 + r;
      if (share == 0 && row < args.rows) store_no_state(args, done / args.num_m, row);
    }
  }

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  tc_fence_before();
  __syncthreads();
  if (PAIR && *abort_flag) let_copies_land();  // their barriers lie with the leader, and wait for both CTAs
  if constexpr (PAIR) cluster_sync_all();  // no CTA frees TMEM while its pair may still use it
  tc_fence_after();
  if (warp == 1) {
    if constexpr (PAIR)
      tmem_dealloc_pair(tmem_base, S::TMEM_COLS);
    else
      tmem_dealloc(tmem_base, S::TMEM_COLS);
  }
}

// ---------------------------------------------------------------------------
// FP32 operands: each value as three bf16 (24 bits of mantissa in 3 x 8), six products
// ---------------------------------------------------------------------------
//
//   x = h + m + l,  h = bf16(x), m = bf16(x - h), l = bf16(x - h - m)   (exact)
//   x y = hh' + hm' + mh' + hl' + lh' + mm'  + terms below 2^-24 of |x y|
//
// Six tensor-core products of 16 cycles a column replace the 64 FMA cycles that
// the CUDA cores need: 128 rows x 128 columns x 64 deep take 1540 cycles of MMA
// against 4096 of FMA.  The hidden states are split once, into scratch; the head
// is split on its way into shared memory, 5.5 operations a value:
//   warps 0..15  two groups take turns: load a 64-deep step of head rows into
//                registers, write it as three swizzled bf16 tiles
//   warp 16      issues the products
//   warps 17..20 thread = row: scan
//   warp 21      loads the hidden states' three tiles by TMA
// Bound by shared memory at 128 columns: the products read 192 KB a step, the
// tiles' writes are 96 KB (2300 cycles at 128 bytes a cycle).  22 warps leave 80
// registers a thread: a list of 9 to 32 alternatives spills (500 to 700 bytes), and
// 97 rows x 32003 x 1024 take 160 us with 20 alternatives in place of 63 with 5.
// The accumulator cuts off below its last bit at every step, so the five small
// products, 5 of 6 steps, have an accumulator of their own, 2^-8 as large.
struct LogprobF32Shape {
  static constexpr int BM = 128, BN = 128, BK = 64, STAGES = 2, THREADS = 22 * 32;
  static constexpr uint32_t TILE = 128 * BK * 2;  // one bf16 tile of 128 rows
  static constexpr uint32_t TMEM_COLS = 512;  // two tiles of 128 columns: h h', and the small products
  static constexpr size_t smem(int top) { return 1024 + STAGES * 6 * TILE + 256 + list_bytes(top); }
};

// out[p][row][dim_out]: part p of the rows' values, eight a thread; dim_out = dim rounded up to 8.
__global__ void __launch_bounds__(256)
    split_rows_kernel(const float* __restrict__ x, long long ldx, int rows, int dim, int dim_out, __nv_bfloat16* out) {
  const long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  const int per_row = dim_out / 8;
  if (i >= static_cast<long long>(rows) * per_row) return;
  const int row = static_cast<int>(i / per_row), k = static_cast<int>(i % per_row) * 8;
  float v[8];
  load8<float, true>(x + row * ldx, k, dim, true, v);
  uint4 h, m, l;
  split3(v[0], v[1], h.x, m.x, l.x);
  split3(v[2], v[3], h.y, m.y, l.y);
  split3(v[4], v[5], h.z, m.z, l.z);
  split3(v[6], v[7], h.w, m.w, l.w);
  const long long plane = static_cast<long long>(rows) * dim_out, at = static_cast<long long>(row) * dim_out + k;
  *reinterpret_cast<uint4*>(out + at) = h;
  *reinterpret_cast<uint4*>(out + plane + at) = m;
  *reinterpret_cast<uint4*>(out + 2 * plane + at) = l;
}

template <bool CAP, int K>
__global__ void __launch_bounds__(LogprobF32Shape::THREADS, 1)
    token_logprobs_f32_tc_kernel(const __grid_constant__ CUtensorMap tma_a, const __grid_constant__ LogprobArgs args) {
  using S = LogprobF32Shape;
  constexpr int BM = S::BM, BN = S::BN, BK = S::BK, STAGES = S::STAGES;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + STAGES * 6 * S::TILE);
  uint64_t* empty = full + STAGES;
  uint64_t* tfull = empty + STAGES;
  uint64_t* tempty = tfull + 2;
  uint64_t* drain = tempty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float* area = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(full) + 256);  // of the lists

  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const int units = args.num_m * args.splits;
  const int num_kb = (args.dim + BK - 1) / BK;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 257);  // a group of splitting threads, and the TMA warp
      mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&tfull[i], 1);
      mbar_init(&tempty[i], 4);  // one arrive per epilogue warp
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 16) {
    tmem_alloc(tmem_slot, S::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp < 16) {
    // thread: elements 4 j .. 4 j + 3 of both halves of head rows r0, r0 + 32, ..,
    // of every other step; odd rows take their halves in the other order, so that a
    // warp's stores meet every bank
    const int stage = warp >> 3, r0 = (threadIdx.x & 255) >> 3, j = threadIdx.x & 7, half0 = (r0 & 1) * 32;
    float4 next[8];
    int unit = blockIdx.x, c = 0, c_end = 0, kb = 0;  // the step: unit, its tile's first column, 64 of dim
    const float* head = nullptr;                      // this thread's first element of the tile
    uint32_t there = 0;                               // bit i: its i-th row exists
    auto tile = [&] {
      head = static_cast<const float*>(args.head) + (c + r0) * args.ldw + 4 * j;
      there = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) there |= (r0 + 32 * i < args.tile && c + r0 + 32 * i < args.vocab ? 1u : 0u) << i;
    };
    auto begin = [&] {
      if (unit < units) {
        c = run_begin(args, unit / args.num_m);
        c_end = run_begin(args, unit / args.num_m + 1);
        tile();
      }
    };
    auto advance = [&] {
      if (++kb < num_kb) return;
      kb = 0;
      c += args.tile;
      if (c < c_end) {
        tile();
      } else {
        unit += gridDim.x;
        begin();
      }
    };
    const long long step = 32 * args.ldw;
    auto load = [&] {
      if (unit >= units) return;
      const int k = kb * BK + 4 * j;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int half = (i & 1) ? 32 - half0 : half0;
        next[i] = (there >> (i / 2) & 1u) && k + half < args.dim
                      ? *reinterpret_cast<const float4*>(head + (i / 2) * step + kb * BK + half)
                      : make_float4(0.f, 0.f, 0.f, 0.f);
      }
    };
    begin();
    if (stage == 1 && unit < units) advance();
    load();
    uint32_t phase = 0;
    bool ok = true;
    while (unit < units) {
      ok = __all_sync(0xffffffffu, mbar_wait(&empty[stage], phase ^ 1, args.status, kTimeoutProducer));
      if (!ok) break;
      uint8_t* dst = smem + stage * 6 * S::TILE;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = r0 + 32 * (i / 2), chunk = ((i & 1) ? 32 - half0 : half0) / 8 + j / 2;
        uint2 h, m, l;
        split3(next[i].x, next[i].y, h.x, m.x, l.x);
        split3(next[i].z, next[i].w, h.y, m.y, l.y);
        uint8_t* p = dst + 3 * S::TILE + r * 128 + ((chunk ^ (r & 7)) << 4) + (j & 1) * 8;
        *reinterpret_cast<uint2*>(p) = h;
        *reinterpret_cast<uint2*>(p + S::TILE) = m;
        *reinterpret_cast<uint2*>(p + 2 * S::TILE) = l;
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      mbar_arrive(&full[stage]);
      phase ^= 1;
      advance();
      if (unit < units) advance();
      load();
    }
    if (!ok) *abort_flag = 1;
  } else if (warp == 16) {
    const uint32_t idesc = idesc_bf16_f32(BM, (args.tile + 15) / 16 * 16);
    const uint64_t desc = smem_desc_k128(smem_u32(smem));
    auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
      return __all_sync(0xffffffffu, mbar_wait(bar, parity, args.status, kTimeoutMma));
    };
    int stage = 0, local = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int unit = blockIdx.x; ok && unit < units; unit += gridDim.x) {
      const int split = unit / args.num_m;
      const int c_end = run_begin(args, split + 1);
      for (int c = run_begin(args, split); ok && c < c_end; c += args.tile, ++local) {
        const int acc = local & 1;
        ok = wait(&tempty[acc], ((local >> 1) & 1) ^ 1);
        tc_fence_after();
        for (int kb = 0; ok && kb < num_kb; ++kb) {
          ok = wait(&full[stage], phase);
          if (!ok) break;
          tc_fence_after();
          if (elect_one()) {
            const uint64_t a = desc + stage * (6 * S::TILE >> 4), b = a + (3 * S::TILE >> 4);
            constexpr int A[6] = {0, 2, 0, 1, 1, 0}, B[6] = {0, 0, 2, 1, 0, 1};  // h h', then l h', h l', m m', m h', h m'
            const uint32_t d = tmem_base + acc * 2 * BN;
#pragma unroll
            for (int k = 0; k < BK / 16; ++k)
#pragma unroll
              for (int p = 0; p < 6; ++p)
                umma_bf16(p == 0 ? d : d + BN, a + ((A[p] * S::TILE + k * 32) >> 4), b + ((B[p] * S::TILE + k * 32) >> 4),
                          idesc, (kb > 0 || k > 0 || p > 1) ? 1u : 0u);
            umma_commit(&empty[stage]);
          }
          __syncwarp();
          if (++stage == STAGES) stage = 0, phase ^= 1;
        }
        if (ok && elect_one()) umma_commit(&tfull[acc]);
        __syncwarp();
      }
    }
    if (elect_one()) {
      if (!ok) *abort_flag = 1;
      umma_commit(drain);
      mbar_wait(drain, 0, args.status, kTimeoutDrain);
    }
    __syncwarp();
  } else if (warp == 21) {
    const int a_box = hidden_box(args.rows);
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int unit = blockIdx.x; ok && unit < units; unit += gridDim.x) {
      const int m = unit % args.num_m, split = unit / args.num_m;
      const int c_end = run_begin(args, split + 1);
      for (int c = run_begin(args, split); ok && c < c_end; c += args.tile)
        for (int kb = 0; ok && kb < num_kb; ++kb) {
          ok = __all_sync(0xffffffffu, mbar_wait(&empty[stage], phase ^ 1, args.status, kTimeoutProducer));
          if (ok && elect_one()) {
            mbar_arrive_expect_tx(&full[stage], 3 * a_box * BK * 2);
            for (int p = 0; p < 3; ++p)  // rows behind the last hold the next part's: their scores are not read
              tma_load_2d(smem + (stage * 6 + p) * S::TILE, &tma_a, &full[stage], kb * BK, p * args.rows + m * BM);
          }
          __syncwarp();
          if (++stage == STAGES) stage = 0, phase ^= 1;
        }
    }
    if (!ok) *abort_flag = 1;
  } else {
    const int q = warp & 3, r = q * 32 + lane;  // TMEM lane quarter; row of the tile
    int local = 0, done = blockIdx.x;  // done: the first unit without a state
    bool ok = true;
    for (int unit = blockIdx.x; ok && unit < units; unit += gridDim.x) {
      const int split = unit / args.num_m, row = unit % args.num_m * BM + r;
      const int c_end = run_begin(args, split + 1);
      const bool any = row - lane < args.rows;  // some row of this warp exists
      RowState st;
      TopList<K> list;
      list.clear(args.top);
      for (int c0 = run_begin(args, split); c0 < c_end; c0 += args.tile, ++local) {
        const int acc = local & 1;
        ok = __all_sync(0xffffffffu, mbar_wait(&tfull[acc], (local >> 1) & 1, args.status, kTimeoutEpilogue));
        if (!ok) {
          *abort_flag = 1;
          break;
        }
        tc_fence_after();
        const uint32_t taddr = tmem_base + acc * 2 * BN + (static_cast<uint32_t>(q * 32) << 16);
        if (any) {
          const int cols = min(args.tile, c_end - c0);
#pragma unroll 1
          for (int c = 0; c < cols; c += 32) {
            float x[32];
#pragma unroll
            for (int half = 0; half < 32; half += 16) {
              uint32_t v[16], w[16];
              tmem_ld16(taddr + c + half, v);
              tmem_ld16(taddr + BN + c + half, w);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 16; ++e) x[half + e] = __uint_as_float(v[e]) + __uint_as_float(w[e]);
            }
            if (row < args.rows) scan32<CAP>(st, list, x, c0 + c, cols - c, args.softcap, args.top, area, r);
            __syncwarp();
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&tempty[acc]);
      }
      if (ok && row < args.rows) store_state(args, st, list, split, row);
      if (ok) done += gridDim.x;
    }
    for (; done < units; done += gridDim.x) {  // a wait failed
      const int row = done % args.num_m * BM + r;
      if (row < args.rows) store_no_state(args, done / args.num_m, row);
    }
  }

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) let_copies_land();  // their barriers wait for the splitting warps too
  tc_fence_after();
  if (warp == 16) tmem_dealloc(tmem_base, S::TMEM_COLS);
}

}  // namespace clef
