// Entry points of the packed-prompt operators: rotary positions with several
// axes, causal attention over packed sequences, token log probabilities.
// Declared in include/clef_b200.h beside the other single-kernel entry points.

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <initializer_list>
#include <set>
#include <type_traits>

#include "attention_packed.cuh"
#include "attention_packed_f32_sm100.cuh"
#include "attention_packed_sm100.cuh"
#include "common.cuh"
#include "host.cuh"
#include "rope_axes.cuh"
#include "token_logprobs.cuh"
#include "token_logprobs_sm100.cuh"

using bf16 = __nv_bfloat16;

namespace clef {

// Runs an entry point's body; no exception leaves the C ABI.
template <typename F>
static int op_guarded(F&& f) {
  try {
    f();
    return CLEF_OK;
  } catch (const Error& e) {
    set_global_error(e.what());
    if (e.code == CLEF_ECUDA) (void)cudaGetLastError();  // a failed allocation is not the next launch's error
    return e.code;
  } catch (const std::exception& e) {
    set_global_error(e.what());
    return CLEF_EINVAL;
  } catch (...) {
    set_global_error("unknown failure");
    return CLEF_EINVAL;
  }
}

// A kernel that follows a host pointer, or one into another GPU's memory,
// faults: refuse such a pointer before the launch.
static void require_on_device(std::initializer_list<const void*> pointers) {
  const int dev = current_device();
  for (const void* p : pointers) {
    if (!p) continue;
    cudaPointerAttributes at{};
    CUDA_CHECK(cudaPointerGetAttributes(&at, p));
    REQUIRE((at.type == cudaMemoryTypeDevice && at.device == dev) || at.type == cudaMemoryTypeManaged,
            "an operand is not in the current device's memory");
  }
}

// So does one that reads a value across its type's alignment.
static void require_aligned(std::initializer_list<const void*> pointers, int bytes) {
  for (const void* p : pointers)
    REQUIRE(reinterpret_cast<uintptr_t>(p) % bytes == 0, "an operand is not aligned to its values' size");
}

// Dynamic shared memory beyond the default is a per-device attribute of a kernel.
template <typename K>
static void allow_smem(K kern, size_t bytes) {
  static std::mutex mu;
  static std::set<std::pair<int, const void*>> done;
  const std::pair<int, const void*> key{current_device(), reinterpret_cast<const void*>(kern)};
  std::lock_guard<std::mutex> lock(mu);
  if (done.count(key)) return;
  CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes)));
  done.insert(key);
}

static int size_of(int dtype) {
  REQUIRE(dtype == CLEF_DTYPE_BF16 || dtype == CLEF_DTYPE_F32, "dtype must be CLEF_DTYPE_BF16 or CLEF_DTYPE_F32");
  return dtype == CLEF_DTYPE_BF16 ? 2 : 4;
}

// Stream-ordered scratch of one call, freed on the stream when the call's kernels are enqueued.
struct OpScratch {
  cudaStream_t st;
  void* p = nullptr;
  OpScratch(size_t bytes, cudaStream_t s) : st(s) {
    CUDA_CHECK(cudaMallocFromPoolAsync(&p, bytes, op_scratch_pool(current_device()), st));
  }
  ~OpScratch() {
    if (p) cudaFreeAsync(p, st);
  }
};

static void rope_frequencies(RopeAxesArgs& a, int rot, double theta, int axes, const int32_t* sections,
                             int interleaved) {
  const int half = rot / 2;
  a.half = half;
  // powers by repeated products of one 64-bit-mantissa root: off by 2^-57 at most
  const long double step = std::pow(static_cast<long double>(theta), -2.0L / rot);
  long double turn = 18446744073709551616.0L / 6.283185307179586476925286766559L;  // 2^64 / 2 pi
  for (int i = 0; i < half; ++i, turn *= step) {
    a.turn[i] = static_cast<unsigned long long>(turn);
    a.axis[i] = 0;
  }
  if (axes == 1) return;
  if (interleaved) {  // pair i turns with axis i % axes while that axis has pairs left, else with axis 0
    for (int i = 0; i < half; ++i)
      if (i / axes < sections[i % axes]) a.axis[i] = static_cast<unsigned char>(i % axes);
  } else {
    int i = 0;
    for (int ax = 0; ax < axes; ++ax)
      for (int n = 0; n < sections[ax]; ++n) a.axis[i++] = static_cast<unsigned char>(ax);
  }
}

template <typename T, int LANES>
static void launch_rope(const RopeAxesArgs& a, cudaStream_t st) {
  // all heads in one block where 512 threads hold them, else in groups of equal size
  const int heads = a.heads[0] + a.heads[1], groups = (heads * LANES + 511) / 512;
  const int threads = ((heads + groups - 1) / groups * LANES + 31) / 32 * 32;
  // a block's tokens share its weights and the start of its pipeline; few tokens spread over the SMs instead
  const int span = std::max(1, std::min(16, static_cast<int>(static_cast<long long>(a.tokens) * groups /
                                                             (12 * sm_count(current_device())))));
  const size_t smem = RopeShape<T>::ring(threads) + sizeof(float2) * span * a.half;
  allow_smem(rope_axes_kernel<T, LANES>, RopeShape<T>::ring(512) + sizeof(float2) * 16 * kRopeMaxHalf);
  rope_axes_kernel<T, LANES><<<dim3((a.tokens + span - 1) / span, groups), threads, smem, st>>>(a, span);
}

template <typename T>
static void rope_axes(const RopeAxesArgs& a, cudaStream_t st) {
  constexpr int kVec = 16 / sizeof(T);
  bool vec = a.d % (2 * kVec) == 0 && a.half % kVec == 0;
  for (int i = 0; i < 2; ++i)
    if (a.heads[i])
      vec = vec && aligned16(a.x[i]) && aligned16(a.out[i]) && (!a.w[i] || aligned16(a.w[i])) && a.ldx[i] % kVec == 0 &&
            a.ldo[i] % kVec == 0 && (a.heads[i] == 1 || (a.hsx[i] % kVec == 0 && a.hso[i] % kVec == 0));
  if (vec) {
    if (a.d <= 8 * kVec)
      launch_rope<T, 4>(a, st);
    else if (a.d <= 16 * kVec)
      launch_rope<T, 8>(a, st);
    else if (a.d <= 32 * kVec)
      launch_rope<T, 16>(a, st);
    else
      launch_rope<T, 32>(a, st);
  } else {
    const long long items = static_cast<long long>(a.tokens) * (a.heads[0] + a.heads[1]);
    rope_axes_any_kernel<T><<<static_cast<int>((items + 7) / 8), 256, 8 * a.d * sizeof(float), st>>>(a);
  }
  CUDA_CHECK(cudaGetLastError());
}

// bf16 [tokens][heads][d] with token stride ld and head stride hs: boxes of 64
// elements of one head x 64 tokens, 128-byte swizzle, zeros outside.
static CUtensorMap tmap_bf16_heads(const void* ptr, int tokens, int heads, int d, long long ld, long long hs) {
  CUtensorMap m;
  if (heads == 1) hs = (d + 7) / 8 * 8;  // never stepped
  cuuint64_t dims[3] = {static_cast<cuuint64_t>(d), static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(tokens)};
  cuuint64_t strides[2] = {static_cast<cuuint64_t>(hs) * 2, static_cast<cuuint64_t>(ld) * 2};
  cuuint32_t box[3] = {64, 1, 64};
  cuuint32_t es[3] = {1, 1, 1};
  CUresult r = tma_encode_fn()(&m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(ptr), dims, strides, box, es,
                               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) throw Error(CLEF_EINVAL, "cuTensorMapEncodeTiled rejected an attention operand");
  return m;
}

template <typename T, int DP>
static void launch_packed_simt(const AttnPackedArgs<T>& a, cudaStream_t st) {
  constexpr size_t smem = AttnPackedSimtShape<DP>::SMEM;
  const auto rows = [](const void* p, long long ld, long long hs, int heads) {
    return aligned16(p) && ld % 4 == 0 && (heads == 1 || hs % 4 == 0);
  };
  const bool vec = a.d % 4 == 0 && rows(a.q, a.ldq, a.hsq, a.H) && rows(a.k, a.ldk, a.hsk, a.Hk) && rows(a.v, a.ldv, a.hsv, a.Hk);
  allow_smem(attn_packed_simt_kernel<T, DP>, smem);
  attn_packed_simt_kernel<T, DP><<<dim3((a.tokens + 63) / 64, a.H), 256, smem, st>>>(a, vec);
  CUDA_CHECK(cudaGetLastError());
}

// Heads whose tiles run side by side: all of them let the longest tiles of
// every head start first (24 records of 16384 rows, 32 heads of 128: 300 us
// against 320 us eight heads at a time), as long as the keys and values that
// they read stay within three quarters of L2 (one sequence of 16384, 16 heads
// of 256: all at once 1680 us, four or eight 1600 us).
static int packed_heads_at_once(const AttnPackedArgs<bf16>& a) {
  const long long kv_bytes = 4LL * a.tokens * a.d;
  int kv = static_cast<int>(std::max(1LL, std::min<long long>(a.Hk, (96LL << 20) / std::max(1LL, kv_bytes))));
  while (a.Hk % kv) --kv;
  return kv * (a.H / a.Hk);
}

template <int D, bool CAP>
static void launch_packed_tc(const AttnPackedMaps& maps, const AttnPackedArgs<bf16>& a, cudaStream_t st) {
  using Sh = AttnPackedTcShape<D>;
  allow_smem(attn_packed_tc_kernel<D, CAP>, Sh::SMEM);
  const int heads = packed_heads_at_once(a);
  attn_packed_tc_kernel<D, CAP><<<dim3(heads, (a.tokens + 127) / 128, a.H / heads), Sh::THREADS, Sh::SMEM, st>>>(maps, a);
  CUDA_CHECK(cudaGetLastError());
}

template <int D, bool CAP>
static void launch_packed_f32_tc(const AttnPackedArgs<float>& a, cudaStream_t st) {
  using Sh = AttnPackedF32Shape<D>;
  const auto rows = [](const void* p, long long ld, long long hs, int heads) {
    return !p || (aligned16(p) && ld % 4 == 0 && (heads == 1 || hs % 4 == 0));
  };
  SplitHeadsArgs sp{};
  sp.x[0] = a.q, sp.x[1] = a.k, sp.x[2] = a.v;
  sp.ld[0] = a.ldq, sp.ld[1] = a.ldk, sp.ld[2] = a.ldv;
  sp.hs[0] = a.hsq, sp.hs[1] = a.hsk, sp.hs[2] = a.hsv;
  sp.heads[0] = a.H, sp.heads[1] = sp.heads[2] = a.Hk;
  sp.tokens = a.tokens;
  sp.d = a.d;
  sp.d8 = (a.d + 7) / 8 * 8;
  sp.vec = a.d % 4 == 0 && rows(a.q, a.ldq, a.hsq, a.H) && rows(a.k, a.ldk, a.hsk, a.Hk) && rows(a.v, a.ldv, a.hsv, a.Hk);
  const size_t row = static_cast<size_t>(a.tokens) * sp.d8;  // elements of a head of one part
  OpScratch scratch(3 * row * (a.H + 2 * a.Hk) * sizeof(bf16), st);
  sp.out[0] = static_cast<bf16*>(scratch.p);
  sp.out[1] = sp.out[0] + 3 * row * a.H;
  sp.out[2] = sp.out[1] + 3 * row * a.Hk;
  const long long groups = static_cast<long long>(row / 8) * (a.H + 2 * a.Hk);
  REQUIRE(groups < (1LL << 38), "too many rows for one call");
  AttnPackedF32Maps maps;
  maps.q = tmap_bf16_heads(sp.out[0], 3 * a.tokens, a.H, sp.d8, static_cast<long long>(a.H) * sp.d8, sp.d8);
  maps.k = tmap_bf16_heads(sp.out[1], 3 * a.tokens, a.Hk, sp.d8, static_cast<long long>(a.Hk) * sp.d8, sp.d8);
  maps.v = tmap_bf16_heads(sp.out[2], 3 * a.tokens, a.Hk, sp.d8, static_cast<long long>(a.Hk) * sp.d8, sp.d8);
  split_heads_kernel<<<static_cast<int>((groups + 255) / 256), 256, 0, st>>>(sp);
  CUDA_CHECK(cudaGetLastError());
  const bool vec = a.d % 4 == 0 && rows(a.gate, a.ldg, a.hsg, a.H) && rows(a.out, a.ldo, a.hso, a.H);
  allow_smem(attn_packed_f32_tc_kernel<D, CAP>, Sh::SMEM);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute early[1];
  early[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3(a.H, (a.tokens + 127) / 128);
  cfg.blockDim = dim3(Sh::THREADS);
  cfg.dynamicSmemBytes = Sh::SMEM;
  cfg.stream = st;
  cfg.attrs = early;
  cfg.numAttrs = 1;
  CUDA_CHECK(cudaLaunchKernelEx(&cfg, attn_packed_f32_tc_kernel<D, CAP>, maps, a, vec, sp.vec));
}

template <typename T>
static void attention_packed(const AttnPackedArgs<T>& a, cudaStream_t st) {
  if constexpr (sizeof(T) == 2) {
    // TMA needs 16-byte aligned rows; everything else runs on the CUDA cores
    const auto rows = [](const void* p, long long ld, long long hs, int heads) {
      return !p || (aligned16(p) && ld > 0 && ld % 8 == 0 && (heads == 1 || (hs > 0 && hs % 8 == 0)));
    };
    if (a.d % 8 == 0 && rows(a.q, a.ldq, a.hsq, a.H) && rows(a.k, a.ldk, a.hsk, a.Hk) && rows(a.v, a.ldv, a.hsv, a.Hk) &&
        rows(a.gate, a.ldg, a.hsg, a.H) && rows(a.out, a.ldo, a.hso, a.H)) {
      AttnPackedMaps maps;
      maps.q = tmap_bf16_heads(a.q, a.tokens, a.H, a.d, a.ldq, a.hsq);
      maps.k = tmap_bf16_heads(a.k, a.tokens, a.Hk, a.d, a.ldk, a.hsk);
      maps.v = tmap_bf16_heads(a.v, a.tokens, a.Hk, a.d, a.ldv, a.hsv);
      maps.gate = a.gate ? tmap_bf16_heads(a.gate, a.tokens, a.H, a.d, a.ldg, a.hsg) : maps.q;
      maps.out = tmap_bf16_heads(a.out, a.tokens, a.H, a.d, a.ldo, a.hso);
      const bool cap = a.softcap > 0.f;
      if (a.d <= 64)
        cap ? launch_packed_tc<64, true>(maps, a, st) : launch_packed_tc<64, false>(maps, a, st);
      else if (a.d <= 128)
        cap ? launch_packed_tc<128, true>(maps, a, st) : launch_packed_tc<128, false>(maps, a, st);
      else
        cap ? launch_packed_tc<256, true>(maps, a, st) : launch_packed_tc<256, false>(maps, a, st);
      return;
    }
  }
  if constexpr (sizeof(T) == 4) {
    // Splitting costs a launch.  Heads above 64 gain from a few rows on: 16 rows, captured,
    // take 14.4 us against 17.8 on the CUDA cores at 16 heads of 128, 14.7 against 18.2 at 64
    // (27.8 against 25.1 at 256, where one CTA an SM makes two rounds of the heads).  Heads of
    // 64, 2 to 64 of them, gain from a second tile of 64 rows on when captured (96 rows: 11
    // against 14 us), but a program that launches each call pays 2 us for the launch
    // (128 rows: 27 against 25, 192 rows: 27 against 31).
    if (a.d <= 128 && a.tokens > (a.d <= 64 ? 128 : 8)) {
      const bool cap = a.softcap > 0.f;
      if (a.d <= 64)
        cap ? launch_packed_f32_tc<64, true>(a, st) : launch_packed_f32_tc<64, false>(a, st);
      else
        cap ? launch_packed_f32_tc<128, true>(a, st) : launch_packed_f32_tc<128, false>(a, st);
      return;
    }
  }
  if (a.d <= 64)
    launch_packed_simt<T, 64>(a, st);
  else if (a.d <= 128)
    launch_packed_simt<T, 128>(a, st);
  else
    launch_packed_simt<T, 256>(a, st);
}

// Cuts the vocabulary into runs of equal columns: as many as leave the fewest
// rounds of columns on `workers`, where a run costs 64 columns besides (its
// first columns fill a new list, its state is stored and joined).  A run is a
// multiple of `step` columns and, with equal_tiles, of its tile.
static void logprob_runs(LogprobArgs& a, int tile, int step, bool equal_tiles, int workers) {
  long long least = INT64_MAX;
  for (int s = 1; s <= kLogprobMaxSplits; ++s) {
    const long long share = (static_cast<long long>(a.vocab) + s - 1) / s;  // columns of a run
    const long long tiles = (share + tile - 1) / tile;
    const long long width = equal_tiles ? ((share + tiles - 1) / tiles + step - 1) / step * step : tile;
    const long long run = equal_tiles ? tiles * width : (share + step - 1) / step * step;
    const long long splits = (a.vocab + run - 1) / run;
    const long long cost = (a.num_m * splits + workers - 1) / workers * (run + 64);
    if (cost < least) {
      least = cost;
      a.splits = static_cast<int>(splits);
      a.run = static_cast<int>(run);
      a.tile = static_cast<int>(width);
    }
    if (share <= step) break;
  }
}

// Clusters of two CTAs of the pair kernel that fit the device at once.
template <bool CAP, int K>
static int logprob_pairs(int dev, cudaLaunchConfig_t cfg) {
  static std::mutex mu;
  static std::map<int, int> fits;
  std::lock_guard<std::mutex> lock(mu);
  auto it = fits.find(dev);
  if (it != fits.end()) return it->second;
  cfg.gridDim = dim3(sm_count(dev) / 2 * 2);
  cfg.dynamicSmemBytes = LogprobShape<true>::smem(kTopMax);
  int n = 0;
  CUDA_CHECK(cudaOccupancyMaxActiveClusters(&n, token_logprobs_tc_kernel<true, CAP, K>, &cfg));
  REQUIRE(n > 0, "no CTA-pair cluster fits on this device");
  fits[dev] = n;
  return n;
}

template <typename T, bool CAP, int K>
static void token_logprobs(FinishArgs f, cudaStream_t st) {
  LogprobArgs& a = f.l;
  const int dev = current_device();
  constexpr int kVec = 16 / sizeof(T);
  const bool vec = a.dim % kVec == 0 && a.ldh % kVec == 0 && a.ldw % kVec == 0 && aligned16(a.hidden) && aligned16(a.head);
  const bool tc = vec;  // 16-byte aligned rows
  const bool pair = tc && sizeof(T) == 2 && a.rows > 128;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  int workers = sm_count(dev);
  if (pair) {
    allow_smem(token_logprobs_tc_kernel<true, CAP, K>, LogprobShape<true>::smem(kTopMax));
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.blockDim = dim3(192);
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    workers = logprob_pairs<CAP, K>(dev, cfg);
  }
  const int bm = pair ? 256 : 128;
  a.num_m = (a.rows + bm - 1) / bm;
  if (!tc)
    logprob_runs(a, 128, 128, false, workers);
  else if (pair)
    logprob_runs(a, 256, 32, false, workers);
  else
    logprob_runs(a, sizeof(T) == 2 ? 256 : 128, 8, true, workers);
  const int grid = static_cast<int>(std::min<long long>(static_cast<long long>(a.num_m) * a.splits, workers));
  const size_t states = static_cast<size_t>(a.splits) * a.rows;
  // FP32 on the tensor cores: the hidden states' three parts behind the states and lists
  const int dim_split = (a.dim + 7) / 8 * 8;
  const size_t state_bytes = (states * (4 + 2 * static_cast<size_t>(a.top)) * 4 + 255) / 256 * 256;
  const size_t split_bytes = tc && sizeof(T) == 4 ? 3 * static_cast<size_t>(a.rows) * dim_split * 2 : 0;
  OpScratch scratch(state_bytes + split_bytes, st);
  a.part = static_cast<float4*>(scratch.p);
  a.list_x = reinterpret_cast<float*>(a.part + states);
  a.list_id = reinterpret_cast<int32_t*>(a.list_x + states * a.top);
  if constexpr (sizeof(T) == 2) {
    if (tc) {
      a.copies = a.rows > 64 ? 1 : a.rows > 32 ? 2 : 4;
      const CUtensorMap ta = tmap_bf16(a.hidden, a.rows, a.dim, a.ldh, hidden_box(a.rows));
      const CUtensorMap tb = tmap_bf16(a.head, a.vocab, a.dim, a.ldw, pair ? 128 : a.tile);
      const CUtensorMap tb16 = tmap_bf16(a.head, a.vocab, a.dim, a.ldw, 16);
      if (pair) {
        cfg.gridDim = dim3(2 * grid);
        cfg.dynamicSmemBytes = LogprobShape<true>::smem(a.top);
        CUDA_CHECK(cudaLaunchKernelEx(&cfg, token_logprobs_tc_kernel<true, CAP, K>, ta, tb, tb16, a));
      } else {
        allow_smem(token_logprobs_tc_kernel<false, CAP, K>, LogprobShape<false>::smem(kTopMax));
        token_logprobs_tc_kernel<false, CAP, K><<<grid, 192, LogprobShape<false>::smem(a.top), st>>>(ta, tb, tb16, a);
        CUDA_CHECK(cudaGetLastError());
      }
    }
  }
  if constexpr (sizeof(T) == 4) {
    if (tc) {
      allow_smem(token_logprobs_f32_tc_kernel<CAP, K>, LogprobF32Shape::smem(kTopMax));
      bf16* parts = reinterpret_cast<bf16*>(static_cast<uint8_t*>(scratch.p) + state_bytes);
      const long long runs8 = static_cast<long long>(a.rows) * (dim_split / 8);
      split_rows_kernel<<<static_cast<int>((runs8 + 255) / 256), 256, 0, st>>>(static_cast<const float*>(a.hidden), a.ldh,
                                                                               a.rows, a.dim, dim_split, parts);
      CUDA_CHECK(cudaGetLastError());
      const CUtensorMap ta = tmap_bf16(parts, 3ULL * a.rows, dim_split, dim_split, hidden_box(a.rows));
      token_logprobs_f32_tc_kernel<CAP, K><<<grid, LogprobF32Shape::THREADS, LogprobF32Shape::smem(a.top), st>>>(ta, a);
      CUDA_CHECK(cudaGetLastError());
    }
  }
  if (!tc) {
    allow_smem(token_logprobs_simt_kernel<T, CAP, K>, logprob_simt_smem(kTopMax));
    token_logprobs_simt_kernel<T, CAP, K><<<grid, 256, logprob_simt_smem(a.top), st>>>(a);
    CUDA_CHECK(cudaGetLastError());
  }
  auto finish = [&](auto kern) {
    allow_smem(kern, static_cast<size_t>(kLogprobMaxSplits) * kTopMax * 8);
    // it may start while the kernel before it ends, and waits for that one itself
    cudaLaunchConfig_t fin = {};
    cudaLaunchAttribute early[1];
    early[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early[0].val.programmaticStreamSerializationAllowed = 1;
    fin.gridDim = dim3(a.rows);
    fin.blockDim = dim3(128);
    fin.dynamicSmemBytes = static_cast<size_t>(a.splits) * a.top * 8;
    fin.stream = st;
    fin.attrs = early;
    fin.numAttrs = 1;
    CUDA_CHECK(cudaLaunchKernelEx(&fin, kern, f));
  };
  if (vec)
    finish(token_logprobs_finish_kernel<T, true, CAP>);
  else
    finish(token_logprobs_finish_kernel<T, false, CAP>);
}

}  // namespace clef

extern "C" {

int clef_op_token_logprobs(int dtype, const void* hidden, int64_t ldh, const void* lm_head, int64_t ldw, int rows, int vocab,
                           int dim, float softcap, const int32_t* targets, int n_targets, float* logprobs, float* entropy,
                           int top, int32_t* top_ids, float* top_logprobs, void* stream) {
  using namespace clef;
  return op_guarded([&] {
    const int size = size_of(dtype);
    REQUIRE(rows >= 0 && vocab > 0 && dim > 0, "rows must not be negative, vocab and dim must be positive");
    REQUIRE(vocab <= 1 << 30 && dim <= 1 << 20 && rows <= 1 << 24, "at most 2^24 rows, 2^30 tokens and 2^20 dimensions");
    REQUIRE(ldh >= dim && ldw >= dim, "row strides must be at least dim");
    REQUIRE(softcap >= 0.f && std::isfinite(softcap), "softcap must not be negative (0 = off)");
    REQUIRE(n_targets >= 0 && n_targets <= 1 << 20, "n_targets must be in [0, 2^20]");
    REQUIRE(top >= 0 && top <= kTopMax && top <= vocab, "top must be in [0, min(32, vocab)]");
    if (rows == 0) return;
    REQUIRE(hidden && lm_head, "null operand");
    REQUIRE(n_targets == 0 || (targets && logprobs), "targets need logprobs");
    REQUIRE(top == 0 || (top_ids && top_logprobs), "top alternatives need their outputs");
    REQUIRE(n_targets > 0 || top > 0 || entropy, "no output was asked for");
    require_aligned({hidden, lm_head}, size);
    require_aligned({n_targets ? targets : nullptr, n_targets ? logprobs : nullptr, entropy, top ? top_ids : nullptr,
                     top ? top_logprobs : nullptr},
                    4);
    require_on_device({hidden, lm_head, n_targets ? targets : nullptr, n_targets ? logprobs : nullptr, entropy,
                       top ? top_ids : nullptr, top ? top_logprobs : nullptr});
    FinishArgs f{};
    f.l.hidden = hidden;
    f.l.head = lm_head;
    f.l.ldh = ldh;
    f.l.ldw = ldw;
    f.l.rows = rows;
    f.l.vocab = vocab;
    f.l.dim = dim;
    f.l.softcap = softcap;
    f.l.top = top;
    f.targets = targets;
    f.n_targets = n_targets;
    f.logprobs = logprobs;
    f.entropy = entropy;
    f.top_ids = top_ids;
    f.top_logprobs = top_logprobs;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    auto run = [&](auto* type, auto cap) {
      using T = std::remove_pointer_t<decltype(type)>;
      if (top <= 8)
        token_logprobs<T, decltype(cap)::value, 8>(f, st);
      else
        token_logprobs<T, decltype(cap)::value, kTopMax>(f, st);
    };
    if (dtype == CLEF_DTYPE_BF16)
      softcap > 0.f ? run(static_cast<bf16*>(nullptr), std::true_type{}) : run(static_cast<bf16*>(nullptr), std::false_type{});
    else
      softcap > 0.f ? run(static_cast<float*>(nullptr), std::true_type{}) : run(static_cast<float*>(nullptr), std::false_type{});
  });
}

int clef_op_attention_packed(int dtype, const void* q, int64_t ldq, int64_t hsq, const void* k, int64_t ldk, int64_t hsk,
                             const void* v, int64_t ldv, int64_t hsv, const void* gate, int64_t ldg, int64_t hsg, void* out,
                             int64_t ldo, int64_t hso, const int32_t* cu_seqlens, int n_seqs, int tokens, int hq, int hkv,
                             int d, float softcap, int window, void* stream) {
  using namespace clef;
  return op_guarded([&] {
    const int size = size_of(dtype);
    REQUIRE(n_seqs >= 0 && tokens >= 0, "sequences and tokens must not be negative");
    REQUIRE(tokens <= 65535 * 128, "at most 8388480 tokens");
    REQUIRE(hq > 0 && hkv > 0 && hq % hkv == 0, "query heads must be a multiple of key/value heads");
    REQUIRE(hq <= 65535, "at most 65535 query heads");
    REQUIRE(d > 0 && d <= 256, "attention head size must be in [1, 256]");
    REQUIRE(softcap >= 0.f && std::isfinite(softcap), "softcap must not be negative (0 = off)");
    REQUIRE(window >= 0, "window must not be negative (0 = off)");
    if (n_seqs == 0 || tokens == 0) return;
    REQUIRE(q && k && v && out && cu_seqlens, "null operand");
    const auto rows = [&](int heads, int64_t ld, int64_t hs) {
      return (heads == 1 || hs >= d) && (tokens == 1 || ld >= d) && ld >= 0 && hs >= 0;
    };
    REQUIRE(rows(hq, ldq, hsq) && rows(hkv, ldk, hsk) && rows(hkv, ldv, hsv) && (!gate || rows(hq, ldg, hsg)) &&
                rows(hq, ldo, hso),
            "token and head strides must be at least head_dim");
    require_aligned({q, k, v, gate, out}, size);
    require_aligned({cu_seqlens}, 4);
    require_on_device({q, k, v, gate, out, cu_seqlens});
    auto call = [&](auto* type) {
      using T = std::remove_pointer_t<decltype(type)>;
      AttnPackedArgs<T> a{};
      a.q = static_cast<const T*>(q);
      a.k = static_cast<const T*>(k);
      a.v = static_cast<const T*>(v);
      a.gate = static_cast<const T*>(gate);
      a.out = static_cast<T*>(out);
      a.ldq = ldq, a.hsq = hsq, a.ldk = ldk, a.hsk = hsk, a.ldv = ldv, a.hsv = hsv;
      a.ldg = ldg, a.hsg = hsg, a.ldo = ldo, a.hso = hso;
      a.cu = cu_seqlens;
      a.n_seqs = n_seqs;
      a.tokens = tokens;
      a.H = hq;
      a.Hk = hkv;
      a.d = d;
      a.softcap = softcap;
      a.window = window;
      attention_packed<T>(a, static_cast<cudaStream_t>(stream));
    };
    if (dtype == CLEF_DTYPE_BF16)
      call(static_cast<bf16*>(nullptr));
    else
      call(static_cast<float*>(nullptr));
  });
}

int clef_op_qk_norm_rope_axes(int dtype, const void* q, int64_t ldq, int64_t hsq, const void* k, int64_t ldk, int64_t hsk,
                              void* q_out, int64_t ldqo, int64_t hsqo, void* k_out, int64_t ldko, int64_t hsko,
                              const int32_t* positions, int64_t ldp, int axes, const int32_t* sections, int interleaved,
                              int tokens, int hq, int hkv, int d, int rot, float rope_theta, const void* q_norm,
                              const void* k_norm, float eps, void* stream) {
  using namespace clef;
  return op_guarded([&] {
    const int size = size_of(dtype);
    REQUIRE(tokens >= 0 && hq >= 0 && hkv >= 0 && hq + hkv > 0, "tokens and heads must not be negative");
    REQUIRE(hq <= 65536 && hkv <= 65536, "at most 65536 heads");
    REQUIRE(d > 0 && d <= 2 * kRopeMaxHalf, "head_dim must be in [1, 256]");
    REQUIRE(rot > 0 && rot % 2 == 0 && rot <= d, "invalid partial rotary dimension");
    REQUIRE(std::isfinite(rope_theta) && rope_theta >= 1.f, "rope_theta must be at least 1");
    REQUIRE(axes >= 1 && axes <= 8, "axes must be in [1, 8]");
    if (axes > 1) {
      REQUIRE(sections, "several axes need their sections");
      long long sum = 0;
      for (int i = 0; i < axes; ++i) {
        REQUIRE(sections[i] >= 0 && sections[i] <= rot / 2, "a section must be in [0, rot / 2]");
        REQUIRE(!interleaved || i == 0 || i + static_cast<long long>(axes) * (sections[i] - 1) < rot / 2,
                "interleaved sections: an axis has more pairs than every axes-th one");
        sum += sections[i];
      }
      REQUIRE(sum == rot / 2, "sections must add up to rot / 2 frequency pairs");
    }
    if (tokens == 0) return;
    REQUIRE((hq == 0 || (q && q_out)) && (hkv == 0 || (k && k_out)) && positions, "null operand");
    const auto rows = [&](int heads, int64_t ld, int64_t hs) {
      return heads == 0 || ((heads == 1 || hs >= d) && (tokens == 1 || ld >= d) && ld >= 0 && hs >= 0);
    };
    REQUIRE(rows(hq, ldq, hsq) && rows(hq, ldqo, hsqo) && rows(hkv, ldk, hsk) && rows(hkv, ldko, hsko),
            "token and head strides must be at least head_dim");
    REQUIRE(axes == 1 || ldp >= tokens, "the positions' axis stride is below the token count");
    REQUIRE(static_cast<long long>(tokens) * (hq + hkv) < (1LL << 33), "tokens * heads must be below 2^33");
    require_aligned({hq ? q : nullptr, hq ? q_out : nullptr, hkv ? k : nullptr, hkv ? k_out : nullptr, hq ? q_norm : nullptr,
                     hkv ? k_norm : nullptr},
                    size);
    require_aligned({positions}, 4);
    require_on_device({hq ? q : nullptr, hq ? q_out : nullptr, hkv ? k : nullptr, hkv ? k_out : nullptr, positions,
                       hq ? q_norm : nullptr, hkv ? k_norm : nullptr});
    RopeAxesArgs a{};
    a.x[0] = q, a.x[1] = k;
    a.out[0] = q_out, a.out[1] = k_out;
    a.w[0] = q_norm, a.w[1] = k_norm;
    a.ldx[0] = ldq, a.ldx[1] = ldk, a.hsx[0] = hsq, a.hsx[1] = hsk;
    a.ldo[0] = ldqo, a.ldo[1] = ldko, a.hso[0] = hsqo, a.hso[1] = hsko;
    a.heads[0] = hq, a.heads[1] = hkv;
    a.pos = positions;
    a.ldp = ldp;
    a.tokens = tokens;
    a.d = d;
    a.eps = eps;
    rope_frequencies(a, rot, rope_theta, axes, sections, interleaved);
    if (dtype == CLEF_DTYPE_BF16)
      rope_axes<bf16>(a, static_cast<cudaStream_t>(stream));
    else
      rope_axes<float>(a, static_cast<cudaStream_t>(stream));
  });
}

}  // extern "C"
