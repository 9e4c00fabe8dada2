// Host-side pieces shared by the library's translation units: the error type
// and checks behind the C ABI's status codes, device properties, TMA
// descriptor encoding and the scratch pool of the single-op entry points.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <map>
#include <mutex>
#include <stdexcept>
#include <string>
#include <utility>

#include "../../include/clef_b200.h"

namespace clef {

// ===========================================================================
// errors
// ===========================================================================

struct Error : std::runtime_error {
  int code;
  Error(int c, const std::string& m) : std::runtime_error(m), code(c) {}
};

#define CUDA_CHECK(expr)                                                                                 \
  do {                                                                                                   \
    cudaError_t e_ = (expr);                                                                             \
    if (e_ != cudaSuccess) throw ::clef::Error(CLEF_ECUDA, std::string(#expr) + ": " + cudaGetErrorString(e_)); \
  } while (0)
#define NCCL_CHECK(expr)                                                                                   \
  do {                                                                                                     \
    ncclResult_t r_ = (expr);                                                                              \
    if (r_ != ncclSuccess) throw ::clef::Error(CLEF_ENCCL, std::string(#expr) + ": " + ncclGetErrorString(r_)); \
  } while (0)
#define REQUIRE(cond, msg)                                  \
  do {                                                      \
    if (!(cond)) throw ::clef::Error(CLEF_EINVAL, (msg));   \
  } while (0)

inline std::mutex g_error_mutex;
inline std::string g_last_error;

inline void set_global_error(const std::string& m) {
  std::lock_guard<std::mutex> lock(g_error_mutex);
  g_last_error = m;
}

// ===========================================================================
// device properties, TMA descriptor encoding
// ===========================================================================

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

inline int sm_count(int device) {
  static std::mutex mu;
  static std::map<int, int> cache;
  std::lock_guard<std::mutex> lock(mu);
  auto it = cache.find(device);
  if (it != cache.end()) return it->second;
  int n = 0;
  CUDA_CHECK(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device));
  cache[device] = n;
  return n;
}

inline int current_device() {
  int d = 0;
  CUDA_CHECK(cudaGetDevice(&d));
  return d;
}

inline PFN_cuTensorMapEncodeTiled_v12000 tma_encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  });
  if (!fn) throw Error(CLEF_ECUDA, "cuTensorMapEncodeTiled is unavailable from the driver");
  return fn;
}

// Row-major bf16 [rows, cols] with row stride ld elements; box 64 columns x box_rows, 128-byte swizzle.
inline CUtensorMap tmap_bf16(const void* ptr, uint64_t rows, uint64_t cols, uint64_t ld, uint32_t box_rows) {
  CUtensorMap m;
  cuuint64_t dims[2] = {cols, rows};
  cuuint64_t strides[1] = {ld * 2};
  cuuint32_t box[2] = {64, box_rows};
  cuuint32_t es[2] = {1, 1};
  CUresult r = tma_encode_fn()(&m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(ptr), dims, strides, box, es,
                               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) throw Error(CLEF_EINVAL, "cuTensorMapEncodeTiled rejected a GEMM operand");
  return m;
}

// A stream-ordered memory pool of this library per device, for the scratch of
// single-op entry points: it keeps its memory between calls (an allocation
// after a synchronize does not map the memory again), and other users of the
// device's default pool are not affected.  A device whose context was reset
// and rebuilt gets a new pool (detected by its default pool's handle).
inline cudaMemPool_t op_scratch_pool(int device) {
  static std::mutex mu;
  static std::map<int, std::pair<cudaMemPool_t, cudaMemPool_t>> pools;  // device -> (default pool seen, ours)
  std::lock_guard<std::mutex> lock(mu);
  cudaMemPool_t def = nullptr;
  CUDA_CHECK(cudaDeviceGetDefaultMemPool(&def, device));
  auto it = pools.find(device);
  if (it != pools.end() && it->second.first == def) return it->second.second;
  cudaMemPoolProps props{};
  props.allocType = cudaMemAllocationTypePinned;
  props.location.type = cudaMemLocationTypeDevice;
  props.location.id = device;
  cudaMemPool_t pool = nullptr;
  CUDA_CHECK(cudaMemPoolCreate(&pool, &props));
  uint64_t keep = ~0ull;
  CUDA_CHECK(cudaMemPoolSetAttribute(pool, cudaMemPoolAttrReleaseThreshold, &keep));
  pools[device] = {def, pool};
  return pool;
}

}  // namespace clef
