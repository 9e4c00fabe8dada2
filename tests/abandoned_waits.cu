// Launches of the packed-prompt kernels whose waits run out: a tensor map with
// boxes shorter than the kernel counts on delivers fewer bytes than it waits
// for.  Every copy stays in bounds and every wait ends after its own limit.
#include "../deciax_b200/csrc/attention_packed_f32_sm100.cuh"
#include "../deciax_b200/csrc/attention_packed_sm100.cuh"
#include "../deciax_b200/csrc/host.cuh"
#include "../deciax_b200/csrc/token_logprobs_sm100.cuh"

using namespace clef;

template <typename F>
static int status_of(F&& f) {
  try {
    f();
    return 0;
  } catch (const std::exception&) {
    return 1;
  }
}

// bf16 [rows][heads][d], boxes of 64 x 1 x box_rows
static CUtensorMap heads_map(const void* ptr, int rows, int heads, int d, int box_rows) {
  CUtensorMap m;
  cuuint64_t dims[3] = {static_cast<cuuint64_t>(d), static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(rows)};
  cuuint64_t strides[2] = {static_cast<cuuint64_t>(d) * 2, static_cast<cuuint64_t>(heads) * d * 2};
  cuuint32_t box[3] = {64, 1, static_cast<cuuint32_t>(box_rows)};
  cuuint32_t es[3] = {1, 1, 1};
  REQUIRE(tma_encode_fn()(&m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(ptr), dims, strides, box, es,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS,
          "tensor map");
  return m;
}

extern "C" {

// 20 rows x 512 columns in two runs of 256, both taken by one CTA; hidden boxes of 8 rows in place of 32.
// part [20][2] float4, list_x and list_id [20][2][top].
int abandoned_logprobs(int fp32, const void* hidden, const void* head, int dim, int top, void* part, void* list_x, void* list_id,
                       const int32_t* targets, float* logprobs, float* entropy, int32_t* top_ids, float* top_logprobs,
                       void* stream) {
  return status_of([&] {
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    FinishArgs f{};
    LogprobArgs& a = f.l;
    a.hidden = hidden, a.head = head;
    a.ldh = a.ldw = dim;
    a.rows = 20, a.vocab = 512, a.dim = dim, a.top = top;
    a.num_m = 1, a.splits = 2, a.run = 256, a.tile = fp32 ? 128 : 256, a.copies = 4;
    a.part = static_cast<float4*>(part);
    a.list_x = static_cast<float*>(list_x);
    a.list_id = static_cast<int32_t*>(list_id);
    f.targets = targets;
    f.n_targets = 1;
    f.logprobs = logprobs, f.entropy = entropy, f.top_ids = top_ids, f.top_logprobs = top_logprobs;
    const size_t lists = 2 * static_cast<size_t>(top) * 8;
    if (fp32) {  // hidden: three parts [3][20][dim], bf16; only waits are tested, so the finish kernel reads the parts as FP32
      auto kern = token_logprobs_f32_tc_kernel<false, 8>;
      const size_t smem = LogprobF32Shape::smem(8);
      CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
      kern<<<1, LogprobF32Shape::THREADS, smem, st>>>(tmap_bf16(hidden, 60, dim, dim, 8), a);
      CUDA_CHECK(cudaGetLastError());
      token_logprobs_finish_kernel<float, true, false><<<20, 128, lists, st>>>(f);
    } else {
      auto kern = token_logprobs_tc_kernel<false, false, 8>;
      const size_t smem = LogprobShape<false>::smem(8);
      CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
      kern<<<1, 192, smem, st>>>(tmap_bf16(hidden, 20, dim, dim, 8), tmap_bf16(head, 512, dim, dim, 256),
                                 tmap_bf16(head, 512, dim, dim, 16), a);
      CUDA_CHECK(cudaGetLastError());
      token_logprobs_finish_kernel<__nv_bfloat16, true, false><<<20, 128, lists, st>>>(f);
    }
    CUDA_CHECK(cudaGetLastError());
  });
}

// One tile, one head of 64: boxes of 32 rows for the keys (which = 1) or the values (2).
// bf16: q, k, v, out [tokens][64]; fp32: q, k, v are three bf16 parts [3][tokens][64] (out and gate FP32).
int abandoned_attention(int fp32, int which, const void* q, const void* k, const void* v, void* out, const int32_t* cu, int tokens,
                        void* stream) {
  return status_of([&] {
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int rows = fp32 ? 3 * tokens : tokens;
    const CUtensorMap mq = heads_map(q, rows, 1, 64, 64), mk = heads_map(k, rows, 1, 64, which == 1 ? 32 : 64),
                      mv = heads_map(v, rows, 1, 64, which == 2 ? 32 : 64);
    auto fill = [&](auto& a) {
      a.ldq = a.ldk = a.ldv = a.ldo = 64;
      a.hsq = a.hsk = a.hsv = a.hso = 64;
      a.cu = cu;
      a.n_seqs = 1, a.tokens = tokens, a.H = a.Hk = 1, a.d = 64;
    };
    if (fp32) {
      AttnPackedArgs<float> a{};
      fill(a);
      a.q = a.k = a.v = a.out = static_cast<float*>(out);
      AttnPackedF32Maps maps{mq, mk, mv};
      using Sh = AttnPackedF32Shape<64>;
      auto kern = attn_packed_f32_tc_kernel<64, false>;
      CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(Sh::SMEM)));
      kern<<<dim3(1, (tokens + 127) / 128), Sh::THREADS, Sh::SMEM, st>>>(maps, a, true, true);
    } else {
      AttnPackedArgs<__nv_bfloat16> a{};
      fill(a);
      a.q = a.k = a.v = a.out = static_cast<__nv_bfloat16*>(out);
      AttnPackedMaps maps{mq, mk, mv, mq, heads_map(out, tokens, 1, 64, 64)};
      using Sh = AttnPackedTcShape<64>;
      auto kern = attn_packed_tc_kernel<64, false>;
      CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(Sh::SMEM)));
      kern<<<dim3(1, (tokens + 127) / 128, 1), Sh::THREADS, Sh::SMEM, st>>>(maps, a);
    }
    CUDA_CHECK(cudaGetLastError());
  });
}

}  // extern "C"
