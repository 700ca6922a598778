// Tensor maps: encoded by the driver, whose entry point is looked up through
// the runtime (the library links no driver stub).
#include <mutex>

#include "tc.cuh"

namespace bloth {

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                 const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                 const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiled encoder() {
  static std::mutex mu;
  static EncodeTiled fn = nullptr;
  std::lock_guard<std::mutex> lk(mu);
  if (fn == nullptr) {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &found) ==
            cudaSuccess &&
        found == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiled>(p);
    else
      cudaGetLastError();
  }
  return fn;
}

int head_map(CUtensorMap* map, const void* p, int64_t sb, int64_t ss, int64_t sh, int B, int64_t S,
             int H, int D, int rows, int dtype) {
  const EncodeTiled enc = encoder();
  if (enc == nullptr) return cuda_status(cudaErrorNotSupported);
  const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)S, (cuuint64_t)H, (cuuint64_t)B};
  // a dimension of one row has no stride of its own: any legal one will do
  const cuuint64_t strides[3] = {(cuuint64_t)(S > 1 ? ss : D) * 2, (cuuint64_t)(H > 1 ? sh : D) * 2,
                                 (cuuint64_t)(B > 1 ? sb : D) * 2};
  const cuuint32_t box[4] = {64, (cuuint32_t)rows, 1, 1};
  const cuuint32_t step[4] = {1, 1, 1, 1};
  const CUresult r =
      enc(map,
          dtype == BLOTH_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
          4, const_cast<void*>(p), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? BLOTH_OK : BLOTH_ERR_ALIGN;
}

}  // namespace bloth
