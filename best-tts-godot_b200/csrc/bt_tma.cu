// bt_tma.cu -- tensor maps for the tiled TMA loads (host side).
#include <cudaTypedefs.h>
#include "bt_ops.h"
#include "bt_internal.h"
#include "bt_tc.h"

namespace bt {

int tma_map(CUtensorMap* map, CUtensorMapDataType type, int rank, const void* base, const uint64_t* dims,
            const uint64_t* strides, const uint32_t* box, bool swizzle) {
  // the driver's encoder through the runtime, so that the library links no
  // driver library and still loads without a GPU
  static PFN_cuTensorMapEncodeTiled_v12000 encode = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess)
      f = nullptr;
    return (PFN_cuTensorMapEncodeTiled_v12000)f;
  }();
  if (!encode) return set_error(BT_ECUDA, "cuTensorMapEncodeTiled is not available");
  const uint32_t ones[5] = {1, 1, 1, 1, 1};
  const CUresult r = encode(map, type, (cuuint32_t)rank, const_cast<void*>(base), dims, strides, box, ones,
                            CU_TENSOR_MAP_INTERLEAVE_NONE,
                            swizzle ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(BT_ECUDA, "cuTensorMapEncodeTiled: error %d", (int)r);
  return BT_OK;
}

}  // namespace bt
