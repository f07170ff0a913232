// Host side of the CTA-pair kernel: 3-D tensor maps.
#include "pair_mma.cuh"

#include <cudaTypedefs.h>

#include <mutex>

namespace veda::cuda::pair
{

bool make_map3(CUtensorMap* map, const void* base, int es, bool is_bf16, int64_t cols, int64_t rows,
               int64_t planes, int64_t ld, int64_t plane, uint32_t bx, uint32_t by,
               Swizzle swizzle)
{
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q{};
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &q) ==
                cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
        {
            fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
        }
    });
    if (fn == nullptr)
    {
        return false;
    }
    const CUtensorMapDataType type = es == 4   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                     : is_bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                               : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    const cuuint64_t dims[3] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows),
                                static_cast<cuuint64_t>(planes)};
    const cuuint64_t strides[2] = {static_cast<cuuint64_t>(ld) * es, static_cast<cuuint64_t>(plane) * es};
    const cuuint32_t box[3] = {bx, by, 1};
    const cuuint32_t estr[3] = {1, 1, 1};
    return fn(map, type, 3, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
              swizzle == Swizzle::k128  ? CU_TENSOR_MAP_SWIZZLE_128B
              : swizzle == Swizzle::k64 ? CU_TENSOR_MAP_SWIZZLE_64B
                                        : CU_TENSOR_MAP_SWIZZLE_NONE,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

} // namespace veda::cuda::pair
