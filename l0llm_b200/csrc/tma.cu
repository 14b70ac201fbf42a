// 2-D tensor maps (tma.cuh).
#include "tma.cuh"

namespace l0b {

l0b_status tensor_map_2d(CUtensorMap* m, CUtensorMapDataType type, size_t elem, const void* ptr, long long width,
                         long long rows, long long stride, int box_w, int box_rows, CUtensorMapSwizzle swizzle) {
    using Fn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                            const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                            CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static const Fn fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess) {
            cudaGetLastError();
            p = nullptr;
        }
        return reinterpret_cast<Fn>(p);
    }();
    L0B_REQUIRE(fn, L0B_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable");
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(width), static_cast<cuuint64_t>(rows)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(stride) * elem};
    const cuuint32_t box[2] = {static_cast<cuuint32_t>(box_w), static_cast<cuuint32_t>(box_rows)};
    const cuuint32_t step[2] = {1, 1};
    const CUresult r = fn(m, type, 2, const_cast<void*>(ptr), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    L0B_REQUIRE(r == CUDA_SUCCESS, L0B_ERR_ARGUMENT,
                "no tensor map for %lld rows of %lld elements, %lld apart (cuTensorMapEncodeTiled: %d)", rows, width, stride,
                static_cast<int>(r));
    return L0B_OK;
}

}  // namespace l0b
