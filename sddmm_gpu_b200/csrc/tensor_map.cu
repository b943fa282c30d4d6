// Tensor maps of the arrays that the tensor-core attention kernels read by tile copies.
#include "tc_utils.cuh"

namespace sddmm {

namespace {
using Encode = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                            const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
Encode encode_entry()
{
    static const Encode found = [] {
        void *f = nullptr;
        cudaDriverEntryPointQueryResult r;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &r) != cudaSuccess || r != cudaDriverEntryPointSuccess) {
            (void)cudaGetLastError();
            f = nullptr;
        }
        return reinterpret_cast<Encode>(f);
    }();
    return found;
}
}  // namespace

bool make_tensor_map(CUtensorMap *map, const HeadArray &a, int dtype, int head_dim, int heads, int64_t rows, int box_rows)
{
    const Encode encode = encode_entry();
    if (!encode || rows < 1 || a.row <= 0 || a.row % 8 || (heads > 1 && (a.head <= 0 || a.head % 8)) || (uintptr_t)a.data % 16) return false;
    const cuuint64_t dims[3] = {(cuuint64_t)head_dim, (cuuint64_t)heads, (cuuint64_t)rows};
    // (one head: its stride is never used, and may be anything)
    const cuuint64_t strides[2] = {(cuuint64_t)(heads > 1 ? a.head * 2 : a.row * 2), (cuuint64_t)a.row * 2};
    if (strides[0] >= (1ull << 40) || strides[1] >= (1ull << 40)) return false;
    const cuuint32_t box[3] = {64, 1, (cuuint32_t)box_rows}, step[3] = {1, 1, 1};
    return encode(map, dtype == 1 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, a.data, dims, strides, box, step,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace sddmm
