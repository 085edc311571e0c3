// Tensor maps of [batch][tokens][heads][dim] bf16 tensors, for copies of 64-column tiles.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <string>

#include "policy_internal.h"

namespace policy {

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                 const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiled encode_tiled()
{
    static const EncodeTiled fn = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess) {
            cudaGetLastError();
            f = nullptr;
        }
        return reinterpret_cast<EncodeTiled>(f);
    }();
    return fn;
}

// Whether strides (of batch, token, head) fit a map: not negative and below 2^40 bytes.  An axis that repeats one
// entry (stride 0) has one in the map, and is addressed by coordinate 0; an axis that a tile runs along cannot repeat.
inline bool map_takes(const int64_t (&shape)[3], const int64_t (&strides)[3], int heads)
{
    constexpr int64_t most = (int64_t{1} << 40) / 2;
    for (int64_t s : strides)
        if (s < 0 || s >= most) return false;
    return (shape[1] <= 1 || strides[1] > 0) && (heads <= 1 || strides[2] > 0);
}

// Tiles of 64 values of `heads` heads and `tokens` tokens: token-major rows, as they lie in the product.
// shape and strides (in values): batch, tokens, heads.  What lies past the tensor is copied as zeros.
inline int make_map(CUtensorMap* map, const void* x, const int64_t (&shape)[3], const int64_t (&strides)[3], int dim, int tokens, int heads)
{
    const EncodeTiled encode = encode_tiled();
    if (!encode) return fail(POLICY_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
    const auto extent = [](int64_t n, int64_t stride) { return static_cast<cuuint64_t>(stride ? n : 1); };
    const auto bytes = [](int64_t stride) { return static_cast<cuuint64_t>(stride ? stride * 2 : 16); };
    const cuuint64_t dims[4] = {static_cast<cuuint64_t>(dim), extent(shape[2], strides[2]), static_cast<cuuint64_t>(shape[1]),
                                extent(shape[0], strides[0])};
    const cuuint64_t steps[3] = {bytes(strides[2]), bytes(strides[1]), bytes(strides[0])};
    const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(heads), static_cast<cuuint32_t>(tokens), 1}, one[4] = {1, 1, 1, 1};
    const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(x), dims, steps, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? POLICY_OK : fail(POLICY_ERR_CUDA, "cuTensorMapEncodeTiled: error " + std::to_string(static_cast<int>(r)));
}

}  // namespace policy
