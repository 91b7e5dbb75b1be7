// Pieces of the tensor-core kernels over paged caches (paged_attention_tc.cu, paged_mass_tc.cu).
#pragma once
#include <cuda.h>

#include "paged_attention.cuh"
#include "tc_common.cuh"

namespace paged {

using namespace tc;

constexpr int kTileQ = 128, kBlock = 128 * 128;       // rows of a query tile; bytes of 64 columns of a tile of 128 rows

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, int x, int y, int z, int u, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(smem_u32(dst)),
                 "l"(map), "r"(x), "r"(y), "r"(z), "r"(u), "r"(smem_u32(bar))
                 : "memory");
}
// [pages or tokens, heads, rows, features] of 16 bits, boxes of 64 features; 128-byte swizzle, what lies beyond the extents reads as zero
inline bool map_4d(CUtensorMap* map, int dt, const void* base, const uint64_t (&dims)[4], uint32_t box1, uint32_t box3) {
    gemvq8::EncodeTiledFn fn = gemvq8::encode_tiled_fn();
    if (!fn) return false;
    cuuint64_t d[4] = {dims[0], dims[1], dims[2], dims[3]};
    cuuint64_t strides[3] = {dims[0] * 2, dims[0] * dims[1] * 2, dims[0] * dims[1] * dims[2] * 2};
    cuuint32_t box[4] = {64, box1, 1, box3};
    cuuint32_t estr[4] = {1, 1, 1, 1};
    return fn(map, dt == RCU_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(base), d, strides, box, estr,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}


// queries by tiles of `tq` tokens with the heads of a group, and rows of pages by 128 or by whole pages
inline bool map_queries(CUtensorMap* map, int dt, const View& p, const void* q, int group, int tq) {
    const uint64_t d[4] = {(uint64_t)p.D, (uint64_t)group, (uint64_t)p.G, (uint64_t)p.T};
    return map_4d(map, dt, q, d, group, tq);
}
inline bool map_pages(CUtensorMap* map, int dt, const View& p, const void* pages, int width) {
    const uint64_t d[4] = {(uint64_t)width, (uint64_t)p.R, (uint64_t)p.G, (uint64_t)p.pages};
    return map_4d(map, dt, pages, d, p.R < kTileK ? p.R : kTileK, 1);
}

}  // namespace paged
