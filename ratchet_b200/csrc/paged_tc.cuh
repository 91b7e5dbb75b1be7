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
template <class T> __device__ __forceinline__ uint32_t pack2(float x, float y);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float x, float y) {
    const __half2 v = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&v);
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float x, float y) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&v);
}
// Weights are taken against the running maximum less this (units of log 2), which stands for the maximum from there on: in the sums, the parts and lse.  f16's smallest
// step is 2^-24, and a weight below half of it vanishes: one row 17 above 20000 others would be all there is (an output of 0.05 was off by 2.8e-4, eleven half steps).
// Against the maximum less 7, weights lie below 2^15 (the maximum moves by steps of more than 8) and are off by 2^-32 of the largest at most; 131000 of them by
// 2^-15 of the sum together.  bf16 has f32's range.
template <class T> struct Above { static constexpr float value = 0.f; };
template <> struct Above<__half> { static constexpr float value = 7.f; };
// whether one of the two 16-bit values is an infinity or NaN
template <class T> __device__ __forceinline__ uint32_t not_finite(uint32_t x);
template <> __device__ __forceinline__ uint32_t not_finite<__half>(uint32_t x) { return __vcmpgeu2(x & 0x7fff7fffu, 0x7c007c00u); }
template <> __device__ __forceinline__ uint32_t not_finite<__nv_bfloat16>(uint32_t x) { return __vcmpgeu2(x & 0x7fff7fffu, 0x7f807f80u); }

// two f32 operations of one instruction
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\tfma.rn.f32x2 x, x, y, z;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
// 2^x for two numbers on the FMA pipe, which the exponential unit (four results a cycle and quarter of an SM) leaves idle.  x = n + f with n whole and
// |f| <= 1/2 (n appears in the low bits of x + 1.5 2^23; a reduction as in Cody and Waite, Software Manual for the Elementary Functions, 1980); 2^f by a
// polynomial of degree 5 with 2^0 = 1, fitted to the least relative error, times 2^n.  Off by 2.2e-7 at most (every f32 f from 2^-5 on tried), as the exponential
// unit's results are (2^-22): sums of weights are f32, and degree 4 (2.6e-6) showed in them.  It costs a prompt of 4096 tokens 0.5 %, the sums nothing.
// x up to 127; below -126 the result is 0; NaN stays NaN.
__device__ __forceinline__ float2 ex2_fma(float2 x) {
    constexpr float kMagic = 12582912.f + 127.f;
    x = make_float2(max_nan(x.x, -127.f), max_nan(x.y, -127.f));
    const float2 t = add2(x, make_float2(kMagic, kMagic));
    const float2 f = fma2(add2(t, make_float2(-kMagic, -kMagic)), make_float2(-1.f, -1.f), x);
    float2 y = fma2(make_float2(0.0013202981790527701f, 0.0013202981790527701f), f, make_float2(0.009674952365458012f, 0.009674952365458012f));
    y = fma2(y, f, make_float2(0.055510472506284714f, 0.055510472506284714f));
    y = fma2(y, f, make_float2(0.24022166430950165f, 0.24022166430950165f));
    y = fma2(y, f, make_float2(0.6931465864181519f, 0.6931465864181519f));
    y = fma2(y, f, make_float2(1.f, 1.f));
    return mul2(y, make_float2(__uint_as_float(__float_as_uint(t.x) << 23), __uint_as_float(__float_as_uint(t.y) << 23)));
}
// A place in a ring of `n` stages, and the parity of its barriers' phase
struct RingAt {
    int n, s, phase;
    __device__ __forceinline__ void go(int k) {
        s += k;
        if (s >= n) {
            s -= n;
            phase ^= 1;
        }
    }
};

// A bounded wait whose common end is one instruction; the rest stays out of line, because these kernels are as long as the instruction cache
static __device__ __noinline__ bool wait_on(uint64_t* bar, int phase, volatile int* abort_flag, int* status) { return gemvq8::mbar_wait(bar, phase, abort_flag, status); }
__device__ __forceinline__ bool wait_warp(uint64_t* bar, int phase, volatile int* abort_flag, int* status) {
    bool ok = gemvq8::mbar_try_wait(bar, phase & 1);
    if (!__all_sync(0xffffffffu, ok)) ok = __all_sync(0xffffffffu, ok || wait_on(bar, phase & 1, abort_flag, status));
    return ok;
}
// lets a copy land before the memory is somebody else's; bounded
static __device__ __noinline__ void land(uint64_t* bar, int phase) {
#pragma unroll 1
    for (int k = 0; k < (1 << 16) && !gemvq8::mbar_test_wait(bar, phase & 1); ++k) {}
}

// Page ids of a sequence, 32 consecutive ones in the warp's lanes
struct PageIds {
    int from = -64, id = 0;
    // id of page i (of the sequence's table) for this lane; `first` .. `first` + 31 covers all lanes' pages, `pages` of them exist
    __device__ __forceinline__ int of(const View& p, int s, int first, int i, int last_first, int pages) {
        if (first < from || last_first >= from + 32) {
            from = first;
            const int at = first + (int)(threadIdx.x & 31);
            id = at < pages ? p.table[(size_t)s * p.MP + at] : 0;
            if (at < pages && (unsigned)id >= (unsigned)p.pages) {
                report_bad(p.status);
                id = 0;
            }
        }
        return __shfl_sync(0xffffffffu, id, i - from);
    }
};

__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, int x, int y, int z, int u, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(smem_u32(dst)),
                 "l"(map), "r"(x), "r"(y), "r"(z), "r"(u), "r"(smem_u32(bar))
                 : "memory");
}
// [pages or tokens, heads, rows, features], boxes of 128 bytes of features; 128-byte swizzle, what lies beyond the extents reads as zero
inline bool map_4d(CUtensorMap* map, int dt, const void* base, const uint64_t (&dims)[4], uint32_t box1, uint32_t box3) {
    gemvq8::EncodeTiledFn fn = gemvq8::encode_tiled_fn();
    if (!fn) return false;
    const uint64_t e = dt_esize(dt);
    cuuint64_t d[4] = {dims[0], dims[1], dims[2], dims[3]};
    cuuint64_t strides[3] = {dims[0] * e, dims[0] * dims[1] * e, dims[0] * dims[1] * dims[2] * e};
    cuuint32_t box[4] = {(cuuint32_t)(128 / e), box1, 1, box3};
    cuuint32_t estr[4] = {1, 1, 1, 1};
    const CUtensorMapDataType type = dt == RCU_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : dt == RCU_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32;
    return fn(map, type, 4, const_cast<void*>(base), d, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// queries by tiles of `tq` tokens with the heads of a group, and rows of pages by 128 or by whole pages
inline bool map_queries(CUtensorMap* map, int dt, const View& p, const void* q, int group, int tq) {
    const uint64_t d[4] = {(uint64_t)p.D, (uint64_t)group, (uint64_t)p.G, (uint64_t)p.T};
    return map_4d(map, dt, q, d, group, tq);
}
inline bool map_slices(CUtensorMap* map, int dt, const View& p, const void* pages, int width, int rows) {
    const uint64_t d[4] = {(uint64_t)width, (uint64_t)p.R, (uint64_t)p.G, (uint64_t)p.pages};
    return map_4d(map, dt, pages, d, rows, 1);
}
inline bool map_pages(CUtensorMap* map, int dt, const View& p, const void* pages, int width) { return map_slices(map, dt, p, pages, width, p.R < kTileK ? p.R : kTileK); }

}  // namespace paged
