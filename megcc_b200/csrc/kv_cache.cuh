// Device helpers of the int8 cache of keys and values: which sequence a packed row belongs to, where a position's
// values lie, 16-bit rows of 8 elements a lane.
//
// The cache holds pages of `page_tokens` positions: whole numbers [pages][kv_heads][page_tokens][d], and an fp32 scale
// for each block of 16 positions of a head. A sequence's table says which page holds its positions 0 .., page_tokens ..,
// and so on.
#pragma once
#include "attention.h"
#include "scaled_s8.cuh"

namespace mb200 {
namespace attn {

using scaled::magnitude;
using scaled::Vec;

// The first i of [0, n) with f(i) > x, n if there is none; f does not decrease. The whole warp asks, 32 places at a time:
// up to 32 sequences one load, up to 1024 two.
template <class F>
__device__ __forceinline__ int first_beyond(int n, long long x, F f) {
    const int lane = threadIdx.x & 31;
    int lo = 0;
    while (n > 0) {
        const int stride = (n + 31) / 32;
        const int at = lo + min((lane + 1) * stride, n) - 1;
        const int below = __popc(__ballot_sync(0xffffffffu, (long long)f(at) <= x));
        const int skip = min(below * stride, n);
        lo += skip;
        if (stride == 1)
            break;
        n = min(stride, n - skip);
    }
    return lo;
}

// The page of a block of positions, or -1
__device__ __forceinline__ int page_of(const mb200_kv_cache& c, int b, int position) {
    const int i = position / c.page_tokens;
    if (i >= c.table_pages)
        return -1;
    const int page = c.block_table[(long long)b * c.table_stride + i];
    return page < c.pages ? page : -1;
}
// rows of d whole numbers, and blocks, in front of a position of a page
__device__ __forceinline__ long long cache_row(const mb200_kv_cache& c, int page, int head, int position) {
    return ((long long)page * c.kv_heads + head) * c.page_tokens + position % c.page_tokens;
}

template <class T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ __half from_float<__half>(float v) {
    return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) {
    return __float2bfloat16_rn(v);
}
template <class T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    const __half2 r = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&r);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 r = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&r);
}

// 8 elements of 16 bits. VEC: they start on a 16-byte boundary
template <bool VEC>
__device__ __forceinline__ uint4 load8(const void* base, long long at) {
    const uint16_t* p = (const uint16_t*)base + at;
    if constexpr (VEC) {
        return *(const uint4*)p;
    } else {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            w[i] = (uint32_t)p[2 * i] | (uint32_t)p[2 * i + 1] << 16;
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
}
template <bool VEC>
__device__ __forceinline__ void store8(void* base, long long at, const uint4& v) {
    uint16_t* p = (uint16_t*)base + at;
    if constexpr (VEC) {
        *(uint4*)p = v;
    } else {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            p[2 * i] = (uint16_t)w[i];
            p[2 * i + 1] = (uint16_t)(w[i] >> 16);
        }
    }
}
template <class T>
__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
    return make_uint4(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7]));
}

}  // namespace attn
}  // namespace mb200
