// int8 operators whose scales are found at run time (one per row of activations) or given per output
// channel: what their kernels share. Activations may be fp32, fp16 or bf16.
//
// A row x is held as whole numbers q with one factor: with amax = max(|x|, 2^-119),
//     scale = RN(amax * RN(1 / 127)),  inv = RN(RN(1 / amax) * 127),  q = the whole number nearest to x * inv
// (the product itself is not rounded, ties go to even). The floor of 2^-119 keeps inv finite and
// scale normal, so a row of zeros is zeros with a scale. A row that holds a NaN or an infinity has
// a NaN for its scale and zeros for its numbers: whatever is computed from it is NaN.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "internal.h"
#include "pdl.h"

namespace mb200 {
namespace scaled {

enum DType : int { DT_F32 = 0, DT_F16 = 1, DT_BF16 = 2 };
inline size_t dtype_bytes(int t) {
    return t == DT_F32 ? 4 : 2;
}
// 2^31 / 128^2: deeper sums may leave an int32
constexpr int kMaxK = 131071;
// of rows and columns: the last tile's indices still fit an int
constexpr int kMaxExtent = 0x7fffffff - 511;

#if defined(__CUDACC__)

// the largest magnitude as the bits of a non-negative float: their order is that of the values,
// with infinity and then the NaNs above every number
struct RowScale {
    float scale, inv;
    uint32_t keep;  // all ones, or zero for a row without a scale
};
__device__ __forceinline__ RowScale row_scale(uint32_t amax_bits) {
    RowScale r;
    const bool finite = amax_bits < 0x7f800000u;
    const float amax = fmaxf(__uint_as_float(amax_bits), 0x1p-119f);
    r.scale = finite ? __fmul_rn(amax, 1.f / 127.f) : __uint_as_float(0x7fffffffu);
    r.inv = finite ? __fmul_rn(__frcp_rn(amax), 127.f) : 0.f;
    r.keep = finite ? 0xffffffffu : 0u;
    return r;
}

// x * inv rounded to a whole number once, in the low byte of the result: adding 1.5 * 2^23 leaves
// no bits behind the point, and |x * inv| <= 127 * (1 + 2^-20) (beyond 2^126 the reciprocal has fewer
// bits than a normal number, 21 at least)
__device__ __forceinline__ uint32_t to_whole(float x, float inv) {
    return __float_as_uint(__fmaf_rn(x, inv, 12582912.f));
}
__device__ __forceinline__ uint32_t pack_whole(float a, float b, float c, float d, float inv) {
    const uint32_t ab = __byte_perm(to_whole(a, inv), to_whole(b, inv), 0x0040);
    const uint32_t cd = __byte_perm(to_whole(c, inv), to_whole(d, inv), 0x0040);
    return __byte_perm(ab, cd, 0x5410);
}

__device__ __forceinline__ float to_float(float v) {
    return v;
}
__device__ __forceinline__ float to_float(__half v) {
    return __half2float(v);
}
__device__ __forceinline__ float to_float(__nv_bfloat16 v) {
    return __bfloat162float(v);
}
__device__ __forceinline__ uint32_t magnitude(float v) {
    return __float_as_uint(v) & 0x7fffffffu;
}

// 16 bytes as floats: 4 fp32, 8 fp16 or bf16
template <class T>
struct Vec;
template <>
struct Vec<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void unpack(const uint4& w, float* v) {
        v[0] = __uint_as_float(w.x), v[1] = __uint_as_float(w.y);
        v[2] = __uint_as_float(w.z), v[3] = __uint_as_float(w.w);
    }
};
template <>
struct Vec<__nv_bfloat16> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void unpack(const uint4& w, float* v) {
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(u[i] << 16);
            v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
        }
    }
};
template <>
struct Vec<__half> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void unpack(const uint4& w, float* v) {
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    }
};
// the largest magnitude of 16 bytes, as the bits of a float (16-bit types compare as they are: the
// order of their bits is that of their values too)
template <class T>
__device__ __forceinline__ uint32_t vec_max(uint32_t so_far, const uint4& w) {
    if (sizeof(T) == 4) {
        return max(max(max(so_far, w.x & 0x7fffffffu), w.y & 0x7fffffffu),
                   max(w.z & 0x7fffffffu, w.w & 0x7fffffffu));
    }
    return __vmaxu2(__vmaxu2(so_far, __vmaxu2(w.x & 0x7fff7fffu, w.y & 0x7fff7fffu)),
                    __vmaxu2(w.z & 0x7fff7fffu, w.w & 0x7fff7fffu));
}
// what vec_max gathered, as the bits of a float
template <class T>
__device__ __forceinline__ uint32_t max_bits(uint32_t m) {
    if (sizeof(T) == 4)
        return m;
    const uint16_t h = (uint16_t)max(m & 0xffffu, m >> 16);
    return magnitude(to_float(*reinterpret_cast<const T*>(&h)));
}

__device__ __forceinline__ void store_as(void* c, int dtype, size_t i, float v) {
    if (dtype == DT_F32)
        ((float*)c)[i] = v;
    else if (dtype == DT_F16)
        ((__half*)c)[i] = __float2half_rn(v);
    else
        ((__nv_bfloat16*)c)[i] = __float2bfloat16_rn(v);
}

// acc * a_scale * b_scale [+ bias], each operation rounded, in this order everywhere
__device__ __forceinline__ float scale_acc(int acc, float sa, float sb) {
    return __fmul_rn(__fmul_rn(__int2float_rn(acc), sa), sb);
}

// `valid` (1 .. 16, or nothing at 0 and below) bytes from any address, zeros behind them. Whole
// 16-byte units are read: each holds at least one of the bytes that are asked for, so none reaches
// into memory that the tensor's own last byte does not share a unit with.
__device__ __forceinline__ uint4 ld_any16(const int8_t* p, int valid) {
    uint4 r = make_uint4(0, 0, 0, 0);
    if (valid <= 0)
        return r;
    const uintptr_t at = (uintptr_t)p;
    const int s = (int)(at & 15);
    const uint4* unit = (const uint4*)(at - s);
    const uint4 lo = *unit;
    const uint4 hi = s + min(valid, 16) > 16 ? unit[1] : r;
    uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    if (s & 8) {
#pragma unroll
        for (int i = 0; i < 6; ++i)
            w[i] = w[i + 2];
    }
    if (s & 4) {
#pragma unroll
        for (int i = 0; i < 5; ++i)
            w[i] = w[i + 1];
    }
    uint32_t* o = &r.x;
    uint32_t out[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        out[i] = __funnelshift_r(w[i], w[i + 1], (s & 3) * 8);
        const int left = valid - 4 * i;
        if (left < 4)
            out[i] &= left <= 0 ? 0u : (1u << (8 * left)) - 1u;
    }
    o[0] = out[0], o[1] = out[1], o[2] = out[2], o[3] = out[3];
    return r;
}

// 16 x 8 sums over 32 bytes of K: A is 16 rows (of weights), B 8 columns (tokens). A thread's words
// are four K bytes each of the rows lane/4 and lane/4 + 8, and of the column lane/4; sums c[0], c[1]
// belong to row lane/4 and the columns 2 * (lane % 4) and one more, c[2], c[3] to row lane/4 + 8.
// Which K bytes a word holds matters only in that A's and B's are the same ones.
__device__ __forceinline__ void mma_16x8x32(
        int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
            "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
            "{%8, %9}, {%0, %1, %2, %3};"
            : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// 64 bytes of K: a thread holds 16 neighbouring bytes of each row and column
__device__ __forceinline__ void mma_64(int (&c)[4], const uint4& lo, const uint4& hi, const uint4& t) {
    mma_16x8x32(c, lo.x, hi.x, lo.y, hi.y, t.x, t.y);
    mma_16x8x32(c, lo.z, hi.z, lo.w, hi.w, t.z, t.w);
}

// bytes between rows of whole numbers that are to lie in shared memory: whole steps, and two rows on other banks
__host__ __device__ constexpr int xs_pitch(int k) {
    return (k + 127) / 128 * 128 + 64;
}
__device__ __forceinline__ uint4 pack_piece(const float (&v)[16], const RowScale& r) {
    uint4 q;
    q.x = pack_whole(v[0], v[1], v[2], v[3], r.inv) & r.keep;
    q.y = pack_whole(v[4], v[5], v[6], v[7], r.inv) & r.keep;
    q.z = pack_whole(v[8], v[9], v[10], v[11], r.inv) & r.keep;
    q.w = pack_whole(v[12], v[13], v[14], v[15], r.inv) & r.keep;
    return q;
}

#endif  // __CUDACC__

// Behind a call of the runtime that has failed
inline cudaError_t why_refused() {
    const cudaError_t e = cudaPeekAtLastError();
    return e != cudaSuccess ? e : cudaErrorUnknown;
}

// Kernels that run in turn ask for the same share of an SM's memory as shared memory, all of it: an SM changes the share
// only when it is empty, so a kernel that asks for more than the one in front cannot begin beside its end.
struct MostShared {
    std::atomic<bool> done[64] = {};
    template <class Kernel>
    void ask(Kernel kernel) {
        int dev = 0;
        if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64 || done[dev].load(std::memory_order_relaxed))
            return;
        // (a preference: the kernel runs without it as well)
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout,
                                 cudaSharedmemCarveoutMaxShared) != cudaSuccess)
            cudaGetLastError();
        done[dev].store(true, std::memory_order_relaxed);
    }
};

// c[m][n] = a[m][k] * b[n][k] (whole numbers) * sa[m] * sb[n] [+ bias[n]]
struct ProductArgs {
    int m, n, k;
    const void* a;  // int8, or with x_dtype >= 0 activations of that type (sa is not read then)
    int x_dtype;    // -1: int8
    long long lda;  // elements
    const int8_t* b;
    long long ldb;
    const float *sa, *sb, *bias;
    void* c;
    int c_dtype;
    long long ldc;
    // b may be read before the kernel in front has ended (pdl.h)
    int b_early;
};

int launch_quantize_rows(
        const void* x, int dtype, int m, int k, long long ldx, int8_t* q, long long ldq, float* scales,
        cudaStream_t st);
// for any operands, made for few rows of a; activations as they are (x_dtype >= 0) as long as shared memory holds them
int launch_product_stream(const ProductArgs& a, cudaStream_t st);
// the tensor-core kernels: int8 operands, 16-byte aligned, rows whole 16-byte units apart
int launch_product_umma(const ProductArgs& a, cudaStream_t st);
// Rows of any alignment to rows `pitch` bytes apart (a multiple of 16, at least k), zeros behind each; two matrices in
// one launch (rows == 0: none)
struct PadRows {
    const int8_t* src;
    long long ld;
    int rows, k;
    int8_t* dst;
    long long pitch;
};
int launch_pad_rows(const PadRows& a, const PadRows& b, cudaStream_t st);

}  // namespace scaled
}  // namespace mb200
