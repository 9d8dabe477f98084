// int8 products for few tokens, and the conversion of activations to int8 rows.
#include "scaled_s8.cuh"

namespace mb200 {
namespace scaled {

namespace {

// ---- rows to whole numbers ----
// HBM: every element is read once and written once as a byte. LANES threads share a row: a warp where
// a row fits its registers (no barrier), else a whole CTA. The first kHeld * LANES vectors of the row stay
// in registers between the maximum and the conversion, what lies behind them is read again.
constexpr int kHeld = 4;
constexpr int kRowThreads = 256;

template <class T, int LANES>
__global__ void __launch_bounds__(kRowThreads) quantize_rows_kernel(
        const T* __restrict__ x, int m, int k, long long ldx, int8_t* __restrict__ q, long long ldq,
        float* __restrict__ scales, int vector_loads, int word_stores) {
    constexpr int N = Vec<T>::N;
    __shared__ uint32_t part[kRowThreads / 32];
    pdl_start();
    const int lane = threadIdx.x % LANES;
    const long long row = (long long)blockIdx.x * (kRowThreads / LANES) + threadIdx.x / LANES;
    if (LANES == 32 && row >= m)
        return;  // (a whole warp; no barrier follows in this form)
    const T* src = x + row * ldx;
    int8_t* dst = q + row * ldq;
    const int nvec = vector_loads ? k / N : 0;  // the elements behind them one by one
    uint4 held[kHeld];
    uint32_t vm = 0;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
        const int v = lane + i * LANES;
        held[i] = v < nvec ? ((const uint4*)src)[v] : make_uint4(0, 0, 0, 0);
        vm = vec_max<T>(vm, held[i]);
    }
    for (int v = lane + kHeld * LANES; v < nvec; v += LANES)
        vm = vec_max<T>(vm, ((const uint4*)src)[v]);
    uint32_t bits = max_bits<T>(vm);
    for (int i = nvec * N + lane; i < k; i += LANES)
        bits = max(bits, magnitude(to_float(src[i])));
    bits = __reduce_max_sync(0xffffffffu, bits);
    if (LANES > 32) {
        if ((threadIdx.x & 31) == 0)
            part[threadIdx.x >> 5] = bits;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kRowThreads / 32; ++w)
            bits = max(bits, part[w]);
    }
    const RowScale r = row_scale(bits);
    if (lane == 0)
        scales[row] = r.scale;
    auto put = [&](int v, const uint4& w) {
        float f[N];
        Vec<T>::unpack(w, f);
        uint32_t o[N / 4];
#pragma unroll
        for (int i = 0; i < N / 4; ++i)
            o[i] = pack_whole(f[4 * i], f[4 * i + 1], f[4 * i + 2], f[4 * i + 3], r.inv) & r.keep;
        if (word_stores) {
            if (N == 8)
                *(uint2*)(dst + (size_t)v * N) = make_uint2(o[0], o[N / 4 - 1]);
            else
                *(uint32_t*)(dst + (size_t)v * N) = o[0];
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i)
                dst[(size_t)v * N + i] = (int8_t)(o[i / 4] >> (8 * (i % 4)));
        }
    };
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
        if (lane + i * LANES < nvec)
            put(lane + i * LANES, held[i]);
    for (int v = lane + kHeld * LANES; v < nvec; v += LANES)
        put(v, ((const uint4*)src)[v]);
    for (int i = nvec * N + lane; i < k; i += LANES)
        dst[i] = (int8_t)(to_whole(to_float(src[i]), r.inv) & r.keep);
}

template <class T>
int quantize_rows(
        const T* x, int m, int k, long long ldx, int8_t* q, long long ldq, float* scales, cudaStream_t st) {
    constexpr int N = Vec<T>::N;
    const int vector_loads = ((uintptr_t)x & 15) == 0 && (m == 1 || ldx % N == 0);
    const int word_stores = ((uintptr_t)q & (N - 1)) == 0 && (m == 1 || ldq % N == 0);
    // (numbers and scales, and what lies between them)
    const uintptr_t q0 = (uintptr_t)q, q1 = q0 + (size_t)(m - 1) * (size_t)ldq + (size_t)k;
    const uintptr_t s0 = (uintptr_t)scales, s1 = s0 + (size_t)m * 4;
    const uintptr_t w0 = q0 < s0 ? q0 : s0, w1 = q1 > s1 ? q1 : s1;
    const Writes writes{(const void*)w0, w1 - w0};
    cudaError_t e;
    if (k <= 32 * kHeld * N && m > 1)
        e = launch_pdl(writes, quantize_rows_kernel<T, 32>, dim3((unsigned)((m - 1) / 8 + 1)),
                       dim3(kRowThreads), 0, st, x, m, k, ldx, q, ldq, scales, vector_loads, word_stores);
    else
        e = launch_pdl(writes, quantize_rows_kernel<T, kRowThreads>, dim3((unsigned)m), dim3(kRowThreads), 0,
                       st, x, m, k, ldx, q, ldq, scales, vector_loads, word_stores);
    if (e != cudaSuccess)
        return set_error(ST_RUNTIME, "quantize_rows: %s", cudaGetErrorString(e));
    return check_launch("quantize_rows");
}

// ---- product for few tokens ----
// HBM: n * k bytes of weights are read once, whatever m. A CTA makes 16 rows of weights times 8 * NT
// tokens; its eight warps take the 64-byte chunks of K in turn and read them straight from global memory into
// the registers of mma.sync (16 neighbouring bytes per thread; which K byte meets which word of the MMA
// does not matter as long as the tokens' are laid out alike), so nothing waits for shared memory or
// a barrier before the sums meet at the end.
constexpr int kWarps = 8;
constexpr int kRows = 16;     // weight rows per CTA
constexpr int kColPitch = 20; // ints per token in the exchange: 2 * 20 = 8 banks apart

template <class XT, int NT, bool ALIGNED>
__global__ void __launch_bounds__(32 * kWarps, NT <= 2 ? 2 : 1) product_stream_kernel(const ProductArgs p, int x_vectors) {
    constexpr bool kFloat = sizeof(XT) > 1;
    constexpr int U = NT == 1 ? 8 : NT == 2 ? 4 : 2;  // chunks in flight per warp
    constexpr int kCols = 8 * NT;
    __shared__ int red[kWarps][kCols][kColPitch];
    __shared__ uint32_t part[kFloat ? kWarps : 1][kCols];
    __shared__ float col_scale[kCols];

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, tig = lane & 3;
    const int n0 = blockIdx.x * kRows;
    const int m0 = blockIdx.y * kCols;
    const int k = p.k, chunks = (k + 63) >> 6;
    const int row_lo = n0 + g, row_hi = n0 + g + 8;
    const int8_t* b_lo = p.b + (size_t)min(row_lo, p.n - 1) * p.ldb;
    const int8_t* b_hi = p.b + (size_t)min(row_hi, p.n - 1) * p.ldb;

    uint4 w[U][2];
    auto load_weights = [&](int c0) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int kk = (c0 + u * kWarps) * 64 + tig * 16;
            if (ALIGNED) {
                w[u][0] = w[u][1] = make_uint4(0, 0, 0, 0);
                if (kk < k) {
                    w[u][0] = ld_stream16(b_lo + kk);
                    w[u][1] = ld_stream16(b_hi + kk);
                }
            } else {
                w[u][0] = ld_any16(b_lo + kk, k - kk);
                w[u][1] = ld_any16(b_hi + kk, k - kk);
            }
        }
    };
    if (p.b_early)
        load_weights(warp);
    pdl_start();
    if (!p.b_early)
        load_weights(warp);

    // a thread's columns of B: tokens m0 + 8 * nt + g
    const XT* a[NT];
    bool have[NT];
    RowScale rs[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int t = m0 + 8 * nt + g;
        have[nt] = t < p.m;
        a[nt] = (const XT*)p.a + (long long)min(t, p.m - 1) * p.lda;
    }
    if constexpr (kFloat) {
        // the rows' scales: every warp has the maximum of its chunks
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            uint32_t bits = 0;
            if (have[nt]) {
                for (int c = warp; c < chunks; c += kWarps) {
                    float v[16];
                    load_piece(a[nt], c * 64 + tig * 16, k, x_vectors, v);
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        bits = max(bits, magnitude(v[i]));
                }
            }
            bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, 1));
            bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, 2));
            if (tig == 0)
                part[warp][8 * nt + g] = bits;
        }
        __syncthreads();
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            uint32_t bits = 0;
#pragma unroll
            for (int i = 0; i < kWarps; ++i)
                bits = max(bits, part[i][8 * nt + g]);
            rs[nt] = row_scale(bits);
            if (warp == 0 && tig == 0)
                col_scale[8 * nt + g] = rs[nt].scale;
        }
    } else {
        if (threadIdx.x < kCols)
            col_scale[threadIdx.x] = m0 + (int)threadIdx.x < p.m ? p.sa[m0 + threadIdx.x] : 0.f;
    }

    int acc[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
        acc[nt][0] = acc[nt][1] = acc[nt][2] = acc[nt][3] = 0;
    for (int c0 = warp; c0 < chunks; c0 += U * kWarps) {
        if (c0 != warp)
            load_weights(c0);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            uint4 t[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int kk = (c0 + u * kWarps) * 64 + tig * 16;
                t[u] = make_uint4(0, 0, 0, 0);
                if constexpr (kFloat) {
                    if (have[nt] && kk < k) {
                        float v[16];
                        load_piece(a[nt], kk, k, x_vectors, v);
                        t[u] = pack_piece(v, rs[nt]);
                    }
                } else if (have[nt]) {
                    if (ALIGNED) {
                        if (kk < k)
                            t[u] = *(const uint4*)((const int8_t*)a[nt] + kk);
                    } else {
                        t[u] = ld_any16((const int8_t*)a[nt] + kk, k - kk);
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
                mma_64(acc[nt], w[u][0], w[u][1], t[u]);
        }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        int(*r)[kColPitch] = red[warp] + 8 * nt + 2 * tig;
        r[0][g] = acc[nt][0];
        r[1][g] = acc[nt][1];
        r[0][g + 8] = acc[nt][2];
        r[1][g + 8] = acc[nt][3];
    }
    __syncthreads();
    const int row = threadIdx.x & 15, n = n0 + row;
    if (n >= p.n)
        return;
    const float sb = p.sb[n], bias = p.bias ? p.bias[n] : 0.f;
    for (int col = threadIdx.x >> 4; col < kCols && m0 + col < p.m; col += 2 * kWarps) {
        int sum = 0;
#pragma unroll
        for (int i = 0; i < kWarps; ++i)
            sum += red[i][col][row];
        float v = scale_acc(sum, col_scale[col], sb);
        if (p.bias)
            v = __fadd_rn(v, bias);
        store_as(p.c, p.c_dtype, (size_t)(m0 + col) * (size_t)p.ldc + n, v);
    }
}

__global__ void __launch_bounds__(256) pad_rows_kernel(
        const int8_t* __restrict__ src, long long ld, int k, int8_t* __restrict__ dst, int units, long long total) {
    pdl_start();
    for (long long i = blockIdx.x * 256LL + threadIdx.x; i < total; i += gridDim.x * 256LL) {
        const long long row = i / units;
        const int at = (int)(i - row * units) * 16;
        ((uint4*)dst)[i] = ld_any16(src + row * ld + at, k - at);
    }
}

template <class XT, int NT>
cudaError_t launch_stream(const ProductArgs& a, bool aligned, int x_vectors, cudaStream_t st) {
    const dim3 grid((unsigned)((a.n - 1) / kRows + 1), (unsigned)((a.m - 1) / (8 * NT) + 1));
    const size_t size = dtype_bytes(a.c_dtype);
    const Writes writes{a.c, ((size_t)(a.m - 1) * (size_t)a.ldc + (size_t)a.n) * size};
    return aligned ? launch_pdl(writes, product_stream_kernel<XT, NT, true>, grid, dim3(32 * kWarps), 0, st, a,
                                x_vectors)
                   : launch_pdl(writes, product_stream_kernel<XT, NT, false>, grid, dim3(32 * kWarps), 0, st, a,
                                x_vectors);
}

template <class XT>
cudaError_t launch_stream_float(const ProductArgs& a, bool aligned, cudaStream_t st) {
    const int x_vectors = ((uintptr_t)a.a & 15) == 0 && (a.m == 1 || a.lda % Vec<XT>::N == 0);
    return a.m <= 8 ? launch_stream<XT, 1>(a, aligned, x_vectors, st)
                    : launch_stream<XT, 2>(a, aligned, x_vectors, st);
}

}  // namespace

int launch_quantize_rows(
        const void* x, int dtype, int m, int k, long long ldx, int8_t* q, long long ldq, float* scales,
        cudaStream_t st) {
    if (dtype == DT_F32)
        return quantize_rows((const float*)x, m, k, ldx, q, ldq, scales, st);
    if (dtype == DT_F16)
        return quantize_rows((const __half*)x, m, k, ldx, q, ldq, scales, st);
    return quantize_rows((const __nv_bfloat16*)x, m, k, ldx, q, ldq, scales, st);
}

int launch_pad_rows(
        const int8_t* src, long long ld, int rows, int k, int8_t* dst, long long pitch, cudaStream_t st) {
    const int units = (int)(pitch / 16);
    const long long total = (long long)rows * units, ctas = (total + 255) / 256;
    const cudaError_t e = launch_pdl(
            Writes{dst, (size_t)total * 16}, pad_rows_kernel, dim3((unsigned)(ctas < 4736 ? ctas : 4736)), dim3(256), 0,
            st, src, ld, k, dst, units, total);
    if (e != cudaSuccess)
        return set_error(ST_RUNTIME, "matmul_s8_scaled: %s", cudaGetErrorString(e));
    return check_launch("matmul_s8_scaled");
}

int launch_product_stream(const ProductArgs& a, cudaStream_t st) {
    const bool b_aligned = ((uintptr_t)a.b & 15) == 0 && (a.n == 1 || a.ldb % 16 == 0) && a.k % 16 == 0;
    cudaError_t e;
    if (a.x_dtype < 0) {
        const bool aligned = b_aligned && ((uintptr_t)a.a & 15) == 0 && (a.m == 1 || a.lda % 16 == 0);
        e = a.m <= 8    ? launch_stream<int8_t, 1>(a, aligned, 0, st)
            : a.m <= 16 ? launch_stream<int8_t, 2>(a, aligned, 0, st)
            : a.m <= 32 ? launch_stream<int8_t, 4>(a, aligned, 0, st)
                        : launch_stream<int8_t, 8>(a, aligned, 0, st);
    } else if (a.x_dtype == DT_F32) {
        e = launch_stream_float<float>(a, b_aligned, st);
    } else if (a.x_dtype == DT_F16) {
        e = launch_stream_float<__half>(a, b_aligned, st);
    } else {
        e = launch_stream_float<__nv_bfloat16>(a, b_aligned, st);
    }
    if (e != cudaSuccess)
        return set_error(ST_RUNTIME, "matmul_s8_scaled: %s", cudaGetErrorString(e));
    return check_launch("matmul_s8_scaled");
}

}  // namespace scaled
}  // namespace mb200
