// int8 products for few tokens, and the conversion of activations to int8 rows.
#include "stream_s8.cuh"
#include "umma_ptx.cuh"

namespace mb200 {
namespace scaled {

namespace {

// ---- rows to whole numbers ----
// HBM: every element is read once and written once as a byte. LANES threads share a row: a warp where
// a row fits its registers (no barrier), else a whole CTA. The first HELD * LANES vectors of the row stay
// in registers between the maximum and the conversion, what lies behind them is read again.
// Vectors are the 16-byte units that the row lies in, zeros around it: with aligned == 0 rows start anywhere in their
// first one, and their numbers go anywhere in a word (4001 x 4095 fp16: 25.8 us; with rows partly in the L2 21.9, and 39.3
// with its numbers stored one by one).
template <class T, int LANES, int HELD, int THREADS>
__global__ void __launch_bounds__(THREADS, THREADS == 512 ? 2 : 0) quantize_rows_kernel(
        const T* __restrict__ x, int m, int k, long long ldx, int8_t* __restrict__ q, long long ldq,
        float* __restrict__ scales, int aligned) {
    constexpr int N = Vec<T>::N;
    __shared__ uint32_t part[THREADS / 32];
    pdl_start();
    const int lane = threadIdx.x % LANES, in_warp = threadIdx.x & 31;
    const long long row = (long long)blockIdx.x * (THREADS / LANES) + threadIdx.x / LANES;
    if (LANES == 32 && row >= m)
        return;  // (a whole warp; no barrier follows in this form)
    // elements of the first unit in front of the row
    const int before = aligned ? 0 : (int)(((uintptr_t)(x + row * ldx) & 15) / sizeof(T));
    const uint4* src = (const uint4*)(x + row * ldx - before);
    int8_t* dst = q + row * ldq - before;
    const unsigned end = (unsigned)before + (unsigned)k;
    const int nvec = (int)((end - 1) / N) + 1, whole = (int)(end / N), first_whole = before > 0;
    auto load = [&](int v) {
        uint4 w = src[v];
        if (v < first_whole || v >= whole) {
            const int from = v == 0 ? before * (int)sizeof(T) : 0;
            const int to = v < whole ? 16 : (int)(end - (unsigned)v * N) * (int)sizeof(T);
            uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int lo = min(max(from - 4 * i, 0), 4), hi = min(max(to - 4 * i, 0), 4);
                u[i] = lo >= hi ? 0u : u[i] >> (8 * lo) << (8 * (lo + 4 - hi)) >> (8 * (4 - hi));
            }
            w = make_uint4(u[0], u[1], u[2], u[3]);
        }
        return w;
    };
    uint4 held[HELD];
    uint32_t vm = 0;
    if (aligned) {
#pragma unroll
        for (int i = 0; i < HELD; ++i) {
            const int v = lane + i * LANES;
            held[i] = v < whole ? src[v] : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < HELD; ++i)
            vm = vec_max<T>(vm, held[i]);
    }
    // (what is not held: the vectors behind, the end of a row, all of a row that starts anywhere)
    const int rest = aligned ? min(whole, HELD * LANES) : 0;
#pragma unroll 4
    for (int v = lane + rest; v < nvec; v += LANES)
        vm = vec_max<T>(vm, load(v));
    uint32_t bits = max_bits<T>(vm);
    bits = __reduce_max_sync(0xffffffffu, bits);
    if (LANES > 32) {
        if (in_warp == 0)
            part[threadIdx.x >> 5] = bits;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < THREADS / 32; ++w)
            bits = max(bits, part[w]);
    }
    const RowScale r = row_scale(bits);
    if (lane == 0)
        scales[row] = r.scale;
    auto convert = [&](uint32_t(&o)[N / 4], const uint4& w) {
        float f[N];
        Vec<T>::unpack(w, f);
#pragma unroll
        for (int i = 0; i < N / 4; ++i)
            o[i] = pack_whole(f[4 * i], f[4 * i + 1], f[4 * i + 2], f[4 * i + 3], r.inv) & r.keep;
    };
    auto put = [&](int v, const uint4& w) {
        uint32_t o[N / 4];
        convert(o, w);
        if (v < whole) {
            if (N == 8)
                *(uint2*)(dst + (size_t)v * N) = make_uint2(o[0], o[N / 4 - 1]);
            else
                *(uint32_t*)(dst + (size_t)v * N) = o[0];
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (i < k - v * N)
                    dst[(size_t)v * N + i] = (int8_t)(o[i / 4] >> (8 * (i % 4)));
        }
    };
    // The words that a lane's bytes lie in up to the last one, which the lane behind it stores with its own first bytes
    // (and lane 0 makes those of the vector in front again). Called by whole warps, for one vector behind the last too.
    auto put_any = [&](int v) {
        uint32_t o[N / 4], in_front[N / 4];
        convert(o, v < nvec ? load(v) : make_uint4(0, 0, 0, 0));
        if (in_warp == 0)
            convert(in_front, v > 0 && v <= nvec ? load(v - 1) : make_uint4(0, 0, 0, 0));
        const uint32_t last = __shfl_up_sync(0xffffffffu, o[N / 4 - 1], 1);
        if (in_warp > 0)
            in_front[N / 4 - 1] = last;
        const int s = (int)((uintptr_t)dst & 3);
#pragma unroll
        for (int i = 0; i < N / 4; ++i)
            o[N / 4 - 1 - i] = __funnelshift_l(i < N / 4 - 1 ? o[N / 4 - 2 - i] : in_front[N / 4 - 1], o[N / 4 - 1 - i],
                                               8 * s);
        int8_t* to = dst + (long long)v * N - s;
        if (v > 1 && v < whole) {
#pragma unroll
            for (int i = 0; i < N / 4; ++i)
                ((uint32_t*)to)[i] = o[i];
        } else if (v <= nvec) {
            const long long at = (long long)v * N - s;
#pragma unroll 1
            for (int b = 0; b < N; ++b) {
                if (at + b >= before && at + b < end)
                    to[b] = (int8_t)o[0];
                o[0] = __funnelshift_r(o[0], N == 8 ? o[N / 4 - 1] : 0, 8);
                if (N == 8)
                    o[N / 4 - 1] >>= 8;
            }
        }
    };
    if (aligned) {
#pragma unroll
        for (int i = 0; i < HELD; ++i)
            if (lane + i * LANES < whole)
                put(lane + i * LANES, held[i]);
#pragma unroll 1
        for (int v = lane + rest; v < nvec; v += LANES)
            put(v, load(v));
    } else {
#pragma unroll 2
        for (int v = lane; v - in_warp <= nvec; v += LANES)
            put_any(v);
    }
}

template <class T>
int quantize_rows(
        const T* x, int m, int k, long long ldx, int8_t* q, long long ldq, float* scales, cudaStream_t st) {
    constexpr int N = Vec<T>::N;
    const int aligned = (((uintptr_t)x & 15) | ((uintptr_t)q & (N - 1))) == 0 &&
                        (m == 1 || (ldx % N == 0 && ldq % N == 0));
    // (numbers and scales, and what lies between them)
    const uintptr_t q0 = (uintptr_t)q, q1 = q0 + (size_t)(m - 1) * (size_t)ldq + (size_t)k;
    const uintptr_t s0 = (uintptr_t)scales, s1 = s0 + (size_t)m * 4;
    const uintptr_t w0 = q0 < s0 ? q0 : s0, w1 = q1 > s1 ? q1 : s1;
    const Writes writes{(const void*)w0, w1 - w0};
    auto launch = [&](auto kernel, int rows, int threads, MostShared& shared) {
        shared.ask(kernel);
        return launch_pdl(writes, kernel, dim3((unsigned)((m - 1) / rows + 1)), dim3((unsigned)threads), 0, st, x, m,
                          k, ldx, q, ldq, scales, aligned);
    };
    // A warp per row where it holds the row and there are rows enough for every SM's warps: 4001 x 4096 fp16 from HBM in
    // 9.2 us (5.3 TB/s), by whole CTAs in 10.2. The CTA grows with the row, so that it holds it as long as that goes:
    // 4096 x 14336 fp32 by 512 threads in 57.3 us (5.1 TB/s), by 256 in 63.9.
    static MostShared shared[5];
    const cudaError_t e =
            m > 1 && k <= 32 * 4 * N        ? launch(quantize_rows_kernel<T, 32, 4, 256>, 8, 256, shared[0])
            : m >= 2048 && k <= 32 * 16 * N ? launch(quantize_rows_kernel<T, 32, 16, 64>, 2, 64, shared[1])
            : k <= 256 * 4 * N              ? launch(quantize_rows_kernel<T, 256, 4, 256>, 1, 256, shared[2])
            : k <= 256 * 8 * N              ? launch(quantize_rows_kernel<T, 256, 8, 256>, 1, 256, shared[3])
                                            : launch(quantize_rows_kernel<T, 512, 8, 512>, 1, 512, shared[4]);
    if (e != cudaSuccess)
        return refused("quantize_rows", e);
    return check_launch("quantize_rows");
}

// ---- product for few tokens ----
// HBM: n * k bytes of weights are read once, whatever m. SHARED: a CTA makes 16 rows of weights times 8 * NT
// tokens; its eight warps take the 128-byte steps of K in turn (stream_s8.cuh) and their sums meet at the end.
// Otherwise each warp makes 16 rows of its own: for short K, where a warp of eight had a step or none, and enough
// rows for the SMs (2 x 12735 x 74: 6.1 us shared).
// int8 tokens come through the ring beside the weights; activations that are still floats are made whole
// numbers first, by every CTA again, while its first weights are on their way.
constexpr int kWarps = 8;
constexpr int kRows = 16;     // weight rows per CTA
constexpr int kColPitch = 20; // ints per token in the exchange: 2 * 20 = 8 banks apart

template <class XT, int NT, bool ALIGNED, bool TOKENS, bool SHARED>
struct Stream {
    static constexpr bool kFloat = sizeof(XT) > 1;
    static constexpr int kCols = 8 * NT;
    static constexpr int kDepth = NT == 1 ? 4 : NT == 2 ? 3 : 2;  // (room for two CTAs per SM)
    typedef Rows<kRows, ALIGNED, true> W;
    typedef Rows<kCols, TOKENS, true> A;
    static constexpr int kStage = W::kBytes + (kFloat ? 0 : A::kBytes);
    static constexpr int kRing = kWarps * kDepth * kStage;
    static constexpr int kCtaRows = SHARED ? kRows : kRows * kWarps;
};

// ALIGNED, TOKENS: rows of weights, of int8 tokens are whole 16-byte units
template <class XT, int NT, bool ALIGNED, bool TOKENS, bool SHARED>
__global__ void __launch_bounds__(32 * kWarps, 2) product_stream_kernel(const ProductArgs p, int x_vectors) {
    typedef Stream<XT, NT, ALIGNED, TOKENS, SHARED> S;
    constexpr bool kFloat = S::kFloat;
    constexpr int kDepth = S::kDepth, kCols = S::kCols;
    extern __shared__ __align__(128) uint8_t dynamic[];  // the rings, then (floats) xs
    __shared__ float col_scale[kCols];
    __shared__ uint32_t part[kFloat ? kCols * kWarps : 1];

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, tig = lane & 3;
    const int n0 = blockIdx.x * S::kCtaRows + (SHARED ? 0 : warp * kRows);
    const int m0 = blockIdx.y * kCols;
    const int k = p.k, steps = (k + kStep - 1) / kStep;
    // this warp's steps: its first one, how far apart they are, how many
    const int first = SHARED ? warp : 0, by = SHARED ? kWarps : 1;
    const int mine = first < steps ? (steps - first + by - 1) / by : 0;
    const uint32_t ring = shared_address(dynamic) + (uint32_t)(warp * kDepth * S::kStage);
    int8_t* xs = (int8_t*)dynamic + S::kRing;
    const int pitch = xs_pitch(k);

    auto b_row = [&](int r) { return p.b + (size_t)min(n0 + r, p.n - 1) * p.ldb; };
    auto a_row = [&](int r) { return (const int8_t*)p.a + (long long)min(m0 + r, p.m - 1) * p.lda; };
    typename S::W w;
    typename S::A a;
    w.open(b_row, k, first);
    if (!kFloat)
        // (no copies for tokens that are not there: every CTA asks for the same few lines)
        a.open([&](int r) { return m0 + r < p.m ? a_row(r) : nullptr; }, k, first);
    auto copy_weights = [&](uint32_t stage, int i) {
        if (i < mine)
            w.template copy<true>(stage, by, k - (first + i * by) * kStep >= S::W::kWhole);
    };
    auto copy_tokens = [&](uint32_t stage, int i) {
        if (!kFloat && i < mine)
            a.template copy<false>(stage + S::W::kBytes, by, k - (first + i * by) * kStep >= S::A::kWhole);
    };
    if (p.b_early)
#pragma unroll 1
        for (int i = 0; i < kDepth - 1; ++i)
            copy_weights(ring + (uint32_t)(i * S::kStage), i);
    pdl_start();
#pragma unroll 1
    for (int i = 0; i < kDepth - 1; ++i) {
        const uint32_t stage = ring + (uint32_t)(i * S::kStage);
        if (!p.b_early)
            copy_weights(stage, i);
        copy_tokens(stage, i);
        copy_commit();
    }
    // scales of what this thread stores in the end
    const int row = threadIdx.x & 15, n = n0 + row;
    const float sb = n < p.n ? p.sb[n] : 0.f, bias = p.bias && n < p.n ? p.bias[n] : 0.f;
    if constexpr (kFloat) {
        rows_to_whole<XT, kWarps>([&](int r) { return (const XT*)p.a + (long long)(m0 + r) * p.lda; },
                                  min(kCols, p.m - m0), k, xs, pitch, col_scale, part, x_vectors);
        __syncthreads();
    } else {
        if (threadIdx.x < kCols)
            col_scale[threadIdx.x] = m0 + (int)threadIdx.x < p.m ? p.sa[m0 + threadIdx.x] : 0.f;
    }
    // rows and columns of this thread's fragments
    const int s_lo = (int)((uintptr_t)b_row(g) & 15), s_hi = (int)((uintptr_t)b_row(g + 8) & 15);
    int s_a[NT];
    const int8_t* x_at[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        s_a[nt] = kFloat ? 0 : (int)((uintptr_t)a_row(8 * nt + g) & 15);
        x_at[nt] = xs + min(8 * nt + g, p.m - 1 - m0) * pitch + tig * 16;
    }
    int acc[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
        acc[nt][0] = acc[nt][1] = acc[nt][2] = acc[nt][3] = 0;
    uint32_t stage = ring, free_stage = ring + (uint32_t)((kDepth - 1) * S::kStage);
#pragma unroll 1
    for (int i = 0; i < mine; ++i) {
        copy_wait<kDepth - 2>();
        __syncwarp();  // all lanes' copies of this step are there, and the last step's stage has been read
        copy_weights(free_stage, i + kDepth - 1);
        copy_tokens(free_stage, i + kDepth - 1);
        copy_commit();
        next_stage<kDepth, S::kStage>(free_stage, ring);
        const int step = first + i * by;
#pragma unroll
        for (int j = 0; j < kStep / 64; ++j) {
            const int piece = 4 * j + tig;
            const uint4 lo = S::W::piece16(stage, g, piece, s_lo), hi = S::W::piece16(stage, g + 8, piece, s_hi);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                uint4 t;
                if constexpr (kFloat) {
                    t = *(const uint4*)(x_at[nt] + step * kStep + 64 * j);
                } else {
                    t = S::A::piece16(stage + S::W::kBytes, 8 * nt + g, piece, s_a[nt]);
                    if (!ALIGNED && step == steps - 1)  // (where rows end with a unit, zeros lie behind it)
                        t = first_bytes(t, k - step * kStep - piece * 16);
                }
                mma_64(acc[nt], lo, hi, t);
            }
        }
        next_stage<kDepth, S::kStage>(stage, ring);
    }
    copy_wait<0>();
    __syncthreads();
    // (the rings are done with)
    int(*red)[kCols][kColPitch] = (int(*)[kCols][kColPitch])dynamic;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        int(*r)[kColPitch] = red[warp] + 8 * nt + 2 * tig;
        r[0][g] = acc[nt][0];
        r[1][g] = acc[nt][1];
        r[0][g + 8] = acc[nt][2];
        r[1][g + 8] = acc[nt][3];
    }
    __syncthreads();
    if (n >= p.n)
        return;
    for (int col = (SHARED ? threadIdx.x : lane) >> 4; col < kCols && m0 + col < p.m; col += SHARED ? 2 * kWarps : 2) {
        int sum = SHARED ? 0 : red[warp][col][row];
        if (SHARED)
#pragma unroll
            for (int i = 0; i < kWarps; ++i)
                sum += red[i][col][row];
        float v = scale_acc(sum, col_scale[col], sb);
        if (p.bias)
            v = __fadd_rn(v, bias);
        store_as(p.c, p.c_dtype, (size_t)(m0 + col) * (size_t)p.ldc + n, v);
    }
}

// Rows of any alignment to rows of whole 16-byte units, a warp per row, or a CTA where there are few
template <int LANES>
__global__ void __launch_bounds__(256) pad_rows_kernel(const PadRows a, const PadRows b) {
    pdl_start();
    const long long job = blockIdx.x * (256LL / LANES) + threadIdx.x / LANES;
    const bool second = job >= a.rows;
    const PadRows& j = second ? b : a;
    const long long row = second ? job - a.rows : job;
    if (row >= j.rows)
        return;
    const int8_t* src = j.src + row * j.ld;
    uint4* dst = (uint4*)(j.dst + row * j.pitch);
#pragma unroll 4
    for (int u = threadIdx.x % LANES; u < (int)(j.pitch / 16); u += LANES)
        dst[u] = ld_any16(src + 16 * u, j.k - 16 * u);
}

template <class XT, int NT, bool ALIGNED, bool TOKENS, bool SHARED>
cudaError_t launch_stream_as(const ProductArgs& a, int x_vectors, cudaStream_t st) {
    typedef Stream<XT, NT, ALIGNED, TOKENS, SHARED> S;
    static umma::KernelReady ready;
    static MostShared shared;
    static_assert(S::kRing >= kWarps * S::kCols * kColPitch * 4, "the exchange lies where the rings were");
    auto kernel = product_stream_kernel<XT, NT, ALIGNED, TOKENS, SHARED>;
    const int smem = S::kRing + (S::kFloat ? (a.m < S::kCols ? a.m : S::kCols) * xs_pitch(a.k) : 0);
    if (!ready.smem(kernel, smem))
        return why_refused();
    shared.ask(kernel);
    const dim3 grid((unsigned)((a.n - 1) / S::kCtaRows + 1), (unsigned)((a.m - 1) / S::kCols + 1));
    const Writes writes{a.c, ((size_t)(a.m - 1) * (size_t)a.ldc + (size_t)a.n) * dtype_bytes(a.c_dtype)};
    return launch_pdl(writes, kernel, grid, dim3(32 * kWarps), (size_t)smem, st, a, x_vectors);
}
template <class XT, int NT, bool ALIGNED, bool TOKENS>
cudaError_t launch_stream(const ProductArgs& a, int x_vectors, cudaStream_t st) {
    // Warps of their own where shared tiles would take several turns on the SMs for a step or two per warp, or up to 2048
    // bytes where rows are whole lines and there are enough for all SMs (20000 x 2048, one token: 9.0 us, by tiles 19.2;
    // with lines that two steps share, 8 x 20000 x 1552, 14.4 to 17.3 us for the shared form's 12.2)
    const long long ctas = ((long long)(a.n - 1) / kRows + 1) * ((a.m - 1) / (8 * NT) + 1);
    const long long own = ((long long)(a.n - 1) / (kRows * kWarps) + 1) * ((a.m - 1) / (8 * NT) + 1);
    if ((a.k <= 8 * kStep && ctas > 2LL * umma::sm_count()) ||
        (a.k <= 16 * kStep && a.k % kStep == 0 && own >= umma::sm_count()))
        return launch_stream_as<XT, NT, ALIGNED, TOKENS, false>(a, x_vectors, st);
    return launch_stream_as<XT, NT, ALIGNED, TOKENS, true>(a, x_vectors, st);
}
template <int NT>
cudaError_t launch_stream_whole(const ProductArgs& a, bool aligned, bool tokens, cudaStream_t st) {
    return !tokens   ? launch_stream<int8_t, NT, false, false>(a, 0, st)
           : aligned ? launch_stream<int8_t, NT, true, true>(a, 0, st)
                     : launch_stream<int8_t, NT, false, true>(a, 0, st);
}

template <class XT>
cudaError_t launch_stream_float(const ProductArgs& a, bool aligned, cudaStream_t st) {
    const int x_vectors = ((uintptr_t)a.a & 15) == 0 && (a.m == 1 || a.lda % Vec<XT>::N == 0);
    return aligned ? launch_stream<XT, 1, true, true>(a, x_vectors, st)
                   : launch_stream<XT, 1, false, true>(a, x_vectors, st);
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

int launch_pad_rows(const PadRows& a, const PadRows& b, cudaStream_t st) {
    const long long rows = (long long)a.rows + b.rows;
    if (rows == 0)
        return ST_SUCCESS;
    // (what is written, and what lies between the two)
    uintptr_t lo = UINTPTR_MAX, hi = 0;
    for (const PadRows* j : {&a, &b})
        if (j->rows) {
            const uintptr_t at = (uintptr_t)j->dst, end = at + (size_t)j->rows * (size_t)j->pitch;
            lo = at < lo ? at : lo;
            hi = end > hi ? end : hi;
        }
    const Writes writes{(const void*)lo, hi - lo};
    static MostShared shared[2];
    shared[0].ask(pad_rows_kernel<256>);
    shared[1].ask(pad_rows_kernel<32>);
    const cudaError_t e = rows < 16LL * umma::sm_count()
                                  ? launch_pdl(writes, pad_rows_kernel<256>, dim3((unsigned)rows), dim3(256), 0, st, a, b)
                                  : launch_pdl(writes, pad_rows_kernel<32>, dim3((unsigned)((rows + 7) / 8)), dim3(256),
                                               0, st, a, b);
    if (e != cudaSuccess)
        return refused("matmul_s8_scaled", e);
    return check_launch("matmul_s8_scaled");
}

int launch_product_stream(const ProductArgs& a, cudaStream_t st) {
    const bool b_aligned = ((uintptr_t)a.b & 15) == 0 && (a.n == 1 || a.ldb % 16 == 0) && a.k % 16 == 0;
    cudaError_t e;
    if (a.x_dtype < 0) {
        const bool tokens = ((uintptr_t)a.a & 15) == 0 && (a.m == 1 || a.lda % 16 == 0);
        e = a.m <= 8    ? launch_stream_whole<1>(a, b_aligned, tokens, st)
            : a.m <= 16 ? launch_stream_whole<2>(a, b_aligned, tokens, st)
                        : launch_stream_whole<4>(a, b_aligned, tokens, st);
    } else if (a.x_dtype == DT_F32) {
        e = launch_stream_float<float>(a, b_aligned, st);
    } else if (a.x_dtype == DT_F16) {
        e = launch_stream_float<__half>(a, b_aligned, st);
    } else {
        e = launch_stream_float<__nv_bfloat16>(a, b_aligned, st);
    }
    if (e != cudaSuccess)
        return refused("matmul_s8_scaled", e);
    return check_launch("matmul_s8_scaled");
}

}  // namespace scaled
}  // namespace mb200
