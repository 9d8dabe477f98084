// Attention of one or a few queries per sequence over the paged int8 cache.
//
// For a key head, the rows are its group's query heads times the queries of a sequence. With the scores as powers of two,
//     t_j = (scale log2(e)) s_k q . k_j,   o = sum 2^(t_j - m) s_v v_j / sum 2^(t_j - m),
// over the positions j that a row sees, in one pass: m is a running maximum that is raised only where a score
// passes it by more than 8 (a vote per block of 16 positions, no reduction), so 2^(t - m) stays below 2^8.
//
// Bound by memory: 2 d bytes per position and key head are all there is to read, and eight rows' products take a
// third of the tensor cores' time at that rate even by mma.sync, whose operands come from registers: whole numbers are
// exact in fp16, where they are made by a byte permutation into 1024 + (v + 128) and a subtraction. Products are taken
// transposed, S^T = K Q^T and O^T = V^T P^T, so that positions and dimensions fill the 16 rows of an MMA and 8 query
// rows its 8 columns: half the instructions and accumulators of the other way round for groups of up to 8. The
// order of dimensions within S's sum is free: a lane takes 16 neighbouring ones with one load. V^T comes by
// ldmatrix.trans over pairs of bytes, whose two dimensions the byte permutation separates. P^T is turned by movmatrix.
//
// Queries are scaled by a power of two of their row, which makes fp16 of bf16 without loss for all elements within 2^-16
// of the row's largest; probabilities are rounded to fp16 (a relative 2^-12, under the results' own 2^-9 or
// 2^-12), after they took their block's scale of V relative to the largest so far, which keeps them in range. Sums and
// accumulators are fp32.
//
// All blocks of all sequences and key heads are one line, cut evenly over the CTAs whatever the lengths, which only
// the device knows. A CTA's warps take its blocks in turn, each through a ring of asynchronous copies of its own. Where a
// head's blocks are cut, the parts go to the workspace and a second kernel joins them in order.
#include "kv_cache.cuh"
#include "umma_ptx.cuh"

namespace mb200 {
namespace attn {
namespace {

constexpr int kWarps = 8, kThreads = 32 * kWarps;
constexpr int kLeast = kWarps;       // blocks a CTA takes at least: one for each warp
constexpr float kAhead = 8.f;        // how far a score may pass the running maximum
constexpr int kLift = 6;             // probabilities are held 2^6 times: 2^8 * 2 * 2^6 < 65504

template <int D>
struct Ring {
    static constexpr int kStage = 2 * kBlock * D + 16;  // keys, values, their two scales
    static constexpr int kStages = D == 128 ? 3 : 6;
    static constexpr int kBytes = kWarps * kStages * kStage;
};
// floats from row to row of the warps' sums: a warp's stores reach all banks
template <int D>
constexpr int kPitch = D + 4;

// How the line of blocks is cut, found alike by both kernels
struct Line {
    long long before, total;  // blocks in front of sequence b (times heads), in all
    int blocks;               // of sequence b
};
struct Shape {
    int rows, tiles, capacity;  // rows of a key head, tiles of them, positions a table has room for
};
__device__ __forceinline__ int blocks_of(const CacheArgs& a, int capacity, int b) {
    const int n = a.lengths[b];
    return n <= 0 ? 0 : (min(n, capacity) + kBlock - 1) / kBlock;
}
__device__ __forceinline__ long long quota_of(long long total, int ctas) {
    const long long q = (total + ctas - 1) / ctas;
    return (q + kLeast - 1) / kLeast * kLeast;
}

__device__ __forceinline__ uint32_t smem_at(const void* p) {
    return umma::smem_u32(p);
}
__device__ __forceinline__ void copy16(uint32_t to, const void* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t to, const void* from) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_end() {
    asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void copies_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(at)
                 : "memory");
    return v;
}
__device__ __forceinline__ float2 lds_f2(uint32_t at) {
    float2 v;
    asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t at, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(at)
                 : "memory");
}
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// two of four bytes v + 128 -> v as fp16: 0x6400 | b is 1024 + b
template <int SELECT>
__device__ __forceinline__ uint32_t two_f16(uint32_t biased) {
    const uint32_t w = __byte_perm(biased, 0x64646464u, SELECT);
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&w), __half2{__ushort_as_half(0x6480), __ushort_as_half(0x6480)});
    return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
    const __half2 r = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&r);
}
// 2^e for -126 <= e <= 127
__device__ __forceinline__ float power_of_two(int e) {
    return __uint_as_float((uint32_t)(e + 127) << 23);
}
// the exponent of a finite, normal magnitude; 0 for zero, infinities and NaNs (nothing is scaled then)
__device__ __forceinline__ int exponent_of(uint32_t magnitude_bits) {
    const int e = (int)(magnitude_bits >> 23);
    return e == 0 || e == 255 ? 0 : max(-120, min(120, e - 127));
}

// rows of the workspace's parts: [cta][first or last][row][D] sums, then [..][row] maxima and totals
struct Parts {
    float* sums;
    float2* stats;
};
__host__ __device__ inline Parts parts_of(void* workspace, int ctas, int rows, int d) {
    float* p = (float*)workspace;
    return Parts{p, (float2*)(p + (size_t)ctas * 2 * rows * d)};
}

// Where row r of a tile lies
__device__ __forceinline__ long long row_at(const CacheArgs& a, const mb200_heads& t, int group, int b, int h, int r) {
    const int i = r / group;
    return ((long long)b * a.queries + i) * t.token_stride + (long long)(h * group + (r - i * group)) * t.head_stride;
}

template <class T, int D, int NT, bool VEC>
__global__ void __launch_bounds__(kThreads, NT == 1 ? 2 : 1) cache_kernel(const CacheArgs a, const Shape shape) {
    constexpr int kRows = 8 * NT, kChunks = D / 64, kTiles = D / 16;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ long long s_from, s_to, s_blk;
    __shared__ int s_b, s_at;
    __shared__ float2 s_stats[kWarps][kRows];
    const int tid = threadIdx.x, lane = tid & 31, warp = umma::uniform_warp_index();
    const int g = lane >> 2, c = lane & 3;
    const int d = a.c.d, group = a.heads / a.c.kv_heads;
    const int lines = a.c.kv_heads * shape.tiles;  // of a sequence: key heads times tiles of rows
    pdl_start();

    // sequences without a position: nothing is seen
    for (int b = blockIdx.x; b < a.c.batch; b += gridDim.x) {
        if (a.lengths[b] > shape.capacity && tid == 0)
            *(volatile int*)a.status = ERR_PAGE;
        if (a.lengths[b] <= 0)
            for (int i = tid; i < a.queries * a.heads * d; i += kThreads) {
                const int e = i % d, th = i / d;
                ((T*)a.out.p)[((long long)b * a.queries + th / a.heads) * a.out.token_stride +
                              (long long)(th % a.heads) * a.out.head_stride + e] = from_float<T>(0.f);
            }
    }

    // this CTA's part of the line
    if (warp == 0) {
        long long total = 0;
        for (int b0 = 0; b0 < a.c.batch; b0 += 32) {
            const int n = b0 + lane < a.c.batch ? blocks_of(a, shape.capacity, b0 + lane) : 0;
            total += __reduce_add_sync(0xffffffffu, n);
        }
        total *= lines;
        const long long quota = quota_of(total, gridDim.x);
        const long long from = quota * blockIdx.x, to = from + quota < total ? from + quota : total;
        long long before = 0;
        int at = 0, n = 0;
        if (from < to) {
            for (int b0 = 0; b0 < a.c.batch; b0 += 32) {
                n = b0 + lane < a.c.batch ? blocks_of(a, shape.capacity, b0 + lane) : 0;
                int sum = n;
#pragma unroll
                for (int s = 1; s < 32; s *= 2) {
                    const int v = __shfl_up_sync(0xffffffffu, sum, s);
                    sum += lane >= s ? v : 0;
                }
                // (a sequence's blocks are counted lines times, one after the other)
                const uint32_t beyond = __ballot_sync(0xffffffffu, (before + sum) * lines > from);
                if (beyond) {
                    const int i = __ffs(beyond) - 1;
                    before += __shfl_sync(0xffffffffu, sum - n, i);
                    n = __shfl_sync(0xffffffffu, n, i);
                    at = b0 + i;
                    break;
                }
                before += __shfl_sync(0xffffffffu, sum, 31);
            }
        }
        if (lane == 0) {
            s_from = from, s_to = to, s_b = at;
            const long long rest = from - before * lines;
            s_at = n ? (int)(rest / n) : 0;
            s_blk = n ? rest % n : 0;
        }
    }
    __syncthreads();
    long long left = s_to - s_from;
    int b = s_b, at = s_at, blk = (int)s_blk;
    bool first = true;
    const uint32_t ring = smem_at(smem) + warp * (Ring<D>::kStages * Ring<D>::kStage);
    // where this lane's 16-byte units of a block go: row r's unit u beside others' so that loads meet all banks
    const int units = d / 16;
    uint32_t to_k[D / 32], to_v[D / 32];
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
        const int x = lane + 32 * i, r = x / units, u = x - r * units;
        to_k[i] = (uint32_t)(r * D + (u ^ (D == 128 ? (r & 1) << 2 : 0)) * 16);
        to_v[i] = (uint32_t)(kBlock * D + r * D + (u ^ (D == 128 ? r & 7 : (r >> 1) & 3)) * 16);
    }
    const int page_blocks = a.c.page_tokens / kBlock;

#pragma unroll 1
    while (left > 0) {
        const int length = min(a.lengths[b], shape.capacity);
        const int all = (max(length, 0) + kBlock - 1) / kBlock;
        if (all == 0) {
            ++b;
            continue;
        }
        const int h = at / shape.tiles, tile = at - h * shape.tiles;
        const int count = (int)(left < all - blk ? left : all - blk);
        const int row0 = tile * kRows, rows = min(kRows, shape.rows - row0);

        // queries: lane (g, c) holds of row g the dimensions 64 i + 16 c .. + 15 as fp16, and its factor
        uint32_t qf[NT][kChunks][8];
        float f0[NT], f1[NT];
        int lim0[NT], lim1[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int r = nt * 8 + g;
            float x[kChunks][16];
            uint32_t most = 0;
#pragma unroll
            for (int i = 0; i < kChunks; ++i) {
                const int dim = 64 * i + 16 * c;
                uint4 lo = make_uint4(0, 0, 0, 0), hi = lo;
                if (r < rows && dim < d) {
                    const long long p = row_at(a, a.q, group, b, h, row0 + r) + dim;
                    lo = load8<VEC>(a.q.p, p);
                    hi = load8<VEC>(a.q.p, p + 8);
                }
                Vec<T>::unpack(lo, *reinterpret_cast<float(*)[8]>(&x[i][0]));
                Vec<T>::unpack(hi, *reinterpret_cast<float(*)[8]>(&x[i][8]));
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    most = max(most, magnitude(x[i][e]));
            }
            most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
            most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
            const int e = exponent_of(most);
            const float down = power_of_two(-e), factor = __fmul_rn(power_of_two(e), a.scale_log2);
#pragma unroll
            for (int i = 0; i < kChunks; ++i)
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    qf[nt][i][j] = pack_f16(__fmul_rn(x[i][2 * j], down), __fmul_rn(x[i][2 * j + 1], down));
            f0[nt] = __shfl_sync(0xffffffffu, factor, 8 * c);
            f1[nt] = __shfl_sync(0xffffffffu, factor, 8 * c + 4);
            // positions that rows 2 c and 2 c + 1 of this tile see
            lim0[nt] = length - a.queries + 1 + (row0 + nt * 8 + 2 * c) / group;
            lim1[nt] = length - a.queries + 1 + (row0 + nt * 8 + 2 * c + 1) / group;
        }
        const int seen_by_all = length - a.queries + 1 + row0 / group;

        float o[NT][kTiles][4], m0[NT], m1[NT], l0[NT], l1[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            m0[nt] = m1[nt] = __uint_as_float(0xff800000u);
            l0[nt] = l1[nt] = 0.f;
#pragma unroll
            for (int t = 0; t < kTiles; ++t)
                o[nt][t][0] = o[nt][t][1] = o[nt][t][2] = o[nt][t][3] = 0.f;
        }
        int top = -121;  // exponent of the largest scale of V so far

        // this warp's blocks: blk + warp, + 8, ..
        const int mine = (count - warp + kWarps - 1) / kWarps;
        // a lane knows the block of the cache of one turn of 32; -1: no page
        auto numbers = [&](int turn) {
            const int i = turn * 32 + lane;
            if (i >= mine)
                return -1;
            const int p = blk + warp + i * kWarps;
            const int page = page_of(a.c, b, p * kBlock);
            if (page < 0) {
                *(volatile int*)a.status = ERR_PAGE;
                return -1;
            }
            return (page * a.c.kv_heads + h) * page_blocks + p % page_blocks;
        };
        int now = numbers(0), next = numbers(1);
        uint32_t no_page = 0;  // of the stages on their way, newest in bit 0
        auto ask = [&](int i) {
            if (i < mine) {
                if (i && (i & 31) == 0) {
                    now = next;
                    next = numbers((i >> 5) + 1);
                }
                const int number = __shfl_sync(0xffffffffu, now, i & 31);
                no_page = no_page << 1 | (number < 0);
                if (number >= 0) {
                    const uint32_t stage = ring + (i % Ring<D>::kStages) * Ring<D>::kStage;
                    const long long off = (long long)number * kBlock * d + lane * 16;
#pragma unroll
                    for (int j = 0; j < D / 32; ++j)
                        if (lane + 32 * j < d) {
                            copy16(stage + to_k[j], a.c.k + off + 512 * j);
                            copy16(stage + to_v[j], a.c.v + off + 512 * j);
                        }
                    if (lane < 2)
                        copy4(stage + 2 * kBlock * D + lane * 4, (lane ? a.c.v_scales : a.c.k_scales) + number);
                }
            }
            copies_end();
        };
#pragma unroll
        for (int i = 0; i < Ring<D>::kStages - 1; ++i)
            ask(i);

#pragma unroll 1
        for (int i = 0; i < mine; ++i) {
            ask(i + Ring<D>::kStages - 1);
            copies_wait<Ring<D>::kStages - 1>();
            __syncwarp();
            const uint32_t stage = ring + (i % Ring<D>::kStages) * Ring<D>::kStage;
            // (stages asked for behind this one: those that there are)
            const bool nothing = no_page >> (min(mine - 1, i + Ring<D>::kStages - 1) - i) & 1;
            float2 scales = lds_f2(stage + 2 * kBlock * D);
            if (nothing)
                scales = make_float2(0.f, 0.f);
            float s[NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
                s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
#pragma unroll
            for (int k = 0; k < kChunks; ++k) {
                const int swizzle = D == 128 ? (g & 1) << 2 : 0;  // (rows g and g + 8 alike)
                const uint4 w0 = lds128(stage + g * D + (((4 * k + c) ^ swizzle) << 4));
                const uint4 w1 = lds128(stage + (g + 8) * D + (((4 * k + c) ^ swizzle) << 4));
                const uint32_t u0[4] = {w0.x, w0.y, w0.z, w0.w}, u1[4] = {w1.x, w1.y, w1.z, w1.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t x0 = u0[j] ^ 0x80808080u, x1 = u1[j] ^ 0x80808080u;
                    const uint32_t frag[4] = {two_f16<0x4140>(x0), two_f16<0x4140>(x1), two_f16<0x4342>(x0),
                                              two_f16<0x4342>(x1)};
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
                        mma_f16(s[nt], frag, qf[nt][k][2 * j], qf[nt][k][2 * j + 1]);
                }
            }
            // scores of positions g and g + 8, rows 2 c and 2 c + 1
            const int p0 = (blk + warp + i * kWarps) * kBlock;
            bool raise = false;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const float k0 = __fmul_rn(scales.x, f0[nt]), k1 = __fmul_rn(scales.x, f1[nt]);
                s[nt][0] = __fmul_rn(s[nt][0], k0), s[nt][1] = __fmul_rn(s[nt][1], k1);
                s[nt][2] = __fmul_rn(s[nt][2], k0), s[nt][3] = __fmul_rn(s[nt][3], k1);
                if (p0 + kBlock > seen_by_all || nothing) {
                    const float hidden = __uint_as_float(0xff800000u);
                    const int u0 = nothing ? INT32_MIN : lim0[nt], u1 = nothing ? INT32_MIN : lim1[nt];
                    s[nt][0] = p0 + g < u0 ? s[nt][0] : hidden, s[nt][1] = p0 + g < u1 ? s[nt][1] : hidden;
                    s[nt][2] = p0 + g + 8 < u0 ? s[nt][2] : hidden, s[nt][3] = p0 + g + 8 < u1 ? s[nt][3] : hidden;
                }
                raise |= fmaxf(s[nt][0], s[nt][2]) > m0[nt] + kAhead || fmaxf(s[nt][1], s[nt][3]) > m1[nt] + kAhead;
            }
            if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float n0 = fmaxf(s[nt][0], s[nt][2]), n1 = fmaxf(s[nt][1], s[nt][3]);
#pragma unroll
                    for (int x = 4; x < 32; x *= 2) {
                        n0 = fmaxf(n0, __shfl_xor_sync(0xffffffffu, n0, x));
                        n1 = fmaxf(n1, __shfl_xor_sync(0xffffffffu, n1, x));
                    }
                    n0 = fmaxf(n0, m0[nt]), n1 = fmaxf(n1, m1[nt]);
                    // (nothing seen so far: there is nothing to scale)
                    const float r0 = n0 == m0[nt] ? 1.f : exp2_fast(m0[nt] - n0);
                    const float r1 = n1 == m1[nt] ? 1.f : exp2_fast(m1[nt] - n1);
                    m0[nt] = n0, m1[nt] = n1;
                    l0[nt] = __fmul_rn(l0[nt], r0), l1[nt] = __fmul_rn(l1[nt], r1);
#pragma unroll
                    for (int t = 0; t < kTiles; ++t) {
                        o[nt][t][0] *= r0, o[nt][t][1] *= r1;
                        o[nt][t][2] *= r0, o[nt][t][3] *= r1;
                    }
                }
            }
            // (a block without a scale makes its sums NaN whatever they count)
            const uint32_t size = magnitude(scales.y);
            const int ev = size >= 0x7f800000u ? top : max(-120, (int)(size >> 23) - 127);
            if (ev > top) {
                // (first block: the sums are zero)
                const float r = top == -121 ? 1.f : power_of_two(max(-126, top - ev));
                top = ev;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int t = 0; t < kTiles; ++t)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            o[nt][t][e] *= r;
            }
            const float lift = __fmul_rn(scales.y, power_of_two(kLift - top));
            uint32_t pb[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const float none = __uint_as_float(0xff800000u);
                const float z0 = m0[nt] == none ? 0.f : m0[nt], z1 = m1[nt] == none ? 0.f : m1[nt];
                float p[4] = {exp2_fast(s[nt][0] - z0), exp2_fast(s[nt][1] - z1), exp2_fast(s[nt][2] - z0),
                              exp2_fast(s[nt][3] - z1)};
                l0[nt] += p[0] + p[2], l1[nt] += p[1] + p[3];
                // (what is not seen stays 0 whatever the block's scale)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    p[e] = p[e] == 0.f ? 0.f : __fmul_rn(p[e], lift);
                pb[nt][0] = movmatrix_trans(pack_f16(p[0], p[1]));
                pb[nt][1] = movmatrix_trans(pack_f16(p[2], p[3]));
            }
#pragma unroll
            for (int t = 0; t < kTiles; t += 2) {
                // lanes 0-7, 8-15: positions 0-7, 8-15 of unit t; 16-23, 24-31: of unit t + 1
                const int r = lane & 15, u = t + (lane >> 4);
                uint32_t v[4];
                ldmatrix_x4_trans(stage + kBlock * D + r * D + ((u ^ (D == 128 ? r & 7 : (r >> 1) & 3)) << 4), v);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    v[e] ^= 0x80808080u;
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const uint32_t frag[4] = {two_f16<0x4240>(v[2 * x]), two_f16<0x4341>(v[2 * x]),
                                              two_f16<0x4240>(v[2 * x + 1]), two_f16<0x4341>(v[2 * x + 1])};
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
                        mma_f16(o[nt][t + x], frag, pb[nt][0], pb[nt][1]);
                }
            }
            __syncwarp();
        }
        copies_wait<0>();

        // ---- the warps' sums become one ----
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int x = 4; x < 32; x *= 2) {
                l0[nt] += __shfl_xor_sync(0xffffffffu, l0[nt], x);
                l1[nt] += __shfl_xor_sync(0xffffffffu, l1[nt], x);
            }
            if (g == 0) {
                s_stats[warp][nt * 8 + 2 * c] = make_float2(m0[nt], l0[nt]);
                s_stats[warp][nt * 8 + 2 * c + 1] = make_float2(m1[nt], l1[nt]);
            }
        }
        __syncthreads();  // (nobody reads the rings any more)
        const int active = min(kWarps, count);
        float* sums = (float*)smem;  // [warp][row][kPitch]
        if (warp < active) {
            const float up = power_of_two(top - kLift < -126 ? -126 : top - kLift);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int t = 0; t < kTiles; ++t) {
                    float* p = sums + (warp * kRows + nt * 8 + 2 * c) * kPitch<D> + 16 * t + 2 * g;
                    *(float2*)p = make_float2(o[nt][t][0] * up, o[nt][t][2] * up);
                    *(float2*)(p + kPitch<D>) = make_float2(o[nt][t][1] * up, o[nt][t][3] * up);
                }
        }
        __syncthreads();
        const bool whole = blk == 0 && count == all;
        const Parts parts = parts_of(a.workspace, gridDim.x, kRows, D);
        const long long part = ((long long)blockIdx.x * 2 + !first) * kRows;
        for (int i = tid; i < rows * d; i += kThreads) {
            const int r = i / d, e = i - r * d;
            float m = __uint_as_float(0xff800000u);
            for (int w = 0; w < active; ++w)
                m = fmaxf(m, s_stats[w][r].x);
            const float z = m == __uint_as_float(0xff800000u) ? 0.f : m;
            float sum = 0.f, total = 0.f;
            for (int w = 0; w < active; ++w) {
                const float2 st = s_stats[w][r];
                const float f = exp2_fast(st.x - z);
                total += st.y * f;
                sum += sums[(w * kRows + r) * kPitch<D> + e] * f;
            }
            if (whole) {
                ((T*)a.out.p)[row_at(a, a.out, group, b, h, row0 + r) + e] =
                        from_float<T>(total == 0.f ? 0.f : __fdiv_rn(sum, total));
            } else {
                parts.sums[(part + r) * D + e] = sum;
                if (e == 0)
                    parts.stats[part + r] = make_float2(m, total);
            }
        }
        __syncthreads();
        first = false;
        left -= count;
        blk = 0;
        if (++at == lines) {
            at = 0;
            ++b;
        }
    }
}

// A row of a head whose blocks were cut: the parts in their order
template <class T, int D>
__global__ void __launch_bounds__(D) join_kernel(const CacheArgs a, const Shape shape, int ctas, int tile_rows) {
    __shared__ long long s_before, s_total;
    const int lines = a.c.kv_heads * shape.tiles;
    const int b = blockIdx.x / lines, at = blockIdx.x - b * lines;
    const int h = at / shape.tiles, tile = at - h * shape.tiles;
    const int r = blockIdx.y, row = tile * tile_rows + r, e = threadIdx.x;
    pdl_start();
    if (threadIdx.x < 32) {
        long long total = 0, before = 0;
        for (int b0 = 0; b0 < a.c.batch; b0 += 32) {
            const int i = b0 + (int)threadIdx.x;
            const int n = i < a.c.batch ? blocks_of(a, shape.capacity, i) : 0;
            total += __reduce_add_sync(0xffffffffu, n);
            before += __reduce_add_sync(0xffffffffu, i < b ? n : 0);
        }
        if (threadIdx.x == 0)
            s_before = before * lines, s_total = total * lines;
    }
    __syncthreads();
    const int blocks = blocks_of(a, shape.capacity, b);
    if (blocks == 0 || row >= shape.rows || e >= a.c.d)
        return;
    const long long quota = quota_of(s_total, ctas);
    const long long from = s_before + (long long)at * blocks, to = from + blocks - 1;
    const int c0 = (int)(from / quota), c1 = (int)(to / quota);
    if (c0 == c1)
        return;
    const Parts parts = parts_of(a.workspace, ctas, tile_rows, D);
    const long long first = ((long long)c0 * 2 + (c0 * quota < from)) * tile_rows + r;
    auto part = [&](int c) { return c == c0 ? first : (long long)c * 2 * tile_rows + r; };
    float m = __uint_as_float(0xff800000u);
#pragma unroll 8
    for (int c = c0; c <= c1; ++c)
        m = fmaxf(m, parts.stats[part(c)].x);
    const float z = m == __uint_as_float(0xff800000u) ? 0.f : m;
    float sum = 0.f, total = 0.f;
#pragma unroll 8
    for (int c = c0; c <= c1; ++c) {
        const float2 st = parts.stats[part(c)];
        const float f = exp2_fast(st.x - z);
        total += st.y * f;
        sum += parts.sums[part(c) * D + e] * f;
    }
    const int group = a.heads / a.c.kv_heads;
    ((T*)a.out.p)[row_at(a, a.out, group, b, h, row) + e] = from_float<T>(total == 0.f ? 0.f : __fdiv_rn(sum, total));
}

// How a call is launched: by its sizes alone, so that a captured one serves any lengths
struct Plan {
    int d, nt, rows, tiles, ctas;
    long long capacity, most;  // positions of a table, blocks in all that a call may have
    size_t bytes;
};
Plan plan_of(const mb200_kv_cache& c, int heads, int queries) {
    Plan p{};
    p.d = c.d <= 64 ? 64 : 128;
    p.rows = heads / c.kv_heads * queries;
    p.nt = p.rows <= 8 ? 1 : 2;
    p.tiles = (p.rows + 8 * p.nt - 1) / (8 * p.nt);
    p.capacity = (long long)c.table_pages * c.page_tokens;
    if (p.capacity > 0x7fffffff - kBlock)
        p.capacity = 0x7fffffff - kBlock;
    p.most = (p.capacity + kBlock - 1) / kBlock * c.batch * c.kv_heads * p.tiles;
    const long long useful = (p.most + kLeast - 1) / kLeast, resident = umma::sm_count() * (p.nt == 1 ? 2 : 1);
    p.ctas = (int)(useful < resident ? useful : resident);
    if (p.ctas < 1)
        p.ctas = 1;
    p.bytes = p.ctas == 1 ? 0 : align_up((size_t)p.ctas * 2 * 8 * p.nt * (p.d + 2) * sizeof(float), 256);
    return p;
}

template <class T, int D, int NT, bool VEC>
int launch(const CacheArgs& a, const Plan& p, cudaStream_t st) {
    constexpr int kSums = kWarps * 8 * NT * kPitch<D> * 4;
    constexpr int kSmem = Ring<D>::kBytes > kSums ? Ring<D>::kBytes : kSums;
    const Shape shape{p.rows, p.tiles, (int)p.capacity};
    static umma::KernelReady ready;
    if (!ready.smem(cache_kernel<T, D, NT, VEC>, kSmem))
        return refused("attention_cache_s8", cudaGetLastError());
    const Writes anything{nullptr, SIZE_MAX};
    cudaError_t e = launch_pdl(anything, cache_kernel<T, D, NT, VEC>, dim3((unsigned)p.ctas), dim3(kThreads), kSmem, st, a,
                               shape);
    if (e == cudaSuccess && p.ctas > 1)
        e = launch_pdl(anything, join_kernel<T, D>,
                       dim3((unsigned)(a.c.batch * a.c.kv_heads * p.tiles), (unsigned)(p.rows < 8 * NT ? p.rows : 8 * NT)),
                       dim3(D), 0, st, a, shape, p.ctas, 8 * NT);
    return e != cudaSuccess ? refused("attention_cache_s8", e) : check_launch("attention_cache_s8");
}
template <class T, int D>
int launch_rows(const CacheArgs& a, const Plan& p, bool vec, cudaStream_t st) {
    if (p.nt == 1)
        return vec ? launch<T, D, 1, true>(a, p, st) : launch<T, D, 1, false>(a, p, st);
    return vec ? launch<T, D, 2, true>(a, p, st) : launch<T, D, 2, false>(a, p, st);
}

}  // namespace

size_t attention_cache_workspace(const mb200_kv_cache& c, int heads, int queries) {
    return plan_of(c, heads, queries).bytes;
}

int launch_attention_cache(const CacheArgs& a, int dtype, cudaStream_t st) {
    const Plan p = plan_of(a.c, a.heads, a.queries);
    const bool vec = ((uintptr_t)a.q.p & 15) == 0 && a.q.token_stride % 8 == 0 && a.q.head_stride % 8 == 0;
    if (dtype == MB200_DTYPE_F16)
        return p.d == 64 ? launch_rows<__half, 64>(a, p, vec, st) : launch_rows<__half, 128>(a, p, vec, st);
    return p.d == 64 ? launch_rows<__nv_bfloat16, 64>(a, p, vec, st) : launch_rows<__nv_bfloat16, 128>(a, p, vec, st);
}

}  // namespace attn
}  // namespace mb200
