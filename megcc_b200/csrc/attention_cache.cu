// Attention of one or a few queries per sequence over the paged int8 cache.
//
// For a key head, the rows are its group's query heads times the queries of a sequence. With the scores as powers of two,
//     t_j = (scale log2(e)) s_k q . k_j,   o = sum 2^(t_j - m) s_v v_j / sum 2^(t_j - m),
// over the positions j that a row sees, in one pass: m is a running maximum that is raised only where a score
// passes it by more than 8 (a vote per block of 16 positions, no reduction), so 2^(t - m) stays below 2^8.
//
// Bound by memory: 2 d bytes per position and key head are all there is to read, and what each byte costs in
// instructions decides whether that is reached. Products are taken transposed, S^T = K Q^T and O^T = V^T P^T, so that positions
// and dimensions fill the 16 rows of an mma.sync and 8 query rows its 8 columns: half the instructions and accumulators of
// the other way round for groups of up to 8.
//   S: keys are multiplied as they lie, int8 by int8 (m16n8k32, as fast as fp16's k16): queries become whole numbers of 23 bits
// of their row's power of two, three planes of int8, whose sums are exact. The order of dimensions within a sum is free:
// a lane takes 16 neighbouring ones with one load.
//   O: values become fp16, which holds them exactly: a byte permutation makes 1024 + (v + 128) of them, and a subtraction v.
// V^T comes by ldmatrix.trans over pairs of bytes, whose two dimensions the same permutation separates. P^T is turned by
// movmatrix. P is rounded to fp16 (2^-12, where results have 2^-9), for fp16 results held as two such numbers, after it
// took its block's scale of V relative to the largest so far, which keeps it in range.
//
// All blocks of all sequences and key heads are one line of rounds (a step of 32 positions for each of a CTA's warps),
// cut evenly over the CTAs whatever the lengths, which only the device knows. Each warp has a ring of asynchronous copies of
// its own. Where a head's rounds are cut, the parts go to the workspace and a second kernel joins them in order.
#include <type_traits>

#include "kv_cache.cuh"
#include "umma_ptx.cuh"

namespace mb200 {
namespace attn {
namespace {

constexpr int kWarps = 4, kThreads = 32 * kWarps;
constexpr int kStep = 2;                   // blocks of a warp's step
constexpr int kRound = kWarps * kStep;     // blocks of a CTA's round
constexpr float kAhead = 8.f;              // how far a score may pass the running maximum
constexpr int kLift = 6;                   // probabilities are held 2^6 times: 2^8 * 2 * 2^6 < 65504
constexpr int kCtasPerSm = 2;

template <int D>
struct Ring {
    static constexpr int kHalf = kStep * kBlock * D;   // keys, then values
    static constexpr int kStage = 2 * kHalf + 128;     // ... and their four scales (stages begin on whole lines)
    static constexpr int kStages = D == 128 ? 3 : 5;
    static constexpr int kBytes = kWarps * kStages * kStage;
};
// floats from row to row of the warps' sums: a warp's stores reach all banks
template <int D>
constexpr int kPitch = D + 4;

struct Shape {
    int rows, tiles, capacity;  // rows of a key head, tiles of them, positions a table has room for
};
// How the line is cut, found alike by both kernels
__device__ __forceinline__ int blocks_of(const CacheArgs& a, int capacity, int b) {
    const int n = a.lengths[b];
    return n <= 0 ? 0 : (min(n, capacity) + kBlock - 1) / kBlock;
}
__device__ __forceinline__ int rounds_of(const CacheArgs& a, int capacity, int b) {
    return b < a.c.batch ? (blocks_of(a, capacity, b) + kRound - 1) / kRound : 0;
}
__device__ __forceinline__ long long quota_of(long long total, int ctas) {
    return (total + ctas - 1) / ctas;
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
__device__ __forceinline__ void mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
            "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%0, %1, %2, %3};"
            : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
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

// Queries as whole numbers of 23 bits: hi 2^16 + mid 2^8 + lo times 2^(e - 21), e the exponent of the row's largest
constexpr int kPlanes = 3;
__device__ __forceinline__ void planes_of(const float (&x)[4], float up, uint32_t (&w)[kPlanes]) {
    uint32_t b[4][kPlanes];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int q = __float2int_rn(__fmul_rn(x[i], up));
        const int q1 = (q - (int)(int8_t)q) >> 8;
        b[i][2] = (uint32_t)q, b[i][1] = (uint32_t)q1, b[i][0] = (uint32_t)((q1 - (int)(int8_t)q1) >> 8);
    }
#pragma unroll
    for (int p = 0; p < kPlanes; ++p)
        w[p] = __byte_perm(__byte_perm(b[0][p], b[1][p], 0x0040), __byte_perm(b[2][p], b[3][p], 0x0040), 0x5410);
}

// FULL: d == D
template <class T, int D, int NT, bool VEC, bool FULL>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) cache_kernel(const CacheArgs a, const Shape shape) {
    using R = Ring<D>;
    constexpr int kRows = 8 * NT, kChunks = D / 64, kTiles = D / 16;
    constexpr bool kFine = std::is_same<T, __half>::value;  // P as two fp16 numbers
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ long long s_from, s_to, s_rest;
    __shared__ int s_b;
    __shared__ float2 s_stats[kWarps][kRows];
    const int tid = threadIdx.x, lane = tid & 31, warp = umma::uniform_warp_index();
    const int g = lane >> 2, c = lane & 3;
    const int d = FULL ? D : a.c.d, group = a.heads / a.c.kv_heads;
    const int lines = a.c.kv_heads * shape.tiles;  // of a sequence: key heads times tiles of rows
    const float none = __uint_as_float(0xff800000u);
    pdl_start();

    // this CTA's part of the line
    if (warp == 0) {
        long long total = 0;
        int mine = 0;
        for (int b0 = 0; b0 < a.c.batch; b0 += 32) {
            mine = rounds_of(a, shape.capacity, b0 + lane);
            total += __reduce_add_sync(0xffffffffu, mine);
        }
        total *= lines;
        const long long quota = quota_of(total, gridDim.x);
        const long long from = quota * blockIdx.x, to = from + quota < total ? from + quota : total;
        long long before = 0;
        int at = 0;
        if (from < to) {
            for (int b0 = 0; b0 < a.c.batch; b0 += 32) {
                const int n = a.c.batch <= 32 ? mine : rounds_of(a, shape.capacity, b0 + lane);
                int sum = n;
#pragma unroll
                for (int s = 1; s < 32; s *= 2) {
                    const int v = __shfl_up_sync(0xffffffffu, sum, s);
                    sum += lane >= s ? v : 0;
                }
                const uint32_t beyond = __ballot_sync(0xffffffffu, (before + sum) * lines > from);
                if (beyond) {
                    const int i = __ffs(beyond) - 1;
                    before += __shfl_sync(0xffffffffu, sum - n, i);
                    at = b0 + i;
                    break;
                }
                before += __shfl_sync(0xffffffffu, sum, 31);
            }
        }
        if (lane == 0)
            s_from = from, s_to = to, s_b = at, s_rest = from - before * lines;
    }
    __syncthreads();
    long long left = s_to - s_from;
    int b = s_b, at = 0, blk = 0;
    if (left > 0) {
        const int n = rounds_of(a, shape.capacity, b);
        at = (int)(s_rest / n);
        blk = (int)(s_rest - (long long)at * n) * kRound;
    }
    bool first = true;
    const uint32_t ring = smem_at(smem) + warp * (R::kStages * R::kStage);
    // where this lane's 16-byte units of a block go: row r's unit u beside others' so that loads meet all banks
    constexpr int kUnits = D / 32;  // of a lane
    const int units = d / 16;
    uint32_t to_k[kUnits], to_v[kUnits];
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
        const int x = lane + 32 * i, r = x / units, u = x - r * units;
        to_k[i] = (uint32_t)(r * D + (u ^ (D == 128 ? (r & 1) << 2 : 0)) * 16);
        to_v[i] = (uint32_t)(R::kHalf + r * D + (u ^ (D == 128 ? r & 7 : (r >> 1) & 3)) * 16);
    }
    const uint32_t at_k = (uint32_t)(g * D + ((c ^ (D == 128 ? (g & 1) << 2 : 0)) << 4));  // (rows g and g + 8 alike)
    const int vr = lane & 15;
    // lanes 0-7, 8-15: positions 0-7, 8-15 of an even unit; 16-23, 24-31: of the next one
    const uint32_t at_v = (uint32_t)(R::kHalf + vr * D), swizzle_v = D == 128 ? vr & 7 : (vr >> 1) & 3;
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
        const int rounds = (all - blk + kRound - 1) / kRound;
        const int take = (int)(left < rounds ? left : rounds);
        const int count = min(all - blk, take * kRound);
        const int row0 = tile * kRows, rows = min(kRows, shape.rows - row0);

        // this warp's steps: blocks blk + 2 warp, + 8, .. and the one behind each
        const int mine = (count - warp * kStep + kRound - 1) / kRound;
        const int first_blk = blk + warp * kStep;
        // a lane knows a block of one turn of 16 steps; -1: no page, or behind the last
        auto numbers = [&](int turn) {
            const int p = first_blk + (turn * 16 + (lane >> 1)) * kRound + (lane & 1);
            if (p >= blk + count)
                return -1;
            const int page = page_of(a.c, b, p * kBlock);
            if (page < 0) {
                *(volatile int*)a.status = ERR_PAGE;
                return -1;
            }
            return (page * a.c.kv_heads + h) * page_blocks + p % page_blocks;
        };
        int now = numbers(0), next = mine > 16 ? numbers(1) : -1;
        uint32_t there = 0;  // blocks of the stages on their way, two bits each, the newest lowest
        uint32_t stage_in = ring;
        auto ask = [&](int i) {
            if (i < mine) {
                if (i && (i & 15) == 0) {
                    now = next;
                    next = numbers((i >> 4) + 1);
                }
                const int n0 = __shfl_sync(0xffffffffu, now, 2 * (i & 15)), n1 = __shfl_sync(0xffffffffu, now, 2 * (i & 15) + 1);
                there = there << 2 | (n0 >= 0 ? 1u : 0u) | (n1 >= 0 ? 2u : 0u);
                auto block = [&](int number, int half) {
                    const long long off = (long long)number * (kBlock * d) + lane * 16;
                    const int8_t *k = a.c.k + off, *v = a.c.v + off;
                    const uint32_t to = stage_in + half * (kBlock * D);
#pragma unroll
                    for (int j = 0; j < kUnits; ++j)
                        if (FULL || lane + 32 * j < d) {
                            copy16(to + to_k[j], k + 512 * j);
                            copy16(to + to_v[j], v + 512 * j);
                        }
                };
                if (n0 >= 0)
                    block(n0, 0);
                if (n1 >= 0)
                    block(n1, 1);
                const int n = lane & 1 ? n1 : n0;
                if (lane < 4 && n >= 0)
                    copy4(stage_in + 2 * R::kHalf + lane * 4, (lane & 2 ? a.c.v_scales : a.c.k_scales) + n);
                stage_in = stage_in + R::kStage == ring + R::kStages * R::kStage ? ring : stage_in + R::kStage;
            }
            copies_end();
        };
#pragma unroll
        for (int i = 0; i < R::kStages - 1; ++i)
            ask(i);

        // queries: lane (g, c) holds of row g the dimensions 64 i + 16 c .. + 15, and its factor
        uint32_t qf[NT][kPlanes][kChunks][4];
        float f0[NT], f1[NT];
        int lim0[NT], lim1[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int r = nt * 8 + g;
            float x[kChunks][4][4];
            uint32_t most = 0;
#pragma unroll
            for (int i = 0; i < kChunks; ++i) {
                const int dim = 64 * i + 16 * c;
                uint4 lo = make_uint4(0, 0, 0, 0), hi = lo;
                if (r < rows && (FULL || dim < d)) {
                    const long long p = row_at(a, a.q, group, b, h, row0 + r) + dim;
                    lo = load8<VEC>(a.q.p, p);
                    hi = load8<VEC>(a.q.p, p + 8);
                }
                Vec<T>::unpack(lo, &x[i][0][0]);
                Vec<T>::unpack(hi, &x[i][2][0]);
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    most = max(most, magnitude(x[i][e / 4][e % 4]));
            }
            most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
            most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
            const int e = exponent_of(most);
            const bool finite = most < 0x7f800000u;
            const int shift = min(126, 21 - e);
            const float up = finite ? power_of_two(shift) : 0.f;
            // (a row with a NaN or an infinity has no whole numbers: all of it is NaN)
            const float factor = finite ? __fmul_rn(power_of_two(-shift), a.scale_log2) : __uint_as_float(0x7fffffffu);
#pragma unroll
            for (int i = 0; i < kChunks; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    uint32_t w[kPlanes];
                    planes_of(x[i][j], up, w);
#pragma unroll
                    for (int p = 0; p < kPlanes; ++p)
                        qf[nt][p][i][j] = w[p];
                }
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
            m0[nt] = m1[nt] = none;
            l0[nt] = l1[nt] = 0.f;
#pragma unroll
            for (int t = 0; t < kTiles; ++t)
                o[nt][t][0] = o[nt][t][1] = o[nt][t][2] = o[nt][t][3] = 0.f;
        }
        int top = -121;  // exponent of the largest scale of V so far
        uint32_t stage = ring;

#pragma unroll 1
        for (int i = 0; i < mine; ++i) {
            ask(i + R::kStages - 1);
            copies_wait<R::kStages - 1>();
            __syncwarp();
            // (stages asked for behind this one: those that there are)
            const uint32_t have = there >> 2 * (min(mine - 1, i + R::kStages - 1) - i) & 3;
            const uint4 sc = lds128(stage + 2 * R::kHalf);
            const float ks[2] = {have & 1 ? __uint_as_float(sc.x) : 0.f, have & 2 ? __uint_as_float(sc.y) : 0.f};
            const float vs[2] = {have & 1 ? __uint_as_float(sc.z) : 0.f, have & 2 ? __uint_as_float(sc.w) : 0.f};
            // scores of positions g and g + 8 of both blocks, rows 2 c and 2 c + 1
            float s[kStep][NT][4];
#pragma unroll
            for (int x = 0; x < kStep; ++x) {
                int acc[NT][kPlanes][4];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int p = 0; p < kPlanes; ++p)
                        acc[nt][p][0] = acc[nt][p][1] = acc[nt][p][2] = acc[nt][p][3] = 0;
#pragma unroll
                for (int k = 0; k < kChunks; ++k) {
                    // (unit 4 k + c: with the swizzle's 4, k and the other half change places)
                    const uint32_t key = (stage + x * (kBlock * D) + at_k) ^ (k << 6);
                    const uint4 w0 = lds128(key), w1 = lds128(key + 8 * D);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int p = 0; p < kPlanes; ++p) {
                            mma_s8(acc[nt][p], w0.x, w1.x, w0.y, w1.y, qf[nt][p][k][0], qf[nt][p][k][1]);
                            mma_s8(acc[nt][p], w0.z, w1.z, w0.w, w1.w, qf[nt][p][k][2], qf[nt][p][k][3]);
                        }
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    const float k0 = __fmul_rn(ks[x], f0[nt]), k1 = __fmul_rn(ks[x], f1[nt]);
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        s[x][nt][e] = __fmul_rn(__fmaf_rn((float)acc[nt][0][e], 65536.f, (float)(acc[nt][1][e] * 256 + acc[nt][2][e])),
                                                e & 1 ? k1 : k0);
                }
            }
            const int p0 = (first_blk + i * kRound) * kBlock;
            if (p0 + kStep * kBlock > seen_by_all || have != 3) {
#pragma unroll
                for (int x = 0; x < kStep; ++x)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int p = p0 + x * kBlock + g + (e & 2 ? 8 : 0);
                            const bool seen = (have >> x & 1) && p < (e & 1 ? lim1[nt] : lim0[nt]);
                            s[x][nt][e] = seen ? s[x][nt][e] : none;
                        }
            }
            bool raise = false;
            float n0[NT], n1[NT];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                n0[nt] = fmaxf(fmaxf(s[0][nt][0], s[0][nt][2]), fmaxf(s[1][nt][0], s[1][nt][2]));
                n1[nt] = fmaxf(fmaxf(s[0][nt][1], s[0][nt][3]), fmaxf(s[1][nt][1], s[1][nt][3]));
                raise |= n0[nt] > m0[nt] + kAhead || n1[nt] > m1[nt] + kAhead;
            }
            if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                    for (int x = 4; x < 32; x *= 2) {
                        n0[nt] = fmaxf(n0[nt], __shfl_xor_sync(0xffffffffu, n0[nt], x));
                        n1[nt] = fmaxf(n1[nt], __shfl_xor_sync(0xffffffffu, n1[nt], x));
                    }
                    const float t0 = fmaxf(n0[nt], m0[nt]), t1 = fmaxf(n1[nt], m1[nt]);
                    // (nothing seen so far: there is nothing to scale)
                    const float r0 = t0 == m0[nt] ? 1.f : exp2_fast(m0[nt] - t0);
                    const float r1 = t1 == m1[nt] ? 1.f : exp2_fast(m1[nt] - t1);
                    m0[nt] = t0, m1[nt] = t1;
                    l0[nt] = __fmul_rn(l0[nt], r0), l1[nt] = __fmul_rn(l1[nt], r1);
#pragma unroll
                    for (int t = 0; t < kTiles; ++t) {
                        o[nt][t][0] *= r0, o[nt][t][1] *= r1;
                        o[nt][t][2] *= r0, o[nt][t][3] *= r1;
                    }
                }
            }
            // (a block without a scale makes its sums NaN whatever they count)
            int ev = top;
#pragma unroll
            for (int x = 0; x < kStep; ++x) {
                const uint32_t size = magnitude(vs[x]);
                ev = max(ev, size >= 0x7f800000u ? top : max(-120, (int)(size >> 23) - 127));
            }
            if (ev > top) {
                // (first step: the sums are zero)
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
            const float unit = power_of_two(kLift - top);
            uint32_t hi[kStep][NT][2], lo[kStep][NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const float z0 = m0[nt] == none ? 0.f : m0[nt], z1 = m1[nt] == none ? 0.f : m1[nt];
#pragma unroll
                for (int x = 0; x < kStep; ++x) {
                    const float lift = __fmul_rn(vs[x], unit);
                    float p[4] = {exp2_fast(s[x][nt][0] - z0), exp2_fast(s[x][nt][1] - z1), exp2_fast(s[x][nt][2] - z0),
                                  exp2_fast(s[x][nt][3] - z1)};
                    l0[nt] += p[0] + p[2], l1[nt] += p[1] + p[3];
                    // (what is not seen stays 0 whatever the block's scale)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        p[e] = p[e] == 0.f ? 0.f : __fmul_rn(p[e], lift);
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const uint32_t w = pack_f16(p[2 * e], p[2 * e + 1]);
                        hi[x][nt][e] = movmatrix_trans(w);
                        if constexpr (kFine) {
                            const float2 back = __half22float2(*reinterpret_cast<const __half2*>(&w));
                            lo[x][nt][e] = movmatrix_trans(pack_f16(p[2 * e] - back.x, p[2 * e + 1] - back.y));
                        }
                    }
                }
            }
#pragma unroll
            for (int t = 0; t < kTiles; t += 2) {
#pragma unroll
                for (int x = 0; x < kStep; ++x) {
                    uint32_t v[4];
                    ldmatrix_x4_trans(stage + x * (kBlock * D) + at_v + (((t + (lane >> 4)) ^ swizzle_v) << 4), v);
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        v[e] ^= 0x80808080u;
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        const uint32_t frag[4] = {two_f16<0x4240>(v[2 * y]), two_f16<0x4341>(v[2 * y]),
                                                  two_f16<0x4240>(v[2 * y + 1]), two_f16<0x4341>(v[2 * y + 1])};
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            if constexpr (kFine)
                                mma_f16(o[nt][t + y], frag, lo[x][nt][0], lo[x][nt][1]);
                            mma_f16(o[nt][t + y], frag, hi[x][nt][0], hi[x][nt][1]);
                        }
                    }
                }
            }
            __syncwarp();
            stage = stage + R::kStage == ring + R::kStages * R::kStage ? ring : stage + R::kStage;
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
        const int active = min(kWarps, (count + kStep - 1) / kStep);
        float* sums = (float*)smem;  // [warp][row][kPitch]
        if (warp < active) {
            const float up = power_of_two(max(-126, top - kLift));
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
            float m = none;
            for (int w = 0; w < active; ++w)
                m = fmaxf(m, s_stats[w][r].x);
            const float z = m == none ? 0.f : m;
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
        left -= take;
        blk = 0;
        if (++at == lines) {
            at = 0;
            ++b;
        }
    }
    // sequences without a position: nothing is seen
    for (b = blockIdx.x; b < a.c.batch; b += gridDim.x) {
        if (a.lengths[b] > shape.capacity && tid == 0)
            *(volatile int*)a.status = ERR_PAGE;
        if (a.lengths[b] <= 0)
            for (int i = tid; i < a.queries * a.heads * d; i += kThreads) {
                const int e = i % d, th = i / d;
                ((T*)a.out.p)[((long long)b * a.queries + th / a.heads) * a.out.token_stride +
                              (long long)(th % a.heads) * a.out.head_stride + e] = from_float<T>(0.f);
            }
    }
}

// Joins the parts of what was cut, in their order: for each item (a sequence's key head and tile of rows), or, where there are more
// of those than CTAs, for each CTA whose part of the line begins inside an item, the first of that item. With many parts to
// an item a CTA has one row and its groups of D threads share the parts; else each group has a row of its own.
constexpr int kJoinThreads = 512, kJoinParts = 512;
template <class T, int D>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(
        const CacheArgs a, const Shape shape, int ctas, int tile_rows, int by_item, int share) {
    constexpr int kGroups = kJoinThreads / D;
    __shared__ long long s_before, s_total;
    __shared__ int s_b;
    __shared__ float s_max[kJoinThreads / 32], s_factor[kJoinParts], s_sum[kGroups][D];
    const int lines = a.c.kv_heads * shape.tiles;
    const int tid = threadIdx.x, e = tid % D, mine = tid / D;
    const int cut = blockIdx.x + 1;
    const float none = __uint_as_float(0xff800000u);
    // (lengths are not the kernel's in front, and all others have ended: see pdl.h)
    if (tid < 32) {
        long long total = 0, before = 0;
        int b = -1;
        for (int b0 = 0; b0 < a.c.batch; b0 += 32)
            total += __reduce_add_sync(0xffffffffu, rounds_of(a, shape.capacity, b0 + tid));
        total *= lines;
        const long long position = cut * quota_of(total, ctas);
        if (by_item) {
            b = blockIdx.x / lines;
            for (int b0 = 0; b0 < b; b0 += 32)
                before += __reduce_add_sync(0xffffffffu, b0 + tid < b ? rounds_of(a, shape.capacity, b0 + tid) : 0);
        }
        for (int b0 = 0; b0 < a.c.batch && position < total && !by_item; b0 += 32) {
            const int n = rounds_of(a, shape.capacity, b0 + tid);
            int sum = n;
#pragma unroll
            for (int s = 1; s < 32; s *= 2) {
                const int v = __shfl_up_sync(0xffffffffu, sum, s);
                sum += tid >= s ? v : 0;
            }
            const uint32_t beyond = __ballot_sync(0xffffffffu, (before + sum) * lines > position);
            if (beyond) {
                const int i = __ffs(beyond) - 1;
                before += __shfl_sync(0xffffffffu, sum - n, i);
                b = b0 + i;
                break;
            }
            before += __shfl_sync(0xffffffffu, sum, 31);
        }
        if (tid == 0)
            s_before = before * lines, s_total = total, s_b = b;
    }
    __syncthreads();
    const int b = s_b;
    long long quota = 1, from = 0, to = 0;
    int at = 0;
    const int rounds = b < 0 ? 0 : rounds_of(a, shape.capacity, b);
    if (rounds > 0) {
        quota = quota_of(s_total, ctas);
        at = by_item ? (int)blockIdx.x - b * lines : (int)((cut * quota - s_before) / rounds);
        from = s_before + (long long)at * rounds, to = from + rounds - 1;
    }
    const int c0 = (int)(from / quota), c1 = (int)(to / quota);
    pdl_start();
    if (c0 == c1 || (!by_item && (from == cut * quota || c0 + 1 != cut)))
        return;
    const int h = at / shape.tiles, tile = at - h * shape.tiles;
    const int rows = min(tile_rows, shape.rows - tile * tile_rows);
    const int r = share ? (int)blockIdx.y : (int)blockIdx.y * kGroups + mine;
    const int groups = share ? kGroups : 1, group_at = share ? mine : 0;
    const Parts parts = parts_of(a.workspace, ctas, tile_rows, D);
    const long long first = ((long long)c0 * 2 + (c0 * quota < from)) * tile_rows;
    auto part = [&](int c) { return (c == c0 ? first : (long long)c * 2 * tile_rows) + r; };
    float sum = 0.f, total = 0.f, m = none;
    if (share) {
        if (r >= rows)
            return;
        for (int c = c0 + tid; c <= c1; c += kJoinThreads)
            m = fmaxf(m, parts.stats[part(c)].x);
#pragma unroll
        for (int x = 1; x < 32; x *= 2)
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
        if ((tid & 31) == 0)
            s_max[tid >> 5] = m;
        __syncthreads();
#pragma unroll
        for (int x = 0; x < kJoinThreads / 32; ++x)
            m = fmaxf(m, s_max[x]);
        const float z = m == none ? 0.f : m;
        for (int base = c0; base <= c1; base += kJoinParts) {
            const int n = min(kJoinParts, c1 + 1 - base);
            __syncthreads();
            float weight = 0.f;
            if (tid < n) {
                const float2 st = parts.stats[part(base + tid)];
                const float f = exp2_fast(st.x - z);
                s_factor[tid] = f;
                weight = st.y * f;
            }
#pragma unroll
            for (int x = 1; x < 32; x *= 2)
                weight += __shfl_xor_sync(0xffffffffu, weight, x);
            total += weight;
            __syncthreads();
#pragma unroll 8
            for (int i = group_at; i < n; i += groups)
                sum += parts.sums[part(base + i) * D + e] * s_factor[i];
        }
        s_sum[mine][e] = sum;
        if ((tid & 31) == 0)
            s_max[tid >> 5] = total;
        __syncthreads();
        if (mine)
            return;
        sum = total = 0.f;
#pragma unroll
        for (int x = 0; x < kGroups; ++x)
            sum += s_sum[x][e];
#pragma unroll
        for (int x = 0; x < kJoinThreads / 32; ++x)
            total += s_max[x];
    } else {
        if (r >= rows)
            return;
#pragma unroll 8
        for (int c = c0; c <= c1; ++c)
            m = fmaxf(m, parts.stats[part(c)].x);
        const float z = m == none ? 0.f : m;
#pragma unroll 8
        for (int c = c0; c <= c1; ++c) {
            const float2 st = parts.stats[part(c)];
            const float f = exp2_fast(st.x - z);
            total += st.y * f;
            sum += parts.sums[part(c) * D + e] * f;
        }
    }
    if (e < a.c.d)
        ((T*)a.out.p)[row_at(a, a.out, a.heads / a.c.kv_heads, b, h, tile * tile_rows + r) + e] =
                from_float<T>(total == 0.f ? 0.f : __fdiv_rn(sum, total));
}

// How a call is launched: by its sizes alone, so that a captured one serves any lengths
struct Plan {
    int d, nt, rows, tiles, ctas;
    long long capacity, most;  // positions of a table, rounds that a call may have
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
    p.most = (p.capacity + kRound * kBlock - 1) / (kRound * kBlock) * c.batch * c.kv_heads * p.tiles;
    const long long resident = umma::sm_count() * kCtasPerSm;
    p.ctas = (int)(p.most < resident ? p.most : resident);
    if (p.ctas < 1)
        p.ctas = 1;
    p.bytes = p.ctas == 1 ? 0 : align_up((size_t)p.ctas * 2 * 8 * p.nt * (p.d + 2) * sizeof(float), 256);
    return p;
}

template <class T, int D, int NT, bool VEC, bool FULL>
int launch(const CacheArgs& a, const Plan& p, cudaStream_t st) {
    constexpr int kSums = kWarps * 8 * NT * kPitch<D> * 4;
    constexpr int kSmem = Ring<D>::kBytes > kSums ? Ring<D>::kBytes : kSums;
    const auto kernel = cache_kernel<T, D, NT, VEC, FULL>;
    const Shape shape{p.rows, p.tiles, (int)p.capacity};
    static umma::KernelReady ready;
    if (!ready.smem(kernel, kSmem))
        return refused("attention_cache_s8", cudaGetLastError());
    const Writes anything{nullptr, SIZE_MAX};
    cudaError_t e = launch_pdl(anything, kernel, dim3((unsigned)p.ctas), dim3(kThreads), kSmem, st, a, shape);
    if (e == cudaSuccess && p.ctas > 1) {
        const int rows = p.rows < 8 * NT ? p.rows : 8 * NT, groups = kJoinThreads / D;
        const long long items = (long long)a.c.batch * a.c.kv_heads * p.tiles;
        const bool by_item = items < p.ctas, share = items * 8 <= p.ctas;
        e = launch_pdl(anything, join_kernel<T, D>,
                       dim3((unsigned)(by_item ? items : p.ctas - 1), (unsigned)(share ? rows : (rows + groups - 1) / groups)),
                       dim3(kJoinThreads), 0, st, a, shape, p.ctas, 8 * NT, (int)by_item, (int)share);
    }
    return e != cudaSuccess ? refused("attention_cache_s8", e) : check_launch("attention_cache_s8");
}
template <class T, int D>
int launch_rows(const CacheArgs& a, const Plan& p, bool vec, cudaStream_t st) {
    // (odd heads and queries at odd places by one variant: either costs a few per cent)
    if (p.nt == 1)
        return vec && a.c.d == D ? launch<T, D, 1, true, true>(a, p, st) : launch<T, D, 1, false, false>(a, p, st);
    return vec && a.c.d == D ? launch<T, D, 2, true, true>(a, p, st) : launch<T, D, 2, false, false>(a, p, st);
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
