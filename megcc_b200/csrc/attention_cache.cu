// Attention of one or a few queries per sequence over the paged int8 cache.
//
// For a key head, the rows are its group's query heads times the queries of a sequence. With the scores as powers of two,
//     t_j = (scale log2(e)) s_k q . k_j,   o = sum 2^(t_j - m) s_v v_j / sum 2^(t_j - m),
// over the positions j that a row sees, in one pass: m is a running maximum that is raised only where a score
// passes it by more than 8 (a vote per step of 32 positions, no reduction), so 2^(t - m) stays below 2^8.
//
// Bound by memory: 2 d bytes per position and key head are all there is to read, and what each byte costs in
// instructions decides whether that is reached. Products are taken transposed, S^T = K Q^T and O^T = V^T P^T, so that positions
// and dimensions fill the 16 rows of an mma.sync and 8 query rows its 8 columns: half the instructions and accumulators of
// the other way round for groups of up to 8.
//   S: keys are multiplied as they lie, int8 by int8 (m16n8k32, as fast as fp16's k16): queries become whole numbers of 22 bits
// of their row's power of two, three planes of int8, whose sums are exact. The order of dimensions within a sum is free:
// a lane takes 16 neighbouring ones with one load.
//   O: values become fp16, which holds them exactly: a byte permutation makes 1024 + (v + 128) of them, and a subtraction v.
// V^T comes by ldmatrix.trans over pairs of bytes, whose two dimensions the same permutation separates. P^T is turned by
// movmatrix. P takes its block's scale of V and is rounded to fp16 (2^-12, where results have 2^-9), for fp16 results held as
// two such numbers. What keeps it in range there is a power of two of each row's own, of the largest product of a probability
// and a scale that the row has met: blocks that a row does not see, or that weigh nothing, take no bits from the others
// whatever their scales.
//
// All blocks of all sequences and key heads are one line of rounds (a step of 32 positions for each of a CTA's warps),
// cut evenly over the CTAs whatever the lengths, which only the device knows. Each warp has a ring of asynchronous copies of
// its own. Where a head's rounds are cut, the parts go to the workspace and a second kernel joins them in order.
//
// One query over 131071 positions, 32 over 8 heads of 128 (269 MB): 55 us, of which the first kernel reads at 5.2 TB/s. 48
// sequences of up to 8192 positions, 32 over 4 heads, fp16 (212 MB): 52 us.
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
constexpr int kIdleRows = 1024;

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

// 1 / x of a power of two whose inverse is a normal number
__device__ __forceinline__ float inverse_power(float x) {
    return __uint_as_float((254u << 23) - __float_as_uint(x));
}
// The exponent of a block's scale of V, -120 at least. (One that is no number makes its sums NaN whatever they count.)
__device__ __forceinline__ float exponent_of_scale(float scale) {
    const uint32_t size = magnitude(scale);
    return size >= 0x7f800000u ? -120.f : (float)max(-120, (int)(size >> 23) - 127);
}
// A row whose scores have passed its maximum m, or whose scores with their scales' exponents have passed w: n and u are this
// lane's largest of either. Returns what the row's sums are multiplied by. k is at least -110, where 2^-126, the smallest
// scale, still leaves P 16 bits, and at most 127: w - m is no larger.
__device__ __forceinline__ float raised(float n, float u, float& m, float& l, float& w, float& up) {
#pragma unroll
    for (int x = 4; x < 32; x *= 2) {
        n = fmaxf(n, __shfl_xor_sync(0xffffffffu, n, x));
        u = fmaxf(u, __shfl_xor_sync(0xffffffffu, u, x));
    }
    const float t = fmaxf(n, m);
    w = fmaxf(u, w);
    if (t == __uint_as_float(0xff800000u))  // (nothing seen so far: there is nothing to scale)
        return 1.f;
    const int before = kLift + 127 - (int)(__float_as_uint(up) >> 23);
    const int k = max(-110, min(127, __float2int_ru(w - t)));
    const float down = t == m ? 1.f : exp2_fast(m - t);
    const float r = k == before ? down : exp2_fast((m - t) + (float)(before - k));
    l = __fmul_rn(l, down);
    m = t;
    up = power_of_two(kLift - k);
    return r;
}

// The workspace: averages [cta][first or last][row][D] of what was cut, then [..][row] maxima and totals, then for each CTA
// the item (a sequence's key head and tile of rows) inside which its part of the line begins
struct Cut {
    int b, at;              // b < 0: it begins with an item, or there is none
    long long from, quota;  // the item's place in the line; rounds of a CTA
    int rounds, unused;
};
struct Parts {
    float* sums;
    float2* stats;
    Cut* cuts;
};
__host__ __device__ inline Parts parts_of(void* workspace, int ctas, int rows, int d) {
    float* p = (float*)workspace;
    const size_t n = (size_t)ctas * 2 * rows;
    return Parts{p, (float2*)(p + n * d), (Cut*)(p + n * (d + 2))};
}
inline size_t parts_bytes(int ctas, int rows, int d) {
    return (size_t)ctas * 2 * rows * (d + 2) * sizeof(float) + (size_t)ctas * sizeof(Cut);
}

// Where row r of a tile lies
__device__ __forceinline__ long long row_at(const CacheArgs& a, const mb200_heads& t, int group, int b, int h, int r) {
    const int i = r / group;
    return ((long long)b * a.queries + i) * t.token_stride + (long long)(h * group + (r - i * group)) * t.head_stride;
}

// Queries as whole numbers Q of 22 bits, hi 2^16 + mid 2^8 + lo (lo, mid in -128 .. 127) times 2^(e - 20), e the exponent of the
// row's largest (from -106 on; below that 2^-126, since the inverse has to be a number as well): 1.5 * 2^23 + 0x8080 added
// in the multiplication leaves, in the sum's bytes, lo + 128, mid + 128 and hi + 64 (|hi| < 64).
constexpr int kPlanes = 3;
__device__ __forceinline__ void planes_of(const float (&x)[4], float up, uint32_t (&w)[kPlanes]) {
    uint32_t b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        b[i] = __float_as_uint(__fmaf_rn(x[i], up, 12615808.f));
    const uint32_t l0 = __byte_perm(b[0], b[1], 0x5140), l1 = __byte_perm(b[2], b[3], 0x5140);
    const uint32_t h0 = __byte_perm(b[0], b[1], 0x0062), h1 = __byte_perm(b[2], b[3], 0x0062);
    w[2] = __byte_perm(l0, l1, 0x5410) ^ 0x80808080u;
    w[1] = __byte_perm(l0, l1, 0x7632) ^ 0x80808080u;
    const uint32_t t = __byte_perm(h0, h1, 0x5410) ^ 0x40404040u;
    w[0] = t | (t & 0x40404040u) << 1;
}

// 4 results; VEC: they start on an 8-byte boundary
template <class T, bool VEC>
__device__ __forceinline__ void store4(void* base, long long at, const float4& v) {
    uint16_t* p = (uint16_t*)base + at;
    const uint32_t lo = pack2<T>(v.x, v.y), hi = pack2<T>(v.z, v.w);
    if constexpr (VEC) {
        *(uint2*)p = make_uint2(lo, hi);
    } else {
        p[0] = (uint16_t)lo, p[1] = (uint16_t)(lo >> 16);
        p[2] = (uint16_t)hi, p[3] = (uint16_t)(hi >> 16);
    }
}

// FULL: d == D; VEC: queries and results start on 16-byte boundaries
template <class T, int D, int NT, bool VEC, bool FULL>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) cache_kernel(const CacheArgs a, const Shape shape) {
    using R = Ring<D>;
    constexpr int kRows = 8 * NT, kChunks = D / 64, kTiles = D / 16;
    constexpr bool kFine = std::is_same<T, __half>::value;  // P as two fp16 numbers
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ long long s_from, s_to, s_rest, s_quota;
    __shared__ int s_b;
    __shared__ float2 s_stats[kWarps][kRows];
    __shared__ float2 s_weight[kWarps][kRows];
    __shared__ float s_down[kWarps][kRows];
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
            s_from = from, s_to = to, s_b = at, s_rest = from - before * lines, s_quota = quota;
    }
    __syncthreads();
    long long left = s_to - s_from;
    int b = s_b, at = 0, blk = 0;
    if (left > 0) {
        const int n = rounds_of(a, shape.capacity, b);
        at = (int)(s_rest / n);
        blk = (int)(s_rest - (long long)at * n) * kRound;
    }
    const Parts parts = parts_of(a.workspace, gridDim.x, kRows, D);
    if (tid == 0 && a.workspace) {
        Cut cut{};
        cut.b = left > 0 && blk > 0 ? b : -1;
        cut.at = at, cut.from = s_from - blk / kRound, cut.quota = s_quota;
        cut.rounds = left > 0 ? rounds_of(a, shape.capacity, b) : 0;
        parts.cuts[blockIdx.x] = cut;
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
        const int length = a.lengths[b];
        const int all = blocks_of(a, shape.capacity, b);
        if (all == 0) {
            ++b;
            continue;
        }
        const int h = at / shape.tiles, tile = at - h * shape.tiles;
        const int rounds = (all - blk + kRound - 1) / kRound;
        const int take = (int)(left < rounds ? left : rounds);
        const int count = min(all - blk, take * kRound);
        const int row0 = tile * kRows, rows = min(kRows, shape.rows - row0);

        const int32_t* table = a.c.block_table + (long long)b * a.c.table_stride;
        // this warp's steps: blocks blk + 2 warp, + 8, .. and the one behind each
        const int mine = (count - warp * kStep + kRound - 1) / kRound;
        const int first_blk = blk + warp * kStep;
        // a lane knows a block of one turn of 16 steps; -1: no page, or behind the last
        auto numbers = [&](int turn) {
            const int p = first_blk + (turn * 16 + (lane >> 1)) * kRound + (lane & 1);
            if (p >= blk + count)
                return -1;
            const int i = p / page_blocks;
            const int page = table[i];  // (i < table_pages: lengths end with the table)
            if ((unsigned)page >= (unsigned)a.c.pages) {
                *(volatile int*)a.status = ERR_PAGE;
                return -1;
            }
            return (page * a.c.kv_heads + h) * page_blocks + p - i * page_blocks;
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

        // positions that a row sees, whether the table has them or not
        auto limit = [&](int row) {
            const int i = row / group;
            return min(length - a.queries + 1, 0x7fffffff - i) + i;
        };
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
            const bool finite = most < 0x7f800000u;
            const int shift = min(126, 20 + 127 - (int)(most >> 23));
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
            lim0[nt] = limit(row0 + nt * 8 + 2 * c);
            lim1[nt] = limit(row0 + nt * 8 + 2 * c + 1);
        }
        const int seen_by_all = limit(row0);

        // of rows 2 c and 2 c + 1: maximum of the scores, sum of the powers, maximum of scores and their block's exponent
        // of V, and 2^(kLift - k): the sums hold 2^(kLift - k) times what they are, with m + k >= w
        float o[NT][kTiles][4], m0[NT], m1[NT], l0[NT], l1[NT], w0[NT], w1[NT], up0[NT], up1[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            m0[nt] = m1[nt] = w0[nt] = w1[nt] = none;
            l0[nt] = l1[nt] = 0.f;
            up0[nt] = up1[nt] = 1.f;
#pragma unroll
            for (int t = 0; t < kTiles; ++t)
                o[nt][t][0] = o[nt][t][1] = o[nt][t][2] = o[nt][t][3] = 0.f;
        }
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
            float n0[NT], n1[NT], u0[NT], u1[NT];
            const float e0 = exponent_of_scale(vs[0]), e1 = exponent_of_scale(vs[1]);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const float a0 = fmaxf(s[0][nt][0], s[0][nt][2]), b0 = fmaxf(s[1][nt][0], s[1][nt][2]);
                const float a1 = fmaxf(s[0][nt][1], s[0][nt][3]), b1 = fmaxf(s[1][nt][1], s[1][nt][3]);
                n0[nt] = fmaxf(a0, b0), n1[nt] = fmaxf(a1, b1);
                u0[nt] = fmaxf(a0 + e0, b0 + e1), u1[nt] = fmaxf(a1 + e0, b1 + e1);
                raise |= n0[nt] > m0[nt] + kAhead || n1[nt] > m1[nt] + kAhead;
                raise |= u0[nt] > w0[nt] + kAhead || u1[nt] > w1[nt] + kAhead;
            }
            if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    const float r0 = raised(n0[nt], u0[nt], m0[nt], l0[nt], w0[nt], up0[nt]);
                    const float r1 = raised(n1[nt], u1[nt], m1[nt], l1[nt], w1[nt], up1[nt]);
#pragma unroll
                    for (int t = 0; t < kTiles; ++t) {
                        o[nt][t][0] *= r0, o[nt][t][1] *= r1;
                        o[nt][t][2] *= r0, o[nt][t][3] *= r1;
                    }
                }
            }
            uint32_t hi[kStep][NT][2], lo[kStep][NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const float z0 = m0[nt] == none ? 0.f : m0[nt], z1 = m1[nt] == none ? 0.f : m1[nt];
#pragma unroll
                for (int x = 0; x < kStep; ++x) {
                    float p[4] = {exp2_fast(s[x][nt][0] - z0), exp2_fast(s[x][nt][1] - z1), exp2_fast(s[x][nt][2] - z0),
                                  exp2_fast(s[x][nt][3] - z1)};
                    l0[nt] += p[0] + p[2], l1[nt] += p[1] + p[3];
                    // (what is not seen stays 0 whatever the block's scale; what is seen is none if that is none, also with p = 0)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        p[e] = s[x][nt][e] == none ? 0.f : __fmul_rn(__fmul_rn(p[e], e & 1 ? up1[nt] : up0[nt]), vs[x]);
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
                s_down[warp][nt * 8 + 2 * c] = inverse_power(up0[nt]);
                s_down[warp][nt * 8 + 2 * c + 1] = inverse_power(up1[nt]);
            }
        }
        __syncthreads();  // (nobody reads the rings any more)
        const int active = min(kWarps, (count + kStep - 1) / kStep);
        float* sums = (float*)smem;  // [warp][row][kPitch]
        if (warp < active) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int t = 0; t < kTiles; ++t) {
                    float* p = sums + (warp * kRows + nt * 8 + 2 * c) * kPitch<D> + 16 * t + 2 * g;
                    *(float2*)p = make_float2(o[nt][t][0], o[nt][t][2]);
                    *(float2*)(p + kPitch<D>) = make_float2(o[nt][t][1], o[nt][t][3]);
                }
        }
        // each warp's weight in a row: what its maximum lies below the largest, over the total, and the power of two that its sums
        // are held away from what they are. In this order nothing on the way to an average is larger than the values are
        const bool whole = blk == 0 && count == all;
        if (tid < kRows) {
            float m = none;
#pragma unroll
            for (int w = 0; w < kWarps; ++w)
                m = fmaxf(m, w < active ? s_stats[w][tid].x : none);
            const float z = m == none ? 0.f : m;
            float total = 0.f, f[kWarps];
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float2 st = s_stats[w][tid];
                f[w] = w < active ? exp2_fast(st.x - z) : 0.f;
                total += w < active ? st.y * f[w] : 0.f;
            }
            // (nothing seen: zeros)
            const float over = total == 0.f ? 0.f : __fdiv_rn(1.f, total);
#pragma unroll
            for (int w = 0; w < kWarps; ++w)
                s_weight[w][tid] = make_float2(__fmul_rn(f[w], over), s_down[w][tid]);
            if (!whole)
                parts.stats[((long long)blockIdx.x * 2 + !first) * kRows + tid] = make_float2(m, total);
        }
        __syncthreads();
        for (int i = tid; i < rows * (D / 4); i += kThreads) {
            const int r = i / (D / 4), e = i % (D / 4) * 4;
            float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kWarps; ++w)
                if (w < active) {
                    const float4 v = *(const float4*)(sums + (w * kRows + r) * kPitch<D> + e);
                    const float2 f = s_weight[w][r];
                    sum.x = __fmaf_rn(v.x * f.x, f.y, sum.x), sum.y = __fmaf_rn(v.y * f.x, f.y, sum.y);
                    sum.z = __fmaf_rn(v.z * f.x, f.y, sum.z), sum.w = __fmaf_rn(v.w * f.x, f.y, sum.w);
                }
            if (!whole)
                *(float4*)(parts.sums + (((long long)blockIdx.x * 2 + !first) * kRows + r) * D + e) = sum;
            else if (FULL || e < d)
                store4<T, VEC>(a.out.p, row_at(a, a.out, group, b, h, row0 + r) + e, sum);
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
    // sequences without a position: nothing is seen. kIdleRows rows of one (a query's heads) at a time, a warp each
    const int all_rows = a.queries * a.heads, pieces = (all_rows - 1) / kIdleRows + 1;
    for (long long x = blockIdx.x; x < (long long)a.c.batch * pieces; x += gridDim.x) {
        const int idle = pieces == 1 ? (int)x : (int)(x / pieces), length = a.lengths[idle];
        const unsigned r0 = (unsigned)(x - (long long)idle * pieces) * kIdleRows, r1 = min(r0 + kIdleRows, (unsigned)all_rows);
        if (length > shape.capacity && tid == 0 && r0 == 0)
            *(volatile int*)a.status = ERR_PAGE;
        if (length <= 0)
            for (unsigned r = r0 + warp; r < r1; r += kWarps) {
                const unsigned i = r / a.heads;
                T* p = (T*)a.out.p + ((long long)idle * a.queries + i) * a.out.token_stride +
                       (long long)(r - i * a.heads) * a.out.head_stride;
                for (int e = lane; e < d; e += 32)
                    p[e] = from_float<T>(0.f);
            }
    }
}

// Joins the parts of an item that was cut, in their order: the first CTA whose part of the line begins inside it names it. One
// row a CTA; its warps share the parts (D / 4 lanes each), all of whose weights every warp finds for itself.
constexpr int kJoinWarps = 8;
template <class T, int D, bool VEC>
__global__ void __launch_bounds__(32 * kJoinWarps) join_kernel(const CacheArgs a, const Shape shape, int ctas, int tile_rows) {
    constexpr int kLanes = D / 4, kAtOnce = 32 / kLanes, kStride = kJoinWarps * kAtOnce;
    __shared__ float4 s_sum[kJoinWarps * kAtOnce][kLanes];
    const int cta = blockIdx.x + 1, r = blockIdx.y;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const Parts parts = parts_of(a.workspace, ctas, tile_rows, D);
    pdl_start();
    const Cut cut = parts.cuts[cta];
    if (cut.b < 0)
        return;
    const int c0 = (int)(cut.from / cut.quota), c1 = (int)((cut.from + cut.rounds - 1) / cut.quota);
    const int h = cut.at / shape.tiles, tile = cut.at - h * shape.tiles;
    if (c0 + 1 != cta || tile * tile_rows + r >= shape.rows)
        return;
    const long long first = ((long long)c0 * 2 + (c0 * cut.quota < cut.from)) * tile_rows;
    auto part = [&](int i) { return (i == 0 ? first : (long long)(c0 + i) * 2 * tile_rows) + r; };
    const int n = c1 + 1 - c0;
    const float none = __uint_as_float(0xff800000u);
    const int sub = warp * kAtOnce + lane / kLanes, e = lane % kLanes;
    auto average = [&](int i) {
        return i < n ? *(const float4*)(parts.sums + part(i) * D + 4 * e) : make_float4(0.f, 0.f, 0.f, 0.f);
    };
    // (the first 32 parts are on their way while the weights are found)
    float4 ahead[32 / kStride];
#pragma unroll
    for (int x = 0; x < 32 / kStride; ++x)
        ahead[x] = average(x * kStride + sub);
    const float2 nothing = make_float2(none, 0.f), mine = lane < n ? parts.stats[part(lane)] : nothing;
    float m = mine.x, total = mine.y;
    for (int i = lane + 32; i < n; i += 32) {
        const float2 st = parts.stats[part(i)];
        const float t = fmaxf(m, st.x), z = t == none ? 0.f : t;
        total = __fmul_rn(total, exp2_fast(m - z)) + st.y * exp2_fast(st.x - z);
        m = t;
    }
    float most = m;
#pragma unroll
    for (int x = 1; x < 32; x *= 2)
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, x));
    const float z = most == none ? 0.f : most;
    total = __fmul_rn(total, exp2_fast(m - z));
#pragma unroll
    for (int x = 1; x < 32; x *= 2)
        total += __shfl_xor_sync(0xffffffffu, total, x);
    const float over = total == 0.f ? 0.f : __fdiv_rn(1.f, total);
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](const float4& v, float weight) {
        sum.x = __fmaf_rn(v.x, weight, sum.x), sum.y = __fmaf_rn(v.y, weight, sum.y);
        sum.z = __fmaf_rn(v.z, weight, sum.z), sum.w = __fmaf_rn(v.w, weight, sum.w);
    };
    const float f = __fmul_rn(mine.y * exp2_fast(mine.x - z), over);
#pragma unroll
    for (int x = 0; x < 32 / kStride; ++x)
        add(ahead[x], __shfl_sync(0xffffffffu, f, x * kStride + sub));
    for (int base = 32; base < n; base += 32) {
        const float2 st = base + lane < n ? parts.stats[part(base + lane)] : nothing;
        const float g = __fmul_rn(st.y * exp2_fast(st.x - z), over);
#pragma unroll
        for (int x = 0; x < 32 / kStride; ++x)
            add(average(base + x * kStride + sub), __shfl_sync(0xffffffffu, g, x * kStride + sub));
    }
    s_sum[sub][e] = sum;
    __syncthreads();
    if (threadIdx.x >= kLanes || 4 * e >= a.c.d)
        return;
    sum = s_sum[0][e];
#pragma unroll
    for (int x = 1; x < kJoinWarps * kAtOnce; ++x) {
        const float4 v = s_sum[x][e];
        sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
    }
    store4<T, VEC>(a.out.p, row_at(a, a.out, a.heads / a.c.kv_heads, cut.b, h, tile * tile_rows + r) + 4 * e, sum);
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
    // (sequences of one round are never cut)
    p.bytes = p.ctas == 1 || p.capacity <= kRound * kBlock ? 0 : align_up(parts_bytes(p.ctas, 8 * p.nt, p.d), 256);
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
    if (e == cudaSuccess && p.bytes)
        e = launch_pdl(anything, join_kernel<T, D, VEC>,
                       dim3((unsigned)(p.ctas - 1), (unsigned)(p.rows < 8 * NT ? p.rows : 8 * NT)), dim3(32 * kJoinWarps), 0,
                       st, a, shape, p.ctas, 8 * NT);
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
    auto aligned = [](const mb200_heads& t) {
        return ((uintptr_t)t.p & 15) == 0 && t.token_stride % 8 == 0 && t.head_stride % 8 == 0;
    };
    const bool vec = aligned(a.q) && aligned(a.out);
    if (dtype == MB200_DTYPE_F16)
        return p.d == 64 ? launch_rows<__half, 64>(a, p, vec, st) : launch_rows<__half, 128>(a, p, vec, st);
    return p.d == 64 ? launch_rows<__nv_bfloat16, 64>(a, p, vec, st) : launch_rows<__nv_bfloat16, 128>(a, p, vec, st);
}

}  // namespace attn
}  // namespace mb200
