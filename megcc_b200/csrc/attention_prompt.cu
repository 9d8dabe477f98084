// Attention over whole prompts: packed sequences, causal or not, key heads shared by groups of query heads.
//
//     o_i = sum_j 2^(t_ij - m_i) v_j / sum_j 2^(t_ij - m_i),   t_ij = scale log2(e) q_i . k_j
//
// in one pass over the keys. A CTA has two tiles of 128 rows, a row for each of a few query heads of a group (the largest power
// of two that divides it) and token: short prompts fill a tile, and less of one lies beyond the diagonal. Keys and values come in tiles of 128 through a
// ring of TMA loads. Both products are tcgen05.mma kind::f16: S = Q K^T with both operands in shared memory, O += P V with
// P in tensor memory, in the columns of the S it was made of (two S and two O of 128 x 128 fill the 512 columns), and
// V as it lies, the dimension contiguous. Each tile has a warpgroup, a thread per row: it takes its row of S to
// registers, raises the running maximum, writes P and adds up P's sum. The tensor cores serve one tile while the other
// one's powers are computed.
//
// The maximum is raised only where a score passes it by more than 2^8: then the row's O in tensor memory, whose last
// product is complete by the time the next S is, is scaled by the warp that found it. So nothing else stands between
// a tile's S and its P, and O is touched once or twice in a prompt.
//
// What bounds it: a pair of tiles and 128 keys take the tensor cores 2048 clocks (d = 128) and as many powers, at 16 a
// clock and SM, the special-function unit as long; so a part of the powers is computed on the FMA pipe:
// 2^x = 2^n 2^f, n the nearest whole number, 2^f by the polynomial of least relative error on [-1/2, 1/2] (Remez'
// exchange; degree 3 for bf16, 2^-13.7, degree 4 for fp16, 2^-18.5, against P's rounding of 2^-9 and 2^-12).
//
// Rows of other sequences in a sequence's last tile of keys count with p = 0, which is nothing for finite values; the
// rows of V are zeroed where they are, since the padding behind a batch may hold anything. Values that are no
// numbers among a sequence's own must not reach queries in front of them either: where a row's result is not finite, that row is
// computed anew by plain loops over what it sees.
#include <cuda.h>

#include <type_traits>

#include "attention.h"
#include "kv_cache.cuh"
#include "umma_ptx.cuh"

namespace mb200 {
namespace attn {

using namespace umma;

namespace {

constexpr int kTile = 128;           // rows of a tile of queries, and of a tile of keys
constexpr int kRows = 2 * kTile;     // queries of a CTA
constexpr int kThreads = 320;        // two warpgroups with a tile each; a warp for the products, one for the loads
constexpr float kAhead = 8.f;        // how far (a power of two) a score may pass the running maximum
constexpr int kPolyEvery = 4;        // of so many pairs of powers one is a polynomial
constexpr float kLift = 6.f;         // P is held 2^6 times: 2^14 at most, and fp16 has room down to 2^-30
enum : int { ERR_PROMPT_WAIT = 0x203 };

struct PromptMaps {
    CUtensorMap q, k, v;
};
// Maps whose middle dimension is the token's (heads lie further apart than tokens)
struct TokensInside {
    bool q, k, v;
};

template <int D>
struct Smem {
    static constexpr int kPanel = kTile * 128;             // 64 elements of each row
    static constexpr int kOperand = kPanel * (D / 64);
    static constexpr int kStages = D == 128 ? 5 : 8;
    static constexpr int kRing = 2 * kOperand;             // behind the two tiles of Q
    static constexpr int kBars = kRing + kStages * kOperand;
    static constexpr int kBytes = kBars + 256 + 1024;      // (1024: to the swizzle's boundary)
};
static_assert(Smem<128>::kBytes <= 232448, "shared memory of an SM");

// tensor memory: S (and P in its first columns) of both tiles, then O of both
constexpr uint32_t kColS = 0, kColO = 256;

// kind::f16: fp32 accumulators; A K-major, B K-major (keys) or with its columns contiguous (values)
template <class T>
__host__ __device__ constexpr uint32_t idesc_of(int n, bool b_columns) {
    const uint32_t type = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    return (1u << 4) | (type << 7) | (type << 10) | ((b_columns ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) |
           ((uint32_t)(kTile >> 4) << 24);
}
// descriptors, 128-byte swizzle: the high word holds the distance of groups of 8 rows, version and layout; the low one
// the address and, for values, the distance of panels of 64 columns
constexpr uint32_t kDescHi = (1u << 14) | (2u << 29) | (1024 / 16);
__device__ __forceinline__ uint32_t desc_lo(uint32_t at, uint32_t panel) {
    return ((at & 0x3FFFFu) >> 4) | (panel >> 4) << 16;
}

__device__ __forceinline__ void mma_ss(
        uint32_t leader, uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
            "{\n\t.reg .pred p, q;\n\t.reg .b64 a, b;\n\t"
            "mov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\t"
            "setp.ne.b32 p, %5, 0;\n\tsetp.ne.b32 q, %6, 0;\n\t"
            "@q tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, p;\n\t}" ::"r"(d),
            "r"(a_lo), "r"(b_lo), "r"(kDescHi), "r"(idesc), "r"(accumulate), "r"(leader)
            : "memory");
}
__device__ __forceinline__ void mma_ts(
        uint32_t leader, uint32_t d, uint32_t a, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
            "{\n\t.reg .pred p, q;\n\t.reg .b64 b;\n\t"
            "mov.b64 b, {%2, %3};\n\t"
            "setp.ne.b32 p, %5, 0;\n\tsetp.ne.b32 q, %6, 0;\n\t"
            "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t}" ::"r"(d),
            "r"(a), "r"(b_lo), "r"(kDescHi), "r"(idesc), "r"(accumulate), "r"(leader)
            : "memory");
}
__device__ __forceinline__ void tma_load_3d_if(
        uint32_t leader, uint32_t smem, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2) {
    asm volatile(
            "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %6, 0;\n\t"
            "@q cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
            " [%0], [%1, {%3, %4, %5}], [%2];\n\t}" ::"r"(smem),
            "l"((uint64_t)map), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(leader)
            : "memory");
}
__device__ __forceinline__ void arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tmem_ld32_nowait(uint32_t at, uint32_t* v) {
    asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
            "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
            "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
            : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
              "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
              "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
              "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
            : "r"(at)
            : "memory");
}
// (the registers are named so that no use of them moves above the wait)
__device__ __forceinline__ void tmem_ld_wait32(uint32_t* v) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]),
                   "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]),
                   "+r"(v[16]), "+r"(v[17]), "+r"(v[18]), "+r"(v[19]), "+r"(v[20]), "+r"(v[21]), "+r"(v[22]),
                   "+r"(v[23]), "+r"(v[24]), "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]), "+r"(v[29]),
                   "+r"(v[30]), "+r"(v[31])
                 :
                 : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t at, const uint32_t* v) {
    asm volatile(
            "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
            "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(at),
            "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
            "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
            : "memory");
}
__device__ __forceinline__ void fence_before() {
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void fence_after() {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// two at a time
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 r;
    asm("{\n\t.reg .b64 a, b, c, d;\n\t"
        "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
        "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 r;
    asm("{\n\t.reg .b64 a, b, d;\n\t"
        "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
        "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 both(float v) {
    return make_float2(v, v);
}
// the largest of three, or a NaN among them
__device__ __forceinline__ float max_or_nan(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// 2^x of numbers up to 100 without the special-function unit; 2^-126 for what is less
template <class T>
__device__ __forceinline__ float2 exp2_poly(float2 x) {
    constexpr bool fine = std::is_same<T, __half>::value;
    x.x = fmaxf(x.x, -126.f), x.y = fmaxf(x.y, -126.f);
    // 1.5 * 2^23 leaves the nearest whole number in the low bits
    const float2 n = add2(x, both(12582912.f));
    const float2 f = fma2(add2(n, both(-12582912.f)), both(-1.f), x);
    float2 p;
    if constexpr (fine) {
        p = fma2(both(0.009570102207f), f, both(0.05591785908f));
        p = fma2(p, f, both(0.2402474433f));
        p = fma2(p, f, both(0.6931217909f));
        p = fma2(p, f, both(0.9999992847f));
    } else {
        p = fma2(both(0.05517166853f), f, both(0.2426111251f));
        p = fma2(p, f, both(0.6932609677f));
        p = fma2(p, f, both(0.9999280572f));
    }
    return make_float2(__uint_as_float(__float_as_uint(p.x) + (__float_as_uint(n.x) << 23)),
                       __uint_as_float(__float_as_uint(p.y) + (__float_as_uint(n.y) << 23)));
}

// A row of scores -> P in tensor memory and its sum. POLY: a part of the powers by the FMA pipe (nothing is hidden: those are
// not 0)
template <class T, bool POLY>
__device__ __forceinline__ void powers(uint32_t (&s)[kTile], float scale, float shift, uint32_t col_s, float2 (&l)[2]) {
    const float2 z = both(shift), f = both(scale);
#pragma unroll
    for (int x = 0; x < 4; ++x) {
        uint32_t p[16];
#pragma unroll
        for (int y = 0; y < 16; ++y) {
            const int e = 32 * x + 2 * y;
            float2 v = fma2(make_float2(__uint_as_float(s[e]), __uint_as_float(s[e + 1])), f, z);
            v = POLY && y % kPolyEvery == kPolyEvery - 1 ? exp2_poly<T>(v) : make_float2(exp2_fast(v.x), exp2_fast(v.y));
            l[y & 1] = add2(l[y & 1], v);
            p[y] = pack2<T>(v.x, v.y);
        }
        tmem_st16(col_s + 16 * x, p);
    }
}

// The whole warp waits, and goes on or gives up as one: what follows (products, loads of tensor memory, __syncwarp) wants
// all of its lanes
__device__ __forceinline__ bool wait_for(uint32_t bar, uint32_t parity, volatile int* abort, int* status) {
    if (__all_sync(0xffffffffu, mbar_wait_u32(bar, parity, abort)))
        return true;
    *abort = 1;
    *(volatile int*)status = ERR_PROMPT_WAIT;
    return false;
}

// What a CTA works on: rows are tokens times `1 << pack` heads
struct Work {
    int head, kv_head, pack;
    int q0, tokens;   // first token, how many
    int k0, keys;     // first row of the sequence's keys, how many
    int seen;         // keys that the first token sees; each next one sees `step` more
    int step;
    __device__ __forceinline__ int limit(int token) const {  // keys that a token sees
        return max(0, min(keys, seen + token * step));
    }
    __device__ __forceinline__ int tiles(int t) const {  // of keys, for tile t of rows
        const int per = kTile >> pack, n = min(tokens - t * per, per);
        return n <= 0 ? 0 : (limit(t * per + n - 1) + kTile - 1) / kTile;
    }
};

// A row by plain loops: lanes take keys for the scores, dimensions for the sum. The whole warp calls it.
template <class T>
__device__ __noinline__ void row_anew(const PromptArgs& a, long long token, int head, int k0, int n) {
    const int lane = threadIdx.x & 31, kv_head = head / (a.heads / a.kv_heads);
    const uint16_t* q = (const uint16_t*)a.q.p + token * a.q.token_stride + head * a.q.head_stride;
    const uint16_t* k = (const uint16_t*)a.k.p + kv_head * a.k.head_stride;
    const uint16_t* v = (const uint16_t*)a.v.p + kv_head * a.v.head_stride;
    auto value = [](const uint16_t* p) { return scaled::to_float(*reinterpret_cast<const T*>(p)); };
    float m = __uint_as_float(0xff800000u), total = 0.f, sum[kMaxD / 32] = {};
    for (int j0 = 0; j0 < n; j0 += 32) {
        const int j = j0 + lane;
        float t = __uint_as_float(0xff800000u);
        if (j < n) {
            const uint16_t* key = k + (long long)(k0 + j) * a.k.token_stride;
            float s = 0.f;
            for (int e = 0; e < a.d; ++e)
                s = __fmaf_rn(value(q + e), value(key + e), s);
            t = __fmul_rn(s, a.scale_log2);
        }
        float top = t;
#pragma unroll
        for (int x = 1; x < 32; x *= 2)
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
        top = fmaxf(top, m);
        const float z = top == __uint_as_float(0xff800000u) ? 0.f : top;
        const float down = exp2_fast(m - z), p = j < n ? exp2_fast(t - z) : 0.f;
        m = top;
        total = __fmul_rn(total, down) + p;
#pragma unroll
        for (int i = 0; i < kMaxD / 32; ++i)
            sum[i] = __fmul_rn(sum[i], down);
        const int here = min(32, n - j0);
        for (int x = 0; x < here; ++x) {
            const float f = __shfl_sync(0xffffffffu, p, x);
            const uint16_t* r = v + (long long)(k0 + j0 + x) * a.v.token_stride;
#pragma unroll
            for (int i = 0; i < kMaxD / 32; ++i)
                if (lane + 32 * i < a.d)
                    sum[i] = __fmaf_rn(f, value(r + lane + 32 * i), sum[i]);
        }
    }
#pragma unroll
    for (int x = 1; x < 32; x *= 2)
        total += __shfl_xor_sync(0xffffffffu, total, x);
    T* out = (T*)a.out.p + token * a.out.token_stride + head * a.out.head_stride;
#pragma unroll
    for (int i = 0; i < kMaxD / 32; ++i)
        if (lane + 32 * i < a.d)
            out[lane + 32 * i] = from_float<T>(__fdiv_rn(sum[i], total));
}

template <class T, int D>
__global__ void __launch_bounds__(kThreads, 1) prompt_kernel(
        const __grid_constant__ PromptMaps maps, const PromptArgs a, const TokensInside inside) {
    using S = Smem<D>;
    constexpr int kStages = S::kStages;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
    __shared__ int s_work[5], s_never;
    uint64_t* bars = (uint64_t*)(smem + S::kBars);
    uint32_t* tmem_slot = (uint32_t*)(bars + 28);
    volatile int* abort = (volatile int*)(tmem_slot + 1);
    const uint32_t bar0 = smem_u32(bars);
    // barriers: queries [2], S complete [2], P written [2], O complete [2], all products complete, the ring's stages full,
    // and empty
    const uint32_t q_full = bar0, s_full = bar0 + 16, p_full = bar0 + 32, o_full = bar0 + 48, drained = bar0 + 64,
                   full = bar0 + 72, empty = full + 8 * kStages;
    const int warp = uniform_warp_index(), lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(bars + i, 1);
            mbar_init(bars + 2 + i, 1);
            mbar_init(bars + 4 + i, 4);
            mbar_init(bars + 6 + i, 1);
        }
        for (int i = 0; i < 1 + 2 * kStages; ++i)
            mbar_init(bars + 8 + i, 1);
        *abort = 0;
        s_never = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    } else if (threadIdx.x == 128) {
        tma_prefetch_map(&maps.q);
        tma_prefetch_map(&maps.k);
        tma_prefetch_map(&maps.v);
    }
    if (warp == 8) {
        __syncwarp();  // (the whole warp's, .aligned: none of its lanes does anything else in front of this)
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                     "r"(512)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    pdl_start();
    // ---- which queries: with n tokens a CTA, sequence b's have the slots from cu[b] / n + b on, the last ones first ----
    Work w;
    w.pack = a.pack;
    const int packs = a.heads >> a.pack, per_cta = kRows >> a.pack;
    w.head = (int)(blockIdx.x % packs) << a.pack;
    w.kv_head = w.head / (a.heads / a.kv_heads);
    if (warp == 9) {
        const int slot = blockIdx.x / packs;
        const int b = first_beyond(a.batch, slot, [&](int i) { return (long long)a.cu_q[i + 1] / per_cta + i + 1; });
        int first = 0, n = 0, k0 = 0, keys = 0, row0 = 0;
        if (b < a.batch) {
            first = a.cu_q[b];
            n = first < 0 ? 0 : min(a.cu_q[b + 1], a.tokens) - first;
            k0 = a.cu_k[b];
            keys = k0 < 0 ? 0 : max(0, min(a.cu_k[b + 1], a.key_tokens) - k0);
            row0 = ((n + per_cta - 1) / per_cta - 1 - (slot - (first / per_cta + b))) * per_cta;
            if (slot < first / per_cta + b || row0 < 0)
                n = row0 = 0;
        }
        if (lane == 0) {
            s_work[0] = first + row0;
            s_work[1] = max(0, min(n - row0, per_cta));
            s_work[2] = k0;
            s_work[3] = keys;
            // (a sequence's last query sees its last key)
            s_work[4] = a.causal ? max(-0x40000000, keys - n + 1 + row0) : keys;
        }
    }
    fence_before();
    __syncthreads();
    fence_after();
    w.q0 = s_work[0], w.tokens = s_work[1], w.k0 = s_work[2], w.keys = s_work[3], w.seen = s_work[4];
    w.step = a.causal ? 1 : 0;
    const uint32_t tmem = *tmem_slot;
    const int n0 = w.tiles(0), n1 = w.tiles(1), most = max(n0, n1);

    if (warp >= 8) {
        const uint32_t leader = elect_one() ? 1 : 0;
        const uint32_t ring = smem_u32(smem + S::kRing);
        if (warp == 9 && most > 0) {
            // ---- loads: Q0, K, Q1, V, K, V, .. ----
            auto load = [&](const CUtensorMap* map, bool tokens_inside, uint32_t to, uint32_t bar, int head, int row) {
                mbar_expect_tx_if(leader, bar, S::kOperand);
#pragma unroll
                for (int i = 0; i < D / 64; ++i)
                    tma_load_3d_if(leader, to + i * S::kPanel, map, bar, 64 * i, tokens_inside ? row : head,
                                   tokens_inside ? head : row);
            };
            load(&maps.q, inside.q, smem_u32(smem), q_full, w.head, w.q0);
            int i = 0;
            for (; i < 2 * most; ++i) {
                const int s = i % kStages, turn = i / kStages;
                if (turn > 0 && !wait_for(empty + 8 * s, (turn - 1) & 1, abort, a.status))
                    break;
                load(i & 1 ? &maps.v : &maps.k, i & 1 ? inside.v : inside.k, ring + s * S::kOperand, full + 8 * s,
                     w.kv_head, w.k0 + (i >> 1) * kTile);
                if (i == 0)
                    load(&maps.q, inside.q, smem_u32(smem + S::kOperand), q_full + 8, w.head, w.q0 + (kTile >> w.pack));
            }
            // whoever gave up: the copies on their way land before the CTA ends
            for (int x = max(0, i - kStages); x < i; ++x)
                mbar_wait_u32(full + 8 * (x % kStages), (x / kStages) & 1, &s_never);
            for (int t = 0; t < 2; ++t)
                mbar_wait_u32(q_full + 8 * t, 0, &s_never);
        } else if (warp == 8) {
            // ---- products ----
            constexpr uint32_t kIdescS = idesc_of<T>(kTile, false), kIdescO = idesc_of<T>(D, true);
            auto scores = [&](int t, int i) {  // S_t = Q_t K^T with the i-th operand of the ring
                const uint32_t q = desc_lo(smem_u32(smem + t * S::kOperand), 0);
                const uint32_t k = desc_lo(ring + (i % kStages) * S::kOperand, 0);
#pragma unroll
                for (int x = 0; x < D / 16; ++x) {
                    const uint32_t at = (x / 4) * (S::kPanel / 16) + (x % 4) * 2;
                    mma_ss(leader, tmem + kColS + t * kTile, q + at, k + at, kIdescS, x != 0);
                }
                umma_commit_if(leader, s_full + 8 * t);
            };
            bool ok = true;
            auto wait = [&](uint32_t bar, uint32_t parity) {
                if (ok)
                    ok = wait_for(bar, parity, abort, a.status);
                return ok;
            };
            auto operand = [&](int i) { return wait(full + 8 * (i % kStages), (i / kStages) & 1); };
            for (int t = 0; t < 2 && ok; ++t) {
                if (t == 0 ? n0 : n1) {
                    if (wait(q_full + 8 * t, 0) && operand(0)) {
                        fence_after();
                        scores(t, 0);
                    }
                } else if (most > 0) {
                    wait(q_full + 8 * t, 0);
                }
            }
            if (most > 0)
                umma_commit_if(leader, empty);
            const bool foreign = w.keys % kTile != 0 && most * kTile > w.keys;
            for (int j = 0; j < most && ok; ++j) {
                const int iv = 2 * j + 1, ik = 2 * j + 2;
                // (both here, where the warp has time: a wait costs it 160 clocks even if there is nothing to wait for)
                if (!operand(iv) || (j + 1 < most && !operand(ik)))
                    break;
                if (foreign && j == most - 1) {
                    uint8_t* v = smem + S::kRing + (iv % kStages) * S::kOperand;
                    for (int r = w.keys % kTile + (lane >> 3); r < kTile; r += 4)
#pragma unroll
                        for (int i = 0; i < D / 64; ++i)
                            *(uint4*)(v + i * S::kPanel + r * 128 + (lane & 7) * 16) = make_uint4(0, 0, 0, 0);
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                }
                for (int t = 0; t < 2 && ok; ++t) {
                    const int n = t == 0 ? n0 : n1;
                    if (j >= n)
                        continue;
                    if (!wait(p_full + 8 * t, j & 1))
                        break;
                    fence_after();
                    const uint32_t v = desc_lo(ring + (iv % kStages) * S::kOperand, S::kPanel);
#pragma unroll
                    for (int x = 0; x < kTile / 16; ++x)
                        mma_ts(leader, tmem + kColO + t * kTile, tmem + kColS + t * kTile + 8 * x, v + x * (2048 / 16),
                               kIdescO, j > 0 || x != 0);
                    umma_commit_if(leader, o_full + 8 * t);
                    if (j + 1 < n) {
                        // S takes P's columns: the product that reads them has to be complete
                        if (!wait(o_full + 8 * t, j & 1))
                            break;
                        scores(t, ik);
                    }
                }
                umma_commit_if(leader, empty + 8 * (iv % kStages));
                if (j + 1 < most) {
                    // (a tile that needs no more keys still lets them go by)
                    umma_commit_if(leader, empty + 8 * (ik % kStages));
                }
            }
            umma_commit_if(leader, drained);
            mbar_wait_u32(drained, 0, &s_never);
        }
    } else {
        // ---- a row each ----
        const int t = warp >> 2, n = t == 0 ? n0 : n1;
        const int row = t * kTile + (threadIdx.x & (kTile - 1));
        const uint32_t lanes = (uint32_t)(warp & 3) * 32u << 16;
        const uint32_t col_s = tmem + lanes + kColS + t * kTile, col_o = tmem + lanes + kColO + t * kTile;
        const int limit = w.limit(row >> w.pack), first_limit = w.limit((row - lane) >> w.pack);
        const float none = __uint_as_float(0xff800000u);
        // (scores get the scale's sign, and with a scale of 0 become 0: what is hidden counts as -infinity still)
        const float scale = a.scale_log2 == 0.f ? 1.f : fabsf(a.scale_log2), sign = a.scale_log2 == 0.f ? 0.f : -1.f;
        float m = none;
        float2 l[2] = {};
        bool ok = true;
#pragma unroll 1
        for (int j = 0; j < n; ++j) {
            ok = wait_for(s_full + 8 * t, j & 1, abort, a.status);
            if (!ok)
                break;
            fence_after();
            uint32_t s[kTile];
#pragma unroll
            for (int x = 0; x < 4; ++x)
                tmem_ld32_nowait(col_s + 32 * x, s + 32 * x);
#pragma unroll
            for (int x = 0; x < 4; ++x)
                tmem_ld_wait32(s + 32 * x);
            if (a.scale_log2 <= 0.f) {
#pragma unroll
                for (int x = 0; x < kTile; ++x)
                    s[x] = __float_as_uint(__uint_as_float(s[x]) * sign);
            }
            const bool hides = (j + 1) * kTile > first_limit;  // (of the warp's rows the first one sees the least)
            if (hides) {
                const int here = limit - j * kTile;
#pragma unroll
                for (int x = 0; x < kTile; ++x)
                    s[x] = x < here ? s[x] : 0xff800000u;
            }
            float top[4] = {none, none, none, none};
#pragma unroll
            for (int x = 0; x < kTile; x += 2)
                top[x / 2 & 3] = max_or_nan(top[x / 2 & 3], __uint_as_float(s[x]), __uint_as_float(s[x + 1]));
            // (a NaN that a row sees makes all of it NaN)
            const float highest = max_or_nan(max_or_nan(top[0], top[1], top[2]), top[3], m);
            // (each row by itself, so that its result depends on no other one)
            const bool raise = !((highest - m) * scale <= kAhead);
            if (__any_sync(0xffffffffu, raise)) {
                const float down = !raise || highest == m ? 1.f : exp2_fast((m - highest) * scale);
                m = raise ? highest : m;
#pragma unroll
                for (int x = 0; x < 2; ++x)
                    l[x].x *= down, l[x].y *= down;
                if (j > 0) {
#pragma unroll 1
                    for (int x = 0; x < D; x += 16) {
                        uint32_t o[16];
                        tmem_ld16(col_o + x, o);
#pragma unroll
                        for (int y = 0; y < 16; ++y)
                            o[y] = __float_as_uint(__uint_as_float(o[y]) * down);
                        tmem_st16(col_o + x, o);
                    }
                }
            }
            const float shift = kLift - (m == none ? 0.f : m * scale);
            if (hides)
                powers<T, false>(s, scale, shift, col_s, l);
            else
                powers<T, true>(s, scale, shift, col_s, l);
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            fence_before();
            __syncwarp();
            if (lane == 0)
                arrive(p_full + 8 * t);
        }
        // ---- the rows' results: 16-byte units of this warp's rows through its part of Q's shared memory, of which all
        // products are complete ----
        const float total = (l[0].x + l[0].y) + (l[1].x + l[1].y);
        if (ok && n > 0) {
            ok = wait_for(o_full + 8 * t, (n - 1) & 1, abort, a.status);
            fence_after();
        }
        if (ok) {
            const int row0 = row - lane, units = a.d / 8;
            uint8_t* stage = smem + t * S::kOperand + (warp & 3) * (32 * D * 2);
            const float inv = __fdiv_rn(1.f, total);
            bool bad = false;
#pragma unroll 1
            for (int x = 0; x < (n > 0 ? D : 0); x += 32) {
                uint32_t o[32];
                tmem_ld32_nowait(col_o + x, o);
                tmem_ld_wait32(o);
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    float v[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        v[e] = limit > 0 ? __uint_as_float(o[8 * u + e]) * inv : 0.f;
                        bad |= !(fabsf(v[e]) <= 3.402823466e38f);
                    }
                    *(uint4*)(stage + lane * (D * 2) + (((x / 8 + u) ^ (lane & 7)) << 4)) = pack8<T>(v);
                }
            }
            __syncwarp();
            const bool vec = ((uintptr_t)a.out.p & 15) == 0 && a.out.token_stride % 8 == 0 && a.out.head_stride % 8 == 0;
            const int here = min(32, (w.tokens << w.pack) - row0);
            for (int i = lane; i < here * units; i += 32) {
                const int r = i / units, u = i - r * units;
                // (with no tile of keys, queries may still be on their way to the stage)
                const uint4 v = n > 0 ? *(const uint4*)(stage + r * (D * 2) + ((u ^ (r & 7)) << 4)) : make_uint4(0, 0, 0, 0);
                const long long to = (long long)(w.q0 + ((row0 + r) >> w.pack)) * a.out.token_stride +
                                     (w.head + ((row0 + r) & ((1 << w.pack) - 1))) * a.out.head_stride + u * 8;
                if (vec)
                    store8<true>(a.out.p, to, v);
                else
                    store8<false>(a.out.p, to, v);
            }
            __syncwarp();
            for (uint32_t rows = __ballot_sync(0xffffffffu, bad && lane < here); rows; rows &= rows - 1) {
                const int r = row0 + __ffs(rows) - 1, token = r >> w.pack;
                row_anew<T>(a, w.q0 + token, w.head + (r & ((1 << w.pack) - 1)), w.k0, w.limit(token));
            }
        }
    }
    fence_before();
    __syncthreads();
    fence_after();
    __syncwarp();
    if (warp == 8)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

bool tokens_before_heads(const mb200_heads& t, int tokens, int heads, int d) {
    return heads > 1 && tokens > 1 && t.token_stride < t.head_stride;
}
// [tokens][heads][d] in boxes of 64 elements of 128 rows: tokens of 1 << pack heads each
int encode(CUtensorMap* map, bool* tokens_inside, int dtype, const mb200_heads& t, int tokens, int heads, int d, int pack = 0) {
    const DriverApi& api = driver_api();
    if (!api.ok)
        return set_error(ST_RUNTIME, "cuTensorMapEncode* entry points not found in the driver");
    // (of one head, or token, any distance will do; the map wants whole units)
    const cuuint64_t row = (cuuint64_t)d * 2;
    const cuuint64_t head = heads == 1 ? row : (cuuint64_t)t.head_stride * 2;
    const cuuint64_t token = tokens == 1 ? head * heads : (cuuint64_t)t.token_stride * 2;
    const bool in = tokens_before_heads(t, tokens, heads, d);
    *tokens_inside = in;
    cuuint64_t dims[3] = {(cuuint64_t)d, (cuuint64_t)(in ? tokens : heads), (cuuint64_t)(in ? heads : tokens)};
    cuuint64_t strides[2] = {in ? token : head, in ? head : token};
    cuuint32_t box[3] = {64, in ? (cuuint32_t)kTile : 1u << pack, in ? 1u : (cuuint32_t)(kTile >> pack)}, estr[3] = {1, 1, 1};
    const CUresult r = api.tiled(
            map, dtype == MB200_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, t.p, dims,
            strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? ST_SUCCESS : set_error(ST_RUNTIME, "cuTensorMapEncodeTiled failed: %d", (int)r);
}

template <class T, int D>
int launch(const PromptMaps& maps, const PromptArgs& a, const TokensInside& inside, cudaStream_t st) {
    static KernelReady ready;
    if (!ready.smem(prompt_kernel<T, D>, Smem<D>::kBytes))
        return refused("attention_prompt", cudaGetLastError());
    const Writes writes{a.out.p, ((size_t)(a.tokens - 1) * a.out.token_stride + (size_t)(a.heads - 1) * a.out.head_stride +
                                  a.d) * 2};
    const unsigned ctas = (unsigned)attention_prompt_ctas(a.tokens, a.batch, a.heads, a.pack);
    const cudaError_t e = launch_pdl(writes, prompt_kernel<T, D>, dim3(ctas), dim3(kThreads), Smem<D>::kBytes, st, maps, a,
                                     inside);
    return e != cudaSuccess ? refused("attention_prompt", e) : check_launch("attention_prompt");
}

}  // namespace

// log2 of the heads that share a tile. (Queries whose heads lie further apart than tokens would come in another order.)
int attention_prompt_pack(const mb200_heads& q, int tokens, int heads, int kv_heads, int d) {
    int pack = 0;
    if (!tokens_before_heads(q, tokens, heads, d))
        while (pack < 6 && heads / kv_heads % (2 << pack) == 0)
            ++pack;
    return pack;
}
long long attention_prompt_ctas(int tokens, int batch, int heads, int pack) {
    return ((long long)tokens / (kRows >> pack) + batch) * (heads >> pack);
}

int launch_attention_prompt(const PromptArgs& a, int dtype, cudaStream_t st) {
    PromptMaps maps;
    TokensInside inside;
    int rc = encode(&maps.q, &inside.q, dtype, a.q, a.tokens, a.heads, a.d, a.pack);
    const int keys = a.key_tokens > 0 ? a.key_tokens : 1;  // (without keys nothing is loaded)
    if (!rc)
        rc = encode(&maps.k, &inside.k, dtype, a.k, keys, a.kv_heads, a.d);
    if (!rc)
        rc = encode(&maps.v, &inside.v, dtype, a.v, keys, a.kv_heads, a.d);
    if (rc)
        return rc;
    if (dtype == MB200_DTYPE_F16)
        return a.d <= 64 ? launch<__half, 64>(maps, a, inside, st) : launch<__half, 128>(maps, a, inside, st);
    return a.d <= 64 ? launch<__nv_bfloat16, 64>(maps, a, inside, st) : launch<__nv_bfloat16, 128>(maps, a, inside, st);
}

}  // namespace attn
}  // namespace mb200
