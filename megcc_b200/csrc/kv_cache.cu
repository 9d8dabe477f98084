// Keys and values of new tokens into the paged int8 cache, with the position rotation on the way, and cached ones
// back as 16-bit values.
//
// Rotation: pairs (x, y) of a head's first `rot` dimensions are turned by the position's angle,
//     x' = x cos - y sin,  y' = y cos + x sin,
// each product and sum rounded to 32 bits. The cosines and sines are tables of the caller's, since angles of far positions
// need more than 32 bits.
//
// Blocks: the 16 positions of a block and head share a scale, s = max(amax, 2^-119) / 127 of the new values there, or the
// block's scale of before where that is larger and the block keeps older positions. A value's whole number is the one
// nearest to the quotient x / s itself: activations of 16 bits have many quotients that lie within a rounding of the
// middle between two. Where the scale grows, older numbers are made anew, q' = q * (s_before / s) to the nearest; so the
// outcome depends on what was appended together, never on the order in which warps run. A block is one warp's: it
// alone reads and writes it. Keys are turned twice, for the largest of them and for their numbers: held in between they
// took the registers of half of the warps (8191 tokens of 32 + 8 + 8 heads of 128, with reading the blocks back: 94 us, 74 so).
//
// What bounds it: for a step of decoding the launch and the four loads that follow from one another (lengths, page, scale,
// whole numbers): 6 to 7 us with reading the blocks back. For prompts the instructions of the blocks' warps (8191 tokens:
// 2.3 a clock and SM, ALUs half taken, 3.2 TB/s; the floor is 37 us). Reading back is bound by memory (65001 rows of 8
// heads of 128: 71 to 76 us, 5.3 to 5.6 TB/s).
#include "kv_cache.cuh"
#include "umma_ptx.cuh"

namespace mb200 {
namespace attn {
namespace {

constexpr int kWarps = 4;
constexpr int kMostSteps = 8;  // steps of a warp over 16 rows: two rows a step at least (d <= 128)
constexpr int kQuerySteps = kTurnSteps;

// The part of a row that a lane holds: 8 elements from 8 * unit on; `rows` rows at a time, this lane's is `sub`
struct Lane {
    int per_row, rows, sub, unit;
    bool active;
    __device__ explicit Lane(int d) {
        const int lane = threadIdx.x & 31;
        per_row = d / 8;
        rows = 32 / per_row;
        sub = lane / per_row;
        unit = lane - sub * per_row;
        active = sub < rows;
    }
};

// Cosines and sines of the 8 elements that a lane holds (4 pairs of neighbours, or one of 8 pairs each)
struct Angles {
    float c[8], s[8];
};
template <bool VEC>
__device__ __forceinline__ void angles_of(const AppendArgs& a, const Lane& l, int position, Angles& g) {
    const int half = a.rot / 2;
    const int n = a.interleaved ? 4 : 8;
    const int first = a.interleaved ? l.unit * 4 : l.unit * 8 < half ? l.unit * 8 : l.unit * 8 - half;
    const long long at = (long long)position * half + first;
    if (VEC) {
        const float4 c = *(const float4*)(a.cosines + at), s = *(const float4*)(a.sines + at);
        g.c[0] = c.x, g.c[1] = c.y, g.c[2] = c.z, g.c[3] = c.w;
        g.s[0] = s.x, g.s[1] = s.y, g.s[2] = s.z, g.s[3] = s.w;
        if (n == 8) {
            const float4 d = *(const float4*)(a.cosines + at + 4), t = *(const float4*)(a.sines + at + 4);
            g.c[4] = d.x, g.c[5] = d.y, g.c[6] = d.z, g.c[7] = d.w;
            g.s[4] = t.x, g.s[5] = t.y, g.s[6] = t.z, g.s[7] = t.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) {
                g.c[i] = a.cosines[at + i];
                g.s[i] = a.sines[at + i];
            }
    }
}

// A lane's 8 elements as floats, turned where they are among the first `rot`. The whole warp calls it: the other
// half's elements come from the lane that holds them. `turns`: the lane has angles in g.
template <class T>
__device__ __forceinline__ void turned(const AppendArgs& a, const Lane& l, const uint4& raw, bool turns, const Angles& g,
                                       float (&x)[8]) {
    Vec<T>::unpack(raw, x);
    if (!a.cosines)
        return;
    if (a.interleaved) {
        if (turns) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float p = x[2 * i], q = x[2 * i + 1];
                x[2 * i] = __fsub_rn(__fmul_rn(p, g.c[i]), __fmul_rn(q, g.s[i]));
                x[2 * i + 1] = __fadd_rn(__fmul_rn(q, g.c[i]), __fmul_rn(p, g.s[i]));
            }
        }
        return;
    }
    const int units = a.rot / 16;
    const int lane = threadIdx.x & 31;
    const int other = turns ? (l.unit < units ? lane + units : lane - units) : lane;
    uint4 w;
    w.x = __shfl_sync(0xffffffffu, raw.x, other), w.y = __shfl_sync(0xffffffffu, raw.y, other);
    w.z = __shfl_sync(0xffffffffu, raw.z, other), w.w = __shfl_sync(0xffffffffu, raw.w, other);
    if (turns) {
        float y[8];
        Vec<T>::unpack(w, y);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            // (the first half's sines are negative here)
            x[i] = __fadd_rn(__fmul_rn(x[i], g.c[i]), __fmul_rn(y[i], g.s[i]));
        }
    }
}
// (a position beyond the tables has no angle: its elements become NaN)
template <bool VEC>
__device__ __forceinline__ bool take_angles(const AppendArgs& a, const Lane& l, bool valid, long long position, Angles& g) {
    const bool turns = valid && a.cosines && l.unit * 8 < a.rot;
    if (turns) {
        if (position < a.positions) {
            angles_of<VEC>(a, l, (int)position, g);
            if (!a.interleaved && l.unit * 16 < a.rot) {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    g.s[i] = -g.s[i];
            }
        } else {
            *(volatile int*)a.status = ERR_POSITION;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                g.c[i] = g.s[i] = __uint_as_float(0x7fffffffu);
        }
    }
    return turns;
}

// A token's queries, kQuerySteps steps of rows
template <class T, bool VEC>
__device__ __forceinline__ void turn_queries(const AppendArgs& a, const Lane& l, int token, int chunk) {
    int b = token, first = token;
    if (a.cu) {
        b = first_beyond(a.c.batch, token, [&](int i) { return a.cu[i + 1]; });
        if (b >= a.c.batch)
            return;
        first = a.cu[b];
    }
    const int before = a.lengths[b];
    if (before < 0 || first > token)
        return;
    uint4 raw[kQuerySteps];
    const int h0 = chunk * kQuerySteps * l.rows + l.sub;
    const long long in0 = token * a.q.token_stride + h0 * a.q.head_stride + l.unit * 8, in_step = l.rows * a.q.head_stride;
    const long long out0 = token * a.q_out.token_stride + h0 * a.q_out.head_stride + l.unit * 8,
                    out_step = l.rows * a.q_out.head_stride;
#pragma unroll
    for (int i = 0; i < kQuerySteps; ++i) {
        const int h = h0 + i * l.rows;
        raw[i] = make_uint4(0, 0, 0, 0);
        if (l.active && h < a.heads)
            raw[i] = load8<VEC>(a.q.p, in0 + i * in_step);
    }
    Angles g;
    const bool turns = take_angles<VEC>(a, l, l.active, (long long)before + (token - first), g);
#pragma unroll
    for (int i = 0; i < kQuerySteps; ++i) {
        const int h = h0 + i * l.rows;
        float x[8];
        turned<T>(a, l, raw[i], turns, g, x);
        if (l.active && h < a.heads)
            store8<VEC>(a.q_out.p, out0 + i * out_step, pack8<T>(x));
    }
}

__device__ __forceinline__ uint32_t pack4_low(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}
// The whole number nearest to x / s, ties to even, in the low byte: x * RN(1 / s) comes within one of it, and what is left of
// x, which one FMA gives exactly, says on which side
__device__ __forceinline__ uint32_t nearest_quotient(float x, float s, float half, float inv) {
    const float t = __fmaf_rn(x, inv, 12582912.f);
    const float left = __fmaf_rn(-__fsub_rn(t, 12582912.f), s, x);
    const float size = fabsf(left);
    const uint32_t q = __float_as_uint(t);
    const bool off = size > half || (size == half && (q & 1));
    return q + (off ? (left > 0.f ? 1u : 0xffffffffu) : 0u);
}

// The new keys (or values) of a block of a head
template <class T, bool VEC>
__device__ __forceinline__ void append_block(const AppendArgs& a, const Lane& l, int slot, int h, bool keys) {
    // The blocks that a sequence's new tokens touch have the slots from first / 16 + 2 b on: n tokens touch
    // at most (n + 30) / 16 blocks, and the next sequence's slots begin at least (n + 17) / 16 rounded up further on, which
    // is never less.
    int b = slot, j = 0, first = slot, n = 1;
    if (a.cu) {
        b = first_beyond(a.c.batch, slot, [&](int i) { return (long long)a.cu[i + 1] / kBlock + 2LL * (i + 1); });
        if (b >= a.c.batch)
            return;
        first = a.cu[b];
        if (first < 0 || first >= a.tokens)
            return;
        n = min(a.cu[b + 1], a.tokens) - first;
        j = slot - (first / kBlock + 2 * b);
    }
    const int before = a.lengths[b];
    if (before < 0)
        return;
    const long long from = (long long)(before / kBlock + j) * kBlock;
    const long long p0 = from > before ? from : before;
    const long long end = (long long)before + n;
    const long long p1 = from + kBlock < end ? from + kBlock : end;
    if (j < 0 || p0 >= p1)
        return;
    const int count = (int)(p1 - p0), kept = (int)(p0 - from);
    const int token = first + (int)(p0 - before);

    const mb200_heads& src = keys ? a.k : a.v;
    uint4 raw[kMostSteps];
#pragma unroll
    for (int i = 0; i < kMostSteps; ++i) {
        const int t = i * l.rows + l.sub;
        raw[i] = make_uint4(0, 0, 0, 0);
        if (l.active && t < count)
            raw[i] = load8<VEC>(src.p, (token + t) * src.token_stride + h * src.head_stride + l.unit * 8);
    }
    const int page = from <= 0x7fffffff ? page_of(a.c, b, (int)from) : -1;
    int8_t* whole = nullptr;
    float* scale = nullptr;
    uint32_t old_bits = 0;
    if (page >= 0) {
        const long long row = cache_row(a.c, page, h, (int)from);
        whole = (keys ? a.c.k : a.c.v) + row * a.c.d + l.unit * 8;
        scale = (keys ? a.c.k_scales : a.c.v_scales) + row / kBlock;
        if (kept)
            old_bits = __float_as_uint(*scale);
    } else {
        *(volatile int*)a.status = ERR_PAGE;
    }
    // a token's values, turned if they are keys
    auto values = [&](int i, float (&x)[8]) {
        const int t = i * l.rows + l.sub;
        if (keys) {
            Angles g;
            const bool turns = take_angles<VEC>(a, l, l.active && t < count, p0 + t, g);
            turned<T>(a, l, raw[i], turns, g, x);
        } else {
            Vec<T>::unpack(raw[i], x);
        }
        return l.active && t < count;
    };
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < kMostSteps; ++i) {
        if (i * l.rows >= count)  // (the same in all lanes)
            break;
        float x[8];
        if (values(i, x)) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                most = max(most, magnitude(x[e]));
            if (keys && a.k_out.p)
                store8<VEC>(a.k_out.p, (token + i * l.rows + l.sub) * a.k_out.token_stride + h * a.k_out.head_stride + l.unit * 8,
                            pack8<T>(x));
        }
    }
    if (page < 0)
        return;
    most = __reduce_max_sync(0xffffffffu, most);
    // (bits of non-negative numbers, infinity and the NaNs above: a block that holds one of those has a NaN for its scale)
    const uint32_t new_bits = most < 0x7f800000u
                                      ? __float_as_uint(__fdiv_rn(fmaxf(__uint_as_float(most), 0x1p-119f), 127.f))
                                      : 0x7fffffffu;
    const uint32_t bits = max(new_bits, old_bits);
    const float s = __uint_as_float(bits);
    const bool finite = bits < 0x7f800000u;
    const float inv = finite ? __frcp_rn(s) : 0.f, half = __fmul_rn(s, 0.5f);
    const uint32_t mask = finite ? 0xffffffffu : 0u;
#pragma unroll
    for (int i = 0; i < kMostSteps; ++i) {
        if (i * l.rows >= count)
            break;
        float x[8];
        if (values(i, x)) {
            uint32_t q[8];
            bool near = false;  // a quotient that may be on the other side of a middle, or on one
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float y = __fmaf_rn(x[e], inv, 12582912.f);
                near |= fabsf(__fmaf_rn(-__fsub_rn(y, 12582912.f), s, x[e])) >= half;
                q[e] = __float_as_uint(y);
            }
            if (near) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    q[e] = nearest_quotient(x[e], s, half, inv);
            }
            const uint2 w = make_uint2(pack4_low(q[0], q[1], q[2], q[3]) & mask, pack4_low(q[4], q[5], q[6], q[7]) & mask);
            *(uint2*)(whole + (long long)(kept + i * l.rows + l.sub) * a.c.d) = w;
        }
    }
    if (kept && bits != old_bits) {
        const double ratio = finite ? (double)__uint_as_float(old_bits) / (double)s : 0.0;
#pragma unroll 1
        for (int t = l.sub; t < kept; t += l.rows) {
            if (!l.active)
                break;
            uint2* p = (uint2*)(whole + (long long)t * a.c.d);
            const uint2 w = *p;
            uint32_t q[8];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                q[e] = (uint32_t)__double2int_rn((double)(int8_t)(w.x >> (8 * e)) * ratio);
                q[4 + e] = (uint32_t)__double2int_rn((double)(int8_t)(w.y >> (8 * e)) * ratio);
            }
            *p = make_uint2(pack4_low(q[0], q[1], q[2], q[3]), pack4_low(q[4], q[5], q[6], q[7]));
        }
    }
    if ((threadIdx.x & 31) == 0 && (!kept || bits != old_bits))
        *scale = s;
}

template <class T, bool VEC>
__global__ void __launch_bounds__(32 * kWarps, 5) append_kernel(const AppendArgs a) {
    const Lane l(a.c.d);
    pdl_start();
    const unsigned w = blockIdx.x * kWarps + (threadIdx.x >> 5);
    const unsigned blocks = 2u * (unsigned)a.slots * (unsigned)a.c.kv_heads;
    if (w < blocks) {
        const unsigned at = w >> 1;
        append_block<T, VEC>(a, l, (int)(at / a.c.kv_heads), (int)(at % a.c.kv_heads), (w & 1) == 0);
    } else if (a.q.p) {
        const unsigned i = w - blocks;
        const unsigned token = i / a.chunks;
        if (token < (unsigned)a.tokens)
            turn_queries<T, VEC>(a, l, (int)token, (int)(i - token * a.chunks));
    }
}

// ---- reading back ----
constexpr int kReadRows = 16, kReadThreads = 256;

// 16 whole numbers -> 16-bit values
template <class T>
__device__ __forceinline__ void values16(const uint4& w, float s, uint4& lo, uint4& hi) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
    uint32_t r[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
            y[e] = __fmul_rn((float)(int8_t)(u[i] >> (8 * e)), s);
        r[2 * i] = pack2<T>(y[0], y[1]);
        r[2 * i + 1] = pack2<T>(y[2], y[3]);
    }
    lo = make_uint4(r[0], r[1], r[2], r[3]);
    hi = make_uint4(r[4], r[5], r[6], r[7]);
}

// kReadRows packed rows of keys and values a CTA: a lane each finds where one lies, then a thread takes 16 whole numbers of
// both tensors at two places at a time, four loads on their way
template <class T, bool VEC>
__global__ void __launch_bounds__(kReadThreads) read_kernel(const ReadArgs a) {
    __shared__ long long where[kReadRows];  // row of head 0, or -1: in no sequence, or -2: in no page
    pdl_start();
    const int row0 = blockIdx.x * kReadRows;
    if (threadIdx.x < kReadRows) {
        const int row = row0 + threadIdx.x;
        long long at = -1;
        if (row < a.tokens) {
            int b = 0, end = a.c.batch;  // the first sequence that ends behind the row
            while (b < end) {
                const int m = (b + end) / 2;
                if (a.cu[m + 1] <= row)
                    b = m + 1;
                else
                    end = m;
            }
            if (b < a.c.batch) {
                const int first = a.cu[b], start = a.starts ? a.starts[b] : 0;
                if (first <= row) {
                    const long long p = (long long)start + (row - first);
                    const int page = p >= 0 && p <= 0x7fffffff ? page_of(a.c, b, (int)p) : -1;
                    at = page < 0 ? -2 : cache_row(a.c, page, 0, (int)p);
                    if (page < 0)
                        *(volatile int*)a.status = ERR_PAGE;
                }
            }
        }
        where[threadIdx.x] = at;
    }
    __syncthreads();
    const uint32_t units = a.c.d / 16, per_row = units * a.c.kv_heads, all = per_row * kReadRows;
    // (a quotient by n is one product for numbers x with x n < 2^32)
    const bool small = per_row < 16384;
    const uint32_t over_row = 0xffffffffu / per_row + 1, over_units = 0xffffffffu / units + 1;
    auto over = [&](uint32_t x, uint32_t n, uint32_t inverse) { return n == 1 ? x : small ? __umulhi(x, inverse) : x / n; };
#pragma unroll 1
    for (uint32_t first = threadIdx.x; first < all; first += 2 * kReadThreads) {
        uint4 w[4];
        float s[4];
        long long from[2];
        uint32_t r[2], h[2], u[2];
#pragma unroll
        for (int y = 0; y < 2; ++y) {
            const uint32_t x = first + y * kReadThreads;
            r[y] = over(x, per_row, over_row);
            const uint32_t rest = x - r[y] * per_row;
            h[y] = over(rest, units, over_units), u[y] = rest - h[y] * units;
            from[y] = x < all ? where[r[y]] : -1;
            const long long row = from[y] + (long long)h[y] * a.c.page_tokens;
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                w[2 * y + v] = make_uint4(0, 0, 0, 0);
                s[2 * y + v] = 0.f;
                if (from[y] >= 0) {
                    w[2 * y + v] = *(const uint4*)((v ? a.c.v : a.c.k) + row * a.c.d + u[y] * 16);
                    s[2 * y + v] = (v ? a.c.v_scales : a.c.k_scales)[row / kBlock];
                }
            }
        }
#pragma unroll
        for (int y = 0; y < 2; ++y) {
            if (from[y] == -1)
                continue;
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                uint4 lo, hi;
                values16<T>(w[2 * y + v], s[2 * y + v], lo, hi);
                const mb200_heads& dst = v ? a.v : a.k;
                const long long to = (long long)(row0 + (int)r[y]) * dst.token_stride + h[y] * dst.head_stride + u[y] * 16;
                store8<VEC>(dst.p, to, lo);
                store8<VEC>(dst.p, to + 8, hi);
            }
        }
    }
}

bool aligned(const mb200_heads& h) {
    return !h.p || (((uintptr_t)h.p & 15) == 0 && h.token_stride % 8 == 0 && h.head_stride % 8 == 0);
}
// (several tensors are written: whatever comes next waits for the end of the launch)
constexpr Writes kAnything{nullptr, SIZE_MAX};

}  // namespace

int launch_append(const AppendArgs& a, int dtype, cudaStream_t st) {
    const bool vec = aligned(a.k) && aligned(a.v) && aligned(a.q) && aligned(a.k_out) && aligned(a.q_out) &&
                     (((uintptr_t)a.cosines | (uintptr_t)a.sines) & 15) == 0;
    const long long warps = 2LL * a.slots * a.c.kv_heads + (a.q.p ? (long long)a.tokens * a.chunks : 0);
    const dim3 grid((unsigned)((warps + kWarps - 1) / kWarps)), block(32 * kWarps);
    auto kernel = dtype == MB200_DTYPE_F16 ? (vec ? append_kernel<__half, true> : append_kernel<__half, false>)
                                           : (vec ? append_kernel<__nv_bfloat16, true> : append_kernel<__nv_bfloat16, false>);
    const cudaError_t e = launch_pdl(kAnything, kernel, grid, block, 0, st, a);
    return e != cudaSuccess ? refused("kv_append_s8", e) : check_launch("kv_append_s8");
}

int launch_read(const ReadArgs& a, int dtype, cudaStream_t st) {
    const bool vec = aligned(a.k) && aligned(a.v);
    const dim3 grid((unsigned)((a.tokens - 1) / kReadRows + 1)), block(kReadThreads);
    auto kernel = dtype == MB200_DTYPE_F16 ? (vec ? read_kernel<__half, true> : read_kernel<__half, false>)
                                           : (vec ? read_kernel<__nv_bfloat16, true> : read_kernel<__nv_bfloat16, false>);
    const cudaError_t e = launch_pdl(kAnything, kernel, grid, block, 0, st, a);
    return e != cudaSuccess ? refused("kv_read_s8", e) : check_launch("kv_read_s8");
}

}  // namespace attn
}  // namespace mb200
