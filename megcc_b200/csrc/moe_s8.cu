// A mixture-of-experts layer for a few tokens, experts in int8: two kernels for up to four tokens, three for more,
// no exchange between CTAs but what one kernel writes and the next ones read (and a cluster's sums in the last).
//
//   p[t][e] = softmax(logits[t]) over all experts; token t goes to the top_k largest (ties: the lowest
//             index), with p as it is or divided by the sum of the chosen
//   z = (xq[t] . w1[e]) * s_x[t] * s_w1[e]      rows 0 .. f-1 of w1: gate g, rows f .. 2f-1: u
//   h = g / (1 + exp(-g)) * u, held as int8 in groups of 32 neighbours with one scale each
//   y[t] = sum over its experts of p * s_w2[e] * sum over groups of s_h * (hq . w2[e])
//
// Rows become whole numbers by the rule of scaled_s8.cuh. A scale per group of h instead of one per row
// lets the CTA that made 32 hidden units finish them: nothing has to wait for the maximum over all of f.
//
// HBM: the chosen experts' weights, 3 * d * f bytes each, are read once and everything else is small, so
// both kernels stream them through rings of asynchronous copies into mma.sync (stream_s8.cuh), over the ends of
// rows, experts and tiles.
// Up to four tokens every CTA of either kernel works the routing out for itself, a token per warp, while its other
// warps make the tokens whole numbers. More are routed and made whole numbers by a kernel in front, whose results both of
// the others read, the last one ahead of the end of the second. Two of 45 experts of 1920 x 800, by each CTA and by a
// kernel in front: 10 tokens 26.9 and 23.9 us, five 21.9 and 19.2, four 17.2 and 17.8, two 11.8 and 13.0.
#include "moe_s8.h"
#include "stream_s8.cuh"
#include "umma_ptx.cuh"

namespace mb200 {
namespace scaled {

namespace {

constexpr int kWarps = 8, kThreads = 32 * kWarps;
constexpr int kRouteWarps = 32;       // of the kernel in front
constexpr int kUnits = 32;            // hidden units per tile of the first kernel, and per group of h
constexpr int kPitch = 2 * kUnits + 4;  // ints per token in its exchange: 2 * 68 = 8 banks apart
constexpr int kRows = 16;             // rows of w2 per CTA of the second kernel
// dynamic shared memory that a CTA may ask for (227 KB less what the kernels declare themselves, 128 bytes)
constexpr int kMostDynamic = 227 * 1024 - 128;

// Where the tokens go, in shared memory: as large as the call's tokens and experts ask for.
struct Route {
    float* p;      // by slot = token * top + rank
    int* order;    // slots by expert, each with its token in the upper half
    // the passes: an expert and up to `cols` of its slots
    short *pass_expert, *pass_start, *pass_cols;
    int* passes;
    // while it is worked out (in memory that is used for something else afterwards)
    int* expert;       // by slot; -1: no share in the result
    uint32_t* tokens;  // by expert: a bit for each of its tokens
    int* at;           // by expert: where its slots begin
};
constexpr int kMostBuild = up16(4 * kMoeMaxTokens * kMoeMaxTop) + up16(8 * kMoeMaxExperts) + up16(4 * kMoeMaxExperts);
__device__ __forceinline__ Route place_route(uint8_t* at, uint8_t* build, int slots, int experts, int cols) {
    Route r;
    r.p = (float*)at;
    at += up16(4 * slots);
    r.order = (int*)at;
    at += up16(4 * slots);
    const int n = up16(2 * most_passes(slots, experts, cols));
    r.pass_expert = (short*)at;
    r.pass_start = (short*)(at + n);
    r.pass_cols = (short*)(at + 2 * n);
    r.passes = (int*)(at + 3 * n);
    r.expert = (int*)build;
    build += up16(4 * slots);
    r.tokens = (uint32_t*)build;
    r.at = (int*)(build + up16(8 * experts));
    return r;
}

// A float's bits in the order of the values: NaN lowest, then -infinity; 0 is nobody's
__device__ __forceinline__ uint32_t rank_key(float v) {
    const uint32_t b = __float_as_uint(__fadd_rn(v, 0.f));  // (-0 and 0 are the same)
    return v != v ? 1u : (b & 0x80000000u) ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ float key_value(uint32_t key) {
    return __uint_as_float((key & 0x80000000u) ? key & 0x7fffffffu : ~key);
}

// N tokens' experts, by a warp: lane j < top gets the j-th choice's index and p. The first 128 logits are kept in
// registers; of those behind them each choice is the largest that comes behind the one before it (smaller, or
// equal with a higher index). A choice waits for two reductions over the warp (145 ns): two tokens wait together.
struct Choice {
    int expert;
    float p;
};
template <int N>
struct Choices {
    Choice of[N];
};
template <int N>
__device__ __noinline__ Choices<N> choose_experts(
        const float* first, size_t to_next, int experts, int top, int renormalize) {
    constexpr int R = 4;
    const int lane = threadIdx.x & 31;
    const float inf = __uint_as_float(0x7f800000u);
    const float* row[N];
    uint32_t key[N][R];
    bool odd[N];    // a NaN or +infinity among the logits
    float sum[N];   // of all exponentials, where it is asked for
    float top_value[N], mine[N];
    uint32_t last[N];
    int last_e[N], mine_e[N];
#pragma unroll
    for (int n = 0; n < N; ++n) {
        row[n] = first + n * to_next;
        odd[n] = false;
        sum[n] = top_value[n] = mine[n] = 0.f;
        last[n] = ~0u;
        last_e[n] = mine_e[n] = -1;
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int e = i * 32 + lane;
            const float v = e < experts ? row[n][e] : -inf;
            key[n][i] = e < experts ? rank_key(v) : 0u;
            odd[n] |= !(v < inf);
        }
    }
#pragma unroll 1
    for (int j = 0; j < top; ++j) {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            uint32_t best = 0;
            int at = 0;
#pragma unroll
            for (int i = 0; i < R; ++i)
                if (key[n][i] > best) {
                    best = key[n][i];
                    at = i * 32 + lane;
                }
#pragma unroll 1
            for (int e = R * 32 + lane; e < experts; e += 32) {
                const uint32_t k = rank_key(row[n][e]);
                if (k > best && (k < last[n] || (k == last[n] && e > last_e[n]))) {
                    best = k;
                    at = e;
                }
            }
            last[n] = __reduce_max_sync(0xffffffffu, best);
            last_e[n] = (int)__reduce_min_sync(0xffffffffu, best == last[n] ? (uint32_t)at : ~0u);
        }
#pragma unroll
        for (int n = 0; n < N; ++n) {
            if (j == 0) {
                top_value[n] = key_value(last[n]);
                if (!renormalize) {
#pragma unroll
                    for (int i = 0; i < R; ++i)
                        sum[n] += key[n][i] != 0 ? expf(key_value(key[n][i]) - top_value[n]) : 0.f;
                }
            }
            if (lane == j) {
                mine[n] = key_value(last[n]);
                mine_e[n] = last_e[n];
            }
#pragma unroll
            for (int i = 0; i < R; ++i)
                if (i * 32 + lane == last_e[n])
                    key[n][i] = 0;
        }
    }
    Choices<N> c;
#pragma unroll
    for (int n = 0; n < N; ++n) {
        mine[n] = lane < top ? expf(mine[n] - top_value[n]) : 0.f;
#pragma unroll 1
        for (int e = R * 32 + lane; e < experts; e += 32) {
            odd[n] |= !(row[n][e] < inf);
            sum[n] += renormalize ? 0.f : expf(row[n][e] - top_value[n]);
        }
        if (renormalize)
            sum[n] = mine[n];
    }
#pragma unroll
    for (int s = 16; s; s >>= 1)
#pragma unroll
        for (int n = 0; n < N; ++n)
            sum[n] += __shfl_xor_sync(0xffffffffu, sum[n], s);
#pragma unroll
    for (int n = 0; n < N; ++n) {
        float p = __fdiv_rn(mine[n], sum[n]);
        if (top_value[n] == -inf)
            p = 0.f;  // every expert is masked: no share in any
        if (__any_sync(0xffffffffu, odd[n]))
            p = __uint_as_float(0x7fffffffu);
        c.of[n] = {lane >= top || p == 0.f ? -1 : mine_e[n], p};
    }
    return c;
}

// A warp for a token or two in turn (each a chain of 2 us or more); then the slots by expert, cut into passes of
// at most `cols`. Barriers of the CTA stand before and behind. Warps that have no token, with kMoeFew at most, call
// meanwhile().
template <int WARPS, class Meanwhile>
__device__ __forceinline__ void route_tokens(const MoeArgs& a, int cols, const Route& r, Meanwhile meanwhile) {
    constexpr int kThreads = 32 * WARPS;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (a.t > 1)
        for (int e = threadIdx.x; e < 2 * a.e; e += kThreads)
            r.tokens[e] = 0;
    // every WARPS-th token, two at a time while there are two
    constexpr int stride = WARPS;
    auto keep = [&](int t, const Choice& c) {
        if (lane < a.top) {
            r.p[t * a.top + lane] = c.p;
            if (a.t > 1)
                r.expert[t * a.top + lane] = c.expert;
        }
    };
    int t = warp;
    if constexpr (WARPS > kMoeFew * 2) {
#pragma unroll 1
        for (; t + stride < a.t; t += 2 * stride) {
            const Choices<2> c =
                    choose_experts<2>(a.logits + (size_t)t * a.e, (size_t)stride * a.e, a.e, a.top, a.renormalize);
            keep(t, c.of[0]);
            keep(t + stride, c.of[1]);
        }
    }
    if (t < a.t) {
        const Choice c = choose_experts<1>(a.logits + (size_t)t * a.e, 0, a.e, a.top, a.renormalize).of[0];
        keep(t, c);
        if (a.t == 1) {
            // one token: a pass for each of its experts, from the largest p down (any p that is 0 comes last)
            if (c.expert >= 0) {
                r.order[lane] = lane;
                r.pass_expert[lane] = (short)c.expert;
                r.pass_start[lane] = (short)lane;
                r.pass_cols[lane] = 1;
            }
            const uint32_t some = __ballot_sync(0xffffffffu, c.expert >= 0);
            if (lane == 0)
                *r.passes = __popc(some);
        }
    }
    if (a.t <= kMoeFew && warp >= kMoeFew)
        meanwhile();
    __syncthreads();
    if (a.t == 1)
        return;
    // A bit per expert and token: what an expert's slots are follows from them alone, whatever order they come in, so
    // every CTA cuts them into the same passes.
    const int slots = a.t * a.top;
#pragma unroll 1
    for (int s = threadIdx.x; s < slots; s += kThreads) {
        const int token = s / a.top, e = r.expert[s];
        if (e >= 0)
            atomicOr(r.tokens + 2 * e + (token >> 5), 1u << (token & 31));
    }
    __syncthreads();
    if (warp == 0) {
        int before = 0;  // slots in the lower half, passes in the upper one
#pragma unroll 1
        for (int e0 = 0; e0 < a.e; e0 += 32) {
            const int e = e0 + lane;
            const int n = e < a.e ? __popc(r.tokens[2 * e]) + __popc(r.tokens[2 * e + 1]) : 0;
            const int np = (n + cols - 1) / cols;
            int sum = np << 16 | n;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int other = __shfl_up_sync(0xffffffffu, sum, d);
                if (lane >= d)
                    sum += other;
            }
            const int from = before + sum - (np << 16 | n), start = from & 0xffff;
            if (e < a.e)
                r.at[e] = start;
#pragma unroll 1
            for (int i = 0; i < np; ++i) {
                const int to = (from >> 16) + i;
                r.pass_expert[to] = (short)e;
                r.pass_start[to] = (short)(start + i * cols);
                r.pass_cols[to] = (short)min(cols, n - i * cols);
            }
            before += __shfl_sync(0xffffffffu, sum, 31);
        }
        if (lane == 0)
            *r.passes = before >> 16;
    }
    __syncthreads();
#pragma unroll 1
    for (int s = threadIdx.x; s < slots; s += kThreads) {
        const int e = r.expert[s], token = s / a.top;
        if (e >= 0) {
            const uint32_t lower = (1u << (token & 31)) - 1u;
            const int rank_of = token < 32 ? __popc(r.tokens[2 * e] & lower)
                                           : __popc(r.tokens[2 * e]) + __popc(r.tokens[2 * e + 1] & lower);
            r.order[r.at[e] + rank_of] = token << 16 | s;
        }
    }
    __syncthreads();
}

// ---- more than four tokens: the routing, by the first CTA, and a token's whole numbers by each of the others ----
// What bounds it is the chain of choices, top_k times two reductions over a warp.
template <class T>
__global__ void __launch_bounds__(32 * kRouteWarps) moe_route_kernel(const MoeArgs a, int cols, int x_vectors) {
    extern __shared__ __align__(128) uint8_t dynamic[];
    pdl_start();
    if (blockIdx.x > 0) {
        const int t = (int)blockIdx.x - 1, pitch = xs_pitch(a.d);
        rows_to_whole<T, kRouteWarps>([&](int) { return (const T*)a.x + (long long)t * a.ldx; }, 1, a.d,
                                      a.xq + (size_t)t * pitch, pitch, a.sx + t, (uint32_t*)dynamic, x_vectors);
        return;
    }
    const int bytes = route_bytes(a.t * a.top, a.e, cols);
    const Route route = place_route(dynamic, dynamic + bytes, a.t * a.top, a.e, cols);
    route_tokens<kRouteWarps>(a, cols, route, [] {});
    for (int i = threadIdx.x; i < bytes / 16; i += 32 * kRouteWarps)
        a.route[i] = ((const uint4*)dynamic)[i];
}
// what the kernel in front has found
__device__ __forceinline__ void read_route(const MoeArgs& a, int cols, const Route& r) {
    const int units = route_bytes(a.t * a.top, a.e, cols) / 16;
    for (int i = threadIdx.x; i < units; i += kThreads)
        ((uint4*)r.p)[i] = a.route[i];
    __syncthreads();
}

// ---- gate, up, activation, and h as whole numbers ----
// Tiles of 32 hidden units (64 rows of w1), once per pass of their expert; a CTA takes neighbouring ones. Four
// of its eight warps have 16 rows each (gate, gate, up, up) and every other step of d, the other four the same rows
// and the remaining steps; each warp's ring runs on over the ends of tiles. COLS tokens at once; with no more
// tokens than that all of them stay in shared memory for the whole kernel. T: of the activations, up to four tokens;
// int8_t where they are whole numbers already.
template <int COLS, int DEPTH, bool ALIGNED>
struct Up {
    static constexpr int kDepth = DEPTH;
    static constexpr int kHalves = 2;  // warps that share a tile's steps
    typedef Rows<16, ALIGNED, (DEPTH > 3)> W;
    static constexpr int kRing = kWarps * kDepth * W::kBytes;
    static constexpr int kExchange = kHalves * COLS * kPitch;  // ints; two of them, used in turn
    static constexpr int smem(int t, int d, int top, int e) {
        return kRing + 2 * kExchange * 4 + (t < COLS ? t : COLS) * xs_pitch(d) + route_bytes(t * top, e, COLS);
    }
};
static_assert(Up<8, 3, false>::smem(8, kMoeMaxDepthFew, kMoeMaxTop, kMoeMaxExperts) <= kMostDynamic &&
                      Up<8, 4, false>::smem(kMoeMaxTokens, kMoeMaxDepth, kMoeMaxTop, kMoeMaxExperts) <= kMostDynamic &&
                      Up<16, 4, true>::smem(kMoeMaxTokens, kMoeMaxDepth, kMoeMaxTop, kMoeMaxExperts) <= kMostDynamic,
              "every layer that is accepted has room (sixteen columns of rows at odd places: few_columns)");

constexpr int kMostUpCtas = 1024;
constexpr int kMostTiles =
        most_passes(kMoeMaxTokens * kMoeMaxTop, kMoeMaxExperts, 8) * ((kMaxK + kUnits - 1) / kUnits);
static_assert((unsigned long long)kMostTiles * kMostUpCtas <= 0xffffffffull, "tiles are shared out in 32 bits");
// (the second kernel's: a pass's steps, over the warps of a cluster of eight)
static_assert((unsigned long long)kMostTiles * 8 * kWarps <= 0xffffffffull, "steps are shared out in 32 bits");

template <class T, int COLS, int DEPTH, int CTAS, bool ALIGNED>
__global__ void __launch_bounds__(kThreads, CTAS) moe_up_kernel(const MoeArgs a, int x_vectors) {
    typedef Up<COLS, DEPTH, ALIGNED> U;
    constexpr int NT = COLS / 8, kDepth = U::kDepth;
    extern __shared__ __align__(128) uint8_t dynamic[];
    int* exchange = (int*)(dynamic + U::kRing);
    int8_t* xs = (int8_t*)(exchange + 2 * U::kExchange);
    const int pitch = xs_pitch(a.d);
    const Route route = place_route((uint8_t*)xs + min(a.t, COLS) * pitch, dynamic, a.t * a.top, a.e, COLS);
    static_assert(U::kRing >= kMostBuild, "the routing is worked out where the rings will be");
    __shared__ float x_scale[COLS];
    constexpr bool kFew = sizeof(T) > 1;
    __shared__ uint32_t part[kFew ? kMoeFew * (kWarps - kMoeFew) : 1];

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, tig = lane & 3;
    const bool resident = kFew || a.t <= COLS;
    pdl_start();
    if constexpr (kFew) {
        // (the logits are on their way when the routing begins)
        ask_ahead<kThreads>(a.logits, a.t * a.e * 4);
        route_tokens<kWarps>(a, COLS, route, [&] {
            rows_to_whole<T, kWarps - kMoeFew, kMoeFew>([&](int t) { return (const T*)a.x + (long long)t * a.ldx; }, a.t,
                                                        a.d, xs, pitch, x_scale, part, x_vectors);
        });
    } else {
        read_route(a, COLS, route);
    }
    const int blocks = (a.f + kUnits - 1) / kUnits;
    // (kMostTiles in kMostUpCtas CTAs at most: products that 32 bits hold)
    const unsigned tiles = (unsigned)(*route.passes * blocks);
    // as few CTAs as still take as many tiles each as the busiest would
    const unsigned each = (tiles + gridDim.x - 1) / gridDim.x, busy = each ? (tiles + each - 1) / each : 1u;
    if (blockIdx.x >= busy || tiles == 0)
        return;
    const int first = (int)(tiles * blockIdx.x / busy), last = (int)(tiles * (blockIdx.x + 1) / busy);
    const int steps = (a.d + kStep - 1) / kStep;
    const int half = warp >> 2;                        // steps half, half + 2, ...
    const int mine = (steps - half + 1) / U::kHalves;  // (none where there is one step only)
    const uint32_t ring = shared_address(dynamic) + (uint32_t)(warp * kDepth * U::W::kBytes);

    // row r of this warp's 16 in a tile: block of 32 units `b` of a pass
    const int block = warp & 3;
    auto tile_row = [&](int pass, int b, int r) {
        const int u = min(b * kUnits + (block & 1) * 16 + r, a.f - 1);
        return a.w1 + ((size_t)route.pass_expert[pass] * 2 * a.f + (block >> 1) * (size_t)a.f + u) * (size_t)a.d;
    };
    typename U::W w;
    int l_tile = first, l_pass = first / blocks, l_block = first - l_pass * blocks, l_step = 0;
    uint32_t stage_in = ring, stage_out = ring;
    auto copy_next = [&] {
        if (mine && l_tile < last) {
            if (l_step == 0)
                w.open([&](int r) { return tile_row(l_pass, l_block, r); }, a.d, half);
            w.template copy<true>(stage_in, U::kHalves, a.d - (half + l_step * U::kHalves) * kStep >= U::W::kWhole);
            if (++l_step == mine) {
                l_step = 0;
                ++l_tile;
                if (++l_block == blocks) {
                    l_block = 0;
                    ++l_pass;
                }
            }
        }
        next_stage<kDepth, U::W::kBytes>(stage_in, ring);
        copy_commit();
    };
    // tokens of a pass that are whole numbers already (all tokens, where they stay), a warp per row
    auto each_token = [&](int p, auto copy) {
        const int rows = resident ? a.t : route.pass_cols[p];
#pragma unroll 1
        for (int c = warp; c < rows; c += kWarps) {
            const int t = resident ? c : route.order[route.pass_start[p] + c] >> 16;
            copy((uint4*)(xs + c * pitch), (const uint4*)(a.xq + (size_t)t * pitch), x_scale + c, a.sx + t);
        }
    };
    if constexpr (!kFew) {
        // (the first ones ahead of the weights)
        each_token(first / blocks, [&](uint4* to, const uint4* from, float* to_scale, const float* scale) {
            const uint32_t at = shared_address(to);
#pragma unroll 4
            for (int i = lane; i < pitch / 16; i += 32)
                copy_async16(at + 16 * i, from + i);
            if (lane == 0)
                copy_async4(shared_address(to_scale), scale);
        });
        copy_commit();
    }
#pragma unroll 1
    for (int i = 0; i < kDepth - 1; ++i)
        copy_next();

    int pass = first / blocks, b = first - pass * blocks, cols = 0, e = 0;
    const int* order = nullptr;
#pragma unroll 1
    for (int tile = first; tile < last; ++tile) {
        const int u0 = b * kUnits;
        if (b == 0 || tile == first) {
            e = route.pass_expert[pass];
            cols = route.pass_cols[pass];
            order = route.order + route.pass_start[pass];
            if constexpr (!kFew) {
                if (tile == first) {
                    copy_wait<kDepth - 1>();
                    __syncthreads();
                } else if (!resident) {
                    __syncthreads();  // (all warps are done with the last pass's tokens)
                    each_token(pass, [&](uint4* to, const uint4* from, float* to_scale, const float* scale) {
#pragma unroll 8
                        for (int i = lane; i < pitch / 16; i += 32)
                            to[i] = from[i];
                        if (lane == 0)
                            *to_scale = *scale;
                    });
                    __syncthreads();
                }
            }
        }
        // scales of the unit that this lane will finish
        const int u = u0 + lane;
        const float* s1 = a.s1 + (size_t)e * 2 * a.f + min(u, a.f - 1);
        const float s_gate = s1[0], s_up = s1[a.f];
        const int8_t* frag[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int c = min(8 * nt + g, cols - 1);
            frag[nt] = xs + (resident ? order[c] >> 16 : c) * pitch + tig * 16;
        }
        const int s_lo = (int)((uintptr_t)tile_row(pass, b, g) & 15);
        const int s_hi = (int)((uintptr_t)tile_row(pass, b, g + 8) & 15);
        int acc[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
            acc[nt][0] = acc[nt][1] = acc[nt][2] = acc[nt][3] = 0;
#pragma unroll 1
        for (int i = 0; i < mine; ++i) {
            copy_wait<kDepth - 2>();
            __syncwarp();  // all lanes' copies of this step are there, and the last step's stage has been read
            copy_next();
            const uint32_t stage = stage_out;
            next_stage<kDepth, U::W::kBytes>(stage_out, ring);
#pragma unroll
            for (int j = 0; j < kStep / 64; ++j) {
                const uint4 lo = U::W::piece16(stage, g, 4 * j + tig, s_lo);
                const uint4 hi = U::W::piece16(stage, g + 8, 4 * j + tig, s_hi);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
                    mma_64(acc[nt], lo, hi, *(const uint4*)(frag[nt] + (half + i * U::kHalves) * kStep + 64 * j));
            }
        }
        int* red = exchange + (tile & 1) * U::kExchange;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            int* at = red + (half * COLS + 8 * nt + 2 * tig) * kPitch + block * 16 + g;
            at[0] = acc[nt][0];
            at[kPitch] = acc[nt][1];
            at[8] = acc[nt][2];
            at[kPitch + 8] = acc[nt][3];
        }
        __syncthreads();  // (the other exchange's readers are past their reading when this one is passed again)
#pragma unroll 1
        for (int c = warp; c < cols; c += kWarps) {
            int gate = 0, up = 0;
#pragma unroll
            for (int i = 0; i < U::kHalves; ++i) {
                gate += red[(i * COLS + c) * kPitch + lane];
                up += red[(i * COLS + c) * kPitch + kUnits + lane];
            }
            const int slot = order[c] & 0xffff;
            const float sx = x_scale[resident ? order[c] >> 16 : c];
            const float zg = scale_acc(gate, sx, s_gate), zu = scale_acc(up, sx, s_up);
            const float h = u < a.f ? __fmul_rn(__fdiv_rn(zg, __fadd_rn(1.f, expf(-zg))), zu) : 0.f;
            const RowScale r = row_scale(__reduce_max_sync(0xffffffffu, magnitude(h)));
            a.hq[(size_t)slot * (blocks * kUnits) + u] = (int8_t)(to_whole(h, r.inv) & r.keep);
            if (lane == 0)
                a.sh[(size_t)slot * blocks + b] = r.scale;
        }
        if (++b == blocks) {
            b = 0;
            ++pass;
        }
    }
}

// ---- down, and the experts' sum ----
// A CTA, or a cluster of CTAs, makes 16 rows of every token. All its steps, pass after pass in the order of the
// experts' indices, are one sequence, of which each warp takes an equal run; it adds into sums of its own, which meet
// at the end in the order of the warps: no float atomics, the same bits every time. (Neighbouring steps for each warp:
// with every eighth step each warp would open every pass.) Clusters: where d has fewer tiles than the GPU has SMs.
template <int NT, int DEPTH, bool ALIGNED>
struct Down {
    static constexpr int kDepth = DEPTH;
    typedef Rows<kRows, ALIGNED> W;
    typedef Rows<8 * NT, true> H;
    static constexpr int kGroups = kStep / kUnits;
    static constexpr int kScales = kGroups * 8 * NT * 4;
    static constexpr int kStage = W::kBytes + H::kBytes + kScales;
    static constexpr int kRing = kWarps * kDepth * kStage;
    static constexpr int smem(int t, int top, int e) {
        return kRing + kWarps * t * kRows * 4 + route_bytes(t * top, e, 8 * NT);
    }
};
static_assert(Down<1, 3, false>::smem(kMoeMaxTokens, kMoeMaxTop, kMoeMaxExperts) <= kMostDynamic &&
                      Down<2, 3, false>::smem(kMoeMaxTokens, kMoeMaxTop, kMoeMaxExperts) <= kMostDynamic,
              "every layer that is accepted has room");

template <int NT, int DEPTH, int CTAS, bool ALIGNED>
__global__ void __launch_bounds__(kThreads, CTAS) moe_down_kernel(const MoeArgs a, int cluster) {
    typedef Down<NT, DEPTH, ALIGNED> D;
    constexpr int kDepth = D::kDepth, kCols = 8 * NT;
    extern __shared__ __align__(128) uint8_t dynamic[];
    float* sums = (float*)(dynamic + D::kRing);  // [kWarps][a.t][kRows]
    const Route route = place_route((uint8_t*)(sums + kWarps * a.t * kRows), dynamic, a.t * a.top, a.e, kCols);
    static_assert(D::kRing >= kMostBuild, "the routing is worked out where the rings will be");

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, tig = lane & 3;
    const int rank = cluster > 1 ? (int)umma::cluster_rank() : 0;
    const int d0 = (int)blockIdx.x / cluster * kRows;
    // Ahead of the end of the kernel in front: the routing, and with it the first weights. What is read here
    // was written before that kernel began its work, which let this one start behind its own wait for it.
    if (a.t <= kMoeFew)
        route_tokens<kWarps>(a, kCols, route, [] {});
    else
        read_route(a, kCols, route);
    const int groups = (a.f + kUnits - 1) / kUnits, width = groups * kUnits;
    const int steps = (a.f + kStep - 1) / kStep;  // of a pass
    const int total = steps * *route.passes;
    const unsigned runs = (unsigned)(cluster * kWarps), run = (unsigned)(rank * kWarps + warp);
    const int first = (int)((unsigned)total * run / runs), mine = (int)((unsigned)total * (run + 1) / runs) - first;
    float* own = sums + warp * a.t * kRows;
    for (int i = lane; i < a.t * kRows; i += 32)
        own[i] = 0.f;
    const uint32_t ring = shared_address(dynamic) + (uint32_t)(warp * kDepth * D::kStage);

    // A place in the sequence of this warp's steps
    struct At {
        int pass, step;
    };
    auto advance = [&](At& at) {  // is it a pass's first step?
        if (++at.step < steps)
            return false;
        at.step = 0;
        ++at.pass;
        return true;
    };
    const At start = {first / steps, first % steps};
    auto w2_row = [&](int pass, int r) {
        return a.w2 + ((size_t)route.pass_expert[pass] * a.d + min(d0 + r, a.d - 1)) * (size_t)a.f;
    };
    typename D::W w;
    typename D::H h;
    const float* sh_from = nullptr;
    At wl = start, hl = start;
    int w_copied = 0, h_copied = 0;
    bool w_new = true, h_new = true;
    auto copy_weights = [&](uint32_t stage) {
        if (w_copied < mine) {
            if (w_new)
                w.open([&](int r) { return w2_row(wl.pass, r); }, a.f, wl.step);
            w.template copy<true>(stage, 1, a.f - wl.step * kStep >= D::W::kWhole);
            w_new = advance(wl);
        }
        ++w_copied;
    };
    auto copy_hidden = [&](uint32_t stage) {
        if (h_copied < mine) {
            if (h_new) {
                const int* order = route.order + route.pass_start[hl.pass];
                const int cols = route.pass_cols[hl.pass];
                h.open([&](int r) { return r < cols ? a.hq + (size_t)(order[r] & 0xffff) * width : nullptr; }, width,
                       hl.step);
                // a lane copies the scales of a token's groups lane / kCols, and so on
                sh_from = a.sh + (size_t)(order[min(lane % kCols, cols - 1)] & 0xffff) * groups + lane / kCols;
            }
            // (of tokens that are not there: nothing)
            const bool whole = width - hl.step * kStep >= kStep;
            const uint32_t hidden = stage + D::W::kBytes, scales = hidden + D::H::kBytes + 4 * lane;
            h.template copy<false>(hidden, 1, whole);
            const float* from = sh_from + hl.step * D::kGroups;
#pragma unroll
            for (int j = 0; j < D::kGroups; j += 32 / kCols) {
                if (whole) {
                    copy_async4(scales + 4 * kCols * j, from + j);
                } else {
                    const bool some = hl.step * D::kGroups + j + lane / kCols < groups;
                    copy_async4(scales + 4 * kCols * j, some ? from + j : a.sh, some);
                }
            }
            h_new = advance(hl);
        }
        ++h_copied;
        copy_commit();
    };
#pragma unroll 1
    for (int i = 0; i < kDepth - 1; ++i)
        copy_weights(ring + (uint32_t)(i * D::kStage));
    pdl_start();
#pragma unroll 1
    for (int i = 0; i < kDepth - 1; ++i)
        copy_hidden(ring + (uint32_t)(i * D::kStage));
    uint32_t stage = ring, free_stage = ring + (uint32_t)((kDepth - 1) * D::kStage);

    At at = start;
    float acc[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
        acc[nt][0] = acc[nt][1] = acc[nt][2] = acc[nt][3] = 0.f;
    float s_lo = 0.f, s_hi = 0.f;
    int sh_lo = 0, sh_hi = 0;
    bool fresh = true;
#pragma unroll 1
    for (int i = 0; i < mine; ++i) {
        copy_wait<kDepth - 2>();
        __syncwarp();  // all lanes' copies of this step are there, and the last step's stage has been read
        copy_weights(free_stage);
        copy_hidden(free_stage);
        next_stage<kDepth, D::kStage>(free_stage, ring);
        if (fresh) {
            const float* s2 = a.s2 + (size_t)route.pass_expert[at.pass] * a.d;
            s_lo = s2[min(d0 + g, a.d - 1)];
            s_hi = s2[min(d0 + g + 8, a.d - 1)];
            sh_lo = (int)((uintptr_t)w2_row(at.pass, g) & 15);
            sh_hi = (int)((uintptr_t)w2_row(at.pass, g + 8) & 15);
        }
        const uint32_t hidden = stage + D::W::kBytes;
#pragma unroll
        for (int j = 0; j < D::kGroups; ++j) {
            const uint2 lo = D::W::piece8(stage, g, 4 * j + tig, sh_lo);
            const uint2 hi = D::W::piece8(stage, g + 8, 4 * j + tig, sh_hi);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const uint2 q = D::H::piece8(hidden, 8 * nt + g, 4 * j + tig, 0);
                int c[4] = {0, 0, 0, 0};
                mma_16x8x32(c, lo.x, hi.x, lo.y, hi.y, q.x, q.y);
                const uint2 s = lds8(hidden + D::H::kBytes + (j * kCols + 8 * nt + 2 * tig) * 4);
                const float s0 = __uint_as_float(s.x), s1 = __uint_as_float(s.y);
                acc[nt][0] = __fmaf_rn(__int2float_rn(c[0]), s0, acc[nt][0]);
                acc[nt][1] = __fmaf_rn(__int2float_rn(c[1]), s1, acc[nt][1]);
                acc[nt][2] = __fmaf_rn(__int2float_rn(c[2]), s0, acc[nt][2]);
                acc[nt][3] = __fmaf_rn(__int2float_rn(c[3]), s1, acc[nt][3]);
            }
        }
        next_stage<kDepth, D::kStage>(stage, ring);
        const int pass = at.pass;
        fresh = advance(at);
        if (fresh || i + 1 == mine) {
            // this warp's share of the pass, to the sums of its tokens
            const int* order = route.order + route.pass_start[pass];
            const int cols = route.pass_cols[pass];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int c = 8 * nt + 2 * tig + j;
                    if (c < cols) {
                        const float p = route.p[order[c] & 0xffff];
                        float* to = own + (order[c] >> 16) * kRows + g;
                        to[0] = __fmaf_rn(__fmul_rn(acc[nt][j], s_lo), p, to[0]);
                        to[8] = __fmaf_rn(__fmul_rn(acc[nt][2 + j], s_hi), p, to[8]);
                    }
                }
                acc[nt][0] = acc[nt][1] = acc[nt][2] = acc[nt][3] = 0.f;
            }
            __syncwarp();  // the next pass's lanes find them
        }
    }
    __syncthreads();
    auto store = [&](int i, float v) {
        const int t = i / kRows, d = d0 + i % kRows;
        if (d < a.d)
            store_as(a.y, a.dtype, (size_t)t * (size_t)a.ldy + d, v);
    };
#pragma unroll 1
    for (int i = threadIdx.x; i < a.t * kRows; i += kThreads) {
        float v = 0.f;
#pragma unroll
        for (int s = 0; s < kWarps; ++s)
            v += sums[s * a.t * kRows + i];
        if (cluster == 1)
            store(i, v);
        else
            sums[i] = v;  // (what this thread alone has read)
    }
    if (cluster > 1) {
        // each CTA finishes its share of the tokens' rows
        __syncwarp();
        umma::cluster_arrive();
        umma::cluster_wait();
        const uint32_t base = shared_address(sums);
#pragma unroll 1
        for (int i = (rank * kThreads + (int)threadIdx.x) * 4; i < a.t * kRows; i += cluster * kThreads * 4) {
            float v[4] = {0.f, 0.f, 0.f, 0.f};
            for (int c = 0; c < cluster; ++c) {
                const uint4 w = umma::ld_cluster_v4(base + 4u * (uint32_t)i, c);
                v[0] += __uint_as_float(w.x);
                v[1] += __uint_as_float(w.y);
                v[2] += __uint_as_float(w.z);
                v[3] += __uint_as_float(w.w);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j)
                store(i + j, v[j]);
        }
        __syncwarp();
        umma::cluster_arrive();
        umma::cluster_wait();  // the others may still read this CTA's sums
    }
}

// Passes of eight tokens or of sixteen: eight unless an expert has more than that on average (weights that are read
// twice come from the L2 the second time, and passes of sixteen leave room for one CTA per SM only). 64 tokens, eight of
// 64 experts of 2048 x 768: by eight 75 us, by sixteen 90; six of 24 of 1928 x 808: 82 and 68. And eight where sixteen rows
// of tokens leave no room for the rings of weights at odd places and the routing (62 to 64 tokens, 16 of 81 to 127 experts,
// d > 8064). All kernels of a call go by this.
bool first_aligned(const MoeArgs& a) {
    return ((uintptr_t)a.w1 & 15) == 0 && a.d % 16 == 0;
}
bool few_columns(const MoeArgs& a) {
    return a.t <= 8 || a.t * a.top <= 8 * a.e ||
           (!first_aligned(a) && Up<16, 4, false>::smem(a.t, a.d, a.top, a.e) > kMostDynamic);
}

template <class T>
cudaError_t launch_route(const MoeArgs& a, cudaStream_t st) {
    static MostShared shared;
    auto kernel = moe_route_kernel<T>;
    shared.ask(kernel);
    const int cols = few_columns(a) ? 8 : 16;
    const int x_vectors = ((uintptr_t)a.x & 15) == 0 && a.ldx % Vec<T>::N == 0;
    static_assert(kMostBuild >= 4 * kRouteWarps, "a row's maxima lie there");
    return launch_pdl(Writes{a.hq, a.workspace_bytes}, kernel, dim3((unsigned)a.t + 1), dim3(32 * kRouteWarps),
                      (size_t)(route_bytes(a.t * a.top, a.e, cols) + kMostBuild), st, a, cols, x_vectors);
}

template <class T, int COLS, int DEPTH, int CTAS, bool ALIGNED>
cudaError_t launch_up_as(const MoeArgs& a, cudaStream_t st) {
    static umma::KernelReady ready;
    static MostShared shared;
    static umma::ResidentCtas resident;
    auto kernel = moe_up_kernel<T, COLS, DEPTH, CTAS, ALIGNED>;
    const int smem = Up<COLS, DEPTH, ALIGNED>::smem(a.t, a.d, a.top, a.e);
    if (!ready.smem(kernel, smem))
        return why_refused();
    shared.ask(kernel);
    const int x_vectors = ((uintptr_t)a.x & 15) == 0 && (a.t == 1 || a.ldx * sizeof(T) % 16 == 0);
    const long long tiles = (long long)a.t * a.top * ((a.f + kUnits - 1) / kUnits);  // at most
    const Writes writes{a.hq, a.workspace_bytes};
    const long long fit = (long long)umma::sm_count() * resident.per_sm(kernel, kThreads, smem, 0);
    const long long most = fit <= 0 ? 512 : fit < kMostUpCtas ? fit : kMostUpCtas;
    const long long ctas = tiles < most ? tiles : most;
    return launch_pdl(writes, kernel, dim3((unsigned)ctas), dim3(kThreads), (size_t)smem, st, a, x_vectors);
}
template <class T>
cudaError_t launch_up(const MoeArgs& a, cudaStream_t st) {
    const bool aligned = first_aligned(a);
    if (a.t <= kMoeFew)
        return aligned ? launch_up_as<T, 8, 3, 3, true>(a, st) : launch_up_as<T, 8, 3, 3, false>(a, st);
    const cudaError_t e = launch_route<T>(a, st);
    if (e != cudaSuccess)
        return e;
    if (a.t <= 8)
        return aligned ? launch_up_as<int8_t, 8, 3, 3, true>(a, st) : launch_up_as<int8_t, 8, 3, 3, false>(a, st);
    if (few_columns(a))
        return aligned ? launch_up_as<int8_t, 8, 4, 2, true>(a, st) : launch_up_as<int8_t, 8, 4, 2, false>(a, st);
    return aligned ? launch_up_as<int8_t, 16, 4, 2, true>(a, st) : launch_up_as<int8_t, 16, 4, 2, false>(a, st);
}

template <int NT, int DEPTH, int CTAS, bool ALIGNED>
cudaError_t launch_down_as(const MoeArgs& a, cudaStream_t st) {
    static umma::KernelReady ready;
    static umma::ResidentCtas resident;
    static MostShared shared;
    auto kernel = moe_down_kernel<NT, DEPTH, CTAS, ALIGNED>;
    const int smem = Down<NT, DEPTH, ALIGNED>::smem(a.t, a.top, a.e);
    if (!ready.smem(kernel, smem))
        return why_refused();
    shared.ask(kernel);
    const Writes writes{a.y, ((size_t)(a.t - 1) * (size_t)a.ldy + (size_t)a.d) * dtype_bytes(a.dtype)};
    // a CTA for every SM where each warp still has two steps (experts with tokens: at most as many as slots), and all at
    // once (64 tokens, two of 8 experts of 2048 x 1024: 31 us, 37 with 256 CTAs for 148 places)
    const int tiles = (a.d - 1) / kRows + 1, slots = a.t * a.top;
    const long long steps = (long long)(slots < a.e ? slots : a.e) * ((a.f + kStep - 1) / kStep);
    const int fit = umma::sm_count() * resident.per_sm(kernel, kThreads, smem, 0);
    int cluster = 1;
    while (cluster < 8 && tiles * cluster < umma::sm_count() && 2 * tiles * cluster <= fit && steps >= 2LL * 2 * cluster * kWarps)
        cluster *= 2;
    return launch_pdl_cluster(writes, kernel, dim3((unsigned)(tiles * cluster)), dim3(kThreads), (size_t)smem, cluster,
                              st, a, cluster);
}
cudaError_t launch_down(const MoeArgs& a, cudaStream_t st) {
    const bool aligned = ((uintptr_t)a.w2 & 15) == 0 && a.f % 16 == 0;
    // (as deep a ring as leaves room for two CTAs per SM beside their tokens' sums)
    if (a.t <= 8)
        return aligned ? launch_down_as<1, 3, 3, true>(a, st) : launch_down_as<1, 3, 3, false>(a, st);
    if (few_columns(a))
        return aligned ? launch_down_as<1, 3, 2, true>(a, st) : launch_down_as<1, 3, 2, false>(a, st);
    return aligned ? launch_down_as<2, 3, 2, true>(a, st) : launch_down_as<2, 3, 2, false>(a, st);
}

template <class T>
cudaError_t launch_both(const MoeArgs& a, cudaStream_t st) {
    const cudaError_t e = launch_up<T>(a, st);
    return e != cudaSuccess ? e : launch_down(a, st);
}

}  // namespace

int launch_moe(const MoeArgs& a, cudaStream_t st) {
    const cudaError_t e = a.dtype == DT_F32   ? launch_both<float>(a, st)
                          : a.dtype == DT_F16 ? launch_both<__half>(a, st)
                                              : launch_both<__nv_bfloat16>(a, st);
    if (e != cudaSuccess)
        return refused("moe_s8", e);
    return check_launch("moe_s8");
}

}  // namespace scaled
}  // namespace mb200
