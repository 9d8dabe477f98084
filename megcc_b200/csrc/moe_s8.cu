// A mixture-of-experts layer for a few tokens, experts in int8: two kernels, no exchange between CTAs
// but what the first one writes and the second one reads.
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
// both kernels are mma.sync loops that take weights straight from global memory into registers, 16 (8)
// neighbouring bytes per thread, with loads running ahead over the ends of rows, experts and tiles.
// Every CTA of either kernel works the routing out for itself: it is a few thousand logits.
#include "moe_s8.h"
#include "scaled_s8.cuh"
#include "umma_ptx.cuh"

namespace mb200 {
namespace scaled {

namespace {

constexpr int kWarps = 8, kThreads = 32 * kWarps;
constexpr int kMaxSlots = kMoeMaxTokens * kMoeMaxTop;
constexpr int kUnits = 32;            // hidden units per tile of the first kernel, and per group of h
constexpr int kPitch = 2 * kUnits + 4;  // ints per token in its exchange: 2 * 68 = 8 banks apart
constexpr int kRows = 16;             // rows of w2 per CTA of the second kernel

struct Route {
    float p[kMaxSlots];        // by slot = token * top + rank
    short expert[kMaxSlots];   // -1: no share in the result
    short order[kMaxSlots];    // slots by expert
    short count[kMoeMaxExperts], start[kMoeMaxExperts];
    // the passes: an expert and up to `cols` of its slots
    short pass_expert[kMoeMaxPasses], pass_start[kMoeMaxPasses], pass_cols[kMoeMaxPasses];
    int passes;
};

// A float's bits in the order of the values: NaN lowest, then -infinity; 0 is nobody's
__device__ __forceinline__ uint32_t rank_key(float v) {
    const uint32_t b = __float_as_uint(__fadd_rn(v, 0.f));  // (-0 and 0 are the same)
    return v != v ? 1u : (b & 0x80000000u) ? ~b : b | 0x80000000u;
}

// A warp per token in turn; then the slots by expert, cut into passes of at most `cols`.
__device__ void route_tokens(const MoeArgs& a, int cols, Route& r) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int e = threadIdx.x; e < a.e; e += kThreads)
        r.count[e] = 0;
    if (threadIdx.x == 0)
        r.passes = 0;
    constexpr int R = kMoeMaxExperts / 32;
    for (int t = warp; t < a.t; t += kWarps) {
        const float* row = a.logits + (size_t)t * a.e;
        uint32_t key[R];
        float top_value = 0.f, sum = 0.f;
        uint32_t odd = 0;  // a NaN or +infinity among the logits
#pragma unroll
        for (int i = 0; i < R; ++i) {
            key[i] = 0;
            if (i * 32 < a.e) {
                const int e = i * 32 + lane;
                if (e < a.e) {
                    const float v = row[e];
                    key[i] = rank_key(v);
                    odd |= !(v < __uint_as_float(0x7f800000u));
                }
            }
        }
        odd = __any_sync(0xffffffffu, odd);
        float chosen = 0.f;  // the sum of the chosen ones' exponentials
        float mine = 0.f;    // lane j: the j-th choice's
        int mine_e = -1;
        for (int j = 0; j < a.top; ++j) {
            uint32_t best = 0;
            int at = 0;
#pragma unroll
            for (int i = 0; i < R; ++i)
                if (i * 32 < a.e && key[i] > best) {
                    best = key[i];
                    at = i;
                }
            const uint32_t high = __reduce_max_sync(0xffffffffu, best);
            const int e = (int)__reduce_min_sync(0xffffffffu, best == high ? (uint32_t)(at * 32 + lane) : ~0u);
            const uint32_t bits = (high & 0x80000000u) ? high & 0x7fffffffu : ~high;
            const float v = __uint_as_float(bits);
            if (j == 0) {
                // (the first choice is the largest logit) all exponentials, from the keys still in place
                top_value = v;
#pragma unroll
                for (int i = 0; i < R; ++i)
                    if (i * 32 < a.e && i * 32 + lane < a.e) {
                        const uint32_t b = (key[i] & 0x80000000u) ? key[i] & 0x7fffffffu : ~key[i];
                        sum += expf(__uint_as_float(b) - top_value);
                    }
#pragma unroll
                for (int s = 16; s; s >>= 1)
                    sum += __shfl_xor_sync(0xffffffffu, sum, s);
            }
            const float w = expf(v - top_value);
            chosen += w;
            if (lane == j) {
                mine = w;
                mine_e = e;
            }
#pragma unroll
            for (int i = 0; i < R; ++i)
                if (i * 32 + lane == e)
                    key[i] = 0;
        }
        if (lane < a.top) {
            float p = __fdiv_rn(mine, a.renormalize ? chosen : sum);
            if (top_value == -__uint_as_float(0x7f800000u))
                p = 0.f;  // every expert is masked: no share in any
            if (odd)
                p = __uint_as_float(0x7fffffffu);
            r.p[t * a.top + lane] = p;
            r.expert[t * a.top + lane] = p == 0.f ? -1 : mine_e;
        }
    }
    __syncthreads();
    // slots per expert: whole numbers, their order does not matter; one thread counts an expert's
    const int slots = a.t * a.top;
    for (int e = threadIdx.x; e < a.e; e += kThreads) {
        int n = 0;
        for (int s = 0; s < slots; ++s)
            n += r.expert[s] == e;
        r.count[e] = (short)n;
    }
    __syncthreads();
    if (warp == 0) {
        int start = 0, passes = 0;
        for (int e0 = 0; e0 < a.e; e0 += 32) {
            const int e = e0 + lane;
            const int n = e < a.e ? r.count[e] : 0, np = (n + cols - 1) / cols;
            int s = n, q = np;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int s1 = __shfl_up_sync(0xffffffffu, s, d), q1 = __shfl_up_sync(0xffffffffu, q, d);
                if (lane >= d) {
                    s += s1;
                    q += q1;
                }
            }
            if (e < a.e)
                r.start[e] = (short)(start + s - n);
            for (int i = 0; i < np; ++i) {
                const int at = passes + q - np + i;
                r.pass_expert[at] = (short)e;
                r.pass_start[at] = (short)(start + s - n + i * cols);
                r.pass_cols[at] = (short)min(cols, n - i * cols);
            }
            start += __shfl_sync(0xffffffffu, s, 31);
            passes += __shfl_sync(0xffffffffu, q, 31);
        }
        if (lane == 0)
            r.passes = passes;
    }
    __syncthreads();
    for (int e = threadIdx.x; e < a.e; e += kThreads) {
        int at = r.start[e];
        if (r.count[e])
            for (int s = 0; s < slots; ++s)
                if (r.expert[s] == e)
                    r.order[at++] = (short)s;
    }
    __syncthreads();
}

// `cols` rows of x as whole numbers in shared memory, a warp per row
template <class T>
__device__ void quantize_tokens(
        const MoeArgs& a, const short* order, int top, int cols, int8_t* xs, int pitch, float* scale,
        int x_vectors) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int c = warp; c < cols; c += kWarps) {
        const int t = order ? order[c] / top : c;
        const T* row = (const T*)a.x + (long long)t * a.ldx;
        uint32_t bits = 0;
        for (int i = lane * 16; i < a.d; i += 512) {
            float v[16];
            load_piece(row, i, a.d, x_vectors, v);
#pragma unroll
            for (int j = 0; j < 16; ++j)
                bits = max(bits, magnitude(v[j]));
        }
        const RowScale r = row_scale(__reduce_max_sync(0xffffffffu, bits));
        if (lane == 0)
            scale[c] = r.scale;
        for (int i = lane * 16; i < a.d; i += 512) {
            float v[16];
            load_piece(row, i, a.d, x_vectors, v);
            *(uint4*)(xs + c * pitch + i) = pack_piece(v, r);
        }
    }
}

// ---- gate, up, activation, and h as whole numbers ----
// Tiles of 32 hidden units (64 rows of w1), a tile per pass of its expert; a CTA takes neighbouring ones. Its
// warps take the 64-byte chunks of d in turn. COLS tokens at once; with no more tokens than that all of them
// stay in shared memory for the whole kernel.
template <class T, int COLS, bool ALIGNED>
__global__ void __launch_bounds__(kThreads, 2) moe_up_kernel(const MoeArgs a, int pitch, int x_vectors) {
    constexpr int NT = COLS / 8;
    extern __shared__ __align__(16) uint8_t dynamic[];
    int* red = (int*)dynamic;                                    // [kWarps][COLS][kPitch]
    int8_t* xs = (int8_t*)(dynamic + kWarps * COLS * kPitch * 4);  // [COLS][pitch]
    __shared__ Route route;
    __shared__ float x_scale[COLS];

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, tig = lane & 3;
    pdl_start();
    route_tokens(a, COLS, route);
    const bool resident = a.t <= COLS;
    const int blocks = (a.f + kUnits - 1) / kUnits;
    const long long tiles = (long long)route.passes * blocks;
    const int first = (int)(tiles * blockIdx.x / gridDim.x), last = (int)(tiles * (blockIdx.x + 1) / gridDim.x);
    if (first == last)
        return;
    const int chunks = (a.d + 63) >> 6;
    const int mine = warp < chunks ? (chunks - warp + kWarps - 1) / kWarps : 0;  // chunks of this warp

    // loads run one chunk ahead of the MMAs, over the ends of tiles
    uint4 w[2][8];
    int l_tile = first, l_chunk = 0;
    const int8_t* l_row[8];
    auto open_tile = [&](int tile) {
        const int e = route.pass_expert[tile / blocks], u0 = tile % blocks * kUnits;
        const int8_t* w1 = a.w1 + (size_t)e * (2 * (size_t)a.f) * a.d;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int u = min(u0 + 8 * i + g, a.f - 1);
            l_row[i] = w1 + (size_t)u * a.d;
            l_row[4 + i] = w1 + ((size_t)a.f + u) * a.d;
        }
    };
    auto load_next = [&](uint4 (&v)[8]) {
        if (l_tile >= last)
            return;
        const int kk = (warp + l_chunk * kWarps) * 64 + tig * 16;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (ALIGNED)
                v[i] = kk < a.d ? ld_stream16(l_row[i] + kk) : make_uint4(0, 0, 0, 0);
            else
                v[i] = ld_any16(l_row[i] + kk, a.d - kk);
        }
        if (++l_chunk == mine) {
            l_chunk = 0;
            if (++l_tile < last)
                open_tile(l_tile);
        }
    };
    if (mine) {
        open_tile(first);
        load_next(w[0]);
    }
    if (resident)
        quantize_tokens<T>(a, nullptr, 1, a.t, xs, pitch, x_scale, x_vectors);
    __syncthreads();

    int pass = -1, cols = 0, e = 0;
    const short* order = nullptr;
    int buf = 0;
    for (int tile = first; tile < last; ++tile) {
        const int u0 = tile % blocks * kUnits;
        if (tile / blocks != pass) {
            pass = tile / blocks;
            e = route.pass_expert[pass];
            cols = route.pass_cols[pass];
            order = route.order + route.pass_start[pass];
            if (!resident) {
                __syncthreads();  // (the last pass's tokens have been read)
                quantize_tokens<T>(a, order, a.top, cols, xs, pitch, x_scale, x_vectors);
                __syncthreads();
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
            frag[nt] = xs + (resident ? order[c] / a.top : c) * pitch + tig * 16;
        }
        int acc[4][NT][4];
#pragma unroll
        for (int b = 0; b < 4; ++b)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
                acc[b][nt][0] = acc[b][nt][1] = acc[b][nt][2] = acc[b][nt][3] = 0;
        auto multiply = [&](const uint4 (&v)[8], int c) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const uint4 x = *(const uint4*)(frag[nt] + (warp + c * kWarps) * 64);
#pragma unroll
                for (int b = 0; b < 4; ++b)
                    mma_64(acc[b][nt], v[2 * b], v[2 * b + 1], x);
            }
        };
        for (int c = 0; c < mine; ++c) {
            if (buf == 0) {
                load_next(w[1]);
                multiply(w[0], c);
            } else {
                load_next(w[0]);
                multiply(w[1], c);
            }
            buf ^= 1;
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                // units 16 * (b % 2) + g and + 8; gate in front, up behind
                int* at = red + (warp * COLS + 8 * nt + 2 * tig) * kPitch + (b >> 1) * kUnits + 16 * (b & 1) + g;
                at[0] = acc[b][nt][0];
                at[kPitch] = acc[b][nt][1];
                at[8] = acc[b][nt][2];
                at[kPitch + 8] = acc[b][nt][3];
            }
        __syncthreads();
        for (int c = warp; c < cols; c += kWarps) {
            int gate = 0, up = 0;
#pragma unroll
            for (int i = 0; i < kWarps; ++i) {
                gate += red[(i * COLS + c) * kPitch + lane];
                up += red[(i * COLS + c) * kPitch + kUnits + lane];
            }
            const int slot = order[c];
            const float sx = x_scale[resident ? slot / a.top : c];
            const float zg = scale_acc(gate, sx, s_gate), zu = scale_acc(up, sx, s_up);
            const float h = u < a.f ? __fmul_rn(__fdiv_rn(zg, __fadd_rn(1.f, expf(-zg))), zu) : 0.f;
            const RowScale r = row_scale(__reduce_max_sync(0xffffffffu, magnitude(h)));
            a.hq[(size_t)slot * (blocks * kUnits) + u] = (int8_t)(to_whole(h, r.inv) & r.keep);
            if (lane == 0)
                a.sh[(size_t)slot * blocks + u0 / kUnits] = r.scale;
        }
        __syncthreads();
    }
}

// ---- down, and the experts' sum ----
// A CTA makes 16 rows of every token: its warps take the groups of f in turn, expert after expert in the
// order of their indices, and add into sums of their own, which meet at the end in the order of the warps:
// no atomics, the same bits every time.
template <class T, bool ALIGNED>
__global__ void __launch_bounds__(kThreads, 2) moe_down_kernel(const MoeArgs a) {
    constexpr int U = 8;  // groups in flight per warp
    extern __shared__ __align__(16) float sums[];  // [kWarps][a.t][kRows]
    __shared__ Route route;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, tig = lane & 3;
    const int d0 = blockIdx.x * kRows;
    // Ahead of the first kernel's end: the routing and the first weights. What is read here was written before
    // the first kernel began, which let this one start behind its own wait for that.
    route_tokens(a, 8, route);
    const int groups = (a.f + kUnits - 1) / kUnits, width = groups * kUnits;
    const int mine = warp < groups ? (groups - warp + kWarps - 1) / kWarps : 0;
    const int steps = mine * route.passes;
    float* own = sums + warp * a.t * kRows;
    for (int i = lane; i < a.t * kRows; i += 32)
        own[i] = 0.f;
    __syncwarp();

    const int row_lo = min(d0 + g, a.d - 1), row_hi = min(d0 + g + 8, a.d - 1);
    uint2 w[U][2], hq[U];
    float sh[U][2];
    // where the loads are: weights, and what the first kernel writes
    int wp = 0, wu = 0, hp = 0, hu = 0;
    const int8_t *w_lo = nullptr, *w_hi = nullptr;
    const int8_t* h_row = nullptr;
    const float *sh0 = nullptr, *sh1 = nullptr;
    auto load_weights = [&](uint2 (&v)[2]) {
        if (wu == 0) {
            const int8_t* w2 = a.w2 + (size_t)route.pass_expert[wp] * a.d * a.f;
            w_lo = w2 + (size_t)row_lo * a.f;
            w_hi = w2 + (size_t)row_hi * a.f;
        }
        const int kk = (warp + wu * kWarps) * kUnits + tig * 8;
        if (ALIGNED) {
            v[0] = kk < a.f ? ld_stream8(w_lo + kk) : make_uint2(0, 0);
            v[1] = kk < a.f ? ld_stream8(w_hi + kk) : make_uint2(0, 0);
        } else {
            v[0] = ld_any8(w_lo + kk, a.f - kk);
            v[1] = ld_any8(w_hi + kk, a.f - kk);
        }
        if (++wu == mine) {
            wu = 0;
            ++wp;
        }
    };
    auto load_hidden = [&](uint2& q, float (&s)[2]) {
        if (hu == 0) {
            const short* order = route.order + route.pass_start[hp];
            const int end = route.pass_cols[hp] - 1;
            h_row = a.hq + (size_t)order[min(g, end)] * width;
            sh0 = a.sh + (size_t)order[min(2 * tig, end)] * groups;
            sh1 = a.sh + (size_t)order[min(2 * tig + 1, end)] * groups;
        }
        const int group = warp + hu * kWarps;
        q = *(const uint2*)(h_row + group * kUnits + tig * 8);
        s[0] = sh0[group];
        s[1] = sh1[group];
        if (++hu == mine) {
            hu = 0;
            ++hp;
        }
    };
#pragma unroll
    for (int i = 0; i < U; ++i)
        if (i < steps)
            load_weights(w[i]);
    pdl_start();
#pragma unroll
    for (int i = 0; i < U; ++i)
        if (i < steps)
            load_hidden(hq[i], sh[i]);

    int pass = 0, u = 0;
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    float s_lo = 0.f, s_hi = 0.f;
    for (int step = 0; step < steps; step += U) {
#pragma unroll
        for (int i = 0; i < U; ++i) {
            if (step + i < steps) {
                if (u == 0) {
                    const float* s2 = a.s2 + (size_t)route.pass_expert[pass] * a.d;
                    s_lo = s2[row_lo];
                    s_hi = s2[row_hi];
                }
                int c[4] = {0, 0, 0, 0};
                mma_16x8x32(c, w[i][0].x, w[i][1].x, w[i][0].y, w[i][1].y, hq[i].x, hq[i].y);
                acc[0] = __fmaf_rn(__int2float_rn(c[0]), sh[i][0], acc[0]);
                acc[1] = __fmaf_rn(__int2float_rn(c[1]), sh[i][1], acc[1]);
                acc[2] = __fmaf_rn(__int2float_rn(c[2]), sh[i][0], acc[2]);
                acc[3] = __fmaf_rn(__int2float_rn(c[3]), sh[i][1], acc[3]);
                if (step + i + U < steps) {
                    load_weights(w[i]);
                    load_hidden(hq[i], sh[i]);
                }
                if (++u == mine) {
                    // this warp's share of the expert, to the sums of its tokens
                    const short* order = route.order + route.pass_start[pass];
#pragma unroll
                    for (int j = 0; j < 2; ++j)
                        if (2 * tig + j < route.pass_cols[pass]) {
                            const int slot = order[2 * tig + j];
                            const float p = route.p[slot];
                            float* at = own + slot / a.top * kRows + g;
                            at[0] = __fmaf_rn(__fmul_rn(acc[j], s_lo), p, at[0]);
                            at[8] = __fmaf_rn(__fmul_rn(acc[2 + j], s_hi), p, at[8]);
                        }
                    __syncwarp();  // the next expert's lanes find them
                    acc[0] = acc[1] = acc[2] = acc[3] = 0.f;
                    u = 0;
                    ++pass;
                }
            }
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < a.t * kRows; i += kThreads) {
        const int t = i / kRows, d = d0 + i % kRows;
        float v = 0.f;
#pragma unroll
        for (int s = 0; s < kWarps; ++s)
            v += sums[s * a.t * kRows + i];
        if (d < a.d)
            store_as(a.y, a.dtype, (size_t)t * (size_t)a.ldy + d, v);
    }
}

template <class T, int COLS, bool ALIGNED>
cudaError_t launch_up(const MoeArgs& a, cudaStream_t st) {
    static umma::KernelReady ready;
    static umma::ResidentCtas resident;
    auto kernel = moe_up_kernel<T, COLS, ALIGNED>;
    const int pitch = (a.d + 127) / 128 * 128 + 64;  // rows half of all banks apart
    const int smem = kWarps * COLS * kPitch * 4 + COLS * pitch;
    if (!ready.smem(kernel, smem))
        return cudaErrorInvalidValue;
    const int x_vectors = ((uintptr_t)a.x & 15) == 0 && (a.t == 1 || a.ldx % Vec<T>::N == 0);
    const long long slots = (long long)a.t * a.top;
    const long long tiles = slots * ((a.f + kUnits - 1) / kUnits);  // at most
    const long long fit = (long long)umma::sm_count() * resident.per_sm(kernel, kThreads, smem + (int)sizeof(Route), 0);
    const Writes writes{a.hq, a.workspace_bytes};
    return launch_pdl(writes, kernel, dim3((unsigned)(tiles < fit ? tiles : fit)), dim3(kThreads), (size_t)smem, st,
                      a, pitch, x_vectors);
}

template <class T>
cudaError_t launch_both(const MoeArgs& a, cudaStream_t st) {
    const bool up16 = ((uintptr_t)a.w1 & 15) == 0 && a.d % 16 == 0;
    const bool down8 = ((uintptr_t)a.w2 & 7) == 0 && a.f % 8 == 0;
    cudaError_t e = a.t <= 8 ? (up16 ? launch_up<T, 8, true>(a, st) : launch_up<T, 8, false>(a, st))
                             : (up16 ? launch_up<T, 16, true>(a, st) : launch_up<T, 16, false>(a, st));
    if (e != cudaSuccess)
        return e;
    const int smem = kWarps * a.t * kRows * 4;
    const dim3 grid((unsigned)((a.d - 1) / kRows + 1));
    const Writes writes{a.y, ((size_t)(a.t - 1) * (size_t)a.ldy + (size_t)a.d) * dtype_bytes(a.dtype)};
    return down8 ? launch_pdl(writes, moe_down_kernel<T, true>, grid, dim3(kThreads), (size_t)smem, st, a)
                 : launch_pdl(writes, moe_down_kernel<T, false>, grid, dim3(kThreads), (size_t)smem, st, a);
}

}  // namespace

int launch_moe(const MoeArgs& a, cudaStream_t st) {
    const cudaError_t e = a.dtype == DT_F32   ? launch_both<float>(a, st)
                          : a.dtype == DT_F16 ? launch_both<__half>(a, st)
                                              : launch_both<__nv_bfloat16>(a, st);
    if (e != cudaSuccess)
        return set_error(ST_RUNTIME, "moe_s8: %s", cudaGetErrorString(e));
    return check_launch("moe_s8");
}

}  // namespace scaled
}  // namespace mb200
