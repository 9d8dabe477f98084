// int8 products with a scale per row and per output channel on the tensor cores (tcgen05.mma kind::i8).
//
// Both operands are K-major, 128 bytes of K per pipeline stage, brought by tiled TMA loads with the
// 128-byte swizzle; sums stay exact in int32 in tensor memory. The epilogue multiplies by the two scales in
// fp32, adds the bias, rounds once and turns the tile round in shared memory, 64 bytes of 32 rows at a time, from where
// the TMA stores it (or, where rows of the result do not begin and end with 16-byte units, the warp).
//
// Two kernels:
//   pair   256 x 256 tiles (or x 192, x 128, where those come out even) on pairs of SMs (cta_group::2), persistent, two
//          accumulator buffers. What bounds wide
//          products is the SM's shared memory: per 128 bytes of K a 128 x 128 tile of one SM writes and reads 64 KB
//          for 256 clocks of MMAs, 512 clocks at 128 B/clk; the pair's 256 x 256 the same bytes per SM
//          for 512 clocks of MMAs.
//   split  128 x 128 tiles, K cut over the 1, 2, 4 or 8 CTAs of a cluster where there are few tiles: there
//          the weights' way from HBM bounds, and every SM has to take part in it. The partial sums meet in
//          shared memory (whole numbers: in any order the same).
#include <limits.h>

#include "scaled_s8.cuh"
#include "umma_pair.cuh"

namespace mb200 {
namespace scaled {

using namespace umma;

namespace {

constexpr int ERR_SHARED_WINDOW = 0x106;

constexpr int kBM = 128;  // rows per CTA
constexpr int kBK = 128;  // K bytes per stage
constexpr int kTileBytes = kBM * kBK;  // of 128 rows

struct UmmaArgs {
    int m, n, k_steps;
    int m_tiles, n_tiles;
    const float *sa, *sb, *bias;
    void* c;
    long long ldc;
    int vector_stores;  // rows of c begin at 16-byte units
    // pair: and end with one, so that the TMA may store them: it writes whole units, over what stands behind a row's last
    // element within its unit
    int tma_stores;
    int b_early;
    int bn;          // pair: columns of a tile, 256, 192 or 128
    // split:
    int a_rows;      // rows of A's box
    int a_bytes;     // of a stage, B's part behind it
    int stages;
    int csplit;      // CTAs per tile
    int* status;
};

template <class T>
struct Out;
template <>
struct Out<float> {
    static __device__ __forceinline__ uint4 unit4(const float* v) {
        return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
    }
    static __device__ __forceinline__ float one(float v) {
        return v;
    }
};
template <>
struct Out<__half> {
    static __device__ __forceinline__ uint32_t two(float a, float b) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static __device__ __forceinline__ uint4 unit4(const float* v) {
        return make_uint4(two(v[0], v[1]), two(v[2], v[3]), 0, 0);
    }
    static __device__ __forceinline__ __half one(float v) {
        return __float2half_rn(v);
    }
};
template <>
struct Out<__nv_bfloat16> {
    static __device__ __forceinline__ uint32_t two(float a, float b) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static __device__ __forceinline__ uint4 unit4(const float* v) {
        return make_uint4(two(v[0], v[1]), two(v[2], v[3]), 0, 0);
    }
    static __device__ __forceinline__ __nv_bfloat16 one(float v) {
        return __float2bfloat16_rn(v);
    }
};

// What a lane needs of the scales for 32 rows times 64 columns of sums. tcgen05.ld 16x256b hands it, of each 16 rows, the
// rows lane / 4 and lane / 4 + 8, and of each eight columns 2 * (lane % 4) and the one behind: so four rows' and sixteen
// columns' scales stay in registers, where a row per lane would read all 64 columns' from shared memory, which the
// MMAs and the TMA keep busy (fp32 results of 6970 x 4576 x 1264: 49.7 us, 51.5 so).
struct Sides {
    float row[4];
    float2 scale[8], bias[8];
    // rows: the lane's own row's scale; scale, bias: of the 64 columns, in shared memory
    __device__ __forceinline__ void take(float rows, const float* col_scale, const float* col_bias, bool has_bias) {
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            row[i] = __shfl_sync(0xffffffffu, rows, 8 * i + (lane >> 2));
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            scale[j] = *(const float2*)(col_scale + 8 * j + 2 * (lane & 3));
            bias[j] = has_bias ? *(const float2*)(col_bias + 8 * j + 2 * (lane & 3)) : make_float2(0.f, 0.f);
        }
    }
    __device__ __forceinline__ float2 apply(uint32_t a, uint32_t b, int i, int j, bool has_bias) const {
        float2 v = make_float2(scale_acc((int)a, row[i], scale[j].x), scale_acc((int)b, row[i], scale[j].y));
        if (has_bias)
            v = make_float2(__fadd_rn(v.x, bias[j].x), __fadd_rn(v.y, bias[j].y));
        return v;
    }
};
// 16 lanes of tensor memory times 8 * N columns; 4 * N words per lane of the warp
__device__ __forceinline__ void tmem_ld_16x256b(uint32_t taddr, uint32_t (&v)[16]) {
    asm volatile(
            "tcgen05.ld.sync.aligned.16x256b.x4.b32 "
            "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
            : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
              "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
            : "r"(taddr)
            : "memory");
}
__device__ __forceinline__ void tmem_ld_wait2(uint32_t (&a)[16], uint32_t (&b)[16]) {
    tmem_ld_wait16(a);
    tmem_ld_wait16(b);
}
__device__ __forceinline__ void stmatrix_x4(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c),
                 "r"(d)
                 : "memory");
}

// 32 rows (of the warp's tensor memory lanes) times 64 columns of results, through 2 KB of shared memory to whole
// sectors: 64 bytes of each row at a time. With map_c the TMA stores them; else the warp does.
// `taken()` is called once the sums are in registers.
constexpr int kRoundBytes = 32 * 64;
template <class T, class Taken>
__device__ __forceinline__ void store_columns(
        uint32_t taddr, const Sides& sides, bool has_bias, uint8_t* stage, int row0, int col0, const UmmaArgs& p,
        const CUtensorMap* map_c, Taken taken) {
    constexpr int kUnit = 16 / (int)sizeof(T);  // results per 16 bytes
    constexpr int kCols = 4 * kUnit;            // of a round
    const int lane = threadIdx.x & 31;
    const uint32_t at = smem_u32(stage);
    T* c = (T*)p.c;
#pragma unroll
    for (int h = 0; h < 2; ++h) {  // 32 columns
        uint32_t acc[2][16];
        __syncwarp();
        tmem_ld_16x256b(taddr + (uint32_t)(32 * h), acc[0]);
        tmem_ld_16x256b(taddr + (16u << 16) + (uint32_t)(32 * h), acc[1]);
        tmem_ld_wait2(acc[0], acc[1]);
        if (h == 1)
            taken();
#pragma unroll
        for (int round = 0; round < 32 / kCols; ++round) {
            const int col = col0 + 32 * h + round * kCols;
            if (map_c) {
                // the last round's bytes have left the stage
                if (lane == 0)
                    asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                __syncwarp();
            }
            // (a row's 16-byte units in an order that depends on the row, the TMA's 64-byte swizzle)
#pragma unroll
            for (int q = 0; q < 2; ++q) {  // 16 rows
                if constexpr (sizeof(T) == 2) {
#pragma unroll
                    for (int jj = 0; jj < 2; ++jj) {
                        uint32_t w[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int j = 2 * jj + (i >> 1);
                            const float2 v = sides.apply(acc[q][4 * j + 2 * (i & 1)], acc[q][4 * j + 2 * (i & 1) + 1],
                                                         2 * q + (i & 1), 4 * h + j, has_bias);
                            w[i] = Out<T>::two(v.x, v.y);
                        }
                        const int r = 16 * q + (lane & 15), unit = 2 * jj + (lane >> 4);
                        stmatrix_x4(at + (uint32_t)(r * 64 + ((unit ^ ((r >> 1) & 3)) << 4)), w[0], w[1], w[2], w[3]);
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const int jc = 2 * round + j;
                            const float2 v = sides.apply(acc[q][4 * jc + 2 * i], acc[q][4 * jc + 2 * i + 1], 2 * q + i,
                                                         4 * h + jc, has_bias);
                            const int r = 16 * q + 8 * i + (lane >> 2), unit = 2 * j + ((lane & 3) >> 1);
                            *(float2*)(stage + r * 64 + ((unit ^ ((r >> 1) & 3)) << 4) + 8 * (lane & 1)) = v;
                        }
                }
            }
            if (map_c) {
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0 && row0 < p.m && col < p.n) {
                    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(
                                         (uint64_t)map_c),
                                 "r"(at), "r"(col), "r"(row0)
                                 : "memory");
                    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                }
                continue;
            }
            __syncwarp();
            if (p.vector_stores && col + kCols <= p.n) {
                const int unit = lane & 3;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int r = 8 * i + (lane >> 2);
                    const uint4 v = *(const uint4*)(stage + r * 64 + ((unit ^ ((r >> 1) & 3)) << 4));
                    if (row0 + r < p.m)
                        *(uint4*)(c + (long long)(row0 + r) * p.ldc + col + unit * kUnit) = v;
                }
            } else {
                const int j = lane % kCols;
                T* to = c + (long long)(row0 + lane / kCols) * p.ldc + col + j;
#pragma unroll 1
                for (int r0 = lane / kCols; r0 < 32; r0 += 8 * (32 / kCols)) {
                    T v[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int r = r0 + i * (32 / kCols);
                        v[i] = *(const T*)(stage + r * 64 + (((j / kUnit) ^ ((r >> 1) & 3)) << 4) +
                                           (j % kUnit) * sizeof(T));
                    }
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        if (row0 + r0 + i * (32 / kCols) < p.m && col + j < p.n)
                            *to = v[i];
                        to += (32 / kCols) * p.ldc;
                    }
                }
            }
            __syncwarp();
        }
    }
}

// the epilogue warps' barrier
template <int WARPS>
__device__ __forceinline__ void epilogue_sync() {
    asm volatile("bar.sync 1, %0;" ::"n"(32 * WARPS) : "memory");
}

// Tiles in groups of eight rows of tiles, downwards first: what the SMs work on at one time shares its
// operands in the L2.
struct Tile {
    int m, n;
};
__device__ __forceinline__ Tile tile_at(int i, int m_tiles, int n_tiles) {
    constexpr int kGroup = 8;
    const int group = i / (kGroup * n_tiles), first = group * kGroup;
    const int rows = min(kGroup, m_tiles - first), j = i - group * kGroup * n_tiles;
    return {first + j % rows, j / rows};
}

// ---- pairs of SMs ----
constexpr int kPairBN = 256;
constexpr int kPairStages = 6;
constexpr int kPairWarps = 16;  // epilogue; with eight a tile's epilogue took 4 us, the MMAs of 6 steps of K 2
constexpr int kPairThreads = 64 + 32 * kPairWarps;
constexpr int kStageBytes = 2 * kTileBytes;
constexpr int kPairRoundOff = kPairStages * kStageBytes;                // the epilogue warps' 2 KB each
constexpr int kPairColOff = kPairRoundOff + kPairWarps * kRoundBytes;  // [256] scales, [256] biases
constexpr int kPairBarOff = kPairColOff + 2 * kPairBN * 4;
constexpr int kPairDynamic = kPairBarOff + (2 * kPairStages + 5) * 8 + 16;
static_assert(kPairDynamic <= 232448, "shared memory of one SM");

template <class T>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1) product_pair_kernel(
        const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
        const __grid_constant__ CUtensorMap map_c, const UmmaArgs p) {
    extern __shared__ uint8_t smem_raw[];
    // A kernel without static shared memory has its window on a 1024-byte boundary, as the swizzle wants it; there
    // is no room to move it up, so one that is not there would leave before it touches anything.
    uint8_t* smem = smem_raw;
    if (smem_u32(smem) & 1023) {
        if (threadIdx.x == 0)
            atomicExch(p.status, ERR_SHARED_WINDOW);
        return;
    }
    float* col_scale = (float*)(smem + kPairColOff);
    float* col_bias = col_scale + kPairBN;
    uint64_t* full_bar = (uint64_t*)(smem + kPairBarOff);  // used in the leader only
    uint64_t* empty_bar = full_bar + kPairStages;          // one set per CTA
    uint64_t* acc_full = empty_bar + kPairStages;          // [2], one set per CTA
    uint64_t* acc_empty = acc_full + 2;                    // [2], used in the leader only
    uint64_t* drain_bar = acc_empty + 2;
    uint32_t* tmem_slot = (uint32_t*)(drain_bar + 1);
    volatile int* abort_flag = (volatile int*)(tmem_slot + 1);

    const int warp = uniform_warp_index(), lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const bool leader = rank == 0;
    const int total_tiles = p.m_tiles * p.n_tiles;
    const int first_tile = (int)cluster_id_x(), tile_step = (int)num_clusters_x();

    if (threadIdx.x == 0) {
        for (int s = 0; s < kPairStages; ++s) {
            mbar_init(&full_bar[s], 1);   // the leader's producer; both CTAs' bytes
            mbar_init(&empty_bar[s], 1);  // one commit
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&acc_full[b], 1);
            mbar_init(&acc_empty[b], 2 * kPairWarps);
        }
        mbar_init(drain_bar, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    } else if (threadIdx.x == 64) {
        tma_prefetch_map(&map_a);
        tma_prefetch_map(&map_b);
    }
    if (warp == 1) {
        asm volatile(
                "tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                "r"(2 * kPairBN)
                : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    cluster_sync();  // both CTAs' barriers exist before anything arrives on them
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem_base = *tmem_slot;
    const uint32_t peer_abort = map_to_cta(smem_u32((const void*)abort_flag), rank ^ 1u);

    auto give_up = [&](int code) {
        if (!*abort_flag) {
            *abort_flag = 1;
            atomicExch(p.status, code);
        }
        asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(peer_abort), "r"(1) : "memory");
    };

    if (warp == 0) {
        // ---------------- TMA producer (both CTAs): own 128 rows of A and half of B's 256 ----------------
        if (lane == 0) {
            int s = 0;
            uint32_t phase = 0;
            bool ok = true;
            auto b_row = [&](const Tile& t) { return t.n * p.bn + (int)rank * (p.bn / 2); };
            auto announce = [&](int stage) {
                if (leader)
                    mbar_expect_tx(&full_bar[stage], 2u * (uint32_t)(kTileBytes + p.bn / 2 * kBK));
            };
            // weights of the first stages ahead of the end of the kernel in front
            int ahead = 0;
            if (p.b_early && first_tile < total_tiles) {
                const Tile t = tile_at(first_tile, p.m_tiles, p.n_tiles);
                for (; ahead < min(kPairStages, p.k_steps); ++ahead) {
                    announce(ahead);
                    tma_pair_load_2d(smem + ahead * kStageBytes + kTileBytes, &map_b,
                                     map_to_cta(smem_u32(&full_bar[ahead]), 0), ahead * kBK, b_row(t));
                }
            }
            pdl_start();
            for (int tile = first_tile; tile < total_tiles && ok; tile += tile_step) {
                const Tile t = tile_at(tile, p.m_tiles, p.n_tiles);
                const int m0 = t.m * (2 * kBM) + (int)rank * kBM, n0 = b_row(t);
                for (int it = 0; it < p.k_steps; ++it) {
                    ok = mbar_wait_cluster(&empty_bar[s], phase ^ 1u, abort_flag);
                    if (!ok) {
                        give_up(ERR_PRODUCER_WAIT);
                        break;
                    }
                    uint8_t* at = smem + s * kStageBytes;
                    const uint32_t full_leader = map_to_cta(smem_u32(&full_bar[s]), 0);
                    const bool b_there = tile == first_tile && it < ahead;
                    if (!b_there)
                        announce(s);
                    tma_pair_load_2d(at, &map_a, full_leader, it * kBK, m0);
                    if (!b_there)
                        tma_pair_load_2d(at + kTileBytes, &map_b, full_leader, it * kBK, n0);
                    if (++s == kPairStages) {
                        s = 0;
                        phase ^= 1u;
                    }
                }
            }
        }
    } else if (warp == 1) {
        // ---------------- MMA issuer (leader only) ----------------
        if (leader && lane == 0) {
            const uint32_t idesc = umma_idesc_s8(2 * kBM, p.bn);
            int local = 0, s = 0;
            uint32_t phase = 0;
            bool ok = true;
            const uint64_t a0 = umma_smem_desc(smem_u32(smem), 16, 1024, 2);
            const uint64_t b0 = umma_smem_desc(smem_u32(smem + kTileBytes), 16, 1024, 2);
            for (int tile = first_tile; tile < total_tiles && ok; tile += tile_step, ++local) {
                const int buf = local & 1;
                const uint32_t acc_phase = (uint32_t)(local >> 1) & 1u;
                // both CTAs' epilogues must have drained this accumulator buffer
                ok = mbar_wait_cluster(&acc_empty[buf], acc_phase ^ 1u, abort_flag);
                if (!ok) {
                    give_up(ERR_MMA_ACC_WAIT);
                    break;
                }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t tmem_d = tmem_base + (uint32_t)(buf * kPairBN);
                for (int it = 0; it < p.k_steps; ++it) {
                    ok = mbar_wait_cluster(&full_bar[s], phase, abort_flag);
                    if (!ok) {
                        give_up(ERR_MMA_WAIT);
                        break;
                    }
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint64_t adesc = a0 + (uint64_t)(s * (kStageBytes / 16));
                    const uint64_t bdesc = b0 + (uint64_t)(s * (kStageBytes / 16));
#pragma unroll
                    for (int k = 0; k < kBK / 32; ++k)
                        umma_pair_s8(tmem_d, adesc + k * 2, bdesc + k * 2, idesc, (it | k) != 0 ? 1u : 0u);
                    // the stage is free in both CTAs once these MMAs retire
                    const uint32_t e_local = smem_u32(&empty_bar[s]);
                    umma_pair_commit(e_local);
                    umma_pair_commit(map_to_cta(e_local, 1));
                    if (++s == kPairStages) {
                        s = 0;
                        phase ^= 1u;
                    }
                }
                if (ok) {
                    const uint32_t f_local = smem_u32(&acc_full[buf]);
                    umma_pair_commit(f_local);
                    umma_pair_commit(map_to_cta(f_local, 1));
                }
            }
        }
    } else {
        // ---------------- epilogue (both CTAs): warps 2..17, tensor memory lanes 32 * (warp % 4) ----------------
        const int q = warp & 3, quarter = (warp - 2) >> 2;
        const int et = (int)threadIdx.x - 64;
        uint8_t* stage = smem + kPairRoundOff + (warp - 2) * kRoundBytes;
        int local = 0;
        bool ok = true;
        pdl_start();
        // half of the threads have a column's scale, half its bias; a tile's come while the one before is stored
        const float* sides = et < kPairBN ? p.sb : p.bias;
        const int column = et & (kPairBN - 1);
        float side = 0.f, sa = 0.f;
        auto fetch = [&](int tile) {
            if (tile < total_tiles) {
                const Tile t = tile_at(tile, p.m_tiles, p.n_tiles);
                const int row = t.m * (2 * kBM) + (int)rank * kBM + q * 32 + lane, n = t.n * p.bn + column;
                sa = row < p.m ? p.sa[row] : 0.f;
                side = sides && column < p.bn && n < p.n ? sides[n] : 0.f;
            }
        };
        fetch(first_tile);
        for (int tile = first_tile; tile < total_tiles; tile += tile_step, ++local) {
            const int buf = local & 1;
            const uint32_t acc_phase = (uint32_t)(local >> 1) & 1u;
            const Tile t = tile_at(tile, p.m_tiles, p.n_tiles);
            const int row0 = t.m * (2 * kBM) + (int)rank * kBM + q * 32, n0 = t.n * p.bn;
            epilogue_sync<kPairWarps>();  // (the last tile's have been read)
            (et < kPairBN ? col_scale : col_bias)[column] = side;
            const float row_scale = sa;
            epilogue_sync<kPairWarps>();
            fetch(tile + tile_step);
            ok = mbar_wait_cluster(&acc_full[buf], acc_phase, abort_flag);
            if (!ok)
                give_up(ERR_EPILOGUE_WAIT);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok)
                continue;  // (still meets the others at the barrier in front of the next tile)
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t taddr = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(buf * kPairBN);
            if (quarter * 64 >= p.bn) {
                // (no columns of a narrow tile for this warp)
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                if (lane == 0)
                    mbar_arrive_cluster(map_to_cta(smem_u32(&acc_empty[buf]), 0));
                continue;
            }
            Sides sides;
            sides.take(row_scale, col_scale + quarter * 64, col_bias + quarter * 64, p.bias != nullptr);
            store_columns<T>(taddr + (uint32_t)(quarter * 64), sides, p.bias != nullptr, stage, row0, n0 + quarter * 64, p,
                             p.tma_stores ? &map_c : nullptr, [&] {
                                 // this warp's sums are in registers: one arrival on the leader's barrier
                                 asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                                 __syncwarp();
                                 if (lane == 0)
                                     mbar_arrive_cluster(map_to_cta(smem_u32(&acc_empty[buf]), 0));
                             });
        }
        if (lane == 0)
            asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }

    // ---------------- teardown ----------------
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (*abort_flag) {
        // a wait ran out: let loads in flight land and MMAs retire (both bounded) before
        // the shared memory and tensor memory are given back
        if (warp == 1 && lane == 0 && leader) {
            umma_pair_commit(smem_u32(drain_bar));
            const long long t0 = clock64();
            while (!mbar_try_wait_cluster(drain_bar, 0)) {
                if (clock64() - t0 > kWaitCycles) {
                    atomicExch(p.status, ERR_DRAIN_WAIT);
                    break;
                }
            }
        }
        for (int i = 0; i < 200; ++i)
            __nanosleep(1000);
        __syncthreads();
    }
    // neither CTA may leave while the other can still reach its barriers, shared memory or accumulators
    cluster_sync();
    if (warp == 1) {
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(2 * kPairBN)
                     : "memory");
    }
}

// ---- one tile per CTA, or per cluster ----
constexpr int kSplitBN = 128;
constexpr int kMaxStages = 6;
constexpr int kSplitWarps = 8;  // epilogue
constexpr int kSplitThreads = 64 + 32 * kSplitWarps;
constexpr int kSplitMost = 227 * 1024;
constexpr int kSplitBars = (2 * kMaxStages + 3) * 8 + 16;
constexpr int kSplitSides = (2 * kSplitBN + kBM) * 4;  // scales and biases of columns, scales of rows
// [CTAs of the cluster][their share of the 128 rows][32 units of four columns] of the others' partial sums
constexpr int kPartialBytes = kBM * kSplitBN * 4;
inline int split_dynamic(int stages, int a_bytes, int csplit) {
    return stages * (a_bytes + kTileBytes) + (csplit > 1 ? kPartialBytes : 0) + kSplitSides + kSplitBars + 1024;
}

// The cluster's partial sums of this CTA's share of the rows: a row per warp, four columns per lane. The others'
// have come by bulk copies between the CTAs' shared memories, 16 KB or so in one. (16-byte loads from there took 2.1 us,
// 16-byte stores to there 2.5.)
template <class T, int SPLIT>
__device__ __forceinline__ void finish_rows(
        const uint8_t* own, const uint8_t* partials, int rank, int m0, int n0, const float* col_scale,
        const float* col_bias,
        const float* row_scale, const UmmaArgs& p) {
    constexpr int kShare = kBM / SPLIT;
    const int warp = (int)(threadIdx.x >> 5) - 2, lane = threadIdx.x & 31;
    const int col = n0 + 4 * lane;
    const float4 s = *(const float4*)(col_scale + 4 * lane);
    const float4 b = p.bias ? *(const float4*)(col_bias + 4 * lane) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 2
    for (int r = warp; r < kShare; r += kSplitWarps) {
        const int m = m0 + rank * kShare + r;
        if (m >= p.m)
            break;
        uint32_t v[4] = {0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < SPLIT; ++j) {
            const uint8_t* row = j == rank ? own + (rank * kShare + r) * 512 : partials + (j * kShare + r) * 512;
            const uint4 x = *(const uint4*)(row + ((lane & ~7) + ((lane ^ r) & 7)) * 16);
            v[0] += x.x;
            v[1] += x.y;
            v[2] += x.z;
            v[3] += x.w;
        }
        const float sa = row_scale[rank * kShare + r];
        float f[4] = {scale_acc((int)v[0], sa, s.x), scale_acc((int)v[1], sa, s.y), scale_acc((int)v[2], sa, s.z),
                      scale_acc((int)v[3], sa, s.w)};
        if (p.bias) {
            f[0] = __fadd_rn(f[0], b.x);
            f[1] = __fadd_rn(f[1], b.y);
            f[2] = __fadd_rn(f[2], b.z);
            f[3] = __fadd_rn(f[3], b.w);
        }
        T* c = (T*)p.c + (long long)m * p.ldc + col;
        if (p.vector_stores && col + 4 <= p.n) {
            const uint4 u = Out<T>::unit4(f);
            if (sizeof(T) == 4)
                *(uint4*)c = u;
            else
                *(uint2*)c = make_uint2(u.x, u.y);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (col + j < p.n)
                    c[j] = Out<T>::one(f[j]);
        }
    }
}

template <class T>
__global__ void __launch_bounds__(kSplitThreads, 2) product_split_kernel(
        const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const UmmaArgs p) {
    extern __shared__ uint8_t smem_raw[];
    // (the same offset in all CTAs of a cluster)
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    const int stage_bytes = p.a_bytes + kTileBytes;
    uint8_t* partials = smem + p.stages * stage_bytes;
    float* col_scale = (float*)(partials + (p.csplit > 1 ? kPartialBytes : 0));
    float* col_bias = col_scale + kSplitBN;
    float* row_scale = col_bias + kSplitBN;
    uint64_t* full_bar = (uint64_t*)(row_scale + kBM);
    uint64_t* empty_bar = full_bar + kMaxStages;
    uint64_t* acc_full = empty_bar + kMaxStages;
    uint64_t* part_bar = acc_full + 1;  // the others' partial sums
    uint64_t* drain_bar = part_bar + 1;
    uint32_t* tmem_slot = (uint32_t*)(drain_bar + 1);
    volatile int* abort_flag = (volatile int*)(tmem_slot + 1);
    volatile int* never = (volatile int*)(tmem_slot + 2);

    const int warp = uniform_warp_index(), lane = threadIdx.x & 31;
    const int rank = p.csplit > 1 ? (int)cluster_rank() : 0;
    const Tile t = tile_at((int)blockIdx.x / p.csplit, p.m_tiles, p.n_tiles);
    const int m0 = t.m * kBM, n0 = t.n * kSplitBN;
    const int k0 = (int)((long long)p.k_steps * rank / p.csplit);
    const int k1 = (int)((long long)p.k_steps * (rank + 1) / p.csplit);

    if (threadIdx.x == 0) {
        for (int s = 0; s < p.stages; ++s) {
            mbar_init(&full_bar[s], 1);
            mbar_init(&empty_bar[s], 1);
        }
        mbar_init(acc_full, 1);
        mbar_init(part_bar, 1);
        mbar_init(drain_bar, 1);
        *abort_flag = *never = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        if (p.csplit > 1)
            mbar_expect_tx(part_bar, (uint32_t)((p.csplit - 1) * (kPartialBytes / p.csplit)));
    } else if (threadIdx.x == 64) {
        tma_prefetch_map(&map_a);
        tma_prefetch_map(&map_b);
    }
    if (warp == 1) {
        asm volatile(
                "tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                "r"(kSplitBN)
                : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem_base = *tmem_slot;
    if (p.csplit > 1)
        cluster_arrive();  // (waited for before anything is stored in another CTA: all of them must have begun)

    auto give_up = [&](int code) {
        if (!*abort_flag) {
            *abort_flag = 1;
            atomicExch(p.status, code);
        }
    };

    bool waited = false;  // for the cluster's first barrier
    if (warp == 0) {
        // ---------------- TMA producer ----------------
        if (lane == 0) {
            const uint32_t bytes = (uint32_t)(p.a_rows * kBK + kTileBytes);
            int ahead = k0;
            if (p.b_early)
                for (; ahead < min(k0 + p.stages, k1); ++ahead) {
                    uint8_t* at = smem + (ahead - k0) * stage_bytes;
                    mbar_expect_tx(&full_bar[ahead - k0], bytes);
                    tma_load_2d(at + p.a_bytes, &map_b, &full_bar[ahead - k0], ahead * kBK, n0);
                }
            pdl_start();
            int s = 0;
            uint32_t phase = 0;
            for (int it = k0; it < k1; ++it) {
                const bool ok = mbar_wait(&empty_bar[s], phase ^ 1u, abort_flag);
                if (!ok) {
                    give_up(ERR_PRODUCER_WAIT);
                    break;
                }
                uint8_t* at = smem + s * stage_bytes;
                if (it >= ahead) {
                    mbar_expect_tx(&full_bar[s], bytes);
                    tma_load_2d(at + p.a_bytes, &map_b, &full_bar[s], it * kBK, n0);
                }
                tma_load_2d(at, &map_a, &full_bar[s], it * kBK, m0);
                if (++s == p.stages) {
                    s = 0;
                    phase ^= 1u;
                }
            }
        }
    } else if (warp == 1) {
        // ---------------- MMA issuer (the whole warp waits, one lane issues) ----------------
        const uint32_t leader = elect_one() ? 1u : 0u;
        constexpr uint32_t idesc = umma_idesc_s8(kBM, kSplitBN);
        const uint64_t a0 = umma_smem_desc(smem_u32(smem), 16, 1024, 2);
        const uint64_t b0 = umma_smem_desc(smem_u32(smem + p.a_bytes), 16, 1024, 2);
        const uint32_t a_hi = (uint32_t)(a0 >> 32), b_hi = (uint32_t)(b0 >> 32);
        uint32_t a_lo = (uint32_t)a0, b_lo = (uint32_t)b0, phase = 0, acc = 0;
        const uint32_t full_a = smem_u32(full_bar), empty_a = smem_u32(empty_bar);
        int s = 0;
        bool ok = true;
        for (int it = k0; it < k1; ++it) {
            ok = mbar_wait_u32(full_a + 8 * s, phase, abort_flag);
            if (!ok) {
                give_up(ERR_MMA_WAIT);
                break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
            for (int k = 0; k < kBK / 32; ++k) {
                umma_s8(leader, tmem_base, a_lo + k * 2, a_hi, b_lo + k * 2, b_hi, idesc, acc);
                acc = 1;
            }
            umma_commit_if(leader, empty_a + 8 * s);
            a_lo += (uint32_t)stage_bytes / 16;
            b_lo += (uint32_t)stage_bytes / 16;
            if (++s == p.stages) {
                s = 0;
                phase ^= 1u;
                a_lo = (uint32_t)a0;
                b_lo = (uint32_t)b0;
            }
        }
        if (ok)
            umma_commit_if(leader, smem_u32(acc_full));
        __syncwarp();
    } else {
        // ---------------- epilogue ----------------
        const int q = warp & 3, half = (warp - 2) >> 2;
        const int et = (int)threadIdx.x - 64;
        const int row0 = m0 + q * 32;
        pdl_start();
        if (et < kSplitBN) {
            col_scale[et] = n0 + et < p.n ? p.sb[n0 + et] : 0.f;
            if (p.bias)
                col_bias[et] = n0 + et < p.n ? p.bias[n0 + et] : 0.f;
        } else {
            row_scale[et - kBM] = m0 + et - kBM < p.m ? p.sa[m0 + et - kBM] : 0.f;
        }
        epilogue_sync<kSplitWarps>();
        const float sa = row_scale[q * 32 + lane];
        bool ok = mbar_wait(acc_full, 0, abort_flag);
        if (!ok)
            give_up(ERR_EPILOGUE_WAIT);
        ok = __all_sync(0xffffffffu, ok);
        // Behind the last MMA all loads have landed and been read: the stages are free.
        if (ok) {
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t taddr = tmem_base + ((uint32_t)(q * 32) << 16);
            if (p.csplit == 1) {
                uint8_t* stage = smem + (warp - 2) * kRoundBytes;
                if (row0 < p.m && n0 + half * 64 < p.n) {
                    Sides sides;
                    sides.take(sa, col_scale + half * 64, col_bias + half * 64, p.bias != nullptr);
                    store_columns<T>(taddr + (uint32_t)(half * 64), sides, p.bias != nullptr, stage, row0,
                                     n0 + half * 64, p, nullptr, [] {});
                }
            } else if (row0 < p.m) {
                // the partial sums, [128 rows][32 units of four columns], units in an order by row
                const int row = q * 32 + lane;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t acc[32];
                    __syncwarp();
                    tmem_ld32(taddr + (uint32_t)(half * 64 + 32 * h), acc);
#pragma unroll
                    for (int u = 0; u < 8; ++u)
                        *(uint4*)(smem + row * 512 + ((half * 2 + h) * 8 + (u ^ (row & 7))) * 16) =
                                make_uint4(acc[4 * u], acc[4 * u + 1], acc[4 * u + 2], acc[4 * u + 3]);
                }
            }
        }
        if (p.csplit > 1) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            cluster_wait();  // (all CTAs have begun)
            waited = true;
            epilogue_sync<kSplitWarps>();
            const int share_bytes = kPartialBytes / p.csplit;
            if (ok && warp == 2 && lane < p.csplit && lane != rank)
                // each CTA its share of the rows
                asm volatile(
                        "cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                                map_to_cta(smem_u32(partials + rank * share_bytes), (uint32_t)lane)),
                        "r"(smem_u32(smem + lane * share_bytes)), "r"(share_bytes),
                        "r"(map_to_cta(smem_u32(part_bar), (uint32_t)lane))
                        : "memory");
            __syncwarp();
            ok = mbar_wait_cluster(part_bar, 0, abort_flag);
            if (!ok)
                give_up(ERR_EPILOGUE_WAIT);
            ok = __all_sync(0xffffffffu, ok);
            if (ok) {
                if (p.csplit == 2)
                    finish_rows<T, 2>(smem, partials, rank, m0, n0, col_scale, col_bias, row_scale, p);
                else if (p.csplit == 4)
                    finish_rows<T, 4>(smem, partials, rank, m0, n0, col_scale, col_bias, row_scale, p);
                else
                    finish_rows<T, 8>(smem, partials, rank, m0, n0, col_scale, col_bias, row_scale, p);
            }
        }
    }

    if (p.csplit > 1) {
        // nobody leaves before what it sends has arrived
        __syncwarp();
        if (!waited)
            cluster_wait();
        cluster_arrive();
        cluster_wait();
    }

    // ---------------- teardown ----------------
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (*abort_flag) {
        if (warp == 1 && lane == 0) {
            umma_commit(drain_bar);
            const bool ok = mbar_wait(drain_bar, 0, never);
            if (!ok)
                atomicExch(p.status, ERR_DRAIN_WAIT);
        }
        for (int i = 0; i < 200; ++i)
            __nanosleep(1000);
        __syncthreads();
    }
    if (warp == 1) {
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kSplitBN)
                     : "memory");
    }
}

// a matrix of rows of `cols` elements, `pitch` bytes apart, in boxes of rows of 128 (operands) or 64 bytes (results)
int encode_as(
        CUtensorMap* map, CUtensorMapDataType type, const void* p, int cols, int rows, long long pitch, int box_cols,
        int box_rows, CUtensorMapSwizzle swizzle) {
    const DriverApi& api = driver_api();
    if (!api.ok)
        return set_error(ST_RUNTIME, "cuTensorMapEncode* entry points not found in the driver");
    cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    // (a single row may name any pitch, the map wants whole 16-byte units all the same)
    cuuint64_t strides[1] = {rows == 1 ? (cuuint64_t)cols * 4 / 16 * 16 + 16 : (cuuint64_t)pitch};
    cuuint32_t box[2] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows};
    cuuint32_t estr[2] = {1, 1};
    const CUresult r = api.tiled(
            map, type, 2, (void*)p, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? ST_SUCCESS : set_error(ST_RUNTIME, "cuTensorMapEncodeTiled failed: %d", (int)r);
}

int encode(CUtensorMap* map, const void* p, int k, int rows, long long pitch, int box_rows) {
    return encode_as(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, p, k, rows, pitch, kBK, box_rows,
                     CU_TENSOR_MAP_SWIZZLE_128B);
}

// Which kernel, by the clocks of its busiest SM. A 128-byte step of K takes a 128 x 128 tile's SM 512 clocks and
// a pair's two 560 at 256 columns (shared memory: the bytes of A's and B's rows in and out); in front of the first
// step and behind the last one stand the loads' round trip and the epilogue, with a cluster's exchange where K is split.
struct Choice {
    bool pair;
    int bn, csplit;
};
template <class Fit>
Choice choose(const UmmaArgs& p, int sms, Fit clusters_that_fit) {
    const long long steps = p.k_steps;
    long long best = LLONG_MAX;
    Choice c = {true, kPairBN, 1};
    for (int bn = kPairBN; bn >= 128; bn -= 64) {
        const long long pair_tiles = (long long)((p.m - 1) / (2 * kBM) + 1) * ((p.n - 1) / bn + 1);
        const long long tile = steps * (48 + 256 + bn), least = 12 * bn;  // (the epilogue's)
        const long long t = (pair_tiles + sms / 2 - 1) / (sms / 2) * (tile < least ? least : tile) + 6000;
        if (t < best) {
            best = t;
            c.bn = bn;
        }
    }
    const long long tiles = (long long)((p.m - 1) / kBM + 1) * ((p.n - 1) / kSplitBN + 1);
    for (int split = 1; split <= 8; split *= 2) {
        if (split > steps || (split > 1 && tiles > clusters_that_fit(split)))
            break;
        // one row of tiles reads its weights once: HBM bounds, not the SM that has a tile more (149 tiles of K = 2048 as
        // pairs in two turns 16.7 us, 11.2 so)
        const long long ctas = tiles * split;
        const long long turns16 = p.m <= kBM && split == 1 && ctas > sms ? 16 * ctas / sms + 1 : (ctas + sms - 1) / sms * 16;
        const long long t = turns16 * ((steps + split - 1) / split * 512 + 2500) / 16 + (split > 1 ? 5500 : 1000);
        if (t < best) {
            best = t;
            c = {false, kSplitBN, split};
        }
    }
    return c;
}

template <class T>
int launch(const ProductArgs& a, UmmaArgs p, const Writes& writes, cudaStream_t st) {
    const int sms = sm_count();
    static ClusterCapacity split_capacity;
    static KernelReady split_ready;
    if (!split_ready.smem(product_split_kernel<T>, kSplitMost))
        return check_launch("matmul_s8_scaled smem attribute");
    const Choice choice = choose(p, sms, [&](int split) {
        return split_capacity.clusters(product_split_kernel<T>, split, kSplitThreads, split_dynamic(3, kTileBytes, split));
    });
    CUtensorMap map_a, map_b;
    cudaError_t e;
    if (choice.pair) {
        static KernelReady ready;
        static ClusterCapacity capacity;
        if (!ready.smem(product_pair_kernel<T>, kPairDynamic))
            return check_launch("matmul_s8_scaled smem attribute");
        p.m_tiles = (p.m - 1) / (2 * kBM) + 1;
        p.bn = choice.bn;
        p.n_tiles = (p.n - 1) / p.bn + 1;
        int rc = encode(&map_a, a.a, a.k, a.m, a.lda, kBM);
        if (!rc)
            rc = encode(&map_b, a.b, a.k, a.n, a.ldb, p.bn / 2);
        CUtensorMap map_c = map_b;  // (not used where the TMA does not store)
        p.tma_stores = p.vector_stores && (size_t)a.n * sizeof(T) % 16 == 0;
        if (!rc && p.tma_stores)
            rc = encode_as(&map_c,
                           a.c_dtype == DT_F32   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                           : a.c_dtype == DT_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                           a.c, a.n, a.m, a.ldc * (long long)sizeof(T), 64 / (int)sizeof(T), 32,
                           CU_TENSOR_MAP_SWIZZLE_64B);
        if (rc)
            return rc;
        const long long total = (long long)p.m_tiles * p.n_tiles;
        const int fit = capacity.clusters(product_pair_kernel<T>, 2, kPairThreads, kPairDynamic);
        const int clusters = (int)(total < fit ? total : fit);
        e = launch_pdl(writes, product_pair_kernel<T>, dim3((unsigned)(2 * clusters)), dim3(kPairThreads), kPairDynamic,
                       st, map_a, map_b, map_c, p);
    } else {
        p.m_tiles = (p.m - 1) / kBM + 1;
        p.n_tiles = (p.n - 1) / kSplitBN + 1;
        p.csplit = choice.csplit;
        p.a_rows = p.m >= kBM ? kBM : (p.m + 7) / 8 * 8;
        const long long ctas = (long long)p.m_tiles * p.n_tiles * p.csplit;
        p.a_bytes = (p.a_rows * kBK + 1023) / 1024 * 1024;
        // With more CTAs than SMs two share one, one's epilogue beside the other's loads: half the shared memory for
        // each. Otherwise all of it (61 x 14336 x 4096: 13.0 us, 15.0 with half, although the next product's
        // first weights could then be fetched beside this one)
        const int room = (p.csplit == 1 && ctas > sms ? 112 << 10 : kSplitMost) - split_dynamic(0, 0, p.csplit);
        p.stages = room / (p.a_bytes + kTileBytes);
        if (p.stages > kMaxStages)
            p.stages = kMaxStages;
        int rc = encode(&map_a, a.a, a.k, a.m, a.lda, p.a_rows);
        if (!rc)
            rc = encode(&map_b, a.b, a.k, a.n, a.ldb, kSplitBN);
        if (rc)
            return rc;
        e = launch_pdl_cluster(writes, product_split_kernel<T>, dim3((unsigned)ctas), dim3(kSplitThreads),
                               (size_t)split_dynamic(p.stages, p.a_bytes, p.csplit), p.csplit, st, map_a, map_b, p);
    }
    if (e != cudaSuccess)
        return refused("matmul_s8_scaled", e);
    return check_launch("matmul_s8_scaled");
}

}  // namespace

int launch_product_umma(const ProductArgs& a, cudaStream_t st) {
    UmmaArgs p{};
    p.m = a.m, p.n = a.n;
    p.k_steps = (a.k + kBK - 1) / kBK;
    p.sa = a.sa, p.sb = a.sb, p.bias = a.bias;
    p.c = a.c, p.ldc = a.ldc;
    const size_t size = dtype_bytes(a.c_dtype);
    p.vector_stores = ((uintptr_t)a.c & 15) == 0 && (a.m == 1 || (size_t)a.ldc * size % 16 == 0);
    p.b_early = a.b_early;
    p.status = device_status_word(st);
    if (!p.status)
        return ST_MALLOC;
    const Writes writes{a.c, ((size_t)(a.m - 1) * (size_t)a.ldc + (size_t)a.n) * size};
    return a.c_dtype == DT_F32   ? launch<float>(a, p, writes, st)
           : a.c_dtype == DT_F16 ? launch<__half>(a, p, writes, st)
                                 : launch<__nv_bfloat16>(a, p, writes, st);
}

}  // namespace scaled
}  // namespace mb200
