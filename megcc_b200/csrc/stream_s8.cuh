// Weights streamed through a warp's own ring of shared memory into mma.sync: what the kernels for few
// tokens have in common. HBM is what bounds them, so the ring's only job is to keep enough bytes on their way
// (an SM's share of 6.5 TB/s times a microsecond is 45 KB). Asynchronous copies do that without registers, and
// in order: a ring in registers made the compiler wait for the youngest load with the oldest (0.86 us a
// step of the second expert kernel, the whole latency of a load). A warp fills and reads its ring
// alone, so no barrier of the CTA stands in the stream.
//
// A step is 128 bytes of K of each of 16 rows: whole lines, and few enough instructions per byte (with 64 bytes
// the expert kernels took 100 to 230 of them per KB and were bound by their issue: 33 us for 100 MB). Rows may
// start at any byte: ALIGNED rows are eight 16-byte units, others the nine units that hold their 128 bytes,
// shifted into place when they are read. WIDE: 16 bytes by two 16-byte loads and selects, where loads of shared memory
// bound (12 x 4096 x 4104 in 7.4 us, by five 4-byte loads, four lanes of them on each bank, in 11.7); otherwise by those,
// with half the registers and instructions (two experts of 1928 x 800: 11.4 us, 12.1 with WIDE).
#pragma once
#include "scaled_s8.cuh"

namespace mb200 {
namespace scaled {

constexpr int kStep = 128;

__device__ __forceinline__ void copy_async16(uint32_t smem, const void* p, bool there) {
    asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(smem), "l"(p), "r"(there ? 16 : 0)
                 : "memory");
}
__device__ __forceinline__ void copy_async16(uint32_t smem, const void* p) {
    asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16;" ::"r"(smem), "l"(p) : "memory");
}
__device__ __forceinline__ void copy_async4(uint32_t smem, const void* p) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem), "l"(p) : "memory");
}
__device__ __forceinline__ void copy_async4(uint32_t smem, const void* p, bool there) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem), "l"(p), "r"(there ? 4 : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() {
    asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void copy_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint32_t shared_address(const void* p) {
    return (uint32_t)__cvta_generic_to_shared(p);
}
__device__ __forceinline__ uint4 lds16(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
    return v;
}
__device__ __forceinline__ uint2 lds8(uint32_t at) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at));
    return v;
}
__device__ __forceinline__ uint32_t lds4(uint32_t at) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(at));
    return v;
}

// ROWS rows of a step in shared memory
template <int ROWS, bool ALIGNED, bool WIDE = false>
struct Rows {
    static constexpr int kUnits = ALIGNED ? 8 : 9;
    static constexpr int kPitch = 16 * kUnits;
    static constexpr int kBytes = ROWS * kPitch;
    static constexpr int kCopies = (ROWS * kUnits + 31) / 32;  // of a lane, per step

    // Where a unit lies: a read of 16 (8) bytes by the lanes of two (four) rows meets every bank once. Eight units are
    // rearranged within their row; with nine each row begins a unit further round the banks, so the rows are.
    static __device__ __forceinline__ int unit_at(int row, int unit) {
        if (ALIGNED)
            return row * kPitch + (unit ^ (((row & 1) << 2) | (row & 2))) * 16;
        return (WIDE ? (row & ~7) | (row & 6) >> 1 | (row & 1) << 2 : row) * kPitch + unit * 16;
    }

    // what a lane copies next: its units' places in global memory, and how far their rows go from there
    const int8_t* from[kCopies];
    int left[ALIGNED ? 1 : kCopies];
    uint32_t there;      // a bit per copy: its row is one to read
    const int8_t* any;   // an address for copies of nothing
    int to[kCopies];     // in the stage

    // (once per kernel: the places in the stage)
    __device__ __forceinline__ Rows() {
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int i = 0; i < kCopies; ++i) {
            const int q = lane + 32 * i, r = q / kUnits, u = q % kUnits;
            to[i] = unit_at(r, u);
        }
    }
    // row(r): address of row r, or null for one that is not there (row 0 is); k: its bytes; step: the first
    template <class RowAt>
    __device__ __forceinline__ void open(RowAt row, int k, int step) {
        const int lane = threadIdx.x & 31;
        any = row(0);
        any -= (uintptr_t)any & 15;
        there = 0;
#pragma unroll
        for (int i = 0; i < kCopies; ++i) {
            const int q = lane + 32 * i, r = q / kUnits, u = q % kUnits;
            const int8_t* p = ROWS * kUnits % 32 == 0 || r < ROWS ? row(r) : nullptr;
            if (p)
                there |= 1u << i;
            // (a unit is read if it holds at least one byte of the row)
            const int s = ALIGNED ? 0 : (int)((uintptr_t)p & 15);
            from[i] = (p ? p - s : any) + step * kStep + 16 * u;
            if (!ALIGNED || i == 0)
                left[i] = k + s - 16 * u - step * kStep;
        }
    }
    // The next step; `by`: how many steps further the one behind it is. whole: rows go on for kWhole bytes at
    // least, the same for all lanes (every step but a row's last: those that it has zeros behind). Rows that are not
    // there are left out: what stands in their place is multiplied, and its column of the result not looked at.
    static constexpr int kWhole = 16 * kUnits;
    template <bool ALL_THERE>
    __device__ __forceinline__ void copy(uint32_t stage, int by, bool whole) {
        const int lane = threadIdx.x & 31;
        if (whole) {
#pragma unroll
            for (int i = 0; i < kCopies; ++i)
                if ((ROWS * kUnits % 32 == 0 || lane + 32 * i < ROWS * kUnits) && (ALL_THERE || (there >> i & 1)))
                    copy_async16(stage + to[i], from[i]);
        } else {
#pragma unroll
            for (int i = 0; i < kCopies; ++i)
                if ((ROWS * kUnits % 32 == 0 || lane + 32 * i < ROWS * kUnits) && (ALL_THERE || (there >> i & 1))) {
                    const bool some = left[ALIGNED ? 0 : i] > 0;
                    copy_async16(stage + to[i], some ? from[i] : any, some);
                }
        }
#pragma unroll
        for (int i = 0; i < kCopies; ++i) {
            from[i] += by * kStep;
            if (!ALIGNED || i == 0)
                left[i] -= by * kStep;
        }
    }
    // 16 bytes of row r from byte 16 * part on; s: the row's address modulo 16
    static __device__ __forceinline__ uint4 piece16(uint32_t stage, int r, int part, int s) {
        const uint32_t at = stage + unit_at(r, part);
        if (ALIGNED)
            return lds16(at);
        uint32_t w[8];
        if (WIDE) {
            const uint4 lo = lds16(at), hi = lds16(at + 16);
            w[0] = lo.x, w[1] = lo.y, w[2] = lo.z, w[3] = lo.w, w[4] = hi.x, w[5] = hi.y, w[6] = hi.z, w[7] = hi.w;
#pragma unroll
            for (int i = 0; i < 6; ++i)
                w[i] = s & 8 ? w[i + 2] : w[i];
#pragma unroll
            for (int i = 0; i < 5; ++i)
                w[i] = s & 4 ? w[i + 1] : w[i];
        } else {
#pragma unroll
            for (int i = 0; i < 5; ++i)
                w[i] = lds4(at + (s & ~3) + 4 * i);
        }
        const int bits = (s & 3) * 8;
        return make_uint4(__funnelshift_r(w[0], w[1], bits), __funnelshift_r(w[1], w[2], bits),
                          __funnelshift_r(w[2], w[3], bits), __funnelshift_r(w[3], w[4], bits));
    }
    // 8 bytes from byte 8 * part on
    static __device__ __forceinline__ uint2 piece8(uint32_t stage, int r, int part, int s) {
        if (ALIGNED)
            return lds8(stage + unit_at(r, part >> 1) + (part & 1) * 8);
        // (words: two 8-byte loads and selects took 68 us where these took 63, 40 tokens, 45 experts, 1925 x 803)
        const uint32_t at = stage + unit_at(r, 0) + part * 8 + (s & ~3);
        const uint32_t a = lds4(at), b = lds4(at + 4), c = lds4(at + 8);
        const int bits = (s & 3) * 8;
        return make_uint2(__funnelshift_r(a, b, bits), __funnelshift_r(b, c, bits));
    }
};

// A place in a ring of DEPTH stages
template <int DEPTH, int BYTES>
__device__ __forceinline__ void next_stage(uint32_t& stage, uint32_t ring) {
    stage += BYTES;
    if (stage == ring + (uint32_t)(DEPTH * BYTES))
        stage = ring;
}

// the first `n` bytes (n <= 0: none) of 16
__device__ __forceinline__ uint4 first_bytes(uint4 v, int n) {
    auto cut = [](uint32_t w, int left) { return left >= 4 ? w : left <= 0 ? 0u : w & ((1u << (8 * left)) - 1u); };
    return make_uint4(cut(v.x, n), cut(v.y, n - 4), cut(v.z, n - 8), cut(v.w, n - 12));
}

// Rows of activations as whole numbers (in shared memory, or not), by the threads of a CTA; zeros behind each row up
// to whole steps. WARPS / rows warps (one at least) share a row, so that a few rows' loads are on their way
// together. row(r): a row's address; part: [rows][WARPS] words of shared memory. With FIRST > 0
// the warps from FIRST on do it (WARPS of them; barrier 1 is theirs). A barrier of the CTA has to follow before the
// rows are read. (Loops stay rolled here and in the kernels where their bodies are long: a launch
// fetches its instructions anew, and 115 KB of them cost the expert kernels 5 us each.)
template <class T, int WARPS, int FIRST = 0, class RowAt>
__device__ __forceinline__ void rows_to_whole(
        RowAt row, int rows, int k, int8_t* xs, int pitch, float* scale, uint32_t* part, bool vectors) {
    const int warp = (int)(threadIdx.x >> 5) - FIRST, lane = threadIdx.x & 31;
    const int share = rows >= WARPS ? 1 : rows * 2 >= WARPS ? 2 : rows * 4 >= WARPS ? 4 : WARPS;
    const int stride = share * 512, first = (warp % share * 32 + lane) * 16;
    // Elements taken 16 at a time; the others (of rows that start anywhere: all) 16 bytes at a time, through the
    // units that hold them
    const int in_vectors = vectors ? k & ~15 : 0;
    constexpr int V = Vec<T>::N, N = 16 / V;  // elements of a load, loads of 16 elements
    const int any_first = in_vectors + first / 16 * V, any_stride = share * 32 * V;
#pragma unroll 1
    for (int r = warp / share; r < rows; r += WARPS / share) {
        const T* x = (const T*)row(r);
        uint32_t vm = 0;
#pragma unroll 2
        for (int i = first; i < in_vectors; i += stride) {
            uint4 w[N];
#pragma unroll
            for (int j = 0; j < N; ++j)
                w[j] = ((const uint4*)(x + i))[j];
#pragma unroll
            for (int j = 0; j < N; ++j)
                vm = vec_max<T>(vm, w[j]);
        }
        uint32_t bits = max_bits<T>(vm);
#pragma unroll 1
        for (int i = any_first; i < k; i += any_stride)
            bits = max(bits, max_bits<T>(vec_max<T>(0, ld_any16((const int8_t*)(x + i), (k - i) * (int)sizeof(T)))));
        bits = __reduce_max_sync(0xffffffffu, bits);
        if (lane == 0)
            part[r * WARPS + warp % share] = bits;
    }
    if (FIRST == 0)
        __syncthreads();
    else
        asm volatile("bar.sync 1, %0;" ::"n"(32 * WARPS) : "memory");
    const int end = (k + kStep - 1) / kStep * kStep;
#pragma unroll 1
    for (int r = warp / share; r < rows; r += WARPS / share) {
        const T* x = (const T*)row(r);
        uint32_t bits = 0;
#pragma unroll 1
        for (int w = 0; w < share; ++w)
            bits = max(bits, part[r * WARPS + w]);
        const RowScale s = row_scale(bits);
        if (warp % share == 0 && lane == 0)
            scale[r] = s.scale;
        int8_t* to = xs + r * pitch;
#pragma unroll 1
        for (int i = first; i < in_vectors; i += stride) {
            float v[16];
#pragma unroll
            for (int j = 0; j < N; ++j)
                Vec<T>::unpack(((const uint4*)(x + i))[j], v + V * j);
            *(uint4*)(to + i) = pack_piece(v, s);
        }
#pragma unroll 1
        for (int i = any_first; i < end; i += any_stride) {
            float v[V];
            Vec<T>::unpack(ld_any16((const int8_t*)(x + i), (k - i) * (int)sizeof(T)), v);
#pragma unroll
            for (int j = 0; j < V; j += 4)
                *(uint32_t*)(to + i + j) = pack_whole(v[j], v[j + 1], v[j + 2], v[j + 3], s.inv) & s.keep;
        }
    }
}
// Asks for what the CTA's threads will read soon: `bytes` from p on, into the L1.
template <int THREADS>
__device__ __forceinline__ void ask_ahead(const void* p, int bytes) {
    const uintptr_t first = (uintptr_t)p & ~(uintptr_t)127;
    const int end = (int)((uintptr_t)p - first) + bytes;
#pragma unroll 1
    for (int at = threadIdx.x * 128; at < end; at += THREADS * 128)
        asm volatile("prefetch.global.L1 [%0];" ::"l"(first + at));
}

}  // namespace scaled
}  // namespace mb200
