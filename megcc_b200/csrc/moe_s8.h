// What the mixture-of-experts kernels take, by value.
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#if defined(__CUDACC__)
#define MB200_HD __host__ __device__
#else
#define MB200_HD
#endif

namespace mb200 {
namespace scaled {

constexpr int kMoeMaxTokens = 64, kMoeMaxTop = 16, kMoeMaxExperts = 512;
// the tokens' whole numbers lie in shared memory: eight rows (sixteen with more than eight tokens)
constexpr int kMoeMaxDepthFew = 16384, kMoeMaxDepth = 8192;

// up to here every CTA routes all tokens itself
constexpr int kMoeFew = 4;

// The routing, as the kernels keep it: bytes for `slots` token-expert pairs in passes of `cols` tokens at most
MB200_HD constexpr int up16(int v) {
    return (v + 15) / 16 * 16;
}
// every expert with tokens, and one more for each `cols` slots
MB200_HD constexpr int most_passes(int slots, int experts, int cols) {
    return (slots < experts ? slots : experts) + slots / cols;
}
MB200_HD constexpr int route_bytes(int slots, int experts, int cols) {
    return 2 * up16(4 * slots) + 3 * up16(2 * most_passes(slots, experts, cols)) + 16;
}
struct MoeArgs {
    int t, d, f, e, top, renormalize, dtype;
    const void* x;
    long long ldx;
    const float* logits;
    const int8_t *w1, *w2;
    const float *s1, *s2;
    void* y;
    long long ldy;
    // the hidden layer: [slots][f rounded up to 32] whole numbers, [slots][f / 32 rounded up] scales
    int8_t* hq;
    float* sh;
    // more than kMoeFew tokens: their routing, and they as whole numbers in rows of xs_pitch(d), with their scales
    uint4* route;
    int8_t* xq;
    float* sx;
    size_t workspace_bytes;
};

int launch_moe(const MoeArgs& a, cudaStream_t st);

}  // namespace scaled
}  // namespace mb200
