// What the mixture-of-experts kernels take, by value.
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace mb200 {
namespace scaled {

constexpr int kMoeMaxTokens = 64, kMoeMaxTop = 16, kMoeMaxExperts = 512;
// the tokens' whole numbers lie in shared memory: eight rows (sixteen with more than eight tokens)
constexpr int kMoeMaxDepthFew = 16384, kMoeMaxDepth = 8192;

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
    size_t workspace_bytes;
};

int launch_moe(const MoeArgs& a, cudaStream_t st);

}  // namespace scaled
}  // namespace mb200
