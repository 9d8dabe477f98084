// What the operators on the int8 cache of keys and values and the attention kernels take, by value.
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "../../include/megcc_b200.h"

namespace mb200 {
namespace attn {

constexpr int kBlock = MB200_KV_BLOCK;  // positions of a head that share a scale
constexpr int kMaxD = 128;
constexpr int kTurnSteps = 8;  // steps of rows of queries that a warp turns

// recorded in the device status word
enum : int {
    ERR_PAGE = 0x201,      // a position whose page is not in the table, or not in the pool
    ERR_POSITION = 0x202,  // a position beyond the rotation's tables
};

struct AppendArgs {
    mb200_kv_cache c;
    const int32_t *lengths, *cu;
    int tokens, slots;
    mb200_heads k, v, q, k_out, q_out;  // q.p, k_out.p null: not asked for
    int heads, chunks;                  // chunks: warps a token's queries take
    const float *cosines, *sines;       // null: nothing is turned
    int positions, rot, interleaved;
    int* status;
};
int launch_append(const AppendArgs& a, int dtype, cudaStream_t st);

struct ReadArgs {
    mb200_kv_cache c;
    const int32_t *starts, *cu;
    int tokens;
    mb200_heads k, v;
    int* status;
};
int launch_read(const ReadArgs& a, int dtype, cudaStream_t st);

struct CacheArgs {
    mb200_kv_cache c;
    const int32_t* lengths;
    int heads, queries;
    mb200_heads q, out;  // token stride: from one query of a sequence to the next; sequences lie `queries` tokens apart
    float scale_log2;    // scale * log2(e)
    void* workspace;
    int* status;
};
size_t attention_cache_workspace(const mb200_kv_cache& c, int heads, int queries);
int launch_attention_cache(const CacheArgs& a, int dtype, cudaStream_t st);


struct PromptArgs {
    int batch, tokens, key_tokens, heads, kv_heads, d;
    const int32_t *cu_q, *cu_k;
    mb200_heads q, k, v, out;
    int causal, pack;  // pack: log2 of the query heads of a group that share a tile
    float scale_log2;
    int* status;
};
int attention_prompt_pack(const mb200_heads& q, int tokens, int heads, int kv_heads, int d);
long long attention_prompt_ctas(int tokens, int batch, int heads, int pack);
int launch_attention_prompt(const PromptArgs& a, int dtype, cudaStream_t st);

}  // namespace attn
}  // namespace mb200
