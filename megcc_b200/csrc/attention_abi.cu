// extern "C" entry points of attention with the int8 cache of keys and values (include/megcc_b200.h).
#include <math.h>

#include "attention.h"
#include "internal.h"

using namespace mb200;
using namespace mb200::attn;

namespace {

constexpr float kLog2E = 1.44269504f;

bool misaligned(const void* p, size_t bytes) {
    return ((uintptr_t)p & (bytes - 1)) != 0;
}

int check_dtype(int dtype, const char* what) {
    if (dtype != MB200_DTYPE_F16 && dtype != MB200_DTYPE_BF16)
        return set_error(ST_UNSUPPORTED_DTYPE, "%s: type %d is neither fp16 nor bf16", what, dtype);
    return ST_SUCCESS;
}

int check_d(int d, const char* what) {
    if (d <= 0 || d % 16 != 0)
        return set_error(ST_INVALID_LAYOUT, "%s: heads of %d elements are no multiple of 16", what, d);
    if (d > kMaxD)
        return set_error(ST_OUT_OF_RANGE, "%s: heads of %d elements (at most %d)", what, d, kMaxD);
    return ST_SUCCESS;
}

int check_cache(const mb200_kv_cache* c, const char* what) {
    if (!c)
        return set_error(ST_NULL_PTR, "%s: the cache is NULL", what);
    const int rc = check_d(c->d, what);
    if (rc)
        return rc;
    if (c->pages <= 0 || c->kv_heads <= 0 || c->page_tokens <= 0 || c->page_tokens % kBlock != 0 || c->batch < 0 ||
        c->table_pages <= 0 || (c->batch > 1 && c->table_stride < c->table_pages))
        return set_error(ST_INVALID_LAYOUT, "%s: %d pages of %d positions, %d key heads, %d sequences of %d pages", what,
                         c->pages, c->page_tokens, c->kv_heads, c->batch, c->table_pages);
    // (blocks are counted in an int)
    if ((long long)c->kv_heads * (c->page_tokens / kBlock) > 0x7fffffffLL / c->pages)
        return set_error(ST_OUT_OF_RANGE, "%s: %d pages of %d heads and %d positions have more than 2^31 blocks", what,
                         c->pages, c->kv_heads, c->page_tokens);
    if (!c->k || !c->v || !c->k_scales || !c->v_scales || (!c->block_table && c->batch > 0))
        return set_error(ST_NULL_PTR, "%s: a pointer of the cache is NULL", what);
    if (misaligned(c->k, 16) || misaligned(c->v, 16) || misaligned(c->k_scales, 4) || misaligned(c->v_scales, 4) ||
        misaligned(c->block_table, 4))
        return set_error(ST_INVALID_LAYOUT, "%s: the cache must be 16-byte aligned, scales and table as their types are",
                         what);
    return ST_SUCCESS;
}

// heads of a token, and tokens, must not overlap where they are written; operands may lie in any way
int check_heads(const mb200_heads& t, int tokens, int heads, int d, bool written, const char* name, const char* what) {
    if (!t.p)
        return set_error(ST_NULL_PTR, "%s: %s is NULL", what, name);
    if (misaligned(t.p, 2))
        return set_error(ST_INVALID_LAYOUT, "%s: %s must be aligned as its type is", what, name);
    if (t.token_stride < 0 || t.head_stride < 0)
        return set_error(ST_INVALID_LAYOUT, "%s: strides of %s are negative", what, name);
    if (!written)
        return ST_SUCCESS;
    const bool by_token = (heads == 1 || t.head_stride >= d) &&
                          (tokens == 1 || t.token_stride >= (heads - 1) * t.head_stride + d);
    const bool by_head = (tokens == 1 || t.token_stride >= d) &&
                         (heads == 1 || t.head_stride >= (tokens - 1) * t.token_stride + d);
    if (!by_token && !by_head)
        return set_error(ST_INVALID_LAYOUT, "%s: rows of %s overlap", what, name);
    return ST_SUCCESS;
}

int check_grid(long long blocks, const char* what) {
    if (blocks > 0x7fffffffLL)
        return set_error(ST_OUT_OF_RANGE, "%s: too large for one launch", what);
    return ST_SUCCESS;
}

int status_word(void* stream, int** word) {
    *word = device_status_word((cudaStream_t)stream);
    return *word ? ST_SUCCESS : ST_RUNTIME;
}

int check_attention_cache(const mb200_kv_cache* c, int heads, int queries) {
    const char* what = "attention_cache_s8";
    const int rc = check_cache(c, what);
    if (rc)
        return rc;
    if (heads <= 0 || heads % c->kv_heads != 0 || queries <= 0)
        return set_error(ST_INVALID_LAYOUT, "%s: %d heads over %d key heads, %d queries", what, heads, c->kv_heads, queries);
    // (rows, and CTAs of the second launch, in an int)
    if ((long long)heads * queries > 0x7fffffffLL / (c->batch > 0 ? c->batch : 1))
        return set_error(ST_OUT_OF_RANGE, "%s: %d sequences of %d queries and %d heads", what, c->batch, queries, heads);
    return ST_SUCCESS;
}

// what the TMA takes: whole 16-byte units, heads and tokens apart
int check_units(const mb200_heads& t, int tokens, int heads, const char* name, const char* what) {
    if (misaligned(t.p, 16) || (tokens > 1 && (t.token_stride % 8 != 0 || t.token_stride == 0)) ||
        (heads > 1 && (t.head_stride % 8 != 0 || t.head_stride == 0)))
        return set_error(ST_INVALID_LAYOUT, "%s: %s must be 16-byte aligned, its strides multiples of 8 elements", what, name);
    if (t.token_stride >= 1LL << 38 || t.head_stride >= 1LL << 38)
        return set_error(ST_OUT_OF_RANGE, "%s: strides of %s", what, name);
    return ST_SUCCESS;
}

}  // namespace

extern "C" {

int mb200_kv_append_s8(const mb200_kv_cache* cache, const mb200_kv_append_param* p, void* stream) {
    const char* what = "kv_append_s8";
    if (!p)
        return set_error(ST_NULL_PTR, "%s: parameter block is NULL", what);
    int rc = check_cache(cache, what);
    if (!rc)
        rc = check_dtype(p->dtype, what);
    if (rc)
        return rc;
    const int d = cache->d;
    if (p->tokens < 0 || (!p->cu && p->tokens != cache->batch))
        return set_error(ST_INVALID_LAYOUT, "%s: %d tokens of %d sequences", what, p->tokens, cache->batch);
    if ((p->cosines == nullptr) != (p->sines == nullptr))
        return set_error(ST_NULL_PTR, "%s: cosines without sines", what);
    if (p->cosines && (p->rot_dims <= 0 || p->rot_dims > d || p->rot_dims % 16 != 0 || p->positions <= 0))
        return set_error(ST_INVALID_LAYOUT, "%s: %d elements turned of %d (a multiple of 16), %d positions", what,
                         p->rot_dims, d, p->positions);
    if (p->q.p && !p->cosines)
        return set_error(ST_INVALID_LAYOUT, "%s: queries are only turned, which needs cosines and sines", what);
    if (p->q.p && p->heads <= 0)
        return set_error(ST_INVALID_LAYOUT, "%s: %d query heads", what, p->heads);
    if (p->tokens == 0 || cache->batch == 0)
        return ST_SUCCESS;
    if (!p->lengths)
        return set_error(ST_NULL_PTR, "%s: lengths are NULL", what);
    rc = check_heads(p->k, p->tokens, cache->kv_heads, d, false, "k", what);
    if (!rc)
        rc = check_heads(p->v, p->tokens, cache->kv_heads, d, false, "v", what);
    if (!rc && p->k_out.p)
        rc = check_heads(p->k_out, p->tokens, cache->kv_heads, d, true, "k_out", what);
    if (!rc && p->q.p) {
        rc = check_heads(p->q, p->tokens, p->heads, d, false, "q", what);
        if (!rc)
            rc = check_heads(p->q_out, p->tokens, p->heads, d, true, "q_out", what);
    }
    if (rc)
        return rc;
    if (misaligned(p->lengths, 4) || misaligned(p->cu, 4) || misaligned(p->cosines, 4) || misaligned(p->sines, 4))
        return set_error(ST_INVALID_LAYOUT, "%s: lengths, cu, cosines and sines must be aligned as their types are", what);
    AppendArgs a{};
    a.c = *cache;
    a.lengths = p->lengths, a.cu = p->cu;
    a.tokens = p->tokens;
    const long long slots = p->cu ? p->tokens / kBlock + 2LL * cache->batch : p->tokens;
    a.k = p->k, a.v = p->v, a.q = p->q, a.k_out = p->k_out, a.q_out = p->q_out;
    a.heads = p->heads;
    const int rows = kTurnSteps * (32 / (d / 8));  // that a warp turns
    a.chunks = p->q.p ? (p->heads + rows - 1) / rows : 1;
    a.cosines = p->cosines, a.sines = p->sines;
    a.positions = p->positions, a.rot = p->cosines ? p->rot_dims : 0, a.interleaved = p->interleaved != 0;
    rc = check_grid(slots, what);
    if (!rc)
        rc = check_grid(2 * slots * cache->kv_heads + (p->q.p ? (long long)p->tokens * a.chunks : 0), what);
    if (!rc)
        rc = status_word(stream, &a.status);
    if (rc)
        return rc;
    a.slots = (int)slots;
    return launch_append(a, p->dtype, (cudaStream_t)stream);
}

int mb200_kv_read_s8(
        const mb200_kv_cache* cache, const int32_t* starts, const int32_t* cu, int tokens, int dtype,
        const mb200_heads* k, const mb200_heads* v, void* stream) {
    const char* what = "kv_read_s8";
    int rc = check_cache(cache, what);
    if (!rc)
        rc = check_dtype(dtype, what);
    if (rc)
        return rc;
    if (tokens < 0)
        return set_error(ST_INVALID_LAYOUT, "%s: %d tokens", what, tokens);
    if (tokens == 0 || cache->batch == 0)
        return ST_SUCCESS;
    if (!cu || !k || !v)
        return set_error(ST_NULL_PTR, "%s: cu or a result is NULL", what);
    rc = check_heads(*k, tokens, cache->kv_heads, cache->d, true, "k", what);
    if (!rc)
        rc = check_heads(*v, tokens, cache->kv_heads, cache->d, true, "v", what);
    if (rc)
        return rc;
    if (misaligned(starts, 4) || misaligned(cu, 4))
        return set_error(ST_INVALID_LAYOUT, "%s: starts and cu must be aligned as their types are", what);
    // (what a CTA counts: units of 16 rows of both tensors)
    if (cache->kv_heads > 0x7fffffff / (2 * 16 * 8))
        return set_error(ST_OUT_OF_RANGE, "%s: %d key heads", what, cache->kv_heads);
    ReadArgs a{};
    a.c = *cache;
    a.starts = starts, a.cu = cu, a.tokens = tokens;
    a.k = *k, a.v = *v;
    rc = status_word(stream, &a.status);
    return rc ? rc : launch_read(a, dtype, (cudaStream_t)stream);
}

size_t mb200_attention_cache_s8_workspace_bytes(const mb200_kv_cache* cache, int heads, int queries) {
    if (check_attention_cache(cache, heads, queries) || cache->batch == 0)
        return 0;
    return attention_cache_workspace(*cache, heads, queries);
}

int mb200_attention_cache_s8(
        const mb200_kv_cache* cache, const int32_t* lengths, int heads, int queries, int dtype, const mb200_heads* q,
        float scale, const mb200_heads* out, void* workspace, size_t workspace_bytes, void* stream) {
    const char* what = "attention_cache_s8";
    int rc = check_attention_cache(cache, heads, queries);
    if (!rc)
        rc = check_dtype(dtype, what);
    if (rc || cache->batch == 0)
        return rc;
    if (!isfinite(scale * kLog2E))
        return set_error(ST_INVALID_LAYOUT, "%s: the scale is not finite, or too large", what);
    if (!lengths || !q || !out)
        return set_error(ST_NULL_PTR, "%s: lengths, q or out is NULL", what);
    rc = check_heads(*q, cache->batch * queries, heads, cache->d, false, "q", what);
    if (!rc)
        rc = check_heads(*out, cache->batch * queries, heads, cache->d, true, "out", what);
    if (rc)
        return rc;
    if (misaligned(lengths, 4))
        return set_error(ST_INVALID_LAYOUT, "%s: lengths must be aligned as their type is", what);
    const size_t need = attention_cache_workspace(*cache, heads, queries);
    if (need && !workspace)
        return set_error(ST_NULL_PTR, "%s: needs a workspace of %zu bytes", what, need);
    if (need && (misaligned(workspace, 256) || workspace_bytes < need))
        return set_error(ST_INVALID_LAYOUT, "%s: the workspace must be 256-byte aligned and hold %zu bytes", what, need);
    CacheArgs a{};
    a.c = *cache;
    a.lengths = lengths, a.heads = heads, a.queries = queries;
    a.q = *q, a.out = *out;
    a.scale_log2 = scale * kLog2E;
    a.workspace = need ? workspace : nullptr;
    rc = status_word(stream, &a.status);
    return rc ? rc : launch_attention_cache(a, dtype, (cudaStream_t)stream);
}

int mb200_attention_prompt(
        int batch, const int32_t* cu_q, const int32_t* cu_k, int tokens, int key_tokens, int heads, int kv_heads, int d,
        int dtype, const mb200_heads* q, const mb200_heads* k, const mb200_heads* v, int causal, float scale,
        const mb200_heads* out, void* stream) {
    const char* what = "attention_prompt";
    int rc = check_dtype(dtype, what);
    if (!rc)
        rc = check_d(d, what);
    if (rc)
        return rc;
    if (batch < 0 || tokens < 0 || key_tokens < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 ||
        (!cu_k && key_tokens != tokens))
        return set_error(ST_INVALID_LAYOUT, "%s: %d sequences, %d tokens and %d of keys, %d heads over %d key heads", what,
                         batch, tokens, key_tokens, heads, kv_heads);
    if (!isfinite(scale * kLog2E))
        return set_error(ST_INVALID_LAYOUT, "%s: the scale is not finite, or too large", what);
    if (tokens == 0 || batch == 0)
        return ST_SUCCESS;
    if (!cu_q || !q || !k || !v || !out)
        return set_error(ST_NULL_PTR, "%s: an operand is NULL", what);
    // (no keys at all: there is nothing to look at, and zeros to write)
    const int some = key_tokens > 0 ? key_tokens : 1;
    PromptArgs a{};
    a.q = *q, a.k = key_tokens > 0 ? *k : *q, a.v = key_tokens > 0 ? *v : *q, a.out = *out;
    rc = check_heads(a.q, tokens, heads, d, false, "q", what);
    if (!rc)
        rc = check_heads(a.k, some, kv_heads, d, false, "k", what);
    if (!rc)
        rc = check_heads(a.v, some, kv_heads, d, false, "v", what);
    if (!rc)
        rc = check_heads(a.out, tokens, heads, d, true, "out", what);
    if (!rc)
        rc = check_units(a.q, tokens, heads, "q", what);
    if (!rc)
        rc = check_units(a.k, some, kv_heads, "k", what);
    if (!rc)
        rc = check_units(a.v, some, kv_heads, "v", what);
    if (rc)
        return rc;
    if (misaligned(cu_q, 4) || misaligned(cu_k, 4))
        return set_error(ST_INVALID_LAYOUT, "%s: cu_q and cu_k must be aligned as their types are", what);
    // (rows of the last tiles are counted in an int)
    if (tokens > 0x7fffffff - 512 || key_tokens > 0x7fffffff - 512)
        return set_error(ST_OUT_OF_RANGE, "%s: %d tokens, %d of keys", what, tokens, key_tokens);
    a.pack = attention_prompt_pack(a.q, tokens, heads, kv_heads, d);
    rc = check_grid(attention_prompt_ctas(tokens, batch, heads, a.pack), what);
    if (!rc)
        rc = status_word(stream, &a.status);
    if (rc)
        return rc;
    a.batch = batch, a.tokens = tokens, a.key_tokens = key_tokens;
    a.heads = heads, a.kv_heads = kv_heads, a.d = d;
    a.cu_q = cu_q, a.cu_k = cu_k ? cu_k : cu_q;
    a.causal = causal != 0;
    a.scale_log2 = scale * kLog2E;
    return launch_attention_prompt(a, dtype, (cudaStream_t)stream);
}

}  // extern "C"
