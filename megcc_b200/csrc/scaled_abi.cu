// extern "C" entry points of the int8 operators with scales found at run time (include/megcc_b200.h).
#include "../../include/megcc_b200.h"
#include "moe_s8.h"
#include "scaled_s8.cuh"
#include "umma_ptx.cuh"

using namespace mb200;
using namespace mb200::scaled;

namespace {

int check_dtype(int dtype, const char* what) {
    if (dtype < DT_F32 || dtype > DT_BF16)
        return set_error(ST_UNSUPPORTED_DTYPE, "%s: type %d is none of MB200_DTYPE_*", what, dtype);
    return ST_SUCCESS;
}

int check_extents(const char* what, int m, int n, int k) {
    if (m < 0 || n <= 0 || k <= 0)
        return set_error(ST_INVALID_LAYOUT, "%s: extents %d x %d x %d", what, m, n, k);
    if (k > kMaxK)
        return set_error(ST_OUT_OF_RANGE, "%s: k = %d, sums of more than %d products may leave an int32", what, k,
                         kMaxK);
    if (m > kMaxExtent || n > kMaxExtent)
        return set_error(ST_OUT_OF_RANGE, "%s: extents %d x %d (at most %d)", what, m, n, kMaxExtent);
    return ST_SUCCESS;
}

bool misaligned(const void* p, size_t bytes) {
    return ((uintptr_t)p & (bytes - 1)) != 0;
}

// b may be fetched ahead of the end of the kernel in front
int may_read_early(const void* p, size_t bytes, cudaStream_t st) {
    return is_constant(p) || !last_launch_writes(st, p, bytes);
}

int check_product_sides(
        const char* what, const int8_t* b, const float* b_scales, const float* bias, const void* c, int dtype,
        long long ldc, int m, int n) {
    if (!b || !b_scales || !c)
        return set_error(ST_NULL_PTR, "%s: operand pointer is NULL", what);
    if (ldc < n && m > 1)
        return set_error(ST_INVALID_LAYOUT, "%s: rows of the result overlap", what);
    if (misaligned(b_scales, 4) || misaligned(bias, 4) || misaligned(c, dtype_bytes(dtype)))
        return set_error(ST_INVALID_LAYOUT, "%s: scales, bias and result must be aligned as their types are", what);
    return ST_SUCCESS;
}

int check_workspace(const char* what, const void* workspace, size_t have, size_t need) {
    if (need == 0)
        return ST_SUCCESS;
    if (!workspace)
        return set_error(ST_NULL_PTR, "%s: needs a workspace of %zu bytes", what, need);
    if (misaligned(workspace, 256) || have < need)
        return set_error(ST_INVALID_LAYOUT, "%s: the workspace must be 256-byte aligned and hold %zu bytes", what,
                         need);
    return ST_SUCCESS;
}

// What the TMA takes: 16-byte aligned, rows whole 16-byte units apart
bool rows_fit(const void* p, int rows, long long ld) {
    return !misaligned(p, 16) && (rows == 1 || ld % 16 == 0);
}
// Few rows of activations, or little of everything: the kernel that streams the weights past them, whatever the
// operands' alignment. Both sides measured (us, streamed and by the TMA-fed tiles, weights from HBM), n x k:
//   one row     16384 x 16384 42.4 / 47.4, 65536 x 1024 11.8 / 23.9, 20000 x 2048 8.9 / 10.2, 32000 x 4096 24.9 / 21.7
//   four        16384 x 2048 12.4 / 12.3, 10000 x 1008 8.4 / 6.5, 16384 x 1024 4.6 / 5.0, 6144 x 4096 6.4 / 8.8
//   sixteen     16384 x 2048 12.8 / 11.8, 14336 x 4096 13.8 / 13.5, 4096 x 8192 6.9 / 10.5, 6144 x 4096 7.8 / 9.1
//   24          4096 x 4096 5.4 / 7.8, 8192 x 4096 10.4 / 10.0, 6000 x 1024 7.5 / 4.6, 14336 x 4096 18.8 / 12.5
// Streamed all the same, on the wrong side of a limit that goes by n and k: sixteen rows of 10000 x 1536 (7.3 / 6.4),
// 24 of 6144 x 4096 (9.9 / 9.2).
// Warps of the streaming kernel share K (launch_stream): short K costs them starts and ends, unless each has
// rows of its own, which wants whole lines. Tiles want many columns, enough for all SMs without cutting K.
// `fits`: the tiles' operands need no copies (4100 x 4100, 24 rows, weights in the L2: 11.5 / 15.5).
bool streams(int m, int n, int k, bool fits) {
    const long long weights = (long long)n * k, sms = umma::sm_count();
    if (m <= 32 && !fits)
        return true;
    if (m <= 16) {
        const bool lines = k % 128 == 0;
        if (k <= 1024)
            return lines || k <= 512 || n < 8192;
        return k > 4096 || n < sms * 3 / 5 * 128 || (k <= 2048 && lines && n >= sms * 128);
    }
    if (m <= 32)
        return weights <= 1 << 22 || (weights <= 1 << 25 && (n < 4800 || (n < 8192 && k > 1024)));
    // A pass over the weights per 32 rows, in no more CTAs than the SMs hold at once, or twice as many where the tiles
    // would need a launch more, for copies (148 x 1614 x 66: 6.0 / 7.8)
    const long long passes = ((long long)m + 31) / 32;
    return passes * weights <= 1 << 22 && passes * ((n + 15) / 16) <= (fits ? 2 : 4) * sms;
}
// So few that it makes whole numbers of them itself, every CTA again, which saves a launch and a transition. So, and by a
// kernel in front (us, weights from HBM): 1 x 4096 x 4096 5.1 / 5.8, 1 x 14336 x 4096 13.3 / 15.3, 4 x 4096 x 4096
// 5.6 / 5.9, 8 x 4096 x 1024 4.2 / 4.3. The rule does not look at n, by which the work is done again: 4 x 14336 x 4096
// 21.0 / 15.3, 8 x 4096 x 4096 7.2 / 5.9, 8 x 128000 x 4096 183 / 88.
bool streams_activations(int m, int k) {
    return m <= 8 && (long long)m * k <= 32768;
}
// int8 tokens that no 16-byte copies take are laid out anew in front of many weights, by which each CTA would shift them
// into place again: 24 x 11008 x 4097 24.9 us, 38.2 so
bool lays_out_tokens(int m, int n, int k, const int8_t* a, long long lda) {
    return m > 8 && (long long)n * k >= 1 << 22 && !rows_fit(a, m, lda);
}
// (whole lines: 128 bytes of K then come as one line of the L2, not as parts of two)
long long padded(int k) {
    return ((long long)k + 127) / 128 * 128;
}
size_t padded_bytes(int rows, int k) {
    return align_up((size_t)rows * (size_t)padded(k), 256);
}
// A matrix as the TMA takes it, in the workspace where it is not yet: what is to be done for that
PadRows pad_job(const int8_t** src, long long* ld, int rows, int k, int8_t** ws) {
    PadRows j{};
    if (!rows_fit(*src, rows, *ld)) {
        j = {*src, *ld, rows, k, *ws, padded(k)};
        *src = *ws, *ld = padded(k);
        *ws += padded_bytes(rows, k);
    }
    return j;
}

int check_moe(const mb200_moe_param* p) {
    if (!p)
        return set_error(ST_NULL_PTR, "moe_s8: parameter block is NULL");
    int rc = check_dtype(p->dtype, "moe_s8");
    if (rc)
        return rc;
    if (p->tokens < 0 || p->d <= 0 || p->f <= 0 || p->experts <= 0 || p->top_k <= 0 || p->top_k > p->experts)
        return set_error(ST_INVALID_LAYOUT, "moe_s8: %d tokens, d %d, f %d, %d of %d experts", p->tokens, p->d, p->f,
                         p->top_k, p->experts);
    if (p->tokens > kMoeMaxTokens || p->top_k > kMoeMaxTop || p->experts > kMoeMaxExperts || p->f > kMaxK ||
        p->d > (p->tokens <= 8 ? kMoeMaxDepthFew : kMoeMaxDepth))
        return set_error(ST_OUT_OF_RANGE, "moe_s8: %d tokens (64), d %d (16384, 8192 with more than 8 tokens), "
                         "f %d (131071), %d of %d experts (16 of 512)", p->tokens, p->d, p->f, p->top_k, p->experts);
    return ST_SUCCESS;
}
size_t moe_hidden_bytes(const mb200_moe_param* p) {  // whole numbers of the hidden layer
    return align_up((size_t)p->tokens * p->top_k * align_up((size_t)p->f, 32), 256);
}
size_t moe_scale_bytes(const mb200_moe_param* p) {  // and their groups' scales
    return align_up((size_t)p->tokens * p->top_k * (align_up((size_t)p->f, 32) / 32) * sizeof(float), 256);
}
size_t moe_route_bytes(const mb200_moe_param* p) {
    return align_up((size_t)route_bytes(p->tokens * p->top_k, p->experts, 8), 256);
}
// the tokens as whole numbers, where a kernel of their own makes them, and their scales behind
size_t moe_token_bytes(const mb200_moe_param* p) {
    return p->tokens <= kMoeFew ? 0 : (size_t)p->tokens * (size_t)xs_pitch(p->d);
}
size_t moe_bytes(const mb200_moe_param* p) {
    return moe_hidden_bytes(p) + moe_scale_bytes(p) + moe_route_bytes(p) + moe_token_bytes(p) +
           (p->tokens <= kMoeFew ? 0 : 256);
}

}  // namespace

extern "C" {

int mb200_quantize_rows_s8(
        const void* x, int dtype, int m, int k, long long ldx, int8_t* q, long long ldq, float* scales,
        void* stream) {
    int rc = check_dtype(dtype, "quantize_rows");
    if (rc)
        return rc;
    if (m < 0 || k <= 0)
        return set_error(ST_INVALID_LAYOUT, "quantize_rows: extents %d x %d", m, k);
    if (m == 0)
        return ST_SUCCESS;
    if (!x || !q || !scales)
        return set_error(ST_NULL_PTR, "quantize_rows: tensor pointer is NULL");
    if (m > 1 && (ldx < k || ldq < k))
        return set_error(ST_INVALID_LAYOUT, "quantize_rows: rows overlap");
    if (misaligned(x, dtype_bytes(dtype)) || misaligned(scales, 4))
        return set_error(ST_INVALID_LAYOUT, "quantize_rows: tensors must be aligned as their types are");
    return launch_quantize_rows(x, dtype, m, k, ldx, q, ldq, scales, (cudaStream_t)stream);
}

size_t mb200_matmul_s8_scaled_workspace_bytes(
        int m, int n, int k, const int8_t* a, long long lda, const int8_t* b_packed) {
    if (m <= 0 || n <= 0 || k <= 0 || k > kMaxK)
        return 0;
    if (streams(m, n, k, rows_fit(a, m, lda) && rows_fit(b_packed, n, k)))
        return lays_out_tokens(m, n, k, a, lda) ? padded_bytes(m, k) : 0;
    return (rows_fit(a, m, lda) ? 0 : padded_bytes(m, k)) + (rows_fit(b_packed, n, k) ? 0 : padded_bytes(n, k));
}

int mb200_matmul_s8_scaled(
        int m, int n, int k, const int8_t* a, long long lda, const int8_t* b_packed, const float* a_scales,
        const float* b_scales, const float* bias, void* c, int dtype, long long ldc, void* workspace,
        size_t workspace_bytes, void* stream) {
    int rc = check_dtype(dtype, "matmul_s8_scaled");
    if (!rc)
        rc = check_extents("matmul_s8_scaled", m, n, k);
    if (rc || m == 0)
        return rc;
    if (!a || !a_scales)
        return set_error(ST_NULL_PTR, "matmul_s8_scaled: operand pointer is NULL");
    rc = check_product_sides("matmul_s8_scaled", b_packed, b_scales, bias, c, dtype, ldc, m, n);
    if (rc)
        return rc;
    if (m > 1 && lda < k)
        return set_error(ST_INVALID_LAYOUT, "matmul_s8_scaled: rows of the left operand overlap");
    if (misaligned(a_scales, 4))
        return set_error(ST_INVALID_LAYOUT, "matmul_s8_scaled: scales must be 4-byte aligned");
    rc = check_workspace("matmul_s8_scaled", workspace, workspace_bytes,
                         mb200_matmul_s8_scaled_workspace_bytes(m, n, k, a, lda, b_packed));
    if (rc)
        return rc;
    cudaStream_t st = (cudaStream_t)stream;
    ProductArgs p{};
    p.m = m, p.n = n, p.k = k;
    p.a = a, p.x_dtype = -1, p.lda = lda;
    p.b = b_packed, p.ldb = k, p.sa = a_scales, p.sb = b_scales, p.bias = bias;
    p.c = c, p.c_dtype = dtype, p.ldc = ldc;
    int8_t* ws = (int8_t*)workspace;
    if (streams(m, n, k, rows_fit(a, m, lda) && rows_fit(b_packed, n, k))) {
        if (lays_out_tokens(m, n, k, a, lda)) {
            rc = launch_pad_rows(pad_job(&a, &p.lda, m, k, &ws), PadRows{}, st);
            if (rc)
                return rc;
            p.a = a;
        }
        p.b_early = may_read_early(b_packed, (size_t)n * k, st);
        return launch_product_stream(p, st);
    }
    const PadRows pad_b = pad_job(&p.b, &p.ldb, n, k, &ws), pad_a = pad_job(&a, &p.lda, m, k, &ws);
    p.a = a;
    rc = launch_pad_rows(pad_b, pad_a, st);
    if (rc)
        return rc;
    p.b_early = may_read_early(p.b, (size_t)n * (size_t)p.ldb, st);
    return launch_product_umma(p, st);
}

size_t mb200_linear_s8_workspace_bytes(int m, int n, int k, const int8_t* b_packed) {
    if (m <= 0 || n <= 0 || k <= 0 || k > kMaxK || streams_activations(m, k))
        return 0;
    return padded_bytes(m, k) + align_up((size_t)m * 4, 256) +
           (rows_fit(b_packed, n, k) || streams(m, n, k, false) ? 0 : padded_bytes(n, k));
}

int mb200_linear_s8(
        int m, int n, int k, const void* x, int dtype, long long ldx, const int8_t* b_packed,
        const float* b_scales, const float* bias, void* y, long long ldy, void* workspace,
        size_t workspace_bytes, void* stream) {
    int rc = check_dtype(dtype, "linear_s8");
    if (!rc)
        rc = check_extents("linear_s8", m, n, k);
    if (rc || m == 0)
        return rc;
    if (!x)
        return set_error(ST_NULL_PTR, "linear_s8: operand pointer is NULL");
    rc = check_product_sides("linear_s8", b_packed, b_scales, bias, y, dtype, ldy, m, n);
    if (rc)
        return rc;
    if (m > 1 && ldx < k)
        return set_error(ST_INVALID_LAYOUT, "linear_s8: rows of the activations overlap");
    if (misaligned(x, dtype_bytes(dtype)))
        return set_error(ST_INVALID_LAYOUT, "linear_s8: activations must be aligned as their type is");
    rc = check_workspace("linear_s8", workspace, workspace_bytes,
                         mb200_linear_s8_workspace_bytes(m, n, k, b_packed));
    if (rc)
        return rc;
    cudaStream_t st = (cudaStream_t)stream;
    ProductArgs p{};
    p.m = m, p.n = n, p.k = k;
    p.a = x, p.x_dtype = dtype, p.lda = ldx;
    p.b = b_packed, p.ldb = k, p.sb = b_scales, p.bias = bias;
    p.c = y, p.c_dtype = dtype, p.ldc = ldy;
    if (streams_activations(m, k)) {
        p.b_early = may_read_early(b_packed, (size_t)n * k, st);
        return launch_product_stream(p, st);
    }
    int8_t* ws = (int8_t*)workspace;
    const bool few = streams(m, n, k, rows_fit(b_packed, n, k));
    if (!few) {
        rc = launch_pad_rows(pad_job(&p.b, &p.ldb, n, k, &ws), PadRows{}, st);
        if (rc)
            return rc;
    }
    float* scales = (float*)(ws + padded_bytes(m, k));
    rc = launch_quantize_rows(x, dtype, m, k, ldx, ws, padded(k), scales, st);
    if (rc)
        return rc;
    p.a = ws, p.x_dtype = -1, p.lda = padded(k), p.sa = scales;
    p.b_early = may_read_early(p.b, (size_t)n * (size_t)p.ldb, st);
    return few ? launch_product_stream(p, st) : launch_product_umma(p, st);
}

size_t mb200_moe_s8_workspace_bytes(const mb200_moe_param* p) {
    return check_moe(p) ? 0 : moe_bytes(p);
}

int mb200_moe_s8(
        const mb200_moe_param* p, const void* x, long long ldx, const float* logits, const int8_t* w1,
        const float* w1_scales, const int8_t* w2, const float* w2_scales, void* y, long long ldy, void* workspace,
        size_t workspace_bytes, void* stream) {
    const int rc = check_moe(p);
    if (rc || p->tokens == 0)
        return rc;
    if (!x || !logits || !w1 || !w1_scales || !w2 || !w2_scales || !y || !workspace)
        return set_error(ST_NULL_PTR, "moe_s8: operand pointer is NULL");
    if (p->tokens > 1 && (ldx < p->d || ldy < p->d))
        return set_error(ST_INVALID_LAYOUT, "moe_s8: rows overlap");
    if (misaligned(x, dtype_bytes(p->dtype)) || misaligned(y, dtype_bytes(p->dtype)) || misaligned(logits, 4) ||
        misaligned(w1_scales, 4) || misaligned(w2_scales, 4))
        return set_error(ST_INVALID_LAYOUT, "moe_s8: tensors must be aligned as their types are");
    if (misaligned(workspace, 256) || workspace_bytes < moe_bytes(p))
        return set_error(ST_INVALID_LAYOUT, "moe_s8: the workspace must be 256-byte aligned and hold %zu bytes",
                         moe_bytes(p));
    MoeArgs a{};
    a.t = p->tokens, a.d = p->d, a.f = p->f, a.e = p->experts, a.top = p->top_k;
    a.renormalize = p->renormalize, a.dtype = p->dtype;
    a.x = x, a.ldx = ldx, a.logits = logits;
    a.w1 = w1, a.s1 = w1_scales, a.w2 = w2, a.s2 = w2_scales;
    a.y = y, a.ldy = ldy;
    a.hq = (int8_t*)workspace, a.sh = (float*)((uint8_t*)workspace + moe_hidden_bytes(p));
    a.route = (uint4*)((uint8_t*)a.sh + moe_scale_bytes(p));
    a.xq = (int8_t*)a.route + moe_route_bytes(p);
    a.sx = (float*)(a.xq + moe_token_bytes(p));
    a.workspace_bytes = moe_bytes(p);
    return launch_moe(a, (cudaStream_t)stream);
}

}  // extern "C"
