// extern "C" entry points of the int8 operators with scales found at run time (include/megcc_b200.h).
#include "../../include/megcc_b200.h"
#include "scaled_s8.cuh"

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
    (void)m, (void)n, (void)k, (void)a, (void)lda, (void)b_packed;
    return 0;
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
    (void)workspace, (void)workspace_bytes;
    cudaStream_t st = (cudaStream_t)stream;
    ProductArgs p{};
    p.m = m, p.n = n, p.k = k;
    p.a = a, p.x_dtype = -1, p.lda = lda;
    p.b = b_packed, p.sa = a_scales, p.sb = b_scales, p.bias = bias;
    p.c = c, p.c_dtype = dtype, p.ldc = ldc;
    p.b_early = may_read_early(b_packed, (size_t)n * k, st);
    return launch_product_stream(p, st);
}

size_t mb200_linear_s8_workspace_bytes(int m, int n, int k, const int8_t* b_packed) {
    (void)m, (void)n, (void)k, (void)b_packed;
    return 0;
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
    (void)workspace, (void)workspace_bytes;
    cudaStream_t st = (cudaStream_t)stream;
    ProductArgs p{};
    p.m = m, p.n = n, p.k = k;
    p.a = x, p.x_dtype = dtype, p.lda = ldx;
    p.b = b_packed, p.sb = b_scales, p.bias = bias;
    p.c = y, p.c_dtype = dtype, p.ldc = ldy;
    p.b_early = may_read_early(b_packed, (size_t)n * k, st);
    return launch_product_stream(p, st);
}

}  // extern "C"
