// lcx_mx4.hip - matrices in 4 bits per value: quantisation and products on device memory (include/lcx.h, lcx_mx4_*)
#include "engine.hpp"
#include "mx4_kernels.hpp"

// sizes of the operators: offsets inside the kernels are 64-bit, tile counts must fit a grid
static constexpr int64_t MX_MAX_DIM = (int64_t)1 << 31;

// nothing may leave a C entry point as an exception (the message itself can fail to allocate)
#define MX_ENTRY(body)                                                     \
    try {                                                                  \
        (void)hipGetLastError();                                           \
        body                                                               \
    } catch (...) {                                                        \
        return LCX_ERR_STATE;                                              \
    }

// dtype -> element type
#define MX_FLOATS(dtype, fn, ...)                                          \
    switch (dtype) {                                                       \
        case LCX_F32: return fn<float>(__VA_ARGS__);                       \
        case LCX_BF16: return fn<__bf16>(__VA_ARGS__);                     \
        case LCX_F16: return fn<_Float16>(__VA_ARGS__);                    \
        default: return fail(LCX_ERR_ARG, std::string(#fn) + ": dtype must be LCX_F32, LCX_BF16 or LCX_F16"); \
    }

static int64_t dim_bad(int64_t a, int64_t b, int64_t c = 0) { return a < 0 || b < 0 || c < 0 || a >= MX_MAX_DIM || b >= MX_MAX_DIM || c >= MX_MAX_DIM; }
static bool mx_misaligned(const void* codes, const void* scales) { return ((uintptr_t)codes & 15) != 0 || ((uintptr_t)scales & 3) != 0; }

// threads per row of the element-wise kernels: a power of two in [32, 256] that covers the row's groups of 8 columns
static int mx_tpr_log2(int64_t cols) {
    int lg = 5;
    while (lg < 8 && ((int64_t)8 << lg) < cols) ++lg;
    return lg;
}
static dim3 mx_row_grid(int64_t rows, int64_t cols, int lg) {
    int64_t gy = cdiv(cdiv(cols, 8), (int64_t)1 << lg);
    if (gy > 64) gy = 64;
    return dim3((unsigned)cdiv(rows, 256 >> lg), (unsigned)(gy < 1 ? 1 : gy));
}

template <typename T>
static int mx4_quantize(const void* x, int64_t rows, int64_t cols, int64_t rs, int64_t cs, void* codes, void* scales, hipStream_t st) {
    const int lg = mx_tpr_log2(cols);
    hipLaunchKernelGGL((mx_quantize_kernel<T>), mx_row_grid(rows, cols, lg), dim3(256), 0, st, (const T*)x, rows, cols, rs, cs, (unsigned char*)codes,
                       (unsigned char*)scales, lg);
    KCHECK();
    return LCX_OK;
}

template <typename T>
static int mx4_dequantize(const void* codes, const void* scales, int64_t rows, int64_t cols, void* out, int64_t rs, int64_t cs, hipStream_t st) {
    const int lg = mx_tpr_log2(cols);
    hipLaunchKernelGGL((mx_dequantize_kernel<T>), mx_row_grid(rows, cols, lg), dim3(256), 0, st, (const unsigned char*)codes, (const unsigned char*)scales,
                       rows, cols, (T*)out, rs, cs, lg);
    KCHECK();
    return LCX_OK;
}

template <typename T> static int mx4_zero(void* out, int64_t rows, int64_t cols, int64_t rs, int64_t cs, hipStream_t st) {
    const int64_t b = cdiv(rows * cols, 256);
    hipLaunchKernelGGL((mx_zero_kernel<T>), dim3((unsigned)(b < 4096 ? b : 4096)), dim3(256), 0, st, (T*)out, rows, cols, rs, cs);
    KCHECK();
    return LCX_OK;
}

static int mx_grid(int64_t mtiles, int64_t ntiles, unsigned* g) {
    if (mtiles * ntiles > 0x7fffffffll) return fail(LCX_ERR_ARG, "lcx_mx4: the output is too large for one call");
    *g = (unsigned)(mtiles * ntiles);
    return LCX_OK;
}

template <typename T>
static int mx4_matmul(const void* ac, const void* as, int64_t M, const void* bc, const void* bs, int64_t N, int64_t K, void* out, int64_t rs, int64_t cs,
                      hipStream_t st) {
    if (K == 0) return mx4_zero<T>(out, M, N, rs, cs, st);
    const int64_t mt = cdiv(M, 32);
    unsigned g;
    LCXCHECK(mx_grid(mt, cdiv(N, 32), &g));
    hipLaunchKernelGGL((mx_matmul_kernel<T>), dim3(g), dim3(64), 0, st, (const unsigned char*)ac, (const unsigned char*)as, M, (const unsigned char*)bc,
                       (const unsigned char*)bs, N, K, (T*)out, rs, cs, mt);
    KCHECK();
    return LCX_OK;
}

template <typename T>
static int mx4_linear(const void* x, int64_t M, int64_t xrs, int64_t xcs, const void* wc, const void* ws, int64_t N, int64_t K, void* out, int64_t rs,
                      int64_t cs, hipStream_t st) {
    if (K == 0) return mx4_zero<T>(out, M, N, rs, cs, st);
    const int64_t mt = cdiv(M, 16);
    unsigned g;
    LCXCHECK(mx_grid(mt, cdiv(N, 16), &g));
    hipLaunchKernelGGL((mx_linear_kernel<T>), dim3(g), dim3(64), 0, st, (const T*)x, M, xrs, xcs, (const unsigned char*)wc, (const unsigned char*)ws, N, K,
                       (T*)out, rs, cs, mt);
    KCHECK();
    return LCX_OK;
}

template <typename T>
static int mx4_linear_grad(const void* dy, int64_t M, int64_t yrs, int64_t ycs, const void* wc, const void* ws, int64_t N, int64_t K, void* out, int64_t rs,
                           int64_t cs, hipStream_t st) {
    if (N == 0) return mx4_zero<T>(out, M, K, rs, cs, st);
    const int64_t mt = cdiv(M, 16);
    unsigned g;
    LCXCHECK(mx_grid(mt, cdiv(K, 128), &g));
    hipLaunchKernelGGL((mx_linear_grad_kernel<T>), dim3(g), dim3(64), 0, st, (const T*)dy, M, yrs, ycs, (const unsigned char*)wc, (const unsigned char*)ws, N,
                       K, (T*)out, rs, cs, mt);
    KCHECK();
    return LCX_OK;
}

extern "C" {

int lcx_mx4_layout(int64_t cols, int64_t* code_row, int64_t* scale_row) {
    MX_ENTRY({
        if (cols < 0 || cols >= MX_MAX_DIM) return fail(LCX_ERR_ARG, "lcx_mx4_layout: bad size");
        if (code_row) *code_row = mx_code_row(cols);
        if (scale_row) *scale_row = mx_scale_row(cols);
        return LCX_OK;
    })
}

int lcx_mx4_quantize(const void* x, int dtype, int64_t rows, int64_t cols, int64_t row_stride, int64_t col_stride, void* codes, void* scales, void* stream) {
    MX_ENTRY({
        if (dim_bad(rows, cols)) return fail(LCX_ERR_ARG, "lcx_mx4_quantize: bad sizes");
        if (dtype < LCX_F32 || dtype > LCX_F16) return fail(LCX_ERR_ARG, "lcx_mx4_quantize: bad dtype");
        if (rows == 0 || cols == 0) return LCX_OK;
        if (!x || !codes || !scales) return fail(LCX_ERR_ARG, "lcx_mx4_quantize: null pointer");
        if (mx_misaligned(codes, scales)) return fail(LCX_ERR_ARG, "lcx_mx4_quantize: codes must be 16-byte and scales 4-byte aligned");
        hipStream_t st = (hipStream_t)stream;
        if (dtype == LCX_F64) return mx4_quantize<double>(x, rows, cols, row_stride, col_stride, codes, scales, st);
        MX_FLOATS(dtype, mx4_quantize, x, rows, cols, row_stride, col_stride, codes, scales, st);
    })
}

int lcx_mx4_dequantize(const void* codes, const void* scales, int64_t rows, int64_t cols, void* out, int dtype, int64_t row_stride, int64_t col_stride,
                       void* stream) {
    MX_ENTRY({
        if (dim_bad(rows, cols)) return fail(LCX_ERR_ARG, "lcx_mx4_dequantize: bad sizes");
        if (dtype < LCX_F32 || dtype > LCX_F16) return fail(LCX_ERR_ARG, "lcx_mx4_dequantize: bad dtype");
        if (rows == 0 || cols == 0) return LCX_OK;
        if (!out || !codes || !scales) return fail(LCX_ERR_ARG, "lcx_mx4_dequantize: null pointer");
        if (mx_misaligned(codes, scales)) return fail(LCX_ERR_ARG, "lcx_mx4_dequantize: codes must be 16-byte and scales 4-byte aligned");
        hipStream_t st = (hipStream_t)stream;
        if (dtype == LCX_F64) return mx4_dequantize<double>(codes, scales, rows, cols, out, row_stride, col_stride, st);
        MX_FLOATS(dtype, mx4_dequantize, codes, scales, rows, cols, out, row_stride, col_stride, st);
    })
}

int lcx_mx4_workspace(int op, int dtype, int64_t M, int64_t N, int64_t K, int64_t* bytes) {
    MX_ENTRY({
        if (!bytes || op < 0 || op > 2 || dim_bad(M, N, K)) return fail(LCX_ERR_ARG, "lcx_mx4_workspace: bad argument");
        if (dtype != LCX_F32 && dtype != LCX_BF16 && dtype != LCX_F16) return fail(LCX_ERR_ARG, "lcx_mx4_workspace: bad dtype");
        *bytes = 0;
        return LCX_OK;
    })
}

int lcx_mx4_matmul(const void* a_codes, const void* a_scales, int64_t M, const void* b_codes, const void* b_scales, int64_t N, int64_t K, void* out, int dtype,
                   int64_t row_stride, int64_t col_stride, void* workspace, int64_t workspace_bytes, void* stream) {
    MX_ENTRY({
        if (dim_bad(M, N, K)) return fail(LCX_ERR_ARG, "lcx_mx4_matmul: bad sizes");
        if (dtype != LCX_F32 && dtype != LCX_BF16 && dtype != LCX_F16) return fail(LCX_ERR_ARG, "lcx_mx4_matmul: dtype must be LCX_F32, LCX_BF16 or LCX_F16");
        if (M == 0 || N == 0) return LCX_OK;
        if (!out || (K > 0 && (!a_codes || !a_scales || !b_codes || !b_scales))) return fail(LCX_ERR_ARG, "lcx_mx4_matmul: null pointer");
        if (mx_misaligned(a_codes, a_scales) || mx_misaligned(b_codes, b_scales))
            return fail(LCX_ERR_ARG, "lcx_mx4_matmul: codes must be 16-byte and scales 4-byte aligned");
        (void)workspace; (void)workspace_bytes;
        MX_FLOATS(dtype, mx4_matmul, a_codes, a_scales, M, b_codes, b_scales, N, K, out, row_stride, col_stride, (hipStream_t)stream);
    })
}

int lcx_mx4_linear(const void* x, int dtype, int64_t M, int64_t x_row, int64_t x_col, const void* codes, const void* scales, int64_t N, int64_t K, void* out,
                   int64_t row_stride, int64_t col_stride, void* workspace, int64_t workspace_bytes, void* stream) {
    MX_ENTRY({
        if (dim_bad(M, N, K)) return fail(LCX_ERR_ARG, "lcx_mx4_linear: bad sizes");
        if (dtype != LCX_F32 && dtype != LCX_BF16 && dtype != LCX_F16) return fail(LCX_ERR_ARG, "lcx_mx4_linear: dtype must be LCX_F32, LCX_BF16 or LCX_F16");
        if (M == 0 || N == 0) return LCX_OK;
        if (!out || (K > 0 && (!x || !codes || !scales))) return fail(LCX_ERR_ARG, "lcx_mx4_linear: null pointer");
        if (mx_misaligned(codes, scales)) return fail(LCX_ERR_ARG, "lcx_mx4_linear: codes must be 16-byte and scales 4-byte aligned");
        (void)workspace; (void)workspace_bytes;
        MX_FLOATS(dtype, mx4_linear, x, M, x_row, x_col, codes, scales, N, K, out, row_stride, col_stride, (hipStream_t)stream);
    })
}

int lcx_mx4_linear_grad(const void* dy, int dtype, int64_t M, int64_t dy_row, int64_t dy_col, const void* codes, const void* scales, int64_t N, int64_t K,
                        void* out, int64_t row_stride, int64_t col_stride, void* workspace, int64_t workspace_bytes, void* stream) {
    MX_ENTRY({
        if (dim_bad(M, N, K)) return fail(LCX_ERR_ARG, "lcx_mx4_linear_grad: bad sizes");
        if (dtype != LCX_F32 && dtype != LCX_BF16 && dtype != LCX_F16)
            return fail(LCX_ERR_ARG, "lcx_mx4_linear_grad: dtype must be LCX_F32, LCX_BF16 or LCX_F16");
        if (M == 0 || K == 0) return LCX_OK;
        if (!out || (N > 0 && (!dy || !codes || !scales))) return fail(LCX_ERR_ARG, "lcx_mx4_linear_grad: null pointer");
        if (mx_misaligned(codes, scales)) return fail(LCX_ERR_ARG, "lcx_mx4_linear_grad: codes must be 16-byte and scales 4-byte aligned");
        (void)workspace; (void)workspace_bytes;
        MX_FLOATS(dtype, mx4_linear_grad, dy, M, dy_row, dy_col, codes, scales, N, K, out, row_stride, col_stride, (hipStream_t)stream);
    })
}

}  // extern "C"
