// mx4_kernels.hpp - matrices in 4 bits per value ("mx4"): quantisation, and products whose contraction runs along or across the blocks.
//
// A value is a 4-bit float (sign, 2 exponent bits, 1 mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6); 32 neighbours along a row share one
// power-of-two scale, held as its biased exponent (a byte: 2^(byte - 127); 255 = the whole block is NaN).  4.25 bits per value.
//
// Layout of an R x C matrix:
//   codes  [R][code_row_bytes(C)]   two values a byte, the even column in the low half; rows padded with zeros to 256 columns (128 B)
//   scales [R][scale_row_bytes(C)]  one byte per 32 columns, rows padded to 512 columns (16 B); inside every 16 blocks the byte of
//                                   block 4 s + g sits at 4 g + s.  A lane of the matrix instructions below owns block g = lane / 16 of
//                                   each 128-column step s: one dword holds its scales of four steps, and the instruction picks a byte.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace lcx {

constexpr int MX_BLOCK = 32;
__host__ __device__ inline int64_t mx_code_row(int64_t cols) { return (cols + 255) / 256 * 128; }
__host__ __device__ inline int64_t mx_scale_row(int64_t cols) { return (cols + 511) / 512 * 16; }
// place of block b (of 32 columns) in its row of scales
__host__ __device__ inline int64_t mx_scale_at(int64_t b) { return (b & ~(int64_t)15) + (b & 3) * 4 + ((b >> 2) & 3); }

typedef __attribute__((ext_vector_type(2))) __bf16 mx_bf2;
typedef __attribute__((ext_vector_type(8))) __bf16 mx_bf8;
typedef __attribute__((ext_vector_type(2))) float mx_f2;
typedef __attribute__((ext_vector_type(4))) float mx_f4;
typedef __attribute__((ext_vector_type(4))) unsigned int mx_u4;
typedef __attribute__((ext_vector_type(8))) int mx_i8;

template <typename T> struct MxTerms;                              // bf16 numbers that add up to a T exactly
template <> struct MxTerms<float> { static constexpr int v = 3; };     // 24 significant bits = 8 + 8 + 8
template <> struct MxTerms<_Float16> { static constexpr int v = 2; };  // 11 = 8 + 3
template <> struct MxTerms<__bf16> { static constexpr int v = 1; };

__device__ __forceinline__ float mx_trunc_bf16(float x) { return __uint_as_float(__float_as_uint(x) & 0xffff0000u); }
// x = term 0 + term 1 + term 2, each a bf16 number: the leading 8 significant bits are cut off twice, what remains has at most 8.  Every
// term takes part in the products below, so cutting (rather than rounding) leaves no bias.  An infinity or NaN stays in term 0
// (the remainder would be NaN: zeros instead, the sum is the same).
template <int TERMS> __device__ __forceinline__ void mx_split(float x, float* t) {
    t[0] = TERMS > 1 ? mx_trunc_bf16(x) : x;
    if constexpr (TERMS > 1) {
        const bool finite = (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u;
        // (cutting a NaN's payload could leave an infinity)
        if (!finite) t[0] = x;
        const float r = finite ? x - t[0] : 0.0f;
        t[1] = TERMS > 2 ? mx_trunc_bf16(r) : r;
        if constexpr (TERMS > 2) t[2] = r - t[1];
    }
}

// ---- quantisation ---------------------------------------------------------------------------------------------------------------
// biased exponent of the shared scale from the bits of the largest magnitude: its binade less 2, so that the largest value falls into
// [4, 8) and saturates at 6 in the upper quarter.  At least 2: every value is then zero or a normal float32 / bf16 number (a block
// whose magnitudes are all below 2^-123 loses relative precision, below 2^-127 it is zero).  255 for a block with an infinity or NaN.
__device__ __forceinline__ int mx_scale_of(unsigned int amax_bits) {
    const int e = (int)(amax_bits >> 23);
    if (e == 255) return 255;
    return e < 4 ? 2 : e - 2;
}
// float64 input: magnitudes beyond float32 count as its largest finite number (they saturate), smaller ones are cut to float32 with
// the lost bits ORed into the last place (the 4-bit rounding that follows is then the one of the exact value)
__device__ __forceinline__ float mx_to_f32(double x) {
    const double a = fabs(x);
    if (a > 3.0e38 && a <= 1.7976931348623157e308) return x < 0 ? -3.4028234663852886e38f : 3.4028234663852886e38f;
    float f = (float)x;
    if ((double)f != x && a <= 1.7976931348623157e308) {
        unsigned int u = __float_as_uint(f);
        if (fabs((double)f) > a) u -= 1;                       // toward zero
        f = __uint_as_float(u | 1u);
    }
    return f;
}
__device__ __forceinline__ float mx_to_f32(float x) { return x; }
__device__ __forceinline__ float mx_to_f32(_Float16 x) { return (float)x; }
__device__ __forceinline__ float mx_to_f32(__bf16 x) { return (float)x; }

// eight values and their shared scale -> a dword of codes (round to nearest even, saturating: v_cvt_scalef32_pk_fp4_f32)
__device__ __forceinline__ unsigned int mx_pack8(const float* v, int sc) {
    const float s = __uint_as_float((unsigned int)(sc == 255 ? 254 : sc) << 23);
    unsigned int q = 0;
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[0], v[1], s, 0);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[2], v[3], s, 1);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[4], v[5], s, 2);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[6], v[7], s, 3);
    return q;
}

// x[r * rs + c * cs] -> codes, scales.  Four lanes share a block, each takes 8 columns.  grid (row groups, column chunks)
template <typename T>
__global__ __launch_bounds__(256) void mx_quantize_kernel(const T* __restrict__ x, int64_t rows, int64_t cols, int64_t rs, int64_t cs,
                                                          unsigned char* __restrict__ codes, unsigned char* __restrict__ scales, int tpr_log2) {
    const int64_t crow = mx_code_row(cols), srow = mx_scale_row(cols);
    const int tpr = 1 << tpr_log2;
    const int64_t r = (int64_t)blockIdx.x * (256 >> tpr_log2) + (threadIdx.x >> tpr_log2);
    if (r >= rows) return;                                     // (whole groups of 4 lanes: tpr >= 32)
    for (int64_t c8 = (int64_t)blockIdx.y * tpr + (threadIdx.x & (tpr - 1)); c8 < srow * 4; c8 += (int64_t)gridDim.y * tpr) {
        const int64_t c0 = c8 * 8;
        float v[8];
        unsigned int am = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            v[j] = c0 + j < cols ? mx_to_f32(x[r * rs + (c0 + j) * cs]) : 0.0f;
            const unsigned int u = __float_as_uint(v[j]) & 0x7fffffffu;
            am = u > am ? u : am;
        }
        unsigned int o = (unsigned int)__shfl_xor((int)am, 1);
        am = o > am ? o : am;
        o = (unsigned int)__shfl_xor((int)am, 2);
        am = o > am ? o : am;
        const int sc = mx_scale_of(am);
        if (c8 * 4 < crow) *reinterpret_cast<unsigned int*>(codes + r * crow + c8 * 4) = mx_pack8(v, sc);
        if ((threadIdx.x & 3) == 0) scales[r * srow + mx_scale_at(c8 >> 2)] = (unsigned char)sc;
    }
}

template <typename T> __device__ __forceinline__ T mx_from_f32(float v) { return (T)v; }

// codes, scales -> out[r * rs + c * cs]
template <typename T>
__global__ __launch_bounds__(256) void mx_dequantize_kernel(const unsigned char* __restrict__ codes, const unsigned char* __restrict__ scales,
                                                            int64_t rows, int64_t cols, T* __restrict__ out, int64_t rs, int64_t cs, int tpr_log2) {
    const int64_t crow = mx_code_row(cols), srow = mx_scale_row(cols);
    const int tpr = 1 << tpr_log2;
    const int64_t r = (int64_t)blockIdx.x * (256 >> tpr_log2) + (threadIdx.x >> tpr_log2);
    if (r >= rows) return;
    for (int64_t c8 = (int64_t)blockIdx.y * tpr + (threadIdx.x & (tpr - 1)); c8 * 8 < cols; c8 += (int64_t)gridDim.y * tpr) {
        const unsigned int q = *reinterpret_cast<const unsigned int*>(codes + r * crow + c8 * 4);
        const float s = __uint_as_float((unsigned int)scales[r * srow + mx_scale_at(c8 >> 2)] << 23);
        float v[8];
        mx_f2 p;
        p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, s, 0); v[0] = p[0]; v[1] = p[1];
        p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, s, 1); v[2] = p[0]; v[3] = p[1];
        p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, s, 2); v[4] = p[0]; v[5] = p[1];
        p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, s, 3); v[6] = p[0]; v[7] = p[1];
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (c8 * 8 + j < cols) out[r * rs + (c8 * 8 + j) * cs] = mx_from_f32<T>(v[j]);
    }
}

// ---- products -------------------------------------------------------------------------------------------------------------------
// 4 bits x 4 bits: out[m][n] = sum_k A[m][k] B[n][k] on v_mfma_scale_f32_16x16x128_f8f6f4: a lane holds one block of 32 of its row (16 bytes)
// and that block's scale; float32 sums.  Rows behind the last one repeat it and are not stored.
template <typename TO>
__global__ __launch_bounds__(64) void mx_matmul_kernel(const unsigned char* __restrict__ ac, const unsigned char* __restrict__ as, int64_t M,
                                                       const unsigned char* __restrict__ bc, const unsigned char* __restrict__ bs, int64_t N, int64_t K,
                                                       TO* __restrict__ out, int64_t rs, int64_t cs, int64_t mtiles) {
    constexpr int RT = 2;                                      // 32 x 32 outputs a wave
    const int64_t crow = mx_code_row(K), srow = mx_scale_row(K);
    const int64_t m0 = (int64_t)(blockIdx.x % mtiles) * 16 * RT, n0 = (int64_t)(blockIdx.x / mtiles) * 16 * RT;
    const int l = threadIdx.x & 15, g = threadIdx.x >> 4;
    const unsigned char *pa[RT], *pb[RT], *sa[RT], *sb[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        const int64_t rm = m0 + 16 * i + l < M ? m0 + 16 * i + l : M - 1, rn = n0 + 16 * i + l < N ? n0 + 16 * i + l : N - 1;
        pa[i] = ac + rm * crow + g * 16;
        pb[i] = bc + rn * crow + g * 16;
        sa[i] = as + rm * srow + g * 4;
        sb[i] = bs + rn * srow + g * 4;
    }
    mx_f4 acc[RT][RT] = {};
    for (int64_t s = 0; s * 64 < crow; ++s) {                  // 128 columns a step
        mx_i8 a[RT] = {}, b[RT] = {};
        int xa[RT], xb[RT];
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            const mx_u4 ta = *reinterpret_cast<const mx_u4*>(pa[i] + s * 64), tb = *reinterpret_cast<const mx_u4*>(pb[i] + s * 64);
#pragma unroll
            for (int j = 0; j < 4; ++j) { a[i][j] = (int)ta[j]; b[i][j] = (int)tb[j]; }
            xa[i] = sa[i][(s >> 2) * 16 + (s & 3)];
            xb[i] = sb[i][(s >> 2) * 16 + (s & 3)];
        }
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int j = 0; j < RT; ++j) acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a[i], b[j], acc[i][j], 4, 4, 0, xa[i], 0, xb[j]);
    }
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < RT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int64_t m = m0 + 16 * i + 4 * g + e, n = n0 + 16 * j + l;
                if (m < M && n < N) out[m * rs + n * cs] = mx_from_f32<TO>(acc[i][j][e]);
            }
}

// eight codes of one block -> bf16 (exact: at most 2 significant bits)
__device__ __forceinline__ mx_bf8 mx_unpack8(unsigned int q, float s) {
    const mx_bf2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, s, 0), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, s, 1),
                 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, s, 2), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, s, 3);
    return mx_bf8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// x[t * rs + k * cs], eight k from k0 on, as bf16 terms; zeros outside
template <typename T, int TERMS>
__device__ __forceinline__ void mx_load_terms(const T* __restrict__ x, int64_t t, int64_t nt, int64_t rs, int64_t k0, int64_t nk, int64_t cs, mx_bf8* f) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        float p[3] = {0.0f, 0.0f, 0.0f};
        if (t < nt && k0 + j < nk) mx_split<TERMS>((float)x[t * rs + (k0 + j) * cs], p);
#pragma unroll
        for (int u = 0; u < TERMS; ++u) f[u][j] = (__bf16)p[u];
    }
}

// out[t][n] = sum_k x[t][k] W[n][k], W in 4 bits with its blocks along k: the codes become bf16 in registers, x is split into bf16 terms
// (MxTerms), every product is exact, float32 sums.  A wave owns 16 rows of W and 16 of x.
template <typename T>
__global__ __launch_bounds__(64) void mx_linear_kernel(const T* __restrict__ x, int64_t M, int64_t xrs, int64_t xcs, const unsigned char* __restrict__ wc,
                                                       const unsigned char* __restrict__ ws, int64_t N, int64_t K, T* __restrict__ out, int64_t rs,
                                                       int64_t cs, int64_t mtiles) {
    constexpr int TERMS = MxTerms<T>::v;
    const int64_t crow = mx_code_row(K), srow = mx_scale_row(K);
    const int64_t t0 = (int64_t)(blockIdx.x % mtiles) * 16, n0 = (int64_t)(blockIdx.x / mtiles) * 16;
    const int l = threadIdx.x & 15, g = threadIdx.x >> 4;
    const int64_t rn = n0 + l < N ? n0 + l : N - 1;
    mx_f4 acc = {};
    for (int64_t s = 0; s * 64 < crow; ++s) {
        const mx_u4 q = *reinterpret_cast<const mx_u4*>(wc + rn * crow + s * 64 + g * 16);
        const float sc = __uint_as_float((unsigned int)ws[rn * srow + (s >> 2) * 16 + g * 4 + (s & 3)] << 23);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const mx_bf8 w = mx_unpack8(q[j], sc);
            mx_bf8 f[TERMS];
            mx_load_terms<T, TERMS>(x, t0 + l, M, xrs, s * 128 + g * 32 + j * 8, K, xcs, f);
#pragma unroll
            for (int u = 0; u < TERMS; ++u) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, f[u], acc, 0, 0, 0);
        }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int64_t n = n0 + 4 * g + e, t = t0 + l;
        if (n < N && t < M) out[t * rs + n * cs] = mx_from_f32<T>(acc[e]);
    }
}

// dx[t][k] = sum_n dy[t][n] W[n][k]: the contraction runs ACROSS the blocks.  A lane reads the dword of 8 columns from each of 8 rows of W;
// unpacked, entry m of the eight dwords is what matrix instruction m needs from this lane: column 8 (lane % 16) + m, eight n.  So a
// wave owns 128 columns as 8 tiles and no value crosses lanes.
template <typename T>
__global__ __launch_bounds__(64) void mx_linear_grad_kernel(const T* __restrict__ dy, int64_t M, int64_t yrs, int64_t ycs,
                                                            const unsigned char* __restrict__ wc, const unsigned char* __restrict__ ws, int64_t N, int64_t K,
                                                            T* __restrict__ out, int64_t rs, int64_t cs, int64_t mtiles) {
    constexpr int TERMS = MxTerms<T>::v;
    const int64_t crow = mx_code_row(K), srow = mx_scale_row(K);
    const int64_t t0 = (int64_t)(blockIdx.x % mtiles) * 16, k0 = (int64_t)(blockIdx.x / mtiles) * 128;
    const int l = threadIdx.x & 15, g = threadIdx.x >> 4;
    const int64_t sat = mx_scale_at((k0 + l * 8) >> 5);
    mx_f4 acc[8] = {};
    for (int64_t n0 = 0; n0 < N; n0 += 32) {
        mx_bf8 w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int64_t n = n0 + g * 8 + j;
            // rows behind the last one contribute zeros (their factor in dy is zero, but a NaN scale must not meet it)
            const unsigned int q = n < N ? *reinterpret_cast<const unsigned int*>(wc + n * crow + (k0 >> 1) + l * 4) : 0u;
            const float sc = n < N ? __uint_as_float((unsigned int)ws[n * srow + sat] << 23) : 1.0f;
            const mx_bf8 v = mx_unpack8(q, sc);
#pragma unroll
            for (int m = 0; m < 8; ++m) w[m][j] = v[m];
        }
        mx_bf8 f[TERMS];
        mx_load_terms<T, TERMS>(dy, t0 + l, M, yrs, n0 + g * 8, N, ycs, f);
#pragma unroll
        for (int m = 0; m < 8; ++m)
#pragma unroll
            for (int u = 0; u < TERMS; ++u) acc[m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[m], f[u], acc[m], 0, 0, 0);
    }
#pragma unroll
    for (int m = 0; m < 8; ++m)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int64_t k = k0 + 8 * (4 * g + e) + m, t = t0 + l;
            if (k < K && t < M) out[t * rs + k * cs] = mx_from_f32<T>(acc[m][e]);
        }
}

template <typename T>
__global__ __launch_bounds__(256) void mx_zero_kernel(T* __restrict__ out, int64_t rows, int64_t cols, int64_t rs, int64_t cs) {
    const int64_t n = rows * cols;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) out[(i / cols) * rs + (i % cols) * cs] = (T)0.0f;
}

}  // namespace lcx
