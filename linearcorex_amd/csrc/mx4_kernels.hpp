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

// largest of the four lanes that share a block (quad permutations: no LDS)
__device__ __forceinline__ unsigned int mx_quad_max(unsigned int v) {
    unsigned int o = (unsigned int)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, true);        // lanes 1 0 3 2
    v = o > v ? o : v;
    o = (unsigned int)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, true);                     // lanes 2 3 0 1
    return o > v ? o : v;
}
template <typename T> struct MxRaw8 { T v[8]; };
// eight neighbours of a row; zeros behind the last column
template <typename T, bool VEC>
__device__ __forceinline__ MxRaw8<T> mx_load8(const T* __restrict__ x, int64_t c0, int64_t cols, int64_t cs) {
    MxRaw8<T> r;
    if (VEC && c0 + 8 <= cols) {
        const mx_u4* p = reinterpret_cast<const mx_u4*>(x + c0);
        mx_u4 t[sizeof(T) / 2];
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) t[i] = p[i];
        __builtin_memcpy(&r, t, sizeof(r));
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) r.v[j] = c0 + j < cols ? x[(c0 + j) * cs] : (T)0.0f;
    }
    return r;
}

// x[r * rs + c * cs] -> codes, scales.  Bound: reading x.  Four lanes share a block, each takes 8 columns (16 bytes of a 16-bit type: VEC, when
// rows are contiguous and aligned), a few of them in flight per thread.  grid (row groups, column chunks)
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void mx_quantize_kernel(const T* __restrict__ x, int64_t rows, int64_t cols, int64_t rs, int64_t cs,
                                                          unsigned char* __restrict__ codes, unsigned char* __restrict__ scales, int tpr_log2) {
    constexpr int U = sizeof(T) == 8 ? 1 : 2;
    const int64_t crow = mx_code_row(cols), srow = mx_scale_row(cols);
    const int tpr = 1 << tpr_log2;
    const int64_t r = (int64_t)blockIdx.x * (256 >> tpr_log2) + (threadIdx.x >> tpr_log2);
    if (r >= rows) return;                                     // (whole groups of 4 lanes: tpr >= 32)
    const int64_t stride = (int64_t)gridDim.y * tpr;
    for (int64_t c8 = (int64_t)blockIdx.y * tpr + (threadIdx.x & (tpr - 1)); c8 < srow * 4; c8 += U * stride) {
        MxRaw8<T> raw[U];
#pragma unroll
        for (int u = 0; u < U; ++u) raw[u] = mx_load8<T, VEC>(x + r * rs, (c8 + u * stride) * 8, cols, cs);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t c = c8 + u * stride;
            float v[8];
            unsigned int am = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                v[j] = mx_to_f32(raw[u].v[j]);
                const unsigned int b = __float_as_uint(v[j]) & 0x7fffffffu;
                am = b > am ? b : am;
            }
            const int sc = mx_scale_of(mx_quad_max(am));
            if (c * 4 < crow) *reinterpret_cast<unsigned int*>(codes + r * crow + c * 4) = mx_pack8(v, sc);
            if ((threadIdx.x & 3) == 0 && c < srow * 4) scales[r * srow + mx_scale_at(c >> 2)] = (unsigned char)sc;
        }
    }
}

// the same for a matrix whose ROWS are neighbours in memory (rs == 1: a transposed view).  A block of 8 waves takes 64 rows x 512 columns; lane =
// row, so that every load of a wave is contiguous; a thread holds whole blocks of 32 columns.  Codes cross through LDS (16-byte pieces at piece ^
// (row & 15): a wave writes one piece of 64 rows, then stores whole rows).
template <typename T>
__global__ __launch_bounds__(512) void mx_quantize_across_kernel(const T* __restrict__ x, int64_t rows, int64_t cols, int64_t cs,
                                                                 unsigned char* __restrict__ codes, unsigned char* __restrict__ scales, int64_t rtiles) {
    const int64_t crow = mx_code_row(cols), srow = mx_scale_row(cols);
    __shared__ mx_u4 lc[64][16];
    __shared__ __attribute__((aligned(16))) unsigned char ls[64][16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t r0 = (int64_t)(blockIdx.x % rtiles) * 64, c0 = (int64_t)(blockIdx.x / rtiles) * 512;
    const T* p = x + (r0 + lane < rows ? r0 + lane : rows - 1);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int b = wave * 2 + h;
        const int64_t c = c0 + b * 32;
        T raw[32];
        if (c + 32 <= cols) {
#pragma unroll
            for (int j = 0; j < 32; ++j) raw[j] = p[(c + j) * cs];
        } else {
#pragma unroll
            for (int j = 0; j < 32; ++j) raw[j] = c + j < cols ? p[(c + j) * cs] : (T)0.0f;
        }
        float v[32];
        unsigned int am = 0;
#pragma unroll
        for (int j = 0; j < 32; ++j) {
            v[j] = mx_to_f32(raw[j]);
            const unsigned int u = __float_as_uint(v[j]) & 0x7fffffffu;
            am = u > am ? u : am;
        }
        const int sc = mx_scale_of(am);
        lc[lane][b ^ (lane & 15)] = mx_u4{mx_pack8(v, sc), mx_pack8(v + 8, sc), mx_pack8(v + 16, sc), mx_pack8(v + 24, sc)};
        ls[lane][mx_scale_at(b)] = (unsigned char)sc;
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int r = (threadIdx.x >> 4) + h * 32, piece = threadIdx.x & 15;
        if (r0 + r < rows && c0 / 2 + piece * 16 < crow) *reinterpret_cast<mx_u4*>(codes + (r0 + r) * crow + c0 / 2 + piece * 16) = lc[r][piece ^ (r & 15)];
    }
    if (threadIdx.x < 256 && r0 + (threadIdx.x >> 2) < rows)
        *reinterpret_cast<unsigned int*>(scales + (r0 + (threadIdx.x >> 2)) * srow + c0 / 32 + (threadIdx.x & 3) * 4) =
            *reinterpret_cast<const unsigned int*>(&ls[threadIdx.x >> 2][(threadIdx.x & 3) * 4]);
}

template <typename T> __device__ __forceinline__ T mx_from_f32(float v) { return (T)v; }

__device__ __forceinline__ void mx_values8(unsigned int q, float s, float* v) {
    mx_f2 p;
    p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, s, 0); v[0] = p[0]; v[1] = p[1];
    p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, s, 1); v[2] = p[0]; v[3] = p[1];
    p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, s, 2); v[4] = p[0]; v[5] = p[1];
    p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, s, 3); v[6] = p[0]; v[7] = p[1];
}

// codes, scales -> out[r * rs + c * cs].  Bound: writing out.  VEC: rows of out are contiguous and aligned to 16 bytes
template <typename T, bool VEC>
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
        mx_values8(q, s, v);
        T* p = out + r * rs + c8 * 8 * cs;
        if (VEC && c8 * 8 + 8 <= cols) {
            MxRaw8<T> o;
#pragma unroll
            for (int j = 0; j < 8; ++j) o.v[j] = mx_from_f32<T>(v[j]);
            mx_u4 t[sizeof(T) / 2];
            __builtin_memcpy(t, &o, sizeof(o));
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<mx_u4*>(p)[i] = t[i];
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (c8 * 8 + j < cols) p[j * cs] = mx_from_f32<T>(v[j]);
        }
    }
}

// the same into a matrix whose rows are neighbours in memory (rs == 1): the mirror image of mx_quantize_across_kernel
template <typename T>
__global__ __launch_bounds__(512) void mx_dequantize_across_kernel(const unsigned char* __restrict__ codes, const unsigned char* __restrict__ scales,
                                                                   int64_t rows, int64_t cols, T* __restrict__ out, int64_t cs, int64_t rtiles) {
    const int64_t crow = mx_code_row(cols), srow = mx_scale_row(cols);
    __shared__ mx_u4 lc[64][16];
    __shared__ __attribute__((aligned(16))) unsigned char ls[64][16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t r0 = (int64_t)(blockIdx.x % rtiles) * 64, c0 = (int64_t)(blockIdx.x / rtiles) * 512;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int r = (threadIdx.x >> 4) + h * 32, piece = threadIdx.x & 15;
        mx_u4 q = {0, 0, 0, 0};
        if (r0 + r < rows && c0 / 2 + piece * 16 < crow) q = *reinterpret_cast<const mx_u4*>(codes + (r0 + r) * crow + c0 / 2 + piece * 16);
        lc[r][piece ^ (r & 15)] = q;
    }
    if (threadIdx.x < 256 && r0 + (threadIdx.x >> 2) < rows)
        *reinterpret_cast<unsigned int*>(&ls[threadIdx.x >> 2][(threadIdx.x & 3) * 4]) =
            *reinterpret_cast<const unsigned int*>(scales + (r0 + (threadIdx.x >> 2)) * srow + c0 / 32 + (threadIdx.x & 3) * 4);
    __syncthreads();
    if (r0 + lane >= rows) return;
    T* p = out + r0 + lane;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int b = wave * 2 + h;
        const int64_t c = c0 + b * 32;
        if (c >= cols) break;
        const mx_u4 q = lc[lane][b ^ (lane & 15)];
        const float s = __uint_as_float((unsigned int)ls[lane][mx_scale_at(b)] << 23);
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            float v[8];
            mx_values8(q[d], s, v);
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (c + 8 * d + j < cols) p[(c + 8 * d + j) * cs] = mx_from_f32<T>(v[j]);
        }
    }
}

// ---- products of x (float32, bf16, fp16) with a 4-bit matrix -----------------------------------------------------------------------
// eight codes of one block -> bf16 (exact: at most 2 significant bits)
__device__ __forceinline__ mx_bf8 mx_unpack8(unsigned int q, float s) {
    const mx_bf2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, s, 0), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, s, 1),
                 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, s, 2), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, s, 3);
    return mx_bf8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// x[t * rs + k * cs], eight k from k0 on, as bf16 terms; zeros from nk on.  VEC: cs is 1, the eight values are aligned to 16 bytes and nk is a
// multiple of 8.  t must be a row.
template <typename T, int TERMS, bool VEC>
__device__ __forceinline__ void mx_load_terms(const T* __restrict__ x, int64_t t, int64_t rs, int64_t k0, int64_t nk, int64_t cs, mx_bf8* f) {
    T v[8];
    if constexpr (VEC) {
        if (k0 < nk) {
            const mx_u4* p = reinterpret_cast<const mx_u4*>(x + t * rs + k0);
            mx_u4 r[sizeof(T) / 2];
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; ++i) r[i] = p[i];
            __builtin_memcpy(v, r, sizeof(v));
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = (T)0.0f;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = k0 + j < nk ? x[t * rs + (k0 + j) * cs] : (T)0.0f;
    }
    if constexpr (TERMS == 1) {
#pragma unroll
        for (int j = 0; j < 8; ++j) f[0][j] = (__bf16)v[j];
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float p[3];
            mx_split<TERMS>((float)v[j], p);
#pragma unroll
            for (int u = 0; u < TERMS; ++u) f[u][j] = (__bf16)p[u];
        }
    }
}

// where an output goes: split == 1 the result, else float32 partial sums [split][M][O] (mx_join_kernel adds them up in order)
template <typename T> struct MxOut {
    T* out;
    int64_t rs, cs;
    float* part;
    int64_t M, O;
};
// N consecutive columns o .. of row t
template <typename T, int N>
__device__ __forceinline__ void mx_store(const MxOut<T>& w, int64_t z, int64_t t, int64_t o, const float* v) {
    if (t >= w.M) return;
    if (w.part) {
        float* p = w.part + (z * w.M + t) * w.O + o;
        if (o + N <= w.O && ((uintptr_t)p & 15) == 0) {
#pragma unroll
            for (int j = 0; j < N; j += 4) *reinterpret_cast<mx_f4*>(p + j) = mx_f4{v[j], v[j + 1], v[j + 2], v[j + 3]};
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (o + j < w.O) p[j] = v[j];
        }
        return;
    }
    T* p = w.out + t * w.rs + o * w.cs;
    if (w.cs == 1 && o + N <= w.O && ((uintptr_t)p & (N * sizeof(T) - 1)) == 0) {
        typedef T vec __attribute__((ext_vector_type(N)));
        vec r;
#pragma unroll
        for (int j = 0; j < N; ++j) r[j] = mx_from_f32<T>(v[j]);
        *reinterpret_cast<vec*>(p) = r;
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (o + j < w.O) p[j * w.cs] = mx_from_f32<T>(v[j]);
    }
}
// out[t][o] = sum over the splits, in order
template <typename T>
__global__ __launch_bounds__(256) void mx_join_kernel(const float* __restrict__ part, int split, int64_t M, int64_t O, T* __restrict__ out, int64_t rs,
                                                      int64_t cs) {
    const int64_t n = M * O;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        float v = part[i];
        for (int z = 1; z < split; ++z) v += part[(int64_t)z * n + i];
        out[(i / O) * rs + (i % O) * cs] = mx_from_f32<T>(v);
    }
}

// ---- few rows of x (up to 16: tokens being decoded) -----------------------------------------------------------------------------
// out[t][n] = sum_k x[t][k] W[n][k], W in 4 bits with its blocks along k: the codes become bf16 in registers, x is split into bf16 terms
// (MxTerms), every product is exact, float32 sums.  Bound: reading W (4.25 bits a value).  The waves of a block share 16 RT rows of W and
// split the contraction (128 columns a step), so that a single token still puts every load of W in flight at once; partial sums meet in LDS.
template <typename T, int RT, int WAVES, bool VEC>
__global__ __launch_bounds__(64 * WAVES) void mx_linear_row_kernel(const T* __restrict__ x, int64_t M, int64_t xrs, int64_t xcs,
                                                                   const unsigned char* __restrict__ wc, const unsigned char* __restrict__ ws, int64_t N,
                                                                   int64_t K, MxOut<T> w) {
    constexpr int TERMS = MxTerms<T>::v, U = 4;
    const int64_t crow = mx_code_row(K), srow = mx_scale_row(K);
    const int64_t n0 = (int64_t)blockIdx.x * 16 * RT;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = lane & 15, g = lane >> 4;
    const int64_t t = l < M ? l : M - 1;                       // rows behind the last one repeat it and are not stored
    const unsigned char *pc[RT], *ps[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        const int64_t rn = n0 + 16 * i + l < N ? n0 + 16 * i + l : N - 1;
        pc[i] = wc + rn * crow + g * 16;
        ps[i] = ws + rn * srow + g * 4;
    }
    mx_f4 acc[RT] = {};
    const int64_t steps = (K + 127) / 128;
    for (int64_t s0 = wave; s0 < steps; s0 += U * WAVES) {
        mx_u4 q[U][RT];
        unsigned int sc[U][RT];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t s = s0 + u * WAVES;
            if (s < steps) {
#pragma unroll
                for (int i = 0; i < RT; ++i) {
                    q[u][i] = *reinterpret_cast<const mx_u4*>(pc[i] + s * 64);
                    sc[u][i] = ps[i][(s >> 2) * 16 + (s & 3)];
                }
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t s = s0 + u * WAVES;
            if (s < steps) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    mx_bf8 f[TERMS];
                    mx_load_terms<T, TERMS, VEC>(x, t, xrs, s * 128 + g * 32 + j * 8, K, xcs, f);
#pragma unroll
                    for (int i = 0; i < RT; ++i) {
                        const mx_bf8 a = mx_unpack8(q[u][i][j], __uint_as_float(sc[u][i] << 23));
#pragma unroll
                        for (int e = 0; e < TERMS; ++e) acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, f[e], acc[i], 0, 0, 0);
                    }
                }
            }
        }
    }
    __shared__ mx_f4 red[WAVES][RT][64];
#pragma unroll
    for (int i = 0; i < RT; ++i) red[wave][i][lane] = acc[i];
    __syncthreads();
    for (int i = wave; i < RT; i += WAVES) {
        mx_f4 v = red[0][i][lane];
#pragma unroll
        for (int k = 1; k < WAVES; ++k) v += red[k][i][lane];
        float o[4] = {v[0], v[1], v[2], v[3]};
        mx_store<T, 4>(w, 0, l, n0 + 16 * i + 4 * g, o);
    }
}

// 8 columns of one row of W as bf16, entry m of dword j -> what matrix instruction m takes from this lane: the transposition of an 8 x 8 piece
// that the lane holds whole, two values a dword
__device__ __forceinline__ void mx_unpack_across(const unsigned int* q, const unsigned int* sc, mx_bf8* w) {
    unsigned int u[8][4];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const mx_bf8 v = mx_unpack8(q[j], __uint_as_float(sc[j] << 23));
        __builtin_memcpy(u[j], &v, 16);
    }
#pragma unroll
    for (int m = 0; m < 8; ++m) {
        unsigned int r[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            r[j] = __builtin_amdgcn_perm(u[2 * j + 1][m >> 1], u[2 * j][m >> 1], (m & 1) ? 0x07060302u : 0x05040100u);
        __builtin_memcpy(&w[m], r, 16);
    }
}

// dx[t][k] = sum_n dy[t][n] W[n][k], up to 16 rows: the contraction runs ACROSS the blocks.  A lane reads 16 bytes (32 columns: one block, one
// scale) from each of 8 rows of W; entry m of the eight is what matrix instruction m needs from this lane: column 32 (lane % 16) + m,
// eight n.  So a wave owns 512 columns as 32 tiles and no value crosses lanes.  The waves of a block split the rows, the blocks along
// y too (partial sums to memory).
template <typename T, int WAVES, bool VEC>
__global__ __launch_bounds__(64 * WAVES) void mx_grad_row_kernel(const T* __restrict__ dy, int64_t M, int64_t yrs, int64_t ycs,
                                                                 const unsigned char* __restrict__ wc, const unsigned char* __restrict__ ws, int64_t N,
                                                                 int64_t K, MxOut<T> w) {
    constexpr int TERMS = MxTerms<T>::v;
    const int64_t crow = mx_code_row(K), srow = mx_scale_row(K);
    const int64_t k0 = (int64_t)blockIdx.x * 512;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = lane & 15, g = lane >> 4;
    const int64_t t = l < M ? l : M - 1;
    // (columns behind the row repeat its last 16 bytes and are not stored)
    const int64_t kb = k0 / 2 + l * 16 < crow ? k0 / 2 + l * 16 : crow - 16;
    const int64_t sat = mx_scale_at(kb >> 4);
    mx_f4 acc[32] = {};
    const int64_t steps = (N + 31) / 32, stride = (int64_t)WAVES * gridDim.y;
    for (int64_t s = (int64_t)blockIdx.y * WAVES + wave; s < steps; s += stride) {
        mx_u4 q[8];
        unsigned int sc[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int64_t n = s * 32 + g * 8 + j;
            // rows behind the last one are zeros with a finite scale (their factor in dy is zero too, but must not meet a NaN)
            q[j] = n < N ? *reinterpret_cast<const mx_u4*>(wc + n * crow + kb) : mx_u4{0, 0, 0, 0};
            sc[j] = n < N ? ws[n * srow + sat] : 127u;
        }
        mx_bf8 f[TERMS];
        mx_load_terms<T, TERMS, VEC>(dy, t, yrs, s * 32 + g * 8, N, ycs, f);
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            unsigned int qd[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) qd[j] = q[j][d];
            mx_bf8 a[8];
            mx_unpack_across(qd, sc, a);
#pragma unroll
            for (int m = 0; m < 8; ++m)
#pragma unroll
                for (int e = 0; e < TERMS; ++e) acc[d * 8 + m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[m], f[e], acc[d * 8 + m], 0, 0, 0);
        }
    }
    __shared__ mx_f4 red[WAVES][8][64];
#pragma unroll
    for (int d = 0; d < 4; ++d) {
        if (d) __syncthreads();
#pragma unroll
        for (int m = 0; m < 8; ++m) red[wave][m][lane] = acc[d * 8 + m];
        __syncthreads();
        // lane (l, g) of output row 4 g + e holds columns 32 (4 g + e) + 8 d + m
        for (int e = wave; e < 4; e += WAVES) {
            float o[8];
#pragma unroll
            for (int m = 0; m < 8; ++m) {
                o[m] = red[0][m][lane][e];
#pragma unroll
                for (int k = 1; k < WAVES; ++k) o[m] += red[k][m][lane][e];
            }
            mx_store<T, 8>(w, blockIdx.y, l, k0 + 32 * (4 * g + e) + 8 * d, o);
        }
    }
}

// ---- many rows of x -------------------------------------------------------------------------------------------------------------
// The rows of x meet the matrix instructions as bf16 fragments: 16 rows, 32 of the contraction, 64 lanes x 16 bytes.  Fragment i of the
// contraction holds, for lane group g, eight values from
//   along the blocks   128 (i / 4) + 32 g + 8 (i % 4)      (a lane of W owns one block of each 128 columns, 8 values an instruction)
//   across the blocks  32 i + 8 g
// mx_fragments_kernel lays x out that way once per call, split into its bf16 terms: frag[i][term][tile of 16 rows][lane][8].  A tile of the
// products below is then a contiguous piece of memory, whatever x's type, strides or odd sizes.
template <bool ALONG> __device__ __forceinline__ int64_t mx_frag_k(int64_t i, int g) {
    return ALONG ? (i >> 2) * 128 + g * 32 + (i & 3) * 8 : i * 32 + g * 8;
}
template <typename T, bool ALONG, bool VEC>
__global__ __launch_bounds__(256) void mx_fragments_kernel(const T* __restrict__ x, int64_t M, int64_t xrs, int64_t xcs, int64_t K, int64_t nfrag,
                                                           int64_t tiles, unsigned short* __restrict__ frag, int rows_first) {
    constexpr int TERMS = MxTerms<T>::v;
    // a block takes one tile of 16 rows and 16 groups of 8 values; neighbouring threads read neighbouring memory
    const int64_t tile = blockIdx.x % tiles, c0 = (int64_t)(blockIdx.x / tiles) * 16;
    const int l = rows_first ? threadIdx.x & 15 : threadIdx.x >> 4;
    const int64_t c = c0 + (rows_first ? threadIdx.x >> 4 : threadIdx.x & 15);         // group of 8 along the contraction
    if (c >= nfrag * 4) return;
    const int64_t i = ALONG ? (c >> 4) * 4 + (c & 3) : c >> 2;
    const int g = (int)(ALONG ? (c >> 2) & 3 : c & 3);
    const int64_t t = tile * 16 + l;
    mx_bf8 f[TERMS] = {};
    if (t < M) mx_load_terms<T, TERMS, VEC>(x, t, xrs, c * 8, K, xcs, f);
#pragma unroll
    for (int u = 0; u < TERMS; ++u) *reinterpret_cast<mx_bf8*>(frag + (((i * TERMS + u) * tiles + tile) * 64 + g * 16 + l) * 8) = f[u];
}

typedef __attribute__((address_space(1))) const void* mx_gptr;
typedef __attribute__((address_space(3))) void* mx_lptr;

// block -> (row tile, column tile, split): consecutive blocks go to the 8 XCDs in turn, so each XCD gets a contiguous piece of an order in which
// eight row tiles share a column tile of W
struct MxTile { int64_t a, b; int z; };
__device__ __forceinline__ MxTile mx_tile(int64_t id, int64_t na, int64_t nb, int split) {
    const int64_t total = na * nb * split, per = (total + 7) / 8;
    int64_t p = (id & 7) * per + (id >> 3);
    MxTile r;
    if (p >= total || (id >> 3) >= per) { r.a = -1; r.b = 0; r.z = 0; return r; }
    r.z = (int)(p / (na * nb));
    p -= (int64_t)r.z * na * nb;
    const int64_t grp = p / (8 * nb), left = na - grp * 8 < 8 ? na - grp * 8 : 8;
    p -= grp * 8 * nb;
    r.a = grp * 8 + p % left;
    r.b = p / left;
    return r;
}

// out[t][n] = sum_k x[t][k] W[n][k] for tiles of 16 CT rows of x and 64 RT rows of W.  Bound: the bf16 matrix pipe (TERMS instructions per
// product).  The four waves own 16 RT rows of W each - codes go from memory to registers and become bf16 there, no LDS - and share the fragments
// of x through LDS (JS of them a stage, double buffered).
template <typename T, int CT, int RT, int JS>
__global__ __launch_bounds__(256, 2) void mx_linear_tile_kernel(const unsigned short* __restrict__ frag, int64_t tiles, const unsigned char* __restrict__ wc,
                                                             const unsigned char* __restrict__ ws, int64_t N, int64_t K, MxOut<T> w, int64_t mt,
                                                             int64_t nt, int split) {
    constexpr int TERMS = MxTerms<T>::v, CH = JS * TERMS * CT;             // 1 KB pieces a stage
    const int64_t crow = mx_code_row(K), srow = mx_scale_row(K);
    const MxTile tile = mx_tile(blockIdx.x, mt, nt, split);
    if (tile.a < 0) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = lane & 15, g = lane >> 4;
    const int64_t n0 = tile.b * 64 * RT + wave * 16 * RT;
    const int64_t steps = (K + 127) / 128, per = ((steps + split - 1) / split + 3) / 4 * 4;      // (whole dwords of scales)
    const int64_t s0 = per * tile.z, s1 = s0 + per < steps ? s0 + per : steps;
    __shared__ __attribute__((aligned(16))) unsigned short lds[2][CH * 512];
    const unsigned char *pc[RT], *ps[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        const int64_t rn = n0 + 16 * i + l < N ? n0 + 16 * i + l : N - 1;
        pc[i] = wc + rn * crow + g * 16;
        ps[i] = ws + rn * srow + g * 4;
    }
    auto stage = [&](int64_t f, int b) {                                   // fragments f .. f + JS of the contraction
#pragma unroll
        for (int c = 0; c < (CH + 3) / 4; ++c) {
            const int i = c * 4 + wave;
            if (CH % 4 == 0 || i < CH) {
                const int64_t at = ((f * TERMS + i / CT) * tiles + tile.a * CT + i % CT) * 512;
                __builtin_amdgcn_global_load_lds((mx_gptr)(frag + at + lane * 8), (mx_lptr)(&lds[b][i * 512]), 16, 0, 0);
            }
        }
    };
    mx_f4 acc[RT][CT] = {};
    mx_u4 q[RT];
    unsigned int sd[RT];
    if (s0 < s1) {
        stage(s0 * 4, 0);
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            q[i] = *reinterpret_cast<const mx_u4*>(pc[i] + s0 * 64);
            sd[i] = *reinterpret_cast<const unsigned int*>(ps[i] + (s0 >> 2) * 16);
        }
    }
    __syncthreads();
    int b = 0;
    for (int64_t s = s0; s < s1; ++s) {
        mx_u4 qn[RT];
        unsigned int sn[RT];
#pragma unroll
        for (int i = 0; i < RT; ++i) { qn[i] = q[i]; sn[i] = sd[i]; }
        float sc[RT];
#pragma unroll
        for (int i = 0; i < RT; ++i) sc[i] = __uint_as_float(((sd[i] >> (8 * (s & 3))) & 255u) << 23);
#pragma unroll
        for (int h = 0; h < 4 / JS; ++h) {
            if (h + 1 < 4 / JS) stage(s * 4 + (h + 1) * JS, b ^ 1);
            else if (s + 1 < s1) stage((s + 1) * 4, b ^ 1);
            if (h == 0 && s + 1 < s1) {
#pragma unroll
                for (int i = 0; i < RT; ++i) {
                    qn[i] = *reinterpret_cast<const mx_u4*>(pc[i] + (s + 1) * 64);
                    if (((s + 1) & 3) == 0) sn[i] = *reinterpret_cast<const unsigned int*>(ps[i] + ((s + 1) >> 2) * 16);
                }
            }
#pragma unroll
            for (int jj = 0; jj < JS; ++jj) {
                mx_bf8 a[RT];
#pragma unroll
                for (int i = 0; i < RT; ++i) a[i] = mx_unpack8(q[i][h * JS + jj], sc[i]);
#pragma unroll
                for (int u = 0; u < TERMS; ++u)
#pragma unroll
                    for (int c = 0; c < CT; ++c) {
                        const mx_bf8 f = *reinterpret_cast<const mx_bf8*>(&lds[b][((jj * TERMS + u) * CT + c) * 512 + lane * 8]);
#pragma unroll
                        for (int i = 0; i < RT; ++i) acc[i][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i], f, acc[i][c], 0, 0, 0);
                    }
            }
            __syncthreads();
            b ^= 1;
        }
#pragma unroll
        for (int i = 0; i < RT; ++i) { q[i] = qn[i]; sd[i] = sn[i]; }
    }
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            float o[4] = {acc[i][c][0], acc[i][c][1], acc[i][c][2], acc[i][c][3]};
            mx_store<T, 4>(w, tile.z, (tile.a * CT + c) * 16 + l, n0 + 16 * i + 4 * g, o);
        }
}

// dx[t][k] = sum_n dy[t][n] W[n][k] for tiles of 16 CT rows of dy and 512 columns of W: as mx_grad_row_kernel, 128 columns a wave (a dword of 8
// columns from each of 8 rows, 8 tiles).  Bound: the bf16 matrix pipe; unpacking costs a cycle of the vector pipe per value of W and tile of
// rows, so a tile takes as many rows as the registers hold.  32 JS rows of W (codes, scales) and their fragments of dy a stage, all of them to
// LDS without passing registers, double buffered: the loads of W are 64-byte pieces whose latency nothing else would hide.  The 16-byte
// pieces of a row of codes are stored at piece ^ 4 ((row / 8) % 4): the four lane groups read different banks.
template <int CT, int JS, int TERMS> struct MxGradLds {
    static constexpr int frag = JS * TERMS * CT * 1024, codes = JS * 32 * 256, scales = JS * 32 * 16, stage = frag + codes + scales;
};
template <typename T, int CT, int JS>
__global__ __launch_bounds__(256, 2) void mx_grad_tile_kernel(const unsigned short* __restrict__ frag, int64_t tiles, const unsigned char* __restrict__ wc,
                                                                             const unsigned char* __restrict__ ws, int64_t N, int64_t K, MxOut<T> w, int64_t mt,
                                                                             int64_t nt, int split) {
    constexpr int TERMS = MxTerms<T>::v, CH = JS * TERMS * CT;
    typedef MxGradLds<CT, JS, TERMS> L;
    const int64_t crow = mx_code_row(K), srow = mx_scale_row(K);
    const MxTile tile = mx_tile(blockIdx.x, mt, nt, split);
    if (tile.a < 0) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = lane & 15, g = lane >> 4;
    const int64_t kblk = tile.b * 512, k0 = kblk + wave * 128;
    const int64_t steps = (N + 31) / 32, per = ((steps + split - 1) / split + JS - 1) / JS * JS;
    const int64_t s0 = per * tile.z, s1 = s0 + per < steps ? s0 + per : steps;
    extern __shared__ __attribute__((aligned(16))) unsigned char glds[];
    auto stage = [&](int64_t s, int b) {
        unsigned char* at = glds + b * L::stage;
#pragma unroll
        for (int c = 0; c < (CH + 3) / 4; ++c) {
            const int i = c * 4 + wave;
            if (CH % 4 == 0 || i < CH)
                __builtin_amdgcn_global_load_lds((mx_gptr)(frag + ((s * TERMS + i / CT) * tiles + tile.a * CT + i % CT) * 512 + lane * 8),
                                                 (mx_lptr)(at + i * 1024), 16, 0, 0);
        }
#pragma unroll
        for (int c = 0; c < JS * 2; ++c) {                     // 4 rows of codes a piece
            const int r = (c * 4 + wave) * 4 + lane / 16, piece = (lane & 15) ^ (((r >> 3) & 3) * 4);
            const int64_t n = s * 32 + r < N ? s * 32 + r : N - 1, kb = kblk / 2 + piece * 16 < crow ? kblk / 2 + piece * 16 : crow - 16;
            __builtin_amdgcn_global_load_lds((mx_gptr)(wc + n * crow + kb), (mx_lptr)(at + L::frag + (c * 4 + wave) * 1024), 16, 0, 0);
        }
        if (lane < 32 && wave < JS) {                          // 32 rows of scales a piece
            const int64_t n = s * 32 + wave * 32 + lane < N ? s * 32 + wave * 32 + lane : N - 1;
            __builtin_amdgcn_global_load_lds((mx_gptr)(ws + n * srow + kblk / 32), (mx_lptr)(at + L::frag + L::codes + wave * 512), 16, 0, 0);
        }
    };
    mx_f4 acc[8][CT] = {};
    if (s0 < s1) stage(s0, 0);
    __syncthreads();
    int b = 0;
    // a lane's dword of row 8 g + j, and the byte of its block's scale
    const int qat = L::frag + g * 8 * 256 + (((wave * 4 + (l >> 2)) ^ (g * 4)) * 16) + (l & 3) * 4;
    const int sat = L::frag + L::codes + g * 8 * 16 + (l >> 2) * 4 + wave;
    for (int64_t s = s0; s < s1; s += JS) {
        if (s + JS < s1) stage(s + JS, b ^ 1);
        const unsigned char* at = glds + b * L::stage;
#pragma unroll
        for (int jj = 0; jj < JS; ++jj) {
            if (JS > 1 && s + jj >= s1) break;
            unsigned int q[8], sc[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                q[j] = *reinterpret_cast<const unsigned int*>(at + qat + jj * 32 * 256 + j * 256);
                sc[j] = at[sat + jj * 32 * 16 + j * 16];
            }
            if ((s + jj) * 32 + 32 > N) {
                // rows behind the last one are zeros with a finite scale (their factor in dy is zero too, but must not meet a NaN)
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if ((s + jj) * 32 + g * 8 + j >= N) { q[j] = 0; sc[j] = 127; }
            }
            mx_bf8 a[8];
            mx_unpack_across(q, sc, a);
#pragma unroll
            for (int u = 0; u < TERMS; ++u)
#pragma unroll
                for (int c = 0; c < CT; ++c) {
                    const mx_bf8 f = *reinterpret_cast<const mx_bf8*>(at + ((jj * TERMS + u) * CT + c) * 1024 + lane * 16);
#pragma unroll
                    for (int m = 0; m < 8; ++m) acc[m][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[m], f, acc[m][c], 0, 0, 0);
                }
        }
        __syncthreads();
        b ^= 1;
    }
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float o[8];
#pragma unroll
            for (int m = 0; m < 8; ++m) o[m] = acc[m][c][e];
            mx_store<T, 8>(w, tile.z, (tile.a * CT + c) * 16 + l, k0 + 8 * (4 * g + e), o);
        }
}

// ---- 4 bits x 4 bits -------------------------------------------------------------------------------------------------------------
// out[m][n] = sum_k A[m][k] B[n][k] on v_mfma_scale_f32_16x16x128_f8f6f4: a lane holds one block of 32 of its row (16 bytes) and that block's
// scale; the instruction multiplies codes and scales, float32 sums.  Rows behind the last one repeat it and are not stored.
__device__ __forceinline__ mx_i8 mx_operand(mx_u4 q) { return mx_i8{(int)q[0], (int)q[1], (int)q[2], (int)q[3], 0, 0, 0, 0}; }

// up to 16 rows of A: as mx_linear_row_kernel, bound by reading B
template <typename T, int RT, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void mx_matmul_row_kernel(const unsigned char* __restrict__ ac, const unsigned char* __restrict__ as, int64_t M,
                                                                   const unsigned char* __restrict__ bc, const unsigned char* __restrict__ bs, int64_t N,
                                                                   int64_t K, MxOut<T> w) {
    constexpr int U = 4;
    const int64_t crow = mx_code_row(K), srow = mx_scale_row(K);
    const int64_t n0 = (int64_t)blockIdx.x * 16 * RT;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = lane & 15, g = lane >> 4;
    const int64_t t = l < M ? l : M - 1;
    const unsigned char *pc[RT], *ps[RT], *pa = ac + t * crow + g * 16, *pas = as + t * srow + g * 4;
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        const int64_t rn = n0 + 16 * i + l < N ? n0 + 16 * i + l : N - 1;
        pc[i] = bc + rn * crow + g * 16;
        ps[i] = bs + rn * srow + g * 4;
    }
    mx_f4 acc[RT] = {};
    const int64_t steps = (K + 127) / 128;
    for (int64_t s0 = wave; s0 < steps; s0 += U * WAVES) {
        mx_u4 q[U][RT], qa[U];
        int sc[U][RT], sa[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t s = s0 + u * WAVES;
            if (s < steps) {
                qa[u] = *reinterpret_cast<const mx_u4*>(pa + s * 64);
                sa[u] = pas[(s >> 2) * 16 + (s & 3)];
#pragma unroll
                for (int i = 0; i < RT; ++i) {
                    q[u][i] = *reinterpret_cast<const mx_u4*>(pc[i] + s * 64);
                    sc[u][i] = ps[i][(s >> 2) * 16 + (s & 3)];
                }
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (s0 + u * WAVES < steps) {
#pragma unroll
                for (int i = 0; i < RT; ++i)
                    acc[i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx_operand(q[u][i]), mx_operand(qa[u]), acc[i], 4, 4, 0, sc[u][i], 0, sa[u]);
            }
    }
    __shared__ mx_f4 red[WAVES][RT][64];
#pragma unroll
    for (int i = 0; i < RT; ++i) red[wave][i][lane] = acc[i];
    __syncthreads();
    for (int i = wave; i < RT; i += WAVES) {
        mx_f4 v = red[0][i][lane];
#pragma unroll
        for (int k = 1; k < WAVES; ++k) v += red[k][i][lane];
        float o[4] = {v[0], v[1], v[2], v[3]};
        mx_store<T, 4>(w, 0, l, n0 + 16 * i + 4 * g, o);
    }
}

// Tiles of (WM x 16 RM) rows of A by (WN x 16 RN) rows of B; WM x WN waves of 16 RM x 16 RN outputs.  Bound: the 4-bit matrix pipe (16 cycles an
// instruction of 64 Kflop).  256 columns a stage: 128 bytes of each row come to LDS without passing registers, double buffered; the
// 16-byte pieces of a row are stored at piece ^ (row & 7), which spreads a fragment's sixteen rows over all banks.  Scales go from
// memory to registers, a dword for four steps.
template <typename T, int WM, int WN, int RM, int RN>
__global__ __launch_bounds__(64 * WM * WN, 2) void mx_matmul_tile_kernel(const unsigned char* __restrict__ ac, const unsigned char* __restrict__ as,
                                                                     const unsigned char* __restrict__ bc, const unsigned char* __restrict__ bs, int64_t N,
                                                                     int64_t K, MxOut<T> w, int64_t mt, int64_t nt, int split) {
    constexpr int BM = WM * 16 * RM, BN = WN * 16 * RN, NW = WM * WN, CH = (BM + BN) / 8;      // 1 KB pieces (8 rows x 128 bytes) a stage
    static_assert(CH % NW == 0, "");
    const int64_t crow = mx_code_row(K), srow = mx_scale_row(K), M = w.M;
    const MxTile tile = mx_tile(blockIdx.x, mt, nt, split);
    if (tile.a < 0) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = lane & 15, g = lane >> 4;
    const int64_t m0 = tile.a * BM, n0 = tile.b * BN;
    const int wm = (wave % WM) * 16 * RM, wn = (wave / WM) * 16 * RN;
    const int64_t steps = (K + 255) / 256, per = ((steps + split - 1) / split + 1) / 2 * 2;
    const int64_t s0 = per * tile.z, s1 = s0 + per < steps ? s0 + per : steps;
    extern __shared__ __attribute__((aligned(16))) unsigned char mlds[];   // [2][BM + BN][128]
    const unsigned char* src[CH / NW];
#pragma unroll
    for (int c = 0; c < CH / NW; ++c) {
        const int r = (c * NW + wave) * 8 + lane / 8, piece = (lane & 7) ^ (r & 7);
        if (r < BM) src[c] = ac + (m0 + r < M ? m0 + r : M - 1) * crow + piece * 16;
        else src[c] = bc + (n0 + r - BM < N ? n0 + r - BM : N - 1) * crow + piece * 16;
    }
    const unsigned char *psa[RM], *psb[RN];
#pragma unroll
    for (int i = 0; i < RM; ++i) psa[i] = as + (m0 + wm + 16 * i + l < M ? m0 + wm + 16 * i + l : M - 1) * srow + g * 4;
#pragma unroll
    for (int i = 0; i < RN; ++i) psb[i] = bs + (n0 + wn + 16 * i + l < N ? n0 + wn + 16 * i + l : N - 1) * srow + g * 4;
    auto stage = [&](int64_t s, int b) {
#pragma unroll
        for (int c = 0; c < CH / NW; ++c)
            __builtin_amdgcn_global_load_lds((mx_gptr)(src[c] + s * 128), (mx_lptr)(mlds + b * (BM + BN) * 128 + (c * NW + wave) * 1024), 16, 0, 0);
    };
    mx_f4 acc[RM][RN] = {};
    int sa[RM], sb[RN], san[RM], sbn[RN];
    if (s0 < s1) {
        stage(s0, 0);
#pragma unroll
        for (int i = 0; i < RM; ++i) sa[i] = *reinterpret_cast<const int*>(psa[i] + (s0 >> 1) * 16);
#pragma unroll
        for (int i = 0; i < RN; ++i) sb[i] = *reinterpret_cast<const int*>(psb[i] + (s0 >> 1) * 16);
    }
    __syncthreads();
    int b = 0;
    // two stages (512 columns: one dword of scales) a turn
    for (int64_t s = s0; s < s1; s += 2) {
        const int64_t sn = s + 2 < s1 ? s + 2 : s;
#pragma unroll
        for (int i = 0; i < RM; ++i) san[i] = *reinterpret_cast<const int*>(psa[i] + (sn >> 1) * 16);
#pragma unroll
        for (int i = 0; i < RN; ++i) sbn[i] = *reinterpret_cast<const int*>(psb[i] + (sn >> 1) * 16);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (s + h >= s1) break;
            if (s + h + 1 < s1) stage(s + h + 1, b ^ 1);
            const unsigned char* base = mlds + b * (BM + BN) * 128;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                mx_u4 fa[RM], fb[RN];
#pragma unroll
                for (int i = 0; i < RM; ++i) fa[i] = *reinterpret_cast<const mx_u4*>(base + (wm + 16 * i + l) * 128 + (((j * 4 + g) ^ (l & 7)) * 16));
#pragma unroll
                for (int i = 0; i < RN; ++i) fb[i] = *reinterpret_cast<const mx_u4*>(base + (BM + wn + 16 * i + l) * 128 + (((j * 4 + g) ^ (l & 7)) * 16));
#pragma unroll
                for (int i = 0; i < RM; ++i)
#pragma unroll
                    for (int k = 0; k < RN; ++k) {
                        // outputs transposed (B's rows along the instruction's rows): a lane ends up with four neighbours of one output row
                        if (h == 0 && j == 0) acc[i][k] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx_operand(fb[k]), mx_operand(fa[i]), acc[i][k], 4, 4, 0, sb[k], 0, sa[i]);
                        else if (h == 0) acc[i][k] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx_operand(fb[k]), mx_operand(fa[i]), acc[i][k], 4, 4, 1, sb[k], 1, sa[i]);
                        else if (j == 0) acc[i][k] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx_operand(fb[k]), mx_operand(fa[i]), acc[i][k], 4, 4, 2, sb[k], 2, sa[i]);
                        else acc[i][k] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx_operand(fb[k]), mx_operand(fa[i]), acc[i][k], 4, 4, 3, sb[k], 3, sa[i]);
                    }
            }
            __syncthreads();
            b ^= 1;
        }
#pragma unroll
        for (int i = 0; i < RM; ++i) sa[i] = san[i];
#pragma unroll
        for (int i = 0; i < RN; ++i) sb[i] = sbn[i];
    }
#pragma unroll
    for (int i = 0; i < RM; ++i)
#pragma unroll
        for (int k = 0; k < RN; ++k) {
            float o[4] = {acc[i][k][0], acc[i][k][1], acc[i][k][2], acc[i][k][3]};
            mx_store<T, 4>(w, tile.z, m0 + wm + 16 * i + l, n0 + wn + 16 * k + 4 * g, o);
        }
}

template <typename T>
__global__ __launch_bounds__(256) void mx_zero_kernel(T* __restrict__ out, int64_t rows, int64_t cols, int64_t rs, int64_t cs) {
    const int64_t n = rows * cols;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) out[(i / cols) * rs + (i % cols) * cs] = (T)0.0f;
}

}  // namespace lcx
