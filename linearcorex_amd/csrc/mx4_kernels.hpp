// mx4_kernels.hpp - matrices in 4 bits per value ("mx4"): quantisation, and products whose contraction runs along or across the blocks.
//
// A value is a 4-bit float (sign, 2 exponent bits, 1 mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6); 32 neighbours along a row share one
// power-of-two scale, held as its biased exponent (a byte: 2^(byte - 127); 255 = the whole block is NaN).  4.25 bits per value.
//
// Layout of an R x C matrix: that of the matrix instructions' operands, so that every kernel reads it in whole lines and a fragment needs no
// shuffling.  A fragment is 16 rows x 128 columns (a step): lane 16 g + l of a wave holds the 16 bytes of block 4 s + g (32 columns) of row
// l, two values a byte, the even column in the low half.
//   codes  [row tiles of 16][steps][64 lanes][16 bytes]          steps = columns / 128, rounded up to an even number
//   scales [row tiles of 16][steps / 4][64 lanes][4 bytes]       the lane's scales of four steps: one dword, of which the instructions (or a
//                                                                shift) pick a byte
// Padding rows and columns are zeros with the scale byte 2.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace lcx {

constexpr int MX_BLOCK = 32;
__host__ __device__ inline int64_t mx_steps(int64_t cols) { return (cols + 255) / 256 * 2; }           // 128 columns each
__host__ __device__ inline int64_t mx_quads(int64_t cols) { return (cols + 511) / 512; }               // groups of four steps
__host__ __device__ inline int64_t mx_row_tiles(int64_t rows) { return (rows + 15) / 16; }

typedef __attribute__((ext_vector_type(2))) __bf16 mx_bf2;
typedef __attribute__((ext_vector_type(8))) __bf16 mx_bf8;
typedef __attribute__((ext_vector_type(2))) float mx_f2;
typedef __attribute__((ext_vector_type(4))) float mx_f4;
typedef __attribute__((ext_vector_type(4))) unsigned int mx_u4;
typedef __attribute__((ext_vector_type(8))) int mx_i8;

// the wave's number in its block, known to be the same for all lanes (addresses that depend on it then live in scalar registers)
__device__ __forceinline__ int mx_wave() { return __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)); }

template <typename T> struct MxTerms;                              // bf16 numbers that add up to a T exactly
template <> struct MxTerms<float> { static constexpr int v = 3; };     // 24 significant bits = 8 + 8 + 8
template <> struct MxTerms<_Float16> { static constexpr int v = 2; };  // 11 = 8 + 3
template <> struct MxTerms<__bf16> { static constexpr int v = 1; };

__device__ __forceinline__ float mx_trunc_bf16(float x) { return __uint_as_float(__float_as_uint(x) & 0xffff0000u); }
// x = term 0 + term 1 + term 2, each a bf16 number: the leading 8 significant bits are cut off twice, what remains has at most 8.  Every
// term takes part in the products below, so cutting (rather than rounding) leaves no bias.  An infinity stays in term 0 alone (its
// remainder would be a NaN); a NaN leaves one in the remainder, whatever the cut makes of its payload.  Numbers below 2^-110 reach under
// bf16's last place, 2^-133: the last term is rounded to it.
template <int TERMS> __device__ __forceinline__ void mx_split(float x, float* t) {
    if constexpr (TERMS == 1) {
        t[0] = x;
    } else {
        t[0] = mx_trunc_bf16(x);
        const float r = __builtin_isinf(x) ? 0.0f : x - t[0];
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
// 16 bytes at an address that only the element type aligns
typedef unsigned int mx_u4u __attribute__((ext_vector_type(4), aligned(2)));
typedef float mx_f4u __attribute__((ext_vector_type(4), aligned(4)));
template <typename T, int N> __device__ __forceinline__ void mx_put(T* p, const T* v) {
    if constexpr (N * sizeof(T) % 16 == 0) {
        mx_u4 t[N * sizeof(T) / 16];
        __builtin_memcpy(t, v, sizeof(t));
#pragma unroll
        for (int i = 0; i < (int)(N * sizeof(T) / 16); ++i) reinterpret_cast<mx_u4u*>(p)[i] = t[i];
    } else {
        typedef unsigned int u2u __attribute__((ext_vector_type(2), aligned(2)));
        static_assert(N * sizeof(T) == 8, "");
        u2u t;
        __builtin_memcpy(&t, v, 8);
        *reinterpret_cast<u2u*>(p) = t;
    }
}
// eight neighbours of a row, read or written 16 bytes at a time from any address the element type allows (global memory takes it)
template <typename T> struct MxRaw8 { T v[8]; };
// zeros behind the last column; VEC: the columns are neighbours (cs == 1)
template <typename T, bool VEC, bool ONCE = false>
__device__ __forceinline__ MxRaw8<T> mx_load8(const T* __restrict__ x, int64_t c0, int64_t cols, int64_t cs) {
    MxRaw8<T> r;
    if (VEC && c0 + 8 <= cols) {
        mx_u4 t[sizeof(T) / 2];
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) t[i] = ONCE ? __builtin_nontemporal_load(reinterpret_cast<const mx_u4u*>(x + c0) + i) : reinterpret_cast<const mx_u4u*>(x + c0)[i];
        __builtin_memcpy(&r, t, sizeof(r));
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) r.v[j] = c0 + j < cols ? x[(c0 + j) * cs] : (T)0.0f;
    }
    return r;
}

// From this size on x is read past the caches: it does not fit what earlier kernels have left there to be written back, and loads that would take
// its place wait for that.  Measured (us; through / past the caches; x just written by another kernel, then after others' writes):
// 64 MB of bf16 16.3 / 17.1, 24 / 18; 128 MB 29.2 / 29.9, 44 / 32; 256 MB 65 / 47, 81 / 61; 20 MB of bf16 8.6 / 10.4, 9.2 / 6.6
constexpr int64_t MX_ONCE_BYTES = 128 << 20;

// x[r * rs + c * cs] -> codes, scales.  Bound: reading x.  A block takes 16 rows x 512 columns: a thread 8 columns of each of four steps (16 bytes
// of a 16-bit type each: VEC, where the columns are neighbours), so that it ends up with a whole dword of scales; four lanes share a
// block of 32.  grid (row tile, quad of steps); x holds the columns from quad quad0 on of a matrix of `steps` steps.
// ONCE: x is read past the caches (MX_ONCE_BYTES).  16384 x 8192 bf16 (340 MB read and written): 57 us, 5.9 TB/s; 32 x 4096: 3.4 us.
template <typename T, bool VEC, bool ONCE>
__global__ __launch_bounds__(256) void mx_quantize_kernel(const T* __restrict__ x, int64_t rows, int64_t cols, int64_t rs, int64_t cs,
                                                          unsigned char* __restrict__ codes, unsigned char* __restrict__ scales, int64_t steps, int64_t quads,
                                                          int64_t quad0, unsigned int nquads) {
    const unsigned int rt32 = blockIdx.x / nquads;
    const int64_t rt = rt32, here = blockIdx.x - rt32 * nquads, quad = quad0 + here;
    const int l = threadIdx.x >> 4, c = threadIdx.x & 15;                  // row of the tile, 8 columns of the step
    const int64_t r = rt * 16 + l;
    MxRaw8<T> raw[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        if (r < rows) raw[u] = mx_load8<T, VEC, ONCE>(x + r * rs, here * 512 + u * 128 + c * 8, cols, cs);
        else
#pragma unroll
            for (int j = 0; j < 8; ++j) raw[u].v[j] = (T)0.0f;
    }
    unsigned int sd = 0;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        float v[8];
        unsigned int am = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            v[j] = mx_to_f32(raw[u].v[j]);
            const unsigned int b = __float_as_uint(v[j]) & 0x7fffffffu;
            am = b > am ? b : am;
        }
        const int sc = mx_scale_of(mx_quad_max(am));
        sd |= (unsigned int)sc << (8 * u);
        const int64_t s = quad * 4 + u;
        if (s < steps) *reinterpret_cast<unsigned int*>(codes + (rt * steps + s) * 1024 + (c >> 2) * 256 + l * 16 + (c & 3) * 4) = mx_pack8(v, sc);
    }
    if ((c & 3) == 0) *reinterpret_cast<unsigned int*>(scales + (rt * quads + quad) * 256 + (c >> 2) * 64 + l * 4) = sd;
}

// the same for a matrix whose ROWS are neighbours in memory (rs == 1: a transposed view).  A block of 8 waves takes 64 rows x 512 columns; lane =
// row, so that every load of a wave is contiguous; a thread holds whole blocks of 32 columns and writes its 16 bytes of the fragment.
// 5000 x 10000 float32 (226 MB): 54 us, 4.2 TB/s; mx_quantize_kernel, element by element, takes twice as long (x in the caches: 45 / 91 us).
template <typename T, bool ONCE>
__global__ __launch_bounds__(512) void mx_quantize_across_kernel(const T* __restrict__ x, int64_t rows, int64_t cols, int64_t cs,
                                                                 unsigned char* __restrict__ codes, unsigned char* __restrict__ scales) {
    const int64_t steps = mx_steps(cols), quads = mx_quads(cols);
    __shared__ __attribute__((aligned(16))) unsigned char ls[4][256];      // [row tile][lane][step]
    const int lane = threadIdx.x & 63, wave = mx_wave(), tile = lane >> 4, l = lane & 15;
    const unsigned int groups = (unsigned int)((rows + 63) / 64), q32 = blockIdx.x / groups, rt32 = blockIdx.x - q32 * groups;
    const int64_t quad = q32, rt = (int64_t)rt32 * 4 + tile, r = rt * 16 + l, rts = mx_row_tiles(rows);
    const T* p = x + (r < rows ? r : rows - 1);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int b = wave * 2 + h, s = b >> 2, g = b & 3;
        const int64_t c = quad * 512 + b * 32;
        T raw[32];
        if (c + 32 <= cols) {
#pragma unroll
            for (int j = 0; j < 32; ++j) raw[j] = ONCE ? __builtin_nontemporal_load(&p[(c + j) * cs]) : p[(c + j) * cs];
        } else {
#pragma unroll
            for (int j = 0; j < 32; ++j) raw[j] = c + j < cols ? p[(c + j) * cs] : (T)0.0f;
        }
        float v[32];
        unsigned int am = 0;
#pragma unroll
        for (int j = 0; j < 32; ++j) {
            v[j] = r < rows ? mx_to_f32(raw[j]) : 0.0f;
            const unsigned int u = __float_as_uint(v[j]) & 0x7fffffffu;
            am = u > am ? u : am;
        }
        const int sc = mx_scale_of(am);
        if (rt < rts && quad * 4 + s < steps)
            *reinterpret_cast<mx_u4*>(codes + (rt * steps + quad * 4 + s) * 1024 + (g * 16 + l) * 16) =
                mx_u4{mx_pack8(v, sc), mx_pack8(v + 8, sc), mx_pack8(v + 16, sc), mx_pack8(v + 24, sc)};
        ls[tile][(g * 16 + l) * 4 + s] = (unsigned char)sc;
    }
    __syncthreads();
    const int64_t wt = (int64_t)rt32 * 4 + (threadIdx.x >> 6);
    if (threadIdx.x < 256 && wt < rts)
        *reinterpret_cast<unsigned int*>(scales + (wt * quads + quad) * 256 + lane * 4) = *reinterpret_cast<const unsigned int*>(&ls[threadIdx.x >> 6][lane * 4]);
}

template <typename T> __device__ __forceinline__ T mx_from_f32(float v) { return (T)v; }

__device__ __forceinline__ void mx_values8(unsigned int q, float s, float* v) {
    mx_f2 p;
    p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, s, 0); v[0] = p[0]; v[1] = p[1];
    p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, s, 1); v[2] = p[0]; v[3] = p[1];
    p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, s, 2); v[4] = p[0]; v[5] = p[1];
    p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, s, 3); v[6] = p[0]; v[7] = p[1];
}

// codes, scales -> out[r * rs + c * cs].  Bound: writing out.  Threads as in mx_quantize_kernel; VEC: the columns of out are neighbours.
// 16384 x 8192 bf16: 51-52 us, 6.5 TB/s.  (Stores past the caches: 5000 x 10000 float32 transposed 38 -> 83 us.)
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void mx_dequantize_kernel(const unsigned char* __restrict__ codes, const unsigned char* __restrict__ scales,
                                                            int64_t rows, int64_t cols, T* __restrict__ out, int64_t rs, int64_t cs, int64_t steps, int64_t quads,
                                                            int64_t quad0, unsigned int nquads) {
    const unsigned int rt32 = blockIdx.x / nquads;
    const int64_t rt = rt32, here = blockIdx.x - rt32 * nquads, quad = quad0 + here;
    const int l = threadIdx.x >> 4, c = threadIdx.x & 15;
    const int64_t r = rt * 16 + l;
    if (r >= rows) return;
    const unsigned int sd = *reinterpret_cast<const unsigned int*>(scales + (rt * quads + quad) * 256 + (c >> 2) * 64 + l * 4);
    unsigned int q[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
        q[u] = quad * 4 + u < steps ? *reinterpret_cast<const unsigned int*>(codes + (rt * steps + quad * 4 + u) * 1024 + (c >> 2) * 256 + l * 16 + (c & 3) * 4) : 0u;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const int64_t c0 = here * 512 + u * 128 + c * 8;
        float v[8];
        mx_values8(q[u], __uint_as_float(((sd >> (8 * u)) & 255u) << 23), v);
        T* p = out + r * rs + c0 * cs;
        if (VEC && c0 + 8 <= cols) {
            MxRaw8<T> o;
#pragma unroll
            for (int j = 0; j < 8; ++j) o.v[j] = mx_from_f32<T>(v[j]);
            mx_put<T, 8>(p, o.v);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (c0 + j < cols) p[j * cs] = mx_from_f32<T>(v[j]);
        }
    }
}

// the same into a matrix whose rows are neighbours in memory (rs == 1): the mirror image of mx_quantize_across_kernel.  5000 x 10000 float32:
// 38 us, 6.0 TB/s (element by element 103)
template <typename T>
__global__ __launch_bounds__(512) void mx_dequantize_across_kernel(const unsigned char* __restrict__ codes, const unsigned char* __restrict__ scales,
                                                                   int64_t rows, int64_t cols, T* __restrict__ out, int64_t cs) {
    const int64_t steps = mx_steps(cols), quads = mx_quads(cols);
    const int lane = threadIdx.x & 63, wave = mx_wave(), l = lane & 15;
    const unsigned int rt32 = blockIdx.x / (unsigned int)quads;
    const int64_t quad = blockIdx.x - rt32 * (unsigned int)quads, rt = (int64_t)rt32 * 4 + (lane >> 4), r = rt * 16 + l;
    if (r >= rows) return;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int b = wave * 2 + h, s = b >> 2, g = b & 3;
        const int64_t c = quad * 512 + b * 32;
        if (c >= cols) break;
        const mx_u4 q = *reinterpret_cast<const mx_u4*>(codes + (rt * steps + quad * 4 + s) * 1024 + (g * 16 + l) * 16);
        const float sc = __uint_as_float((unsigned int)scales[(rt * quads + quad) * 256 + (g * 16 + l) * 4 + s] << 23);
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            float v[8];
            mx_values8(q[d], sc, v);
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (c + 8 * d + j < cols) out[r + (c + 8 * d + j) * cs] = mx_from_f32<T>(v[j]);
        }
    }
}

// ---- products of x (float32, bf16, fp16) with a 4-bit matrix -----------------------------------------------------------------------
// The scale operand of the conversions: only the exponent field of the dword counts (sign and mantissa are ignored: checked for every byte
// and exponent), so the byte i of a dword of scales takes one rotation.
__device__ __forceinline__ float mx_scale_operand(unsigned int dword, int i) { return __uint_as_float(__builtin_amdgcn_alignbit(dword, dword, (9 + 8 * i) & 31)); }

// eight codes of one block -> bf16 (exact: at most 2 significant bits)
__device__ __forceinline__ mx_bf8 mx_unpack8(unsigned int q, float s) {
    const mx_bf2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, s, 0), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, s, 1),
                 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, s, 2), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, s, 3);
    return mx_bf8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// eight values as bf16 terms
template <typename T, int TERMS> __device__ __forceinline__ void mx_terms(const MxRaw8<T>& r, mx_bf8* f) {
    if constexpr (TERMS == 1) {
#pragma unroll
        for (int j = 0; j < 8; ++j) f[0][j] = (__bf16)r.v[j];
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float p[3];
            mx_split<TERMS>((float)r.v[j], p);
#pragma unroll
            for (int u = 0; u < TERMS; ++u) f[u][j] = (__bf16)p[u];
        }
    }
}

// where an output goes: split == 1 the result, else float32 partial sums [split][M][O] (t_first: [split][O][M], for an output whose rows are
// neighbours in memory); mx_join_kernel adds them up in order.  oscale (may be null): a factor of every output column.  skip (may be null):
// the whole product is left out if the word is not 0.
template <typename T> struct MxOut {
    T* out;
    int64_t rs, cs;
    float* part;
    int64_t M, O;
    bool t_first;
    const float* oscale;
    const int* skip;
};
// N consecutive columns o .. of row t
template <typename T, int N>
__device__ __forceinline__ void mx_store(const MxOut<T>& w, int64_t z, int64_t t, int64_t o, const float* v) {
    if (t >= w.M) return;
    if (w.part) {
        float* p = w.part + z * w.M * w.O + (w.t_first ? o * w.M + t : t * w.O + o);
        if (!w.t_first && o + N <= w.O) {
            mx_put<float, N>(p, v);
        } else {
            const int64_t ps = w.t_first ? w.M : 1;
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (o + j < w.O) p[j * ps] = v[j];
        }
        return;
    }
    T* p = w.out + t * w.rs + o * w.cs;
    if (w.cs == 1 && o + N <= w.O && !w.oscale) {
        T r[N];
#pragma unroll
        for (int j = 0; j < N; ++j) r[j] = mx_from_f32<T>(v[j]);
        mx_put<T, N>(p, r);
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (o + j < w.O) p[j * w.cs] = mx_from_f32<T>(w.oscale ? v[j] * w.oscale[o + j] : v[j]);
    }
}
// a wave's tiles: acc[i][c] holds rows 16 c + l of t0 and columns 16 i + 4 g .. of o0.  Whole tiles of an ordinary output take the short way:
// one address a lane, the rest constant offsets
template <typename T, int RT, int CT>
__device__ __forceinline__ void mx_store_tile(const MxOut<T>& w, int64_t z, int64_t t0, int64_t o0, int l, int g, const mx_f4 (&acc)[RT][CT]) {
    const bool whole = t0 + 16 * CT <= w.M && o0 + 16 * RT <= w.O && !w.t_first && !w.oscale;
    if (whole && w.part) {
        float* p = w.part + (z * w.M + t0 + l) * w.O + o0 + 4 * g;
#pragma unroll
        for (int c = 0; c < CT; ++c, p += 16 * w.O)
#pragma unroll
            for (int i = 0; i < RT; ++i) *reinterpret_cast<mx_f4u*>(p + 16 * i) = acc[i][c];
    } else if (whole && w.cs == 1) {
        T* p = w.out + (t0 + l) * w.rs + o0 + 4 * g;
#pragma unroll
        for (int c = 0; c < CT; ++c, p += 16 * w.rs)
#pragma unroll
            for (int i = 0; i < RT; ++i) {
                const T r[4] = {mx_from_f32<T>(acc[i][c][0]), mx_from_f32<T>(acc[i][c][1]), mx_from_f32<T>(acc[i][c][2]), mx_from_f32<T>(acc[i][c][3])};
                mx_put<T, 4>(p + 16 * i, r);
            }
    } else {
#pragma unroll
        for (int c = 0; c < CT; ++c)
#pragma unroll
            for (int i = 0; i < RT; ++i) {
                const float o[4] = {acc[i][c][0], acc[i][c][1], acc[i][c][2], acc[i][c][3]};
                mx_store<T, 4>(w, z, t0 + 16 * c + l, o0 + 16 * i + 4 * g, o);
            }
    }
}

// out[t][o] = sum over the splits, in order; four columns a thread, rscale (may be null) a factor of every row.  grid (columns, rows).  Bound:
// reading the parts; two of 2048 x 4096 (84 MB read and written): 13 us, 6.4 TB/s
template <typename T>
__global__ __launch_bounds__(256) void mx_join_kernel(const float* __restrict__ part, int split, int64_t M, int64_t O, T* __restrict__ out, int64_t rs,
                                                      int64_t cs, const float* __restrict__ rscale, const int* __restrict__ skip) {
    const int64_t o = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) * 4, n = M * O;
    if (o >= O || (skip && *skip)) return;
    for (int64_t t = (int64_t)blockIdx.y * blockDim.y + threadIdx.y; t < M; t += (int64_t)gridDim.y * blockDim.y) {
        const float* p = part + t * O + o;
        const float f = rscale ? rscale[t] : 1.0f;
        if (o + 4 <= O) {
            mx_f4 v = *reinterpret_cast<const mx_f4u*>(p);
#pragma unroll 4
            for (int z = 1; z < split; ++z) v += *reinterpret_cast<const mx_f4u*>(p + z * n);
            T* q = out + t * rs + o * cs;
            T r[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) r[j] = mx_from_f32<T>(v[j] * f);
            if (cs == 1) {
                mx_put<T, 4>(q, r);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) q[j * cs] = r[j];
            }
        } else {
            for (int j = 0; o + j < O; ++j) {
                float v = p[j];
                for (int z = 1; z < split; ++z) v += p[z * n + j];
                out[t * rs + (o + j) * cs] = mx_from_f32<T>(v * f);
            }
        }
    }
}

// The factor per column that gives a rounded block back the mean square it had: !FACTOR sums the squares of the N rows before the rounding, FACTOR
// after it and takes the root of the ratio (1 where either sum is 0 or not a number).  64 columns a block; sums in 64 bits.  Once per filled
// block of a shard, as the next kernel: reading the block bounds all three
template <bool FACTOR>
__global__ __launch_bounds__(1024) void mx_square_columns_kernel(const float* __restrict__ x, int64_t N, int64_t cols, int64_t ld, double* __restrict__ sum,
                                                                 float* __restrict__ out) {
    __shared__ double red[16][64];
    const int c = threadIdx.x & 63, g = threadIdx.x >> 6;
    const int64_t col = (int64_t)blockIdx.x * 64 + c;
    double s = 0.0;
    if (col < cols)
        for (int64_t r = g; r < N; r += 16) { const double v = x[r * ld + col]; s += v * v; }
    red[g][c] = s;
    __syncthreads();
    if (g == 0 && col < cols) {
        for (int k = 1; k < 16; ++k) s += red[k][c];
        if (!FACTOR) sum[col] = s;
        else out[col] = s > 0.0 && sum[col] > 0.0 ? (float)sqrt(sum[col] / s) : 1.0f;
    }
}
__global__ __launch_bounds__(256) void mx_scale_columns_kernel(float* __restrict__ x, int64_t rows, int64_t cols, int64_t ld, const float* __restrict__ f) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows * cols; i += (int64_t)gridDim.x * 256) x[(i / cols) * ld + i % cols] *= f[i % cols];
}

// ---- few rows of x (up to 16: tokens being decoded) -----------------------------------------------------------------------------
// out[t][n] = sum_k x[t][k] W[n][k], W in 4 bits with its blocks along k: the codes become bf16 in registers, x is split into bf16 terms
// (MxTerms), every product is exact, float32 sums.  Bound: reading W (4.25 bits a value).  The waves of a block share 16 RT rows of W and
// split the contraction (128 columns a step), so that a single token still puts every load of W in flight at once; partial sums meet in LDS.
// Eight waves: sixteen gain where 512 rows meet 20000 columns (11.6 -> 10.9 us) and lose elsewhere (4-bit 8 x 7000 x 4096 4.8 -> 5.6).
// W out of HBM: 1 x 4096 x 4096 bf16 takes 5.5 us (of which a launch is 3.5), 1 x 28672 x 8192 31 us, 4.0 TB/s (in the caches 5 and 25 us).  Four rows of x
// cost a tenth more; sixteen read x in scattered 16-byte pieces and take 15 us at 14336 x 4096 (2.1 TB/s) where one takes 11.  (x through LDS in
// whole lines: 9 % slower.)
constexpr int MX_ROW_WAVES = 8;
template <typename T, int RT, bool VEC>
__global__ __launch_bounds__(64 * MX_ROW_WAVES) void mx_linear_row_kernel(const T* __restrict__ x, int64_t M, int64_t xrs, int64_t xcs,
                                                                   const unsigned char* __restrict__ wc, const unsigned char* __restrict__ ws, int64_t N,
                                                                   int64_t K, MxOut<T> w) {
    constexpr int TERMS = MxTerms<T>::v, U = 4, WAVES = MX_ROW_WAVES;
    const int64_t ksteps = mx_steps(K), quads = mx_quads(K), rts = mx_row_tiles(N);
    const int64_t n0 = (int64_t)blockIdx.x * 16 * RT;
    const int lane = threadIdx.x & 63, wave = mx_wave(), l = lane & 15, g = lane >> 4;
    const int64_t t = l < M ? l : M - 1;                       // rows behind the last one repeat it and are not stored
    const unsigned char *pc[RT], *ps[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        const int64_t rt = (int64_t)blockIdx.x * RT + i < rts ? (int64_t)blockIdx.x * RT + i : rts - 1;
        pc[i] = wc + rt * ksteps * 1024 + lane * 16;
        ps[i] = ws + rt * quads * 256 + lane * 4;
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
                    q[u][i] = *reinterpret_cast<const mx_u4*>(pc[i] + s * 1024);
                    sc[u][i] = ps[i][(s >> 2) * 256 + (s & 3)];
                }
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t s = s0 + u * WAVES;
            if (s < steps) {
                MxRaw8<T> raw[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) raw[j] = mx_load8<T, VEC>(x + t * xrs, s * 128 + g * 32 + j * 8, K, xcs);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    mx_bf8 f[TERMS];
                    mx_terms<T, TERMS>(raw[j], f);
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
__device__ __forceinline__ void mx_unpack_across(const unsigned int* q, const float* sc, mx_bf8* w) {
    unsigned int u[8][4];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const mx_bf8 v = mx_unpack8(q[j], sc[j]);
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

// ---- many rows of x -------------------------------------------------------------------------------------------------------------
// The rows of x meet the matrix instructions as bf16 fragments: 16 rows, 32 of the contraction, 64 lanes x 16 bytes.  Fragment i of the
// contraction holds, for lane group g, eight values from
//   along the blocks   128 (i / 4) + 32 g + 8 (i % 4)      (a lane of W owns one block of each 128 columns, 8 values an instruction)
//   across the blocks  32 i + 8 g
// mx_fragments_kernel lays x out that way once per call, split into its bf16 terms: frag[i][term][tile of 16 rows][lane][8].  A tile of the
// products below is then a contiguous piece of memory, whatever x's type, strides or odd sizes.  kscale (may be null): a factor of every
// column of W, taken into x here.  Bound: the fragments' stores; 64 x 20000 float32 5.5 us, 2048 x 8192 bf16 (67 MB) 12 us, 5.5 TB/s.
template <bool ALONG> __device__ __forceinline__ int64_t mx_frag_k(int64_t i, int g) {
    return ALONG ? (i >> 2) * 128 + g * 32 + (i & 3) * 8 : i * 32 + g * 8;
}
template <typename T, bool ALONG, bool VEC>
__global__ __launch_bounds__(256) void mx_fragments_kernel(const T* __restrict__ x, int64_t M, int64_t xrs, int64_t xcs, int64_t K, int64_t nfrag,
                                                           int64_t tiles, unsigned short* __restrict__ frag, int rows_first,
                                                           const float* __restrict__ kscale, const int* __restrict__ skip) {
    constexpr int TERMS = MxTerms<T>::v;
    if (skip && *skip) return;
    // a block takes one tile of 16 rows and 16 groups of 8 values; neighbouring threads read neighbouring memory
    const unsigned int grp = blockIdx.x / (unsigned int)tiles;
    const int64_t tile = blockIdx.x - grp * (unsigned int)tiles, c0 = (int64_t)grp * 16;
    const int l = rows_first ? threadIdx.x & 15 : threadIdx.x >> 4;
    const int64_t c = c0 + (rows_first ? threadIdx.x >> 4 : threadIdx.x & 15);         // group of 8 along the contraction
    if (c >= nfrag * 4) return;
    const int64_t i = ALONG ? (c >> 4) * 4 + (c & 3) : c >> 2;
    const int g = (int)(ALONG ? (c >> 2) & 3 : c & 3);
    const int64_t t = tile * 16 + l;
    mx_bf8 f[TERMS] = {};
    if (t < M) {
        MxRaw8<T> r = mx_load8<T, VEC>(x + t * xrs, c * 8, K, xcs);
        if (kscale) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (c * 8 + j < K) r.v[j] = (T)((float)r.v[j] * kscale[c * 8 + j]);
        }
        mx_terms<T, TERMS>(r, f);
    }
#pragma unroll
    for (int u = 0; u < TERMS; ++u) *reinterpret_cast<mx_bf8*>(frag + (((i * TERMS + u) * tiles + tile) * 64 + g * 16 + l) * 8) = f[u];
}

// No instruction is moved across this by the compiler.  The tile kernels below run in slices: the fragments of the next slice are read from LDS
// behind the first matrix instructions of this one, so that a wave never waits for a read it has just issued.  (Left alone, the compiler
// reads each fragment right before its use, and two waves of a SIMD fall into step: neither pipe is fed while they wait.)
__device__ __forceinline__ void mx_fence() { __builtin_amdgcn_sched_barrier(0); }
// Waves in the middle of a stage go before waves at its ends, so that two blocks of a CU take turns at the matrix pipe: 4096 x 8192 x 4096 bf16 193 ->
// 189 us, forward and backward of 2048 x 8192 x 4096 249 -> 241, 64 x 20000 x 20000 float32 134 -> 132.  (No gain in mx_matmul_tile_kernel.)
__device__ __forceinline__ void mx_ahead(bool on) {
    if (on) __builtin_amdgcn_s_setprio(1);
    else __builtin_amdgcn_s_setprio(0);
}

typedef __attribute__((address_space(1))) const void* mx_gptr;
typedef __attribute__((address_space(3))) void* mx_lptr;

// bf16 whose rows are whole lines (neighbouring columns, 16-byte aligned, whole stages of the contraction) goes to LDS without being laid out first:
// that saves a launch and its pass over x (4096 x 8192 x 4096 207 -> 195 us; forward and backward of 2048 x 8192 x 4096 282 -> 252; 24 x 4096 x
// 4096 14.3 -> 11.1).  A stage is P
// pieces of 16 bytes of each row; a load takes 64 / P rows, the lane's piece exchanged with a power-of-two pattern of its row such that the 16
// lanes that read a fragment's column of pieces together touch every bank once: piece p of row r lies at p ^ r (P = 16: a row is all banks)
// or p ^ (r / 2) (P = 8: two rows are).  Rows behind the last repeat it and are not stored.
template <int P> struct MxDirect {
    unsigned int at, end, next;                                // the lane's place in its first load, in the last row; bytes from load to load
    __device__ __forceinline__ MxDirect(int lane, int wave, int64_t stride, int64_t rows) {
        const int r = (wave * 64 + lane) / P, piece = (lane % P) ^ (P == 16 ? r % 16 : (r / 2) % 8);
        at = (unsigned int)(r * stride * 2) + piece * 16;
        const int64_t last = rows - 1 < 127 ? rows - 1 : 127;
        end = (unsigned int)(last * stride * 2) + piece * 16;
        next = (unsigned int)(256 / P * stride * 2);
    }
    __device__ __forceinline__ unsigned int from(int c) const { return at + c * next < end ? at + c * next : end; }
};

// block -> (row tile, column tile, split): consecutive blocks go to the 8 XCDs in turn, so each XCD gets a contiguous piece of an order in which
// eight row tiles share a column tile of W
struct MxTile { int a, b, z; };
__device__ __forceinline__ MxTile mx_tile(unsigned int id, unsigned int na, unsigned int nb, unsigned int split) {
    const unsigned int area = na * nb, total = area * split, per = (total + 7) / 8;       // (all below 2^31)
    unsigned int p = (id & 7) * per + (id >> 3);
    MxTile r = {-1, 0, 0};
    if (p >= total || (id >> 3) >= per) return r;
    const unsigned int z = p / area;
    p -= z * area;
    const unsigned int grp = p / (8 * nb), left = na - grp * 8 < 8 ? na - grp * 8 : 8;
    p -= grp * 8 * nb;
    r.z = (int)z;
    r.b = (int)(p / left);
    r.a = (int)(grp * 8 + (p - (unsigned int)r.b * left));
    return r;
}

// out[t][n] = sum_k x[t][k] W[n][k] for tiles of 16 CT rows of x and 64 RT rows of W.  Bound: the bf16 matrix pipe (TERMS instructions per
// product).  The four waves own 16 RT rows of W each - codes go from memory to registers and become bf16 there, no LDS - and share the fragments
// of x through LDS (JS of them a stage, double buffered: as many as leave room for two blocks a CU).  4096 x 8192 x 4096 bf16: 192-195 us, 1.42
// PFLOP/s, where the instructions alone reach 2.17 on operands that stay in registers; 64 x 20000 x 20000 float32: 115-118 us, 1.32 (three terms).  Of
// 218 us of an earlier form the kernel took 195 without its loads of x, 202 without those of W, 156 without reading LDS.  Tried: tiles of 8 x 8 a
// wave (the accumulators spill), three waves a SIMD (140 against 126 us, float32), all loads of a stage at once (the same here, 10 % slower in the 4-bit tiles).
// DIRECT: frag is x itself (rows `tiles` elements apart), see MxDirect.
template <typename T, int CT, int RT, int JS, bool DIRECT>
__global__ __launch_bounds__(256, 2) void mx_linear_tile_kernel(const unsigned short* __restrict__ frag, int64_t tiles, const unsigned char* __restrict__ wc,
                                                             const unsigned char* __restrict__ ws, int64_t N, int64_t K, MxOut<T> w, int mt, int nt, int split) {
    static_assert(!DIRECT || (MxTerms<T>::v == 1 && JS == 4), "");
    constexpr int TERMS = MxTerms<T>::v, CH = JS * TERMS * CT;             // 1 KB pieces a stage
    const int64_t ksteps = mx_steps(K), quads = mx_quads(K), rts = mx_row_tiles(N);
    if (w.skip && *w.skip) return;
    const MxTile tile = mx_tile(blockIdx.x, mt, nt, split);
    if (tile.a < 0) return;
    const int lane = threadIdx.x & 63, wave = mx_wave(), l = lane & 15, g = lane >> 4;
    const int64_t n0 = (int64_t)tile.b * 64 * RT + wave * 16 * RT;
    const int64_t steps = (K + 127) / 128, per = (steps + split - 1) / split;
    const int64_t s0 = per * tile.z, s1 = s0 + per < steps ? s0 + per : steps;
    __shared__ __attribute__((aligned(16))) unsigned short lds[2][CH * 512];
    const unsigned char *pc[RT], *ps[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        const int64_t rt = n0 / 16 + i < rts ? n0 / 16 + i : rts - 1;      // (tiles behind the last one repeat it and are not stored)
        pc[i] = wc + rt * ksteps * 1024;
        ps[i] = ws + rt * quads * 256;
    }
    // running address of the next stage: scalar, advanced by a constant
    const unsigned char* fp = (const unsigned char*)frag + (DIRECT ? (int64_t)tile.a * CT * 16 * tiles * 2 + s0 * 256 : (s0 * 4 * TERMS * tiles + (int64_t)tile.a * CT) * 1024);
    const int64_t fstage = DIRECT ? 256 : JS * TERMS * tiles * 1024, fterm = tiles * 1024;
    const MxDirect<16> dx(lane, wave, tiles, w.M - (int64_t)tile.a * CT * 16);
    // piece c of the wave's share of the next JS fragments of the contraction
    constexpr int PIECES = (CH + 3) / 4;
    auto stage = [&](int b, int c) {
        const int i = c * 4 + wave;
        if (CH % 4 == 0 || i < CH)
            __builtin_amdgcn_global_load_lds((mx_gptr)(DIRECT ? fp + dx.from(c) : fp + (i / CT) * fterm + (i % CT) * 1024 + lane * 16), (mx_lptr)(&lds[b][i * 512]),
                                             16, 0, 0);
    };
    // fragment i of a stage (step i / CT, tile i % CT)
    const int dlane = l * 256 + ((4 * g) ^ l) * 16;
    auto fragment = [&](int b, int i) {
        return *reinterpret_cast<const mx_bf8*>((const unsigned char*)lds[b] + (DIRECT ? (i % CT) * 4096 + (dlane ^ (i / CT * 16)) : i * 1024 + lane * 16));
    };
    mx_f4 acc[RT][CT] = {};
    mx_u4 q[RT];
    unsigned int sd[RT];
    if (s0 < s1) {
#pragma unroll
        for (int c = 0; c < PIECES; ++c) stage(0, c);
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            q[i] = *reinterpret_cast<const mx_u4*>(pc[i] + s0 * 1024 + lane * 16);
            sd[i] = *reinterpret_cast<const unsigned int*>(ps[i] + (s0 >> 2) * 256 + lane * 4);
        }
    }
    __syncthreads();
    int b = 0;
    for (int64_t s = s0; s < s1; ++s) {
        mx_u4 qn[RT];
        unsigned int sn[RT];
        const int64_t sx = s + 1 < s1 ? s + 1 : s;
        float sc[RT];
#pragma unroll
        for (int i = 0; i < RT; ++i) sc[i] = mx_scale_operand(sd[i], (int)(s & 3));
#pragma unroll
        for (int h = 0; h < 4 / JS; ++h) {
            if (h + 1 < 4 / JS || s + 1 < s1) fp += fstage;    // (behind the last stage: that one again, unused)
            // slices of F fragments
            constexpr int F = CT < 4 ? CT : 4, SL = CH / F;
            mx_bf8 f[2][F], a[2][RT];
#pragma unroll
            for (int c = 0; c < F; ++c) f[0][c] = fragment(b, c);
#pragma unroll
            for (int i = 0; i < RT; ++i) a[0][i] = mx_unpack8(q[i][h * JS], sc[i]);
            mx_ahead(true);
#pragma unroll
            for (int sl = 0; sl < SL; ++sl) {
                const int jj = sl * F / (TERMS * CT), c0 = sl * F % CT;
#pragma unroll
                for (int c = 0; c < F; ++c) {
                    if (c == 1 || F == 1) {
                        mx_fence();
                        // the loads of the next stage, a few a slice: all at once they would fill the address queue and hold the wave up
#pragma unroll
                        for (int p = sl * PIECES / SL; p < (sl + 1) * PIECES / SL; ++p) stage(b ^ 1, p);
                        if (h == 0) {
#pragma unroll
                            for (int i = sl * RT / SL; i < (sl + 1) * RT / SL; ++i) {
                                qn[i] = *reinterpret_cast<const mx_u4*>(pc[i] + sx * 1024 + lane * 16);
                                sn[i] = *reinterpret_cast<const unsigned int*>(ps[i] + (sx >> 2) * 256 + lane * 4);
                            }
                        }
                        if (sl + 1 < SL) {
#pragma unroll
                            for (int n = 0; n < F; ++n) f[(sl + 1) & 1][n] = fragment(b, (sl + 1) * F + n);
                            if ((sl + 1) * F % (TERMS * CT) == 0) {
#pragma unroll
                                for (int i = 0; i < RT; ++i) a[(jj + 1) & 1][i] = mx_unpack8(q[i][h * JS + jj + 1], sc[i]);
                            }
                        }
                    }
#pragma unroll
                    for (int i = 0; i < RT; ++i) acc[i][c0 + c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[jj & 1][i], f[sl & 1][c], acc[i][c0 + c], 0, 0, 0);
                }
                mx_fence();
            }
            mx_ahead(false);
            __syncthreads();
            b ^= 1;
        }
#pragma unroll
        for (int i = 0; i < RT; ++i) { q[i] = qn[i]; sd[i] = sn[i]; }
    }
    mx_store_tile<T, RT, CT>(w, tile.z, (int64_t)tile.a * CT * 16, n0, l, g, acc);
}

// dx[t][k] = sum_n dy[t][n] W[n][k] for tiles of 16 CT rows of dy and 512 columns of W: the contraction runs ACROSS the blocks.  A lane reads the
// dword of 8 columns from each of 8 rows; unpacked, entry m of the eight dwords is what matrix instruction m needs from this lane: column 8
// (lane % 16) + m, eight n.  So a wave owns 128 columns as 8 tiles and no value crosses lanes.  Bound: the bf16 matrix pipe; unpacking
// costs three vector instructions per matrix instruction at CT 4, one step ahead and in between them.  32 JS rows of W (codes, scales) and
// their fragments of dy a stage, all of them to LDS without passing registers: the fragments double buffered, W in three buffers, since it is
// unpacked a step early (AHEAD; with two or three terms the fragments need its registers: 219 against 183 us).  2048 x 8192 x 4096 bf16 in two
// parts: 136-142 us, 0.99 PFLOP/s (154 behind the forward product; 8192 rows: 1.1 PFLOP/s); 64 x 20000 x 20000 float32: 157-163 us, 0.96.  Of 155 us of an earlier form the bf16 kernel took 98 without
// reading W from LDS, 118 without unpacking, 130 without loads.  Row r of block b in row tile p is stored at row r ^ (b | 4 (p % 2)) of its block: the sixteen (block, lane group)
// that a wave reads at once lie in different banks.
template <int CT, int JS, int TERMS> struct MxGradLds {
    static constexpr int frag = JS * TERMS * CT * 1024, codes = JS * 8 * 1024, scales = JS * 2 * 256, wstage = codes + scales, total = 2 * frag + 3 * wstage;
};
// DIRECT: frag is dy itself (rows `tiles` elements apart), see MxDirect.
template <typename T, int CT, int JS, bool DIRECT>
__global__ __launch_bounds__(256, 2) void mx_grad_tile_kernel(const unsigned short* __restrict__ frag, int64_t tiles, const unsigned char* __restrict__ wc,
                                                             const unsigned char* __restrict__ ws, int64_t N, int64_t K, MxOut<T> w, int mt, int nt, int split) {
    static_assert(!DIRECT || (MxTerms<T>::v == 1 && JS == 2), "");
    constexpr int TERMS = MxTerms<T>::v, CH = JS * TERMS * CT;
    constexpr bool AHEAD = TERMS == 1 && JS % 2 == 0;
    typedef MxGradLds<CT, JS, TERMS> L;
    const int64_t ksteps = mx_steps(K), quads = mx_quads(K), rts = mx_row_tiles(N);
    if (w.skip && *w.skip) return;
    const MxTile tile = mx_tile(blockIdx.x, mt, nt, split);
    if (tile.a < 0) return;
    const int lane = threadIdx.x & 63, wave = mx_wave(), l = lane & 15, g = lane >> 4;
    const int64_t k0 = (int64_t)tile.b * 512 + wave * 128;
    const int64_t steps = (N + 31) / 32, per = ((steps + split - 1) / split + JS - 1) / JS * JS;
    const int64_t s0 = per * tile.z, s1 = s0 + per < steps ? s0 + per : steps;
    extern __shared__ __attribute__((aligned(16))) unsigned char glds[];
    // running addresses of the next stage: scalar, advanced by a constant
    const unsigned char* fp = (const unsigned char*)frag + (DIRECT ? (int64_t)tile.a * CT * 16 * tiles * 2 + s0 * 64 : (s0 * TERMS * tiles + (int64_t)tile.a * CT) * 1024);
    const MxDirect<8> dx(lane, wave, tiles, w.M - (int64_t)tile.a * CT * 16);
    const int64_t fterm = tiles * 1024, fstage = DIRECT ? 128 : JS * TERMS * fterm, wtile = ksteps * 1024, stile = quads * 256;
    const unsigned char* wp = wc + (s0 * 2 * ksteps + ((int64_t)tile.b * 4 + wave < ksteps ? (int64_t)tile.b * 4 + wave : ksteps - 1)) * 1024;
    const unsigned char* sp = ws + ((s0 * 2 + (wave < JS * 2 ? wave : 0)) * quads + tile.b) * 256;
    // row tiles from the next stage on.  Those behind the last one: its codes again, whose factors in dy are zero; their scales must not be a
    // NaN, so they are taken from those very zeros, the half fragments of dy
    int64_t left = rts - s0 * 2;
    const unsigned char* zp = (const unsigned char*)frag + ((s0 + (wave >> 1)) * TERMS * tiles + (int64_t)tile.a * CT) * 1024 + (wave & 1) * 512;
    const int wlane[2] = {g * 256 + (l ^ g) * 16, g * 256 + (l ^ (g | 4)) * 16};
    constexpr int FP = (CH + 3) / 4, WP = JS * 2, PIECES = FP + WP + 1;    // loads of a wave: fragments, codes, scales
    auto load_frag = [&](int at, int c) {
        const int i = c * 4 + wave;
        if (CH % 4 == 0 || i < CH)
            __builtin_amdgcn_global_load_lds((mx_gptr)(DIRECT ? fp + dx.from(c) : fp + (i / CT) * fterm + (i % CT) * 1024 + lane * 16), (mx_lptr)(glds + at + i * 1024),
                                             16, 0, 0);
    };
    // fragment i of step jj of the stage at LDS offset at
    const int dlane = l * 128 + (g ^ (l >> 1)) * 16;
    auto fragment = [&](int at, int jj, int i) {
        return *reinterpret_cast<const mx_bf8*>(glds + at + (DIRECT ? i * 2048 + (dlane ^ (jj * 64)) : (jj * TERMS * CT + i) * 1024 + lane * 16));
    };
    auto load_w = [&](int at, int p) {                         // the wave's step of row tile p; p == WP: the scales
        if (p < WP)
            __builtin_amdgcn_global_load_lds((mx_gptr)(wp + (p < left ? p : left - 1) * wtile + wlane[p & 1]), (mx_lptr)(glds + at + (p * 4 + wave) * 1024), 16,
                                             0, 0);
        else if (wave < WP && lane < 16)
            __builtin_amdgcn_global_load_lds((mx_gptr)((DIRECT || wave < left ? sp : zp) + lane * 16), (mx_lptr)(glds + at + L::codes + wave * 256), 16, 0, 0);
    };
    // (behind the last stage: that one again, unused - the addresses stay where they are)
    auto next_frag = [&](bool more) { fp += more ? fstage : 0; };
    auto next_w = [&](bool more) {
        wp += more ? WP * wtile : 0;
        sp += more ? WP * stile : 0;
        zp += more ? JS * TERMS * fterm : 0;
        left -= more ? WP : 0;
    };
    // row 8 g + j of a step is row 8 (g % 2) + j of row tile g / 2
    const int blk = l >> 2, mask = blk | 4 * (g >> 1);
    int qat[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) qat[j] = ((g >> 1) * 4 + wave) * 1024 + blk * 256 + (g & 1) * 128 + (l & 3) * 4 + ((j ^ mask) * 16);
    const int sat = L::codes + (g >> 1) * 256 + blk * 64 + (g & 1) * 32;
    mx_f4 acc[8][CT] = {};
    int f0 = 0, f1 = L::frag, w0 = 2 * L::frag, w1 = w0 + L::wstage, w2 = w1 + L::wstage;
    mx_bf8 a[2][8];
    auto unpack_step = [&](int at, int jj, mx_bf8* to) {                    // the jj-th step of the stage at LDS offset at
        unsigned int q[8];
        mx_u4 d[2];
        float sc[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) q[j] = *reinterpret_cast<const unsigned int*>(glds + at + jj * 8192 + qat[j]);
        d[0] = *reinterpret_cast<const mx_u4*>(glds + at + jj * 512 + sat);
        d[1] = *reinterpret_cast<const mx_u4*>(glds + at + jj * 512 + sat + 16);
#pragma unroll
        for (int j = 0; j < 8; ++j) sc[j] = mx_scale_operand(d[j >> 2][j & 3], wave);
        mx_unpack_across(q, sc, to);
    };
    if (s0 < s1) {
#pragma unroll
        for (int c = 0; c < FP; ++c) load_frag(f0, c);
        next_frag(s0 + JS < s1);
#pragma unroll
        for (int p = 0; p <= WP; ++p) load_w(w0, p);
        next_w(s0 + JS < s1);
#pragma unroll
        for (int p = 0; p <= WP; ++p) load_w(w1, p);
        next_w(s0 + 2 * JS < s1);
    }
    __syncthreads();
    if (AHEAD && s0 < s1) unpack_step(w0, 0, a[0]);
    for (int64_t s = s0; s < s1; s += JS) {
        mx_ahead(true);
#pragma unroll
        for (int jj = 0; jj < JS; ++jj) {                      // (a step behind the last one: the fragments of dy are zeros)
            const int cur = AHEAD ? jj & 1 : 0, nxt = cur ^ 1;
            if (!AHEAD) unpack_step(w0, jj, a[0]);
            // slices of F fragments; the first of the next step's unpacking rides behind the first of them
            constexpr int F = CT < 2 ? CT : 2, SL = TERMS * CT / F;
            mx_bf8 f[2][F];
#pragma unroll
            for (int c = 0; c < F; ++c) f[0][c] = fragment(f0, jj, c);
#pragma unroll
            for (int sl = 0; sl < SL; ++sl) {
                const int c0 = sl * F % CT;
#pragma unroll
                for (int c = 0; c < F; ++c) {
                    if (c == 1 || F == 1) {
                        mx_fence();
                        // the loads of the stages ahead, a few a slice
#pragma unroll
                        for (int p = (jj * SL + sl) * PIECES / (JS * SL); p < (jj * SL + sl + 1) * PIECES / (JS * SL); ++p) {
                            if (p < FP) load_frag(f1, p);
                            else load_w(w2, p - FP);
                        }
                        if (sl + 1 < SL) {
#pragma unroll
                            for (int n = 0; n < F; ++n) f[(sl + 1) & 1][n] = fragment(f0, jj, (sl + 1) * F + n);
                        }
                        if (AHEAD && sl == 0) {
                            if (jj + 1 < JS) unpack_step(w0, jj + 1, a[nxt]);
                            else unpack_step(w1, 0, a[nxt]);
                        }
                    }
#pragma unroll
                    for (int m = 0; m < 8; ++m) acc[m][c0 + c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[cur][m], f[sl & 1][c], acc[m][c0 + c], 0, 0, 0);
                }
                if (!AHEAD || sl > 0) mx_fence();              // (unpacking mixes with the matrix instructions of two slices)
            }
        }
        mx_ahead(false);
        next_frag(s + 2 * JS < s1);
        next_w(s + 3 * JS < s1);
        __syncthreads();
        { const int t = f0; f0 = f1; f1 = t; }
        { const int t = w0; w0 = w1; w1 = w2; w2 = t; }
    }
    // a lane ends up with 32 neighbours of a row: columns 32 g + 8 e + m
    const int64_t t0 = (int64_t)tile.a * CT * 16;
    if (t0 + 16 * CT <= w.M && k0 + 128 <= w.O && !w.t_first && !w.oscale && (w.part || w.cs == 1)) {
        const int64_t at = (t0 + l) * (w.part ? w.O : w.rs) + k0 + 32 * g;
#pragma unroll
        for (int c = 0; c < CT; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float o[8];
                T r[8];
#pragma unroll
                for (int m = 0; m < 8; ++m) { o[m] = acc[m][c][e]; r[m] = mx_from_f32<T>(o[m]); }
                if (w.part) mx_put<float, 8>(w.part + tile.z * w.M * w.O + at + 16 * c * w.O + 8 * e, o);
                else mx_put<T, 8>(w.out + at + 16 * c * w.rs + 8 * e, r);
            }
        return;
    }
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float o[8];
#pragma unroll
            for (int m = 0; m < 8; ++m) o[m] = acc[m][c][e];
            mx_store<T, 8>(w, tile.z, ((int64_t)tile.a * CT + c) * 16 + l, k0 + 8 * (4 * g + e), o);
        }
}

// ---- 4 bits x 4 bits -------------------------------------------------------------------------------------------------------------
// out[m][n] = sum_k A[m][k] B[n][k] on v_mfma_scale_f32_16x16x128_f8f6f4: a lane holds one block of 32 of its row (16 bytes) and that block's
// scale; the instruction multiplies codes and scales, float32 sums.  Rows behind the last one repeat it and are not stored.
__device__ __forceinline__ mx_i8 mx_operand(mx_u4 q) { return mx_i8{(int)q[0], (int)q[1], (int)q[2], (int)q[3], 0, 0, 0, 0}; }

// up to 16 rows of A: as mx_linear_row_kernel, bound by reading B.  8 x 8192 x 8192: 10 us out of HBM, 3.5 TB/s; 6.6
// with B in the caches (its tiles: 13)
template <typename T, int RT>
__global__ __launch_bounds__(64 * MX_ROW_WAVES) void mx_matmul_row_kernel(const unsigned char* __restrict__ ac, const unsigned char* __restrict__ as, int64_t M,
                                                                   const unsigned char* __restrict__ bc, const unsigned char* __restrict__ bs, int64_t N,
                                                                   int64_t K, MxOut<T> w) {
    constexpr int U = 4, WAVES = MX_ROW_WAVES;
    const int64_t ksteps = mx_steps(K), quads = mx_quads(K), rts = mx_row_tiles(N);
    const int64_t n0 = (int64_t)blockIdx.x * 16 * RT;
    const int lane = threadIdx.x & 63, wave = mx_wave(), l = lane & 15, g = lane >> 4;
    const unsigned char *pc[RT], *ps[RT], *pa = ac + lane * 16, *pas = as + lane * 4;      // (one row tile)
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        const int64_t rt = (int64_t)blockIdx.x * RT + i < rts ? (int64_t)blockIdx.x * RT + i : rts - 1;
        pc[i] = bc + rt * ksteps * 1024 + lane * 16;
        ps[i] = bs + rt * quads * 256 + lane * 4;
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
                qa[u] = *reinterpret_cast<const mx_u4*>(pa + s * 1024);
                sa[u] = pas[(s >> 2) * 256 + (s & 3)];
#pragma unroll
                for (int i = 0; i < RT; ++i) {
                    q[u][i] = *reinterpret_cast<const mx_u4*>(pc[i] + s * 1024);
                    sc[u][i] = ps[i][(s >> 2) * 256 + (s & 3)];
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

// Tiles of 16 CT rows of A by 64 RT rows of B.  Bound: the 4-bit matrix pipe (16 cycles an instruction of 64 Kflop) and what feeds it: as in
// mx_linear_tile_kernel the four waves own 16 RT rows of B each, whose fragments and scales go from memory to registers (an instruction's
// operands are 2 KB, and both through LDS would take all of its bandwidth), and share the fragments of A through LDS, two steps a stage,
// double buffered.  A dword of scales serves four steps.  8192 x 8192 x 8192: 267-290 us, 253 at best, 3.8-4.3 PFLOP/s (the instructions alone: 7.5); 1000 x 5003 x 10007: 47
// us, 2.1.  Tried: four stages in flight (spills, 388 us), A's codes row-major in 64-byte pieces (557 against 423 us).
template <typename T, int CT, int RT>
__global__ __launch_bounds__(256, 2) void mx_matmul_tile_kernel(const unsigned char* __restrict__ ac, const unsigned char* __restrict__ as,
                                                               const unsigned char* __restrict__ bc, const unsigned char* __restrict__ bs, int64_t N,
                                                               int64_t K, MxOut<T> w, int mt, int nt, int split) {
    constexpr int CH = CT * 2 / 4;                                         // fragments a wave and stage
    const int64_t ksteps = mx_steps(K), quads = mx_quads(K), mts = mx_row_tiles(w.M), nts = mx_row_tiles(N);
    const MxTile tile = mx_tile(blockIdx.x, mt, nt, split);
    if (tile.a < 0) return;
    const int lane = threadIdx.x & 63, wave = mx_wave(), l = lane & 15, g = lane >> 4;
    const int64_t steps = ksteps / 2, per = ((steps + split - 1) / split + 1) / 2 * 2;     // stages
    const int64_t s0 = per * tile.z, s1 = s0 + per < steps ? s0 + per : steps;
    __shared__ __attribute__((aligned(16))) unsigned char lds[2][CT * 2 * 1024];           // [step][row tile][lane]
    // (row tiles behind the last one repeat it and are not stored)
    const unsigned char *xb[CH], *xsb[CT], *qb[RT], *sb[RT];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int i = c * 4 + wave;
        const int64_t rt = (int64_t)tile.a * CT + i % CT < mts ? (int64_t)tile.a * CT + i % CT : mts - 1;
        xb[c] = ac + (rt * ksteps + i / CT) * 1024;
    }
#pragma unroll
    for (int c = 0; c < CT; ++c) xsb[c] = as + ((int64_t)tile.a * CT + c < mts ? (int64_t)tile.a * CT + c : mts - 1) * quads * 256;
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        int64_t rt = ((int64_t)tile.b * 4 + wave) * RT + i;
        rt = rt < nts ? rt : nts - 1;
        qb[i] = bc + rt * ksteps * 1024;
        sb[i] = bs + rt * quads * 256;
    }
    auto load_a = [&](int64_t s, int b, int c) {                            // piece c of the wave's share of stage s
        __builtin_amdgcn_global_load_lds((mx_gptr)(xb[c] + s * 2048 + lane * 16), (mx_lptr)(&lds[b][(c * 4 + wave) * 1024]), 16, 0, 0);
    };
    mx_f4 acc[RT][CT] = {};
    mx_u4 q[RT][2];
    int sd[RT], sx[CT];
    if (s0 < s1) {
#pragma unroll
        for (int c = 0; c < CH; ++c) load_a(s0, 0, c);
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            q[i][0] = *reinterpret_cast<const mx_u4*>(qb[i] + s0 * 2048 + lane * 16);
            q[i][1] = *reinterpret_cast<const mx_u4*>(qb[i] + s0 * 2048 + 1024 + lane * 16);
            sd[i] = *reinterpret_cast<const int*>(sb[i] + (s0 >> 1) * 256 + lane * 4);
        }
#pragma unroll
        for (int c = 0; c < CT; ++c) sx[c] = *reinterpret_cast<const int*>(xsb[c] + (s0 >> 1) * 256 + lane * 4);
    }
    __syncthreads();
    // two stages (four steps: one dword of scales) a turn
    for (int64_t s = s0; s < s1; s += 2) {
        int sdn[RT], sxn[CT];
        const int64_t sn = s + 2 < s1 ? s + 2 : s;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (h == 1 && s + 1 >= s1) break;
            const int64_t nx = s + h + 1 < s1 ? s + h + 1 : s + h;         // (the last stage loads something it does not use)
            mx_u4 qn[RT][2];
            constexpr int F = 2, SL = 2 * CT / F;
            mx_u4 f[2][F];
            const unsigned char* at = &lds[h][lane * 16];
#pragma unroll
            for (int c = 0; c < F; ++c) f[0][c] = *reinterpret_cast<const mx_u4*>(at + c * 1024);
#pragma unroll
            for (int sl = 0; sl < SL; ++sl) {
                const int j = sl * F / CT, c0 = sl * F % CT;
#pragma unroll
                for (int n = 0; n < F; ++n) {
                    const int c = c0 + n;
                    if (n == 1) {
                        mx_fence();
                        // the loads of the next stage, a few a slice: all at once they would fill the address queue and hold the wave up
#pragma unroll
                        for (int p = sl * CH / SL; p < (sl + 1) * CH / SL; ++p) load_a(nx, h ^ 1, p);
#pragma unroll
                        for (int p = sl * 2 * RT / SL; p < (sl + 1) * 2 * RT / SL; ++p)
                            qn[p / 2][p & 1] = *reinterpret_cast<const mx_u4*>(qb[p / 2] + nx * 2048 + (p & 1) * 1024 + lane * 16);
                        if (h == 1) {
#pragma unroll
                            for (int p = sl * (RT + CT) / SL; p < (sl + 1) * (RT + CT) / SL; ++p) {
                                if (p < RT) sdn[p] = *reinterpret_cast<const int*>(sb[p < RT ? p : 0] + (sn >> 1) * 256 + lane * 4);
                                else sxn[p - RT] = *reinterpret_cast<const int*>(xsb[p < RT ? 0 : p - RT] + (sn >> 1) * 256 + lane * 4);
                            }
                        }
                        if (sl + 1 < SL) {
#pragma unroll
                            for (int e = 0; e < F; ++e) f[(sl + 1) & 1][e] = *reinterpret_cast<const mx_u4*>(at + ((sl + 1) * F + e) * 1024);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < RT; ++i) {
                        // (the byte of the scales is part of the instruction)
                        const mx_i8 A = mx_operand(q[i][j]), B = mx_operand(f[sl & 1][n]);
                        if (h == 0 && j == 0) acc[i][c] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(A, B, acc[i][c], 4, 4, 0, sd[i], 0, sx[c]);
                        else if (h == 0) acc[i][c] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(A, B, acc[i][c], 4, 4, 1, sd[i], 1, sx[c]);
                        else if (j == 0) acc[i][c] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(A, B, acc[i][c], 4, 4, 2, sd[i], 2, sx[c]);
                        else acc[i][c] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(A, B, acc[i][c], 4, 4, 3, sd[i], 3, sx[c]);
                    }
                }
                mx_fence();
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < RT; ++i) { q[i][0] = qn[i][0]; q[i][1] = qn[i][1]; }
        }
#pragma unroll
        for (int i = 0; i < RT; ++i) sd[i] = sdn[i];
#pragma unroll
        for (int c = 0; c < CT; ++c) sx[c] = sxn[c];
    }
    mx_store_tile<T, RT, CT>(w, tile.z, (int64_t)tile.a * CT * 16, ((int64_t)tile.b * 4 + wave) * RT * 16, l, g, acc);
}

template <typename T>
__global__ __launch_bounds__(256) void mx_zero_kernel(T* __restrict__ out, int64_t rows, int64_t cols, int64_t rs, int64_t cs) {
    const int64_t n = rows * cols;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) out[(i / cols) * rs + (i % cols) * cs] = (T)0.0f;
}

}  // namespace lcx
