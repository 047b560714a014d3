// lcx_mx4.hip - matrices in 4 bits per value: quantisation and products on device memory (include/lcx.h, lcx_mx4_*)
#include "engine.hpp"
#include "mx4_kernels.hpp"
#include <algorithm>

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

constexpr int64_t MX_MAX_PIECES = (int64_t)1 << 24;             // blocks of 256 threads that a launch can count

constexpr int MX_CUS = 256;            // blocks are sized for a whole MI355X; the choices below only shift speed

static int64_t dim_bad(int64_t a, int64_t b, int64_t c = 0) { return a < 0 || b < 0 || c < 0 || a >= MX_MAX_DIM || b >= MX_MAX_DIM || c >= MX_MAX_DIM; }
static bool mx_misaligned(const void* codes, const void* scales) { return (((uintptr_t)codes | (uintptr_t)scales) & 15) != 0; }

// a launch counts its threads in 32 bits
static int mx_grid(int64_t mtiles, int64_t ntiles, int threads, unsigned* g) {
    if (mtiles * ntiles > 0xffffffffll / threads) return fail(LCX_ERR_ARG, "lcx_mx4: the matrix is too large for one call");
    *g = (unsigned)(mtiles * ntiles);
    return LCX_OK;
}

template <typename T>
static int mx4_quantize(const void* x, int64_t rows, int64_t cols, int64_t rs, int64_t cs, void* codes, void* scales, hipStream_t st) {
    unsigned char *qc = (unsigned char*)codes, *qs = (unsigned char*)scales;
    unsigned g;
    const int64_t steps = mx_steps(cols), quads = mx_quads(cols);
    const auto once = [&] { return rows * cols * (int64_t)sizeof(T) >= MX_ONCE_BYTES; };          // (of sizes that a launch can count)
    if (rs == 1 && cs != 1) {
        LCXCHECK(mx_grid(cdiv(rows, 64), quads, 512, &g));
        if (once()) hipLaunchKernelGGL((mx_quantize_across_kernel<T, true>), dim3(g), dim3(512), 0, st, (const T*)x, rows, cols, cs, qc, qs);
        else hipLaunchKernelGGL((mx_quantize_across_kernel<T, false>), dim3(g), dim3(512), 0, st, (const T*)x, rows, cols, cs, qc, qs);
    } else {
        LCXCHECK(mx_grid(mx_row_tiles(rows), quads, 256, &g));
#define MX_QUANTIZE(VEC, ONCE)                                                                                                                              \
    hipLaunchKernelGGL((mx_quantize_kernel<T, VEC, ONCE>), dim3(g), dim3(256), 0, st, (const T*)x, rows, cols, rs, cs, qc, qs, steps, quads, (int64_t)0, \
                       (unsigned)quads)
        if (cs != 1) MX_QUANTIZE(false, false);
        else if (once()) MX_QUANTIZE(true, true);
        else MX_QUANTIZE(true, false);
#undef MX_QUANTIZE
    }
    KCHECK();
    return LCX_OK;
}

template <typename T>
static int mx4_dequantize(const void* codes, const void* scales, int64_t rows, int64_t cols, void* out, int64_t rs, int64_t cs, hipStream_t st) {
    const unsigned char *qc = (const unsigned char*)codes, *qs = (const unsigned char*)scales;
    unsigned g;
    if (rs == 1 && cs != 1) {
        LCXCHECK(mx_grid(cdiv(rows, 64), mx_quads(cols), 512, &g));
        hipLaunchKernelGGL((mx_dequantize_across_kernel<T>), dim3(g), dim3(512), 0, st, qc, qs, rows, cols, (T*)out, cs);
    } else {
        LCXCHECK(mx_grid(mx_row_tiles(rows), mx_quads(cols), 256, &g));
        if (cs == 1) hipLaunchKernelGGL((mx_dequantize_kernel<T, true>), dim3(g), dim3(256), 0, st, qc, qs, rows, cols, (T*)out, rs, cs, mx_steps(cols),
                                        mx_quads(cols), (int64_t)0, (unsigned)mx_quads(cols));
        else hipLaunchKernelGGL((mx_dequantize_kernel<T, false>), dim3(g), dim3(256), 0, st, qc, qs, rows, cols, (T*)out, rs, cs, mx_steps(cols),
                                mx_quads(cols), (int64_t)0, (unsigned)mx_quads(cols));
    }
    KCHECK();
    return LCX_OK;
}

template <typename T> static int mx4_zero(void* out, int64_t rows, int64_t cols, int64_t rs, int64_t cs, hipStream_t st) {
    const int64_t b = cdiv(rows * cols, 256);
    hipLaunchKernelGGL((mx_zero_kernel<T>), dim3((unsigned)(b < 4096 ? b : 4096)), dim3(256), 0, st, (T*)out, rows, cols, rs, cs);
    KCHECK();
    return LCX_OK;
}


// ---- products of x with a 4-bit matrix -------------------------------------------------------------------------------------------------
// What one call does: sizes of its tiles, its splits of the contraction and its work space [fragments of x | partial sums].
struct MxPlan {
    bool row = false;                  // up to 16 rows of x: the row kernels
    int ct = 1, rt = 1;                // 16-row tiles of x, of W (linear)
    int64_t mt = 1, nt = 1;            // tiles over the rows of x / over the output columns
    int64_t nfrag = 0;                 // fragments of the contraction
    int split = 1;
    int64_t frag_bytes = 0, part_bytes = 0;
};

// Time of a tile kernel's step on a CU that holds one block (t1 + u1 x its work) or two (t2 + u2 x), in us: the work is the 16-row tiles of x per
// block, times the bf16 terms.  A step is 128 of the contraction (lcx_mx4_matmul: 512).  pair: what a second block a CU costs once.
// (Fitted to products of 256, 512, 768 and 1024 tiles, contractions of 4096 and 8192.)
struct MxStep { double t1, u1, t2, u2, pair; };

// Tile height (16 ct rows of x) and parts of the contraction for M rows, `cols` tiles over the O outputs and `steps`: least time of
//   steps of a part x step time at so many blocks a CU (a second block on some CUs only counts 0.3 and its share of the rest,
//     a later one three quarters; where CUs are left over, a block takes down to 0.85 of the time)
//   + start and outputs of a block, 1 us and 1.3 more per 16 rows
//   + writing the parts and adding them up: 7 TB/s, 3 us for the launch, 0.1 a part
// Within 2.5 % of the best (ct, split) on average, 0.9 % at the median, 26 % at worst (float32 1000 x 5003 x 10007), over 175 sizes from 24 x 4096 x 4096 to
// 512 x 20000 x 20000.  What it weighs, us: bf16 512 x 14336 x 4096 in tiles of ct 2 / 4 / 8: 59 / 51 / 56; float32 64 x 20000 x 20000 in
// 1 / 2 / 3 / 4 / 6 parts: 201 / 155 / 125 / 133 / 130
static double mx_choose(int64_t M, int64_t O, int64_t cols, int64_t steps, int terms, int min_ct, int max_ct, const MxStep& c, int* ct_out, int* split_out) {
    *ct_out = min_ct;
    *split_out = 1;
    double best = 1e300;
    for (int ct = min_ct; ct <= max_ct && (ct == min_ct || 8 * ct < M); ct *= 2) {
        const int64_t tiles = cdiv(M, 16 * ct) * cols;
        const double one = c.t1 + c.u1 * ct * terms, two = c.t2 + c.u2 * ct * terms, fixed = 1.0 + 1.3 * ct;
        // (more than four blocks a CU only pay where the last round's waste is long: products of some 300 us)
        for (int64_t s = 1; s <= 64 && s <= steps && (s == 1 || tiles * s <= (best > 300.0 ? 16 : 4) * MX_CUS); ++s) {
            const int64_t full = tiles * s / MX_CUS, rest = tiles * s % MX_CUS;
            const double b = full == 0 ? 1.0 : (double)full + (rest == 0 ? 0.0 : full == 1 ? 0.3 + 0.7 * (double)rest / MX_CUS : 0.75 + 0.25 * (double)rest / MX_CUS);
            const double step = full == 0 ? one * (0.85 + 0.15 * (double)rest / MX_CUS) : b <= 2.0 ? one + (two - one) * (b - 1.0) : two * 0.5 * b;
            const double t = (double)cdiv(steps, s) * step + (b <= 2.0 ? fixed + c.pair * (b - 1.0) : (fixed + c.pair) * 0.5 * b) +
                             (s > 1 ? (double)(s * M * O) * 8 / 7e6 + 3.0 + 0.1 * (double)s : 0.0);
            if (t < best * 0.98) { best = t; *ct_out = ct; *split_out = (int)s; }
        }
    }
    return best;
}

// what a fit adds to a product: a factor of every column of W (taken into x before it is split, or into the output), and the flag of a trial
// that turned out invalid
struct MxExtra {
    const float *kscale = nullptr, *oscale = nullptr;
    const int* skip = nullptr;
    bool tiles = false;                // no row kernel
};

// M rows of x, C the contraction, O output columns; along: lcx_mx4_linear, else lcx_mx4_linear_grad
template <typename T> static MxPlan mx_plan(bool along, int64_t M, int64_t C, int64_t O, bool tiles = false) {
    constexpr int TERMS = MxTerms<T>::v;
    MxPlan p;
    p.rt = 4;
    p.nt = along ? cdiv(O, 64 * p.rt) : cdiv(O, 512);
    const MxStep step = along        ? TERMS == 1 ? MxStep{0.52, 0.13, 0.42, 0.33, 1.5} : MxStep{0.58, 0.145, 0.4, 0.33, 0.0}
                        : TERMS == 1 ? MxStep{1.7, 0.21, 1.9, 0.48, 4.0}
                                     : MxStep{2.7, 0.19, 2.1, 0.53, 4.0};
    const auto choose = [&] { return mx_choose(M, O, p.nt, cdiv(C, 128), TERMS, M <= 16 ? 1 : 2, along && TERMS == 1 ? 8 : 4, step, &p.ct, &p.split); };
    if (M <= 16 && along && !tiles) {
        // The row kernel or the tiles, whichever takes less time by these models (fitted for K and N from 512 to 28672; 10 %):
        //   row    3.5 us + the steps a CU works through
        //   tiles  mx_choose, or reading W; 8 us for the two launches more
        // Measured, us, row / tiles, W out of HBM (in the caches): 1 x 4096 x 4096 bf16 5.3 / 10.3 (4.9 / 8.6); 16 x 20000 x 20000 bf16
        // 100 / 58 (70 / 42), float32 174 / 67 (135 / 47); 8 x 28672 x 8192 float16 48 / 40 (42 / 29); 1 x 28672 x 8192 bf16 34 / 34 (25 / 25).
        // 2 x 16 rows of W a wave halve the reads of x where there are enough rows to fill the chip.  One / two, us, bf16, W out of HBM:
        //   rows of W x 4096   2048       4096       5120       6144       8192       12288      16384      28672
        //   1 row of x         4.8/5.8    5.3/6.1    6.8/6.2    7.0/6.5    7.4/7.1    10.0/9.9   12.6/11.1  20.0/18.2
        //   13                 6.3/7.1    7.0/7.5    10.9/7.6   11.0/7.9   11.3/8.4   15.5/13.2  19.6/14.0  32.0/23.7
        // (Two are faster from 4097 rows on, but the model of the row kernel then comes out too low for long contractions: float16
        // 16 x 7942 x 8833 would take it, 36 us, instead of the tiles, 24.)
        const int rt = O < 32 * MX_CUS ? 1 : 2;
        const double blocks = (double)cdiv(O, 16 * rt) / MX_CUS;
        const double row = 3.5 + (double)cdiv(C, 128) * (blocks < 1.0 ? 1.0 : blocks) *
                                     ((rt == 2 ? 0.09 : 0.04) + (TERMS == 1 ? 0.0 : TERMS == 2 ? 0.075 : 0.09) +
                                      (TERMS == 1 ? 0.0045 : TERMS == 2 ? 0.002 : 0.0075) * (double)M);
        const double read = (double)O * (double)C * 0.53 / 6e6 + 5.0;
        // (nearly always the row kernel: a microsecond of the call is saved by not looking at the tiles then)
        if (row <= read + 8.0 || row <= choose() + 8.0) {
            p = MxPlan();
            p.row = true;
            p.rt = rt;
            return p;
        }
    } else {
        (void)choose();
    }
    p.mt = cdiv(M, 16 * p.ct);
    p.nfrag = cdiv(C, 128) * 4;
    const int64_t pieces = p.mt * p.ct * cdiv(C, 128);         // (a block of mx_fragments_kernel each)
    p.frag_bytes = pieces < MX_MAX_PIECES ? pieces * 4 * TERMS * 1024 : -1;
    if (p.split > 1) p.part_bytes = (int64_t)p.split * M * O * 4;
    return p;
}
static int64_t mx_plan_bytes(const MxPlan& p) { return round_up(p.frag_bytes, 256) + p.part_bytes; }

static int64_t mx_matmul_bytes(int64_t M, int64_t N, int64_t K);
template <typename T> static int64_t mx_workspace(int op, int64_t M, int64_t N, int64_t K) {
    if (M == 0 || N == 0 || K == 0) return 0;
    if (op == 0) return mx_matmul_bytes(M, N, K);
    const MxPlan p = op & 1 ? mx_plan<T>(true, M, K, N) : mx_plan<T>(false, M, N, K);
    return op > 2 ? p.part_bytes : p.frag_bytes < 0 ? -1 : mx_plan_bytes(p);
}

template <typename T, bool ALONG>
static int mx_fragments(const T* x, int64_t M, int64_t rs, int64_t cs, int64_t C, const MxPlan& p, unsigned short* frag, const MxExtra& ex, hipStream_t st) {
    const int64_t tiles = p.mt * p.ct;
    unsigned g;
    LCXCHECK(mx_grid(tiles, cdiv(p.nfrag * 4, 16), 256, &g));
    const int rows_first = (rs < 0 ? -rs : rs) < (cs < 0 ? -cs : cs);
    if (cs == 1)
        hipLaunchKernelGGL((mx_fragments_kernel<T, ALONG, true>), dim3(g), dim3(256), 0, st, x, M, rs, cs, C, p.nfrag, tiles, frag, 0, ex.kscale, ex.skip);
    else
        hipLaunchKernelGGL((mx_fragments_kernel<T, ALONG, false>), dim3(g), dim3(256), 0, st, x, M, rs, cs, C, p.nfrag, tiles, frag, rows_first,
                           ex.kscale, ex.skip);
    KCHECK();
    return LCX_OK;
}

// rows that the tile kernels take as they are (MxDirect; the offsets inside a tile are 32-bit): C of the contraction, whole stages of it
template <typename T> static bool mx_direct(const MxPlan& p, const T* x, int64_t rs, int64_t cs, int64_t C, int stage) {
    return MxTerms<T>::v == 1 && !p.row && C % stage == 0 && cs == 1 && rs >= 0 && rs < (1 << 23) && rs % 8 == 0 && ((uintptr_t)x & 15) == 0;
}

// the plan without the fragments' space where x is taken as it is; the work space as the plan wants it
static int mx_space(const char* name, MxPlan& p, bool direct, const void* space, int64_t bytes) {
    if (direct) p.frag_bytes = 0;
    if (p.frag_bytes < 0) return fail(LCX_ERR_ARG, std::string(name) + ": x is too large for one call");
    const int64_t want = mx_plan_bytes(p);
    if (bytes < want || (want && (!space || ((uintptr_t)space & 15))))
        return fail(LCX_ERR_ARG, std::string(name) + ": the work space is smaller than lcx_mx4_workspace says or not 16-byte aligned");
    return LCX_OK;
}

template <typename T> static int mx_join(int split, const MxOut<T>& w, hipStream_t st) {
    if (split == 1) return LCX_OK;
    // t_first: the partial sums lie transposed, and so does the output
    const int64_t M = w.t_first ? w.O : w.M, O = w.t_first ? w.M : w.O;
    int bx = 256;
    while (bx > 4 && (int64_t)bx * 2 >= O) bx /= 2;
    const int by = 256 / bx;
    const int64_t gy = cdiv(M, by);
    hipLaunchKernelGGL((mx_join_kernel<T>), dim3((unsigned)cdiv(O, bx * 4), (unsigned)(gy < 32768 ? gy : 32768)), dim3(bx, by), 0, st, w.part, split, M, O, w.out,
                       w.t_first ? w.cs : w.rs, w.t_first ? w.rs : w.cs, w.oscale, w.skip);
    KCHECK();
    return LCX_OK;
}

// fragments of the contraction (linear) and steps (linear_grad) a stage holds, by the height of a tile
template <typename T> constexpr int mx_linear_js(int ct) { return MxTerms<T>::v == 3 && ct == 4 ? 2 : 4; }      // (three terms of four: 96 KB of LDS, one block a CU)
template <typename T> constexpr int mx_grad_js() { return MxTerms<T>::v > 1 ? 1 : 2; }         // (a second step would be 83 KB with two terms: one block a CU)

template <typename T, int CT, bool DIRECT = false>
static int mx_linear_tiles(const MxPlan& p, const unsigned short* frag, int64_t tiles, const unsigned char* wc, const unsigned char* ws, int64_t N, int64_t K, const MxOut<T>& w,
                           hipStream_t st) {
    unsigned g;
    LCXCHECK(mx_grid(8, cdiv(p.mt * p.nt * p.split, 8), 256, &g));
    hipLaunchKernelGGL((mx_linear_tile_kernel<T, CT, 4, mx_linear_js<T>(CT), DIRECT>), dim3(g), dim3(256), 0, st, frag, tiles, wc, ws, N, K, w, (int)p.mt, (int)p.nt, p.split);
    KCHECK();
    return LCX_OK;
}
template <typename T, int CT, bool DIRECT = false>
static int mx_grad_tiles(const MxPlan& p, const unsigned short* frag, int64_t tiles, const unsigned char* wc, const unsigned char* ws, int64_t N, int64_t K, const MxOut<T>& w,
                         hipStream_t st) {
    unsigned g;
    LCXCHECK(mx_grid(8, cdiv(p.mt * p.nt * p.split, 8), 256, &g));
    constexpr int JS = mx_grad_js<T>();
    constexpr size_t lds = MxGradLds<CT, JS, MxTerms<T>::v>::total;
    LCXCHECK(allow_lds(mx_grad_tile_kernel<T, CT, JS, DIRECT>, lds));
    hipLaunchKernelGGL((mx_grad_tile_kernel<T, CT, JS, DIRECT>), dim3(g), dim3(256), lds, st, frag, tiles, wc, ws, N, K, w, (int)p.mt, (int)p.nt, p.split);
    KCHECK();
    return LCX_OK;
}

template <typename T, bool VEC>
static int mx_linear_rows(const MxPlan& p, const T* x, int64_t rs, int64_t cs, const unsigned char* wc, const unsigned char* ws, int64_t N, int64_t K,
                          const MxOut<T>& w, hipStream_t st) {
    unsigned g;
    LCXCHECK(mx_grid(1, cdiv(N, 16 * p.rt), 64 * MX_ROW_WAVES, &g));
#define MX_ROWS(RT) hipLaunchKernelGGL((mx_linear_row_kernel<T, RT, VEC>), dim3(g), dim3(64 * MX_ROW_WAVES), 0, st, x, w.M, rs, cs, wc, ws, N, K, w)
    if (p.rt == 2) MX_ROWS(2);
    else MX_ROWS(1);
#undef MX_ROWS
    KCHECK();
    return LCX_OK;
}

template <typename T>
static int mx4_linear(const void* xv, int64_t M, int64_t xrs, int64_t xcs, const void* wcv, const void* wsv, int64_t N, int64_t K, void* out, int64_t rs,
                      int64_t cs, void* space, int64_t space_bytes, hipStream_t st, const MxExtra& ex = MxExtra()) {
    constexpr int TERMS = MxTerms<T>::v;
    if (K == 0) return mx4_zero<T>(out, M, N, rs, cs, st);
    MxPlan p = mx_plan<T>(true, M, K, N, ex.tiles);
    const T* x = (const T*)xv;
    const bool direct = mx_direct(p, x, xrs, xcs, K, 128);
    LCXCHECK(mx_space("lcx_mx4_linear", p, direct, space, space_bytes));
    const unsigned char *wc = (const unsigned char*)wcv, *ws = (const unsigned char*)wsv;
    unsigned short* frag = (unsigned short*)space;
    MxOut<T> w{(T*)out, rs, cs, p.split > 1 ? (float*)((char*)space + round_up(p.frag_bytes, 256)) : nullptr, M, N, rs == 1 && cs != 1, ex.oscale, ex.skip};
    if (p.row) return xcs == 1 ? mx_linear_rows<T, true>(p, x, xrs, xcs, wc, ws, N, K, w, st)
                                                : mx_linear_rows<T, false>(p, x, xrs, xcs, wc, ws, N, K, w, st);
    if constexpr (TERMS == 1) {
        if (direct) {
            const unsigned short* xb = (const unsigned short*)xv;
            if (p.ct == 1) LCXCHECK((mx_linear_tiles<T, 1, true>(p, xb, xrs, wc, ws, N, K, w, st)));
            else if (p.ct == 2) LCXCHECK((mx_linear_tiles<T, 2, true>(p, xb, xrs, wc, ws, N, K, w, st)));
            else if (p.ct == 4) LCXCHECK((mx_linear_tiles<T, 4, true>(p, xb, xrs, wc, ws, N, K, w, st)));
            else LCXCHECK((mx_linear_tiles<T, 8, true>(p, xb, xrs, wc, ws, N, K, w, st)));
            return mx_join<T>(p.split, w, st);
        }
    }
    LCXCHECK((mx_fragments<T, true>(x, M, xrs, xcs, K, p, frag, ex, st)));
    const int64_t tiles = p.mt * p.ct;
    if (p.ct == 1) LCXCHECK((mx_linear_tiles<T, 1>(p, frag, tiles, wc, ws, N, K, w, st)));
    else if (p.ct == 2) LCXCHECK((mx_linear_tiles<T, 2>(p, frag, tiles, wc, ws, N, K, w, st)));
    else if (p.ct == 4) LCXCHECK((mx_linear_tiles<T, 4>(p, frag, tiles, wc, ws, N, K, w, st)));
    else {
        if constexpr (TERMS == 1) LCXCHECK((mx_linear_tiles<T, 8>(p, frag, tiles, wc, ws, N, K, w, st)));
    }
    return mx_join<T>(p.split, w, st);
}

template <typename T>
static int mx4_linear_grad(const void* dyv, int64_t M, int64_t yrs, int64_t ycs, const void* wcv, const void* wsv, int64_t N, int64_t K, void* out, int64_t rs,
                           int64_t cs, void* space, int64_t space_bytes, hipStream_t st, const MxExtra& ex = MxExtra()) {
    constexpr int TERMS = MxTerms<T>::v;
    if (N == 0) return mx4_zero<T>(out, M, K, rs, cs, st);
    MxPlan p = mx_plan<T>(false, M, N, K, ex.tiles);
    const T* dy = (const T*)dyv;
    const bool direct = mx_direct(p, dy, yrs, ycs, N, 64);
    LCXCHECK(mx_space("lcx_mx4_linear_grad", p, direct, space, space_bytes));
    const unsigned char *wc = (const unsigned char*)wcv, *ws = (const unsigned char*)wsv;
    unsigned short* frag = (unsigned short*)space;
    MxOut<T> w{(T*)out, rs, cs, p.split > 1 ? (float*)((char*)space + round_up(p.frag_bytes, 256)) : nullptr, M, K, rs == 1 && cs != 1, ex.oscale, ex.skip};
    if constexpr (TERMS == 1) {
        if (direct) {
            const unsigned short* yb = (const unsigned short*)dyv;
            if (p.ct == 1) LCXCHECK((mx_grad_tiles<T, 1, true>(p, yb, yrs, wc, ws, N, K, w, st)));
            else if (p.ct == 2) LCXCHECK((mx_grad_tiles<T, 2, true>(p, yb, yrs, wc, ws, N, K, w, st)));
            else LCXCHECK((mx_grad_tiles<T, 4, true>(p, yb, yrs, wc, ws, N, K, w, st)));
            return mx_join<T>(p.split, w, st);
        }
    }
    LCXCHECK((mx_fragments<T, false>(dy, M, yrs, ycs, N, p, frag, ex, st)));
    const int64_t tiles = p.mt * p.ct;
    if (p.ct == 1) LCXCHECK((mx_grad_tiles<T, 1>(p, frag, tiles, wc, ws, N, K, w, st)));
    else if (p.ct == 2) LCXCHECK((mx_grad_tiles<T, 2>(p, frag, tiles, wc, ws, N, K, w, st)));
    else LCXCHECK((mx_grad_tiles<T, 4>(p, frag, tiles, wc, ws, N, K, w, st)));
    return mx_join<T>(p.split, w, st);
}

// ---- 4 bits x 4 bits --------------------------------------------------------------------------------------------------------------------
struct MxMatmulPlan {
    bool row = false;
    int ct = 1, rt = 1, split = 1;
    int64_t mt = 1, nt = 1, part_bytes = 0;
};
static MxMatmulPlan mx_matmul_plan(int64_t M, int64_t N, int64_t K) {
    MxMatmulPlan p;
    if (M <= 16) {
        p.row = true;
        // Two row tiles a block, which halve the reads of A, once one would leave more blocks than CUs.  One / two, us, 8 rows, B out of HBM:
        //   n x 4096   2048 4.3/5.1   4096 4.5/5.3   5120 5.9/5.4   8192 6.8/6.1   12288 8.7/8.7    16384 10.5/9.3   28672 16.7/15.0
        //   n x 8192   2048 6.0/7.6   4096 6.4/8.2   5120 9.7/9.1   8192 11.1/10.2 12288 15.4/15.1  16384 19.4/16.7  28672 31.8/28.7
        // (B in the caches: up to 10 % slower at 10240 and 12288, 5 % from 16384 on)
        p.rt = N <= 16 * MX_CUS ? 1 : 2;
        return p;
    }
    p.nt = cdiv(N, 256);
    mx_choose(M, N, p.nt, cdiv(K, 512), 1, 2, 8, MxStep{1.5, 0.06, 0.9, 0.34, 5.0}, &p.ct, &p.split);
    p.mt = cdiv(M, 16 * p.ct);
    if (p.split > 1) p.part_bytes = (int64_t)p.split * M * N * 4;
    return p;
}

static int64_t mx_matmul_bytes(int64_t M, int64_t N, int64_t K) { return mx_matmul_plan(M, N, K).part_bytes; }

// what a product of these sizes is made of (tools/lcx_probe.h, lcx_test_mx4_plan): {row kernel, 16-row tiles of x, of W, parts}
template <typename T> static void mx_plan_of(int op, int64_t M, int64_t N, int64_t K, int* v) {
    if (op == 0) {
        const MxMatmulPlan p = mx_matmul_plan(M, N, K);
        v[0] = p.row, v[1] = p.ct, v[2] = p.row ? p.rt : 4, v[3] = p.split;
    } else {
        const MxPlan p = op == 1 ? mx_plan<T>(true, M, K, N) : mx_plan<T>(false, M, N, K);
        v[0] = p.row, v[1] = p.ct, v[2] = p.rt, v[3] = p.split;
    }
}
void lcx_mx_plan(int op, int dtype, int64_t M, int64_t N, int64_t K, int* v) {
    if (dtype == LCX_F32) mx_plan_of<float>(op, M, N, K, v);
    else if (dtype == LCX_BF16) mx_plan_of<__bf16>(op, M, N, K, v);
    else mx_plan_of<_Float16>(op, M, N, K, v);
}

template <typename T, int CT, int RT>
static int mx_matmul_tiles(const MxMatmulPlan& p, const unsigned char* ac, const unsigned char* as, const unsigned char* bc, const unsigned char* bs, int64_t N,
                           int64_t K, const MxOut<T>& w, hipStream_t st) {
    unsigned g;
    LCXCHECK(mx_grid(8, cdiv(p.mt * p.nt * p.split, 8), 256, &g));
    hipLaunchKernelGGL((mx_matmul_tile_kernel<T, CT, RT>), dim3(g), dim3(256), 0, st, ac, as, bc, bs, N, K, w, (int)p.mt, (int)p.nt, p.split);
    KCHECK();
    return LCX_OK;
}

template <typename T>
static int mx4_matmul(const void* acv, const void* asv, int64_t M, const void* bcv, const void* bsv, int64_t N, int64_t K, void* out, int64_t rs, int64_t cs,
                      void* space, int64_t space_bytes, hipStream_t st) {
    if (K == 0) return mx4_zero<T>(out, M, N, rs, cs, st);
    const unsigned char *ac = (const unsigned char*)acv, *as = (const unsigned char*)asv, *bc = (const unsigned char*)bcv, *bs = (const unsigned char*)bsv;
    const MxMatmulPlan p = mx_matmul_plan(M, N, K);
    if (space_bytes < p.part_bytes || (p.part_bytes && (!space || ((uintptr_t)space & 15)))) return fail(LCX_ERR_ARG, "lcx_mx4_matmul: the work space is smaller than lcx_mx4_workspace says or not 16-byte aligned");
    MxOut<T> w{(T*)out, rs, cs, p.split > 1 ? (float*)space : nullptr, M, N, rs == 1 && cs != 1, nullptr, nullptr};
    if (p.row) {
        unsigned g;
        LCXCHECK(mx_grid(1, cdiv(N, 16 * p.rt), 64 * MX_ROW_WAVES, &g));
#define MX_ROWS(RT) hipLaunchKernelGGL((mx_matmul_row_kernel<T, RT>), dim3(g), dim3(64 * MX_ROW_WAVES), 0, st, ac, as, M, bc, bs, N, K, w)
        if (p.rt == 2) MX_ROWS(2);
        else MX_ROWS(1);
#undef MX_ROWS
        KCHECK();
        return LCX_OK;
    }
    if (p.ct == 8) LCXCHECK((mx_matmul_tiles<T, 8, 4>(p, ac, as, bc, bs, N, K, w, st)));
    else if (p.ct == 4) LCXCHECK((mx_matmul_tiles<T, 4, 4>(p, ac, as, bc, bs, N, K, w, st)));
    else LCXCHECK((mx_matmul_tiles<T, 2, 4>(p, ac, as, bc, bs, N, K, w, st)));
    return mx_join<T>(p.split, w, st);
}

// ---- the resident shard of a fit in 4 bits (engine.hpp) ----------------------------------------------------------------------------------
// X~ (Npad samples x ldx variables, blocks along the variables).  Rounding to 4 bits changes a variable's mean square by a per cent or so, and
// the algorithm's moments are relative to it (preprocessed data have 1 where nothing is missing or transformed, other values elsewhere): hence one
// float32 factor per variable (xunit) that gives it back the mean square it had, which the passes apply to the small operand or to the
// output.  What is fitted is X~ = values of the 4 bits x factor.
int lcx_mx_shard_alloc(lcx_ctx* h) {
    const int64_t rt = mx_row_tiles(h->Npad);
    const MxPlan a = mx_plan<float>(true, h->Mp, h->ldx, h->Npad, true), b = mx_plan<float>(false, h->Mp, h->Npad, h->ldx, true);
    const int64_t wa = mx_plan_bytes(a), wb = mx_plan_bytes(b);
    const size_t bytes[4] = {(size_t)(rt * mx_steps(h->ldx) * 1024), (size_t)(rt * mx_quads(h->ldx) * 256), (size_t)h->ldx * 4,
                             (size_t)std::max({wa, wb, h->ldx * 8})};             // (ldx doubles: the sums of a block being filled)
    void** to[4] = {&h->xq, &h->xs, (void**)&h->xunit, &h->xwork};
    for (int i = 0; i < 4; ++i) {
        LCXCHECK(dev_alloc(to[i], bytes[i], h->stream));
        h->bytes_resident += bytes[i];
    }
    h->xq_bytes = bytes[0] + bytes[1] + bytes[2];
    h->xwork_bytes = (int64_t)bytes[3];
    return LCX_OK;
}
// columns [c0, c0 + cols) from (and, rounded, back to) the row-major staging block; c0 is a multiple of 512
static int mx_shard_block(lcx_ctx* h, float* stage, int64_t ld, int64_t c0, int64_t cols, bool fill) {
    const int64_t nq = mx_quads(cols);
    unsigned g;
    LCXCHECK(mx_grid(mx_row_tiles(h->Npad), nq, 256, &g));
    unsigned char *qc = (unsigned char*)h->xq, *qs = (unsigned char*)h->xs;
    double* sum = (double*)h->xwork;
    if (fill) {
        hipLaunchKernelGGL((mx_square_columns_kernel<false>), dim3((unsigned)cdiv(cols, 64)), dim3(1024), 0, h->stream, stage, h->N, cols, ld, sum, h->xunit + c0);
        KCHECK();
        // (a staging block is up to 1 GB, just written: MX_ONCE_BYTES)
        hipLaunchKernelGGL((mx_quantize_kernel<float, true, true>), dim3(g), dim3(256), 0, h->stream, stage, h->Npad, cols, ld, (int64_t)1, qc, qs, mx_steps(h->ldx),
                           mx_quads(h->ldx), c0 / 512, (unsigned)nq);
        KCHECK();
    }
    hipLaunchKernelGGL((mx_dequantize_kernel<float, true>), dim3(g), dim3(256), 0, h->stream, qc, qs, h->Npad, cols, stage, ld, (int64_t)1, mx_steps(h->ldx),
                       mx_quads(h->ldx), c0 / 512, (unsigned)nq);
    KCHECK();
    if (fill) {
        hipLaunchKernelGGL((mx_square_columns_kernel<true>), dim3((unsigned)cdiv(cols, 64)), dim3(1024), 0, h->stream, stage, h->N, cols, ld, sum, h->xunit + c0);
    } else {
        hipLaunchKernelGGL(mx_scale_columns_kernel, dim3(4096), dim3(256), 0, h->stream, stage, h->Npad, cols, ld, h->xunit + c0);
    }
    KCHECK();
    return LCX_OK;
}
int lcx_mx_shard_fill(lcx_ctx* h, float* stage, int64_t ld, int64_t c0, int64_t cols) { return mx_shard_block(h, stage, ld, c0, cols, true); }
int lcx_mx_shard_read(lcx_ctx* h, float* stage, int64_t ld, int64_t c0, int64_t cols) { return mx_shard_block(h, stage, ld, c0, cols, false); }
// out [Npad][Mp] = X~ . B, B [ldx][Mp]
int lcx_mx_shard_xbt(lcx_ctx* h, const float* B, float* out, const int* skip) {
    MxExtra ex;
    ex.kscale = h->xunit;
    ex.skip = skip;
    ex.tiles = true;
    return mx4_linear<float>(B, h->Mp, 1, h->Mp, h->xq, h->xs, h->Npad, h->ldx, out, 1, h->Mp, h->xwork, h->xwork_bytes, h->stream, ex);
}
// out [ldx][Mp] = X~^T . Y, Y [Npad][Mp]
int lcx_mx_shard_xty(lcx_ctx* h, const float* Y, float* out, const int* skip) {
    MxExtra ex;
    ex.oscale = h->xunit;
    ex.skip = skip;
    ex.tiles = true;
    return mx4_linear_grad<float>(Y, h->Mp, 1, h->Mp, h->xq, h->xs, h->Npad, h->ldx, out, 1, h->Mp, h->xwork, h->xwork_bytes, h->stream, ex);
}
// name of the kernel of a pass (kind 0: X~ . B, else X~^T . Y), as a profiler shows it
void lcx_mx_shard_kernel(const lcx_ctx* h, int kind, char* buf, int64_t len) {
    const MxPlan p = kind == 0 ? mx_plan<float>(true, h->Mp, h->ldx, h->Npad, true) : mx_plan<float>(false, h->Mp, h->Npad, h->ldx, true);
    if (kind == 0) snprintf(buf, (size_t)len, "lcx::mx_linear_tile_kernel<float, %d, 4, %d, false>", p.ct, mx_linear_js<float>(p.ct));
    else snprintf(buf, (size_t)len, "lcx::mx_grad_tile_kernel<float, %d, %d, false>", p.ct, mx_grad_js<float>());
}

extern "C" {

int lcx_mx4_layout(int64_t rows, int64_t cols, int64_t* code_bytes, int64_t* scale_bytes) {
    MX_ENTRY({
        if (dim_bad(rows, cols)) return fail(LCX_ERR_ARG, "lcx_mx4_layout: bad sizes");
        if (code_bytes) *code_bytes = mx_row_tiles(rows) * mx_steps(cols) * 1024;
        if (scale_bytes) *scale_bytes = mx_row_tiles(rows) * mx_quads(cols) * 256;
        return LCX_OK;
    })
}

int lcx_mx4_quantize(const void* x, int dtype, int64_t rows, int64_t cols, int64_t row_stride, int64_t col_stride, void* codes, void* scales, void* stream) {
    MX_ENTRY({
        if (dim_bad(rows, cols)) return fail(LCX_ERR_ARG, "lcx_mx4_quantize: bad sizes");
        if (dtype < LCX_F32 || dtype > LCX_F16) return fail(LCX_ERR_ARG, "lcx_mx4_quantize: bad dtype");
        if (rows == 0 || cols == 0) return LCX_OK;
        if (!x || !codes || !scales) return fail(LCX_ERR_ARG, "lcx_mx4_quantize: null pointer");
        if (mx_misaligned(codes, scales)) return fail(LCX_ERR_ARG, "lcx_mx4_quantize: codes and scales must be 16-byte aligned");
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
        if (mx_misaligned(codes, scales)) return fail(LCX_ERR_ARG, "lcx_mx4_dequantize: codes and scales must be 16-byte aligned");
        hipStream_t st = (hipStream_t)stream;
        if (dtype == LCX_F64) return mx4_dequantize<double>(codes, scales, rows, cols, out, row_stride, col_stride, st);
        MX_FLOATS(dtype, mx4_dequantize, codes, scales, rows, cols, out, row_stride, col_stride, st);
    })
}

int lcx_mx4_workspace(int op, int dtype, int64_t M, int64_t N, int64_t K, int64_t* bytes) {
    MX_ENTRY({
        if (!bytes || op < 0 || op > 4 || dim_bad(M, N, K)) return fail(LCX_ERR_ARG, "lcx_mx4_workspace: bad argument");
        if (op > 2 && dtype != LCX_BF16) return fail(LCX_ERR_ARG, "lcx_mx4_workspace: only LCX_BF16 is read in place");
        if (dtype != LCX_F32 && dtype != LCX_BF16 && dtype != LCX_F16) return fail(LCX_ERR_ARG, "lcx_mx4_workspace: bad dtype");
        const int64_t b = dtype == LCX_F32 ? mx_workspace<float>(op, M, N, K) : dtype == LCX_BF16 ? mx_workspace<__bf16>(op, M, N, K) : mx_workspace<_Float16>(op, M, N, K);
        if (b < 0) return fail(LCX_ERR_ARG, "lcx_mx4_workspace: x is too large for one call");
        *bytes = b;
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
            return fail(LCX_ERR_ARG, "lcx_mx4_matmul: codes and scales must be 16-byte aligned");
        MX_FLOATS(dtype, mx4_matmul, a_codes, a_scales, M, b_codes, b_scales, N, K, out, row_stride, col_stride, workspace, workspace_bytes,
                  (hipStream_t)stream);
    })
}

int lcx_mx4_linear(const void* x, int dtype, int64_t M, int64_t x_row, int64_t x_col, const void* codes, const void* scales, int64_t N, int64_t K, void* out,
                   int64_t row_stride, int64_t col_stride, void* workspace, int64_t workspace_bytes, void* stream) {
    MX_ENTRY({
        if (dim_bad(M, N, K)) return fail(LCX_ERR_ARG, "lcx_mx4_linear: bad sizes");
        if (dtype != LCX_F32 && dtype != LCX_BF16 && dtype != LCX_F16) return fail(LCX_ERR_ARG, "lcx_mx4_linear: dtype must be LCX_F32, LCX_BF16 or LCX_F16");
        if (M == 0 || N == 0) return LCX_OK;
        if (!out || (K > 0 && (!x || !codes || !scales))) return fail(LCX_ERR_ARG, "lcx_mx4_linear: null pointer");
        if (mx_misaligned(codes, scales)) return fail(LCX_ERR_ARG, "lcx_mx4_linear: codes and scales must be 16-byte aligned");
        MX_FLOATS(dtype, mx4_linear, x, M, x_row, x_col, codes, scales, N, K, out, row_stride, col_stride, workspace, workspace_bytes, (hipStream_t)stream);
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
        if (mx_misaligned(codes, scales)) return fail(LCX_ERR_ARG, "lcx_mx4_linear_grad: codes and scales must be 16-byte aligned");
        MX_FLOATS(dtype, mx4_linear_grad, dy, M, dy_row, dy_col, codes, scales, N, K, out, row_stride, col_stride, workspace, workspace_bytes, (hipStream_t)stream);
    })
}

}  // extern "C"
