/*
 * What the kernels of the linear layer and of the products by expert share: the
 * arguments of a product C[m][n] = sum_k A(m, k) B(n, k) with its epilogue, the
 * activations, and the epilogue itself on eight consecutive columns of a row.
 */
#ifndef ESHKOL_HIP_LINEAR_ARGS_H
#define ESHKOL_HIP_LINEAR_ARGS_H

#include "layer_common.h"

#include <algorithm>

/* How an operand lies in memory: its rows (m or n) apart and k contiguous, or k
 * apart and the rows contiguous. */
enum { ROWS_K = 0, K_ROWS = 1 };
/* What the groups of experts cut: nothing, the rows of A and C, or the contraction. */
enum { GROUP_NONE = 0, GROUP_ROWS = 1, GROUP_K = 2 };

struct LinearEpilogue {
    const void* bias;           /* [experts][N] or NULL                            */
    const uint16_t* residual;
    void* y;                    /* 16-bit, or fp32 where out32                     */
    uint16_t* pre;
    uint64_t ld_res, ldy, ld_pre;
    int bias_wide, act, out32;
};

struct LinearArgs {
    const uint16_t *a, *b;
    uint64_t lda, ldb;          /* elements                                        */
    uint32_t M, N, K;           /* GROUP_ROWS: M all rows; GROUP_K: K all rows     */
    /* how far the contiguous rows of a K_ROWS operand may be read (a multiple of 8) */
    uint32_t a_extent, b_extent;
    LinearEpilogue e;
    /* cut of the contraction: `splits` parts of `part_k` (a multiple of 64); with more
     * than one the sums go to part[split][M][part_ld] and a second launch joins them */
    uint32_t splits, part_k, part_ld;
    float* part;
    const int32_t* offsets;
    uint32_t experts;
    uint64_t b_stride, y_stride;   /* elements per expert: B (GROUP_ROWS), C (GROUP_K) */
    uint32_t tiles_m, tiles_n;
    uint32_t wg_tiles;          /* workgroups of one part: the tiles, rounded up to a multiple of 8 */
};

namespace linear {

/* dz = grad_y act'(pre), and the sums of dz's columns before it is rounded. A workgroup takes 256 columns (32 threads, eight
 * each) of every parts-th eight rows of its expert; its eight rows of threads are joined in LDS. */
struct SlopeArgs {
    const uint16_t *dy, *pre;
    uint16_t* dz;               /* NULL: the sums alone                            */
    float* part;                /* [experts][parts][N], or NULL                    */
    uint64_t ld_dy, ld_pre, ld_dz;
    uint32_t rows, N, parts, experts, across, blocks;      /* across: workgroups per row of parts */
    const int32_t* offsets;
    int act;
};

/* The sums of a bias gradient's parts, in ascending order: a thread takes a column of an expert. */
struct BiasJoin {
    const float* part;          /* [experts][parts][N]                             */
    float* out;                 /* [experts][N]                                    */
    uint32_t N, parts, experts;
};

/* Rows that do not start on 16-byte boundaries, or are no multiple of 16 bytes, copied to ones that do and are (zeros
 * behind their end): `chunks` pieces of 16 bytes of matrices of rows x cols. */
struct AlignArgs {
    const uint16_t* in;
    uint16_t* out;
    uint64_t ld, stride, rows, chunks;
    uint32_t cols, out_ld, blocks;
};

/* A matrix operand as the caller gave it, and whether it has to be copied before the tiled kernel may read it. */
struct Matrix {
    const uint16_t* p;
    uint64_t ld, stride, rows, cols, count;
    bool copy;
    uint64_t copy_bytes;
};

/* What a product is: C[M][N] over K; per expert where group says so. */
struct Shape {
    int fa, fb, group;
    uint64_t M, N, K, experts;
};
/* How a product is run: tiles of a shape that all of a launch share; tiles of 32 or 64 rows; B streamed past at most 64 rows
 * (in parts of K that a second launch joins, or with K whole in a workgroup) */
enum { RUN_TILES, RUN_TILES_32, RUN_TILES_64, RUN_STREAM, RUN_STREAM_WHOLE };
enum { TILE_LARGE, TILE_WIDE, TILE_WIDE_ALONE, TILE_SQUARE, TILE_SQUARE_ALONE };

struct Product {
    Shape s;
    Matrix a, b;
    LinearArgs g;
    int kind, rt;               /* rt: sixteens of rows of RUN_STREAM              */
    uint32_t splits, part_k, part_ld;
    uint64_t part_bytes;
    bool streams() const { return kind == RUN_STREAM || kind == RUN_STREAM_WHOLE; }     /* at any alignment */
    uint64_t copy_bytes() const { return streams() ? 0 : a.copy_bytes + b.copy_bytes; }
};

inline uint32_t tiles_of(uint64_t n, uint32_t t) { return (uint32_t)((n + t - 1) / t); }
inline uint64_t tile_count(const Shape& s, uint32_t bm, uint32_t bn) {
    uint64_t m = tiles_of(s.M, bm);
    if (s.group == GROUP_ROWS) m += std::min(s.experts, s.M);               /* each group may end inside a tile */
    return m * tiles_of(s.N, bn) * (s.group == GROUP_K ? s.experts : 1);
}

/* Queues one or two products with what goes before and behind them (linear_16.h), for one element type each. */
int run_bf16(Product* q, int n, int tile, const SlopeArgs* slope, const BiasJoin* bias, char* ws, hipStream_t st);
int run_f16(Product* q, int n, int tile, const SlopeArgs* slope, const BiasJoin* bias, char* ws, hipStream_t st);

}  // namespace linear

#ifdef __HIPCC__
namespace linear {

using namespace layer;

typedef int v4i_t __attribute__((ext_vector_type(4)));
typedef short v4s_t __attribute__((ext_vector_type(4)));
typedef float v4f_t __attribute__((ext_vector_type(4)));
typedef float v16f_t __attribute__((ext_vector_type(16)));
typedef _Float16 v8h_t __attribute__((ext_vector_type(8)));
typedef __bf16 v8b_t __attribute__((ext_vector_type(8)));

template <bool BF16> struct Half16 { typedef _Float16 T; };
template <> struct Half16<true> { typedef __bf16 T; };

/* e^x through the hardware's 2^x: relative error (|x| + 1) 2^-23 */
__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896341f); }

__device__ __forceinline__ float tanh_of(float z) {
    const float a = fabsf(z);
    /* below 1/4 the series to z^9 (next term below 2^-25 of z); above, no cancellation: 1 - 2 / (e^2a + 1) */
    const float s = z * z;
    float p = fmaf(s, 62.0f / 2835.0f, -17.0f / 315.0f);
    p = fmaf(p, s, 2.0f / 15.0f);
    p = fmaf(p, s, -1.0f / 3.0f);
    const float small = fmaf(z * s, p, z);
    const float big = fmaf(-2.0f, __builtin_amdgcn_rcpf(exp_of(2.0f * a) + 1.0f), 1.0f);
    return a < 0.25f ? small : __builtin_copysignf(big, z);
}
/* 1 - tanh^2 z = 4 e / (1 + e)^2, e = exp(-2 |z|): no difference, so a saturated unit's derivative keeps its digits (as 1 - t^2
 * it is 4e-4 off at |z| = 5, 6e-2 at 8 and 0 from 9 on, where it is 6e-8). Relative error (4 |z| + 11) 2^-24. */
__device__ __forceinline__ float tanh_slope_of(float z) {
    const float e = exp_of(-2.0f * fabsf(z)), r = __builtin_amdgcn_rcpf(1.0f + e);
    return 4.0f * e * r * r;
}
__device__ __forceinline__ float sigmoid_of(float z) { return __builtin_amdgcn_rcpf(1.0f + exp_of(-z)); }

/* z no further out than +-most, where the functions below have long reached their limits, so that an infinity gives
 * the limit and not infinity times 0; NaN stays NaN */
__device__ __forceinline__ float within(float z, float most) { return fabsf(z) > most ? __builtin_copysignf(most, z) : z; }

/* Phi(-a) / phi(a) / sqrt(2 pi) for 0 <= a <= 14 (Phi the normal distribution's integral, phi its density; Phi leaves the range of
 * fp32 at 13.5): t (c1 + c2 t + ... + c8 t^7), t = 1 / (1 + p a). p and the coefficients were fitted for the least relative error,
 * 8.4e-8 over 0 .. 13.5; evaluated in fp32 4e-7. */
__device__ __forceinline__ float normal_ratio(float a) {
    const float t = __builtin_amdgcn_rcpf(fmaf(a, 0.30401892054236973f, 1.0f));
    float p = 0.036861336417387855f;
    p = fmaf(p, t, -0.1552789393030083f);
    p = fmaf(p, t, 0.19210584912500997f);
    p = fmaf(p, t, -0.04306761068848061f);
    p = fmaf(p, t, 0.12352392127006696f);
    p = fmaf(p, t, 0.10243598088911153f);
    p = fmaf(p, t, 0.12217721613835655f);
    return t * fmaf(p, t, 0.12124228790163077f);
}
/* exp(-a^2 / 2): the exponent's two roundings make a relative error of up to a^2 2^-24 */
__device__ __forceinline__ float normal_exp(float a) { return __builtin_amdgcn_exp2f(a * a * -0.72134752044448170f); }

/* z Phi(z) = max(z, 0) - |z| Phi(-|z|), relative error 5e-7 for |z| below 2, 7e-7 below 4. Six coefficients (3.7e-6, 9e-6 at |z| = 11)
 * put one f16 value in 430 on the wrong side of a rounding and gained little: 8192^3 914-917 us and with these 919, the
 * experts' 16384 rows x 1024 x 4096 244-246 and 246. */
__device__ __forceinline__ float gelu_of(float z) {
    const float a = fabsf(z) > 14.0f ? 14.0f : fabsf(z);
    return fmaf(-a, normal_ratio(a) * normal_exp(a), fmaxf(z, 0.0f));
}

/* Phi(z) + z phi(z), the derivative of z Phi(z): with d = phi(a) (R(a) - a), R = Phi(-a) / phi(a), a = |z|, it is d below
 * zero and 1 - d above, one exponential for both terms */
__device__ __forceinline__ float gelu_slope_of(float z) {
    const float a = fabsf(z) > 14.0f ? 14.0f : fabsf(z);
    const float d = normal_exp(a) * fmaf(a, -0.39894228040143268f, normal_ratio(a));
    return z < 0.0f ? d : 1.0f - d;
}

/* eight activations: the choice is made once for all of them */
__device__ __forceinline__ void act8(float (&v)[8], int act) {
#define EACH(expr) do { _Pragma("unroll") for (int i = 0; i < 8; i++) { const float z = v[i]; v[i] = (expr); } } while (0)
    switch (act) {
    case HIP_ACT_TANH: EACH(tanh_of(z)); break;
    case HIP_ACT_RELU: EACH(z < 0.0f ? 0.0f : z); break;        /* NaN stays NaN */
    case HIP_ACT_GELU: EACH(gelu_of(z)); break;
    case HIP_ACT_SILU: EACH((z < -100.0f ? -100.0f : z) * sigmoid_of(z)); break;
    default: break;
    }
}
/* d times the derivatives at z */
__device__ __forceinline__ void slope8(float (&d)[8], const float (&v)[8], int act) {
#define SLOPE(expr) do { _Pragma("unroll") for (int i = 0; i < 8; i++) { const float z = v[i]; d[i] *= (expr); } } while (0)
    switch (act) {
    case HIP_ACT_TANH: SLOPE(tanh_slope_of(z)); break;
    case HIP_ACT_RELU: SLOPE(z > 0.0f ? 1.0f : (z != z ? z : 0.0f)); break;
    case HIP_ACT_GELU: SLOPE(gelu_slope_of(z)); break;
    case HIP_ACT_SILU: SLOPE(({ const float c = within(z, 100.0f), s = sigmoid_of(c); s * fmaf(c, 1.0f - s, 1.0f); })); break;
    default: break;
    }
#undef SLOPE
#undef EACH
}

/* the group of an expert, inside 0 .. rows whatever the offsets hold */
__device__ __forceinline__ void expert_range(const int32_t* offsets, uint32_t e, uint32_t rows, uint32_t* lo, uint32_t* hi) {
    *lo = *hi = 0;
    if (rows == 0) return;                                  /* offsets may be NULL then */
    const int a = offsets[e], b = offsets[e + 1];
    const uint32_t l = a < 0 ? 0u : min((uint32_t)a, rows);
    *lo = l;
    *hi = b < 0 ? l : max(l, min((uint32_t)b, rows));
}

/* eight columns of bias row `expert` from column c on, zeros beyond N */
template <bool BF16>
__device__ __forceinline__ void load_bias(const LinearEpilogue& e, uint32_t expert, uint32_t c, uint32_t N, float (&out)[8]) {
    typedef typename Half16<BF16>::T E;
    if (!e.bias) {
#pragma unroll
        for (int i = 0; i < 8; i++) out[i] = 0.0f;
    } else if (e.bias_wide) load_row<float, float, 8>((const float*)e.bias + (uint64_t)expert * N, c, N, out);
    else load_row<E, float, 8>((const E*)e.bias + (uint64_t)expert * N, c, N, out);
}

/* z = v + bias, pre = z, y = act(z) + residual for columns c .. c + 7 of a row; y_at is the output matrix's
 * first element (its expert's, where C is one per expert). STREAM: stores that do not displace what the L2 holds (the
 * operands other tiles are about to read): 113 -> 104 us for an expert layer's two gradients, 8191 x 1024 x 2048 */
template <bool BF16, bool STREAM = false>
__device__ __forceinline__ void finish_row8(const LinearEpilogue& e, void* y_at, uint64_t row, uint32_t c, uint32_t N,
                                            float (&v)[8], const float (&bias)[8]) {
    typedef typename Half16<BF16>::T E;
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] += bias[i];
    if (e.pre) store_row<E, float, 8, STREAM>((E*)e.pre + row * e.ld_pre, c, N, v);
    act8(v, e.act);
    if (e.residual) {
        float r[8];
        load_row<E, float, 8>((const E*)e.residual + row * e.ld_res, c, N, r);
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] += r[i];
    }
    if (e.out32) store_row<float, float, 8, STREAM>((float*)y_at + row * e.ldy, c, N, v);
    else store_row<E, float, 8, STREAM>((E*)y_at + row * e.ldy, c, N, v);
}

}  // namespace linear
#endif
#endif
