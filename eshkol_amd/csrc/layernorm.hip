/*
 * Layer norm and its gradients (gpu_hip_layers.h).
 *
 * Forward: y = (x - mean) rstd gamma + beta, from the row held in registers: one
 * pass over memory, and no difference of two large sums. A first mean m is the sum
 * over n; the second sweep adds up the deviations from it and their squares,
 *   s = sum (x - m),  q = sum (x - m)^2;  mean = m + s / n,  variance = q / n - (s / n)^2,
 * so m's own rounding drops out: without it a row of one value 1000 and 1000 columns
 * had a mean 6e-5 off, which 1 / sqrt(epsilon) made -0.02 of the output's 0. It costs
 * 0.1 us of one row of 4096 (3.55 -> 3.64) and 1 of 32768 (121.7 -> 122.7).
 *
 * Backward, with h = (x - mean) rstd and t = grad_y gamma:
 *   grad_x = rstd (t - sum t / n - h sum (t h) / n) [+ grad_residual]
 * a row at a time in registers, while every thread adds grad_y h and grad_y of
 * its own columns over the rows its workgroup walks; the workgroups' sums meet in
 * a second launch, in ascending order.
 *
 * Bound by memory: every value is read once and written once. 32768 x 4096 bf16,
 * with a device copy's 5.1 TB/s as the floor: forward 122 us (4.4 TB/s, floor 105; f32
 * 223, floor 211; 16384 x 4096 f64 202, floor 211),
 * backward with the residual's gradient 224 us (4.8 TB/s, floor 210; 7 of them the
 * second launch). 4095 x 1023 fp32 backward 19.5 us (floor 10): two rows per wave,
 * so the launches and the first trip to memory are half of it. One row of 4096: 3.6
 * us on the device.
 */
#include "layer_common.h"

#include <algorithm>

namespace {

using namespace layer;

struct NormArgs {
    const void *x, *gamma, *beta;
    void *y, *mean, *rstd;
    uint64_t rows, ldx, ldy;
    uint32_t cols;
    int wide;                       /* parameters are fp32 */
    double epsilon;
};

/* the sum over the T threads that share a row, through row `at` of the scratch; sums
 * that follow each other take different rows, so that one barrier per sum is enough */
template <int T, class Acc>
__device__ __forceinline__ Acc team_sum(Acc v, Acc (*scratch)[T / 64 > 0 ? T / 64 : 1], int at) {
    v = wave_sum(v);
    if constexpr (T > 64) {
        constexpr int W = T / 64;
        if ((threadIdx.x & 63) == 0) scratch[at][threadIdx.x >> 6] = v;
        __syncthreads();
        v = scratch[at][0];
#pragma unroll
        for (int w = 1; w < W; w++) v += scratch[at][w];
    }
    return v;
}

/* two sums behind one barrier, through the rows behind the first */
template <int T, class Acc>
__device__ __forceinline__ void team_sum2(Acc& u, Acc& v, Acc (*scratch)[T / 64 > 0 ? T / 64 : 1]) {
    u = wave_sum(u);
    v = wave_sum(v);
    if constexpr (T > 64) {
        constexpr int W = T / 64;
        if ((threadIdx.x & 63) == 0) { scratch[1][threadIdx.x >> 6] = u; scratch[2][threadIdx.x >> 6] = v; }
        __syncthreads();
        u = scratch[1][0];
        v = scratch[2][0];
#pragma unroll
        for (int w = 1; w < W; w++) { u += scratch[1][w]; v += scratch[2][w]; }
    }
}
/* The mean and 1 / sqrt(variance + epsilon) of a row from its first mean m and the sums s and q of the deviations from it
 * and of their squares. A mean that is no finite number (a row with an infinity or NaN, or a sum out of range) stays m. */
template <class Acc>
__device__ __forceinline__ void moments(Acc m, Acc s, Acc q, Acc inv_n, Acc epsilon, Acc* mean, Acc* rstd) {
    const Acc c = s * inv_n, v = fma_of(-c, c, q * inv_n);
    *mean = c - c == 0 ? m + c : m;
    *rstd = (Acc)1 / (Acc)sqrt((v < 0 ? (Acc)0 : v) + epsilon);
}

/* Sixteen bytes of a row, kept as four words: a vector of 16-bit elements that lives across a branch is taken apart into a
 * register for each element. */
typedef int words_t __attribute__((ext_vector_type(4)));
template <class E> __device__ __forceinline__ typename Vec16<E>::type elements(words_t w) { return __builtin_bit_cast(typename Vec16<E>::type, w); }
/* element e, widened */
template <class E> __device__ __forceinline__ auto wide_of(words_t w, int e) {
    if constexpr (sizeof(E) == 8) return (double)elements<E>(w)[e];
    else if constexpr (__is_same(E, __bf16)) return __int_as_float((e & 1) ? (w[e >> 1] & (int)0xffff0000) : (w[e >> 1] << 16));
    else return (float)elements<E>(w)[e];
}

/* One 16-byte vector of a row from element c on, zeros behind the row's end. EVEN: rows are whole vectors. */
template <class E, bool EVEN>
__device__ __forceinline__ words_t load_vec(const E* row, uint32_t c, uint32_t n) {
    typedef int unaligned __attribute__((ext_vector_type(4), aligned(2)));     /* global memory takes it at any address */
    constexpr int N = Vec16<E>::N;
    words_t v = {0, 0, 0, 0};
    if (EVEN ? c < n : c + N <= n) v = *(const unaligned*)(row + c);
    else if (!EVEN && c < n) {
        typename Vec16<E>::type part = {};
#pragma unroll
        for (int e = 0; e < N; e++) if (c + e < n) part[e] = row[c + e];
        v = __builtin_bit_cast(words_t, part);
    }
    return v;
}
/* Makes the compiler take a vector's values as new ones: it would otherwise keep the widened copies of one sweep for the
 * next, in twice the registers. It also keeps the loads behind it (the parameters of this vector) from being moved up in
 * front of the sweep, all of a row's at once. */
__device__ __forceinline__ void renew(words_t& w) { asm volatile("" : "+v"(w) :: "memory"); }
/* A thread's place in its row, as a value of this turn of the loop: the addresses of every vector and parameter would
 * otherwise be computed once and kept, in more registers than the row itself. */
__device__ __forceinline__ int position(int t) { asm volatile("" : "+v"(t)); return t; }

template <class E, class Acc, bool EVEN>
__device__ __forceinline__ void store_vec(E* row, uint32_t c, uint32_t n, const Acc (&in)[Vec16<E>::N]) {
    if constexpr (EVEN) {
        typedef typename Vec16<E>::type vec;
        vec v;
#pragma unroll
        for (int e = 0; e < Vec16<E>::N; e++) v[e] = (E)in[e];
        if (c < n) *(vec*)(row + c) = v;
    } else store_row<E, Acc, Vec16<E>::N>(row, c, n, in);
}

/* A row is held by T threads, V vectors of 16 bytes each, as it lies in memory: it is widened again for each of the three
 * sweeps, which costs less than the registers of a wide copy (32768 x 4096 bf16: 117 registers and 166 us with one). T = 64: a row
 * per wave, no barrier. The next row is requested before the current one is worked on. */
template <int DT, int T, int V, bool EVEN>
__global__ __launch_bounds__(T < 256 ? 256 : T)
void norm_kernel(NormArgs a) {
    typedef typename Elem<DT>::T E;
    typedef typename Elem<DT>::Acc Acc;
    constexpr int N = Vec16<E>::N;
    constexpr int PER = T < 256 ? 256 / T : 1;              /* rows per workgroup */
    __shared__ Acc scratch[3][T / 64 > 0 ? T / 64 : 1];
    const int t0 = threadIdx.x % T;
    const Acc inv_n = (Acc)1 / (Acc)a.cols;
    const uint64_t step = (uint64_t)gridDim.x * PER;
    uint64_t row = (uint64_t)blockIdx.x * PER + threadIdx.x / T;
    if (row >= a.rows) return;                              /* whole waves; whole workgroups where they share a row */
    words_t x[V];
#pragma unroll
    for (int i = 0; i < V; i++) x[i] = load_vec<E, EVEN>((const E*)a.x + row * a.ldx, (uint32_t)(t0 + i * T) * N, a.cols);
    for (; row < a.rows; row += step) {
        const int t = position(t0);
        words_t next[V];
        const uint64_t ahead = row + step < a.rows ? row + step : row;
#pragma unroll
        for (int i = 0; i < V; i++) next[i] = load_vec<E, EVEN>((const E*)a.x + ahead * a.ldx, (uint32_t)(t + i * T) * N, a.cols);
        Acc s = 0;
#pragma unroll
        for (int i = 0; i < V; i++)
#pragma unroll
            for (int e = 0; e < N; e++) s += wide_of<E>(x[i], e);
        const Acc first = team_sum<T, Acc>(s, scratch, 0) * inv_n;
        Acc q = 0, mean, rstd;
        s = 0;
#pragma unroll
        for (int i = 0; i < V; i++) {
            renew(x[i]);
#pragma unroll
            for (int e = 0; e < N; e++) {
                const uint32_t c = (uint32_t)(t + i * T) * N + (EVEN ? 0 : e);
                const Acc d = c < a.cols ? wide_of<E>(x[i], e) - first : (Acc)0;
                s += d;
                q = fma_of(d, d, q);
            }
        }
        team_sum2<T, Acc>(s, q, scratch);
        moments(first, s, q, inv_n, (Acc)a.epsilon, &mean, &rstd);
        if (t == 0) {
            if (a.mean) ((Acc*)a.mean)[row] = mean;
            if (a.rstd) ((Acc*)a.rstd)[row] = rstd;
        }
        E* yr = (E*)a.y + row * a.ldy;
#pragma unroll
        for (int i = 0; i < V; i++) {
            const uint32_t c = (uint32_t)(t + i * T) * N;
            renew(x[i]);
            if (c < a.cols) {
                Acc g[N], b[N], o[N];
                load_param<E, Acc, N, EVEN>(a.gamma, a.wide, (Acc)1, c, a.cols, g);
                load_param<E, Acc, N, EVEN>(a.beta, a.wide, (Acc)0, c, a.cols, b);
#pragma unroll
                for (int e = 0; e < N; e++) o[e] = fma_of((wide_of<E>(x[i], e) - mean) * rstd, g[e], b[e]);
                store_vec<E, Acc, EVEN>(yr, c, a.cols, o);
            }
            x[i] = next[i];
        }
    }
}

/* Rows too long for the registers of a workgroup: three passes, the last two
 * mostly from the caches. */
template <int DT>
__global__ __launch_bounds__(1024)
void norm_long_kernel(NormArgs a) {
    typedef typename Elem<DT>::T E;
    typedef typename Elem<DT>::Acc Acc;
    constexpr int N = Vec16<E>::N, T = 1024;
    __shared__ Acc scratch[3][T / 64];
    const Acc inv_n = (Acc)1 / (Acc)a.cols;
    for (uint64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const E* xr = (const E*)a.x + row * a.ldx;
        Acc v[N], s = 0;
        for (uint64_t c = threadIdx.x * N; c < a.cols; c += T * N) {
            load_row<E, Acc, N>(xr, (uint32_t)c, a.cols, v);
#pragma unroll
            for (int e = 0; e < N; e++) s += v[e];
        }
        const Acc first = team_sum<T, Acc>(s, scratch, 0) * inv_n;
        Acc q = 0, mean, rstd;
        s = 0;
        for (uint64_t c = threadIdx.x * N; c < a.cols; c += T * N) {
            load_row<E, Acc, N>(xr, (uint32_t)c, a.cols, v);
#pragma unroll
            for (int e = 0; e < N; e++) {
                const Acc d = c + e < a.cols ? v[e] - first : (Acc)0;
                s += d;
                q = fma_of(d, d, q);
            }
        }
        team_sum2<T, Acc>(s, q, scratch);
        moments(first, s, q, inv_n, (Acc)a.epsilon, &mean, &rstd);
        if (threadIdx.x == 0) {
            if (a.mean) ((Acc*)a.mean)[row] = mean;
            if (a.rstd) ((Acc*)a.rstd)[row] = rstd;
        }
        E* yr = (E*)a.y + row * a.ldy;
        for (uint64_t c = threadIdx.x * N; c < a.cols; c += T * N) {
            Acc g[N], b[N];
            load_row<E, Acc, N>(xr, (uint32_t)c, a.cols, v);
            load_param<E, Acc, N>(a.gamma, a.wide, (Acc)1, (uint32_t)c, a.cols, g);
            load_param<E, Acc, N>(a.beta, a.wide, (Acc)0, (uint32_t)c, a.cols, b);
#pragma unroll
            for (int e = 0; e < N; e++) v[e] = fma_of((v[e] - mean) * rstd, g[e], b[e]);
            store_row<E, Acc, N>(yr, (uint32_t)c, a.cols, v);
        }
    }
}

struct NormBackArgs {
    const void *dy, *x, *gamma, *mean, *rstd, *res;
    void *dx, *part;                /* part: [gridDim.x][2][cols] partial sums, or NULL */
    uint64_t rows, ld_dy, ldx, ld_res, ld_dx;
    uint32_t cols;
    int wide;
};

/* T threads per row and V vectors per thread as above, the next row's values requested before the current row is
 * worked on. Each thread adds grad_y h and grad_y of its columns over the rows it sees; with T = 64 the four waves'
 * sums are joined in LDS at the end. */
template <int DT, int T, int V, bool EVEN>
__global__ __launch_bounds__(T < 256 ? 256 : T)
void norm_back_kernel(NormBackArgs a) {
    typedef typename Elem<DT>::T E;
    typedef typename Elem<DT>::Acc Acc;
    constexpr int N = Vec16<E>::N;
    constexpr int PER = T < 256 ? 256 / T : 1;
    constexpr int W = T / 64 > 0 ? T / 64 : 1;
    __shared__ Acc scratch[2][2][W];
    __shared__ Acc join[PER > 1 ? PER : 1][PER > 1 ? T * V * N : 1];
    const int t0 = threadIdx.x % T;
    const Acc inv_n = (Acc)1 / (Acc)a.cols;
    const uint64_t step = (uint64_t)gridDim.x * PER;
    uint64_t row = (uint64_t)blockIdx.x * PER + threadIdx.x / T;
    Acc sg[V][N], sb[V][N];
#pragma unroll
    for (int i = 0; i < V; i++)
#pragma unroll
        for (int e = 0; e < N; e++) sg[i][e] = sb[i][e] = 0;
    words_t x[V], d[V], r[V];
    Acc mean = 0, rstd = 0;
    auto load = [&](int t, uint64_t at, words_t (&xv)[V], words_t (&dv)[V], words_t (&rv)[V], Acc& m, Acc& s) {
        m = ((const Acc*)a.mean)[at];
        s = ((const Acc*)a.rstd)[at];
#pragma unroll
        for (int i = 0; i < V; i++) {
            const uint32_t c = (uint32_t)(t + i * T) * N;
            xv[i] = load_vec<E, EVEN>((const E*)a.x + at * a.ldx, c, a.cols);
            dv[i] = load_vec<E, EVEN>((const E*)a.dy + at * a.ld_dy, c, a.cols);
            if (a.res) rv[i] = load_vec<E, EVEN>((const E*)a.res + at * a.ld_res, c, a.cols);
        }
    };
    if (row < a.rows) load(t0, row, x, d, r, mean, rstd);
    int turn = 0;
    for (; row < a.rows; row += step, turn ^= 1) {
        const int t = position(t0);
        words_t nx[V], nd[V], nr[V];
        Acc nmean, nrstd;
        load(t, row + step < a.rows ? row + step : row, nx, nd, nr, nmean, nrstd);
        Acc sa = 0, sc = 0;
#pragma unroll
        for (int i = 0; i < V; i++) {
            const uint32_t c = (uint32_t)(t + i * T) * N;
            renew(x[i]);
            if (EVEN && c >= a.cols) continue;
            Acc g[N];
            load_param<E, Acc, N, EVEN>(a.gamma, a.wide, (Acc)1, c, a.cols, g);
#pragma unroll
            for (int e = 0; e < N; e++) {
                const Acc dy = wide_of<E>(d[i], e);
                const Acc h = c + (EVEN ? 0 : e) < a.cols ? (wide_of<E>(x[i], e) - mean) * rstd : (Acc)0;
                sg[i][e] = fma_of(dy, h, sg[i][e]);
                sb[i][e] += dy;
                const Acc tt = dy * g[e];
                sa += tt;
                sc = fma_of(tt, h, sc);
            }
        }
        if (a.dx) {
            sa = wave_sum(sa);
            sc = wave_sum(sc);
            if constexpr (T > 64) {
                if ((threadIdx.x & 63) == 0) { scratch[turn][0][threadIdx.x >> 6] = sa; scratch[turn][1][threadIdx.x >> 6] = sc; }
                __syncthreads();
                sa = scratch[turn][0][0];
                sc = scratch[turn][1][0];
#pragma unroll
                for (int w = 1; w < W; w++) { sa += scratch[turn][0][w]; sc += scratch[turn][1][w]; }
            }
            sa *= inv_n;
            sc *= inv_n;
            E* xo = (E*)a.dx + row * a.ld_dx;
#pragma unroll
            for (int i = 0; i < V; i++) {
                const uint32_t c = (uint32_t)(t + i * T) * N;
                renew(x[i]);
                renew(d[i]);
                if (c >= a.cols) continue;
                Acc g[N], o[N];
                load_param<E, Acc, N, EVEN>(a.gamma, a.wide, (Acc)1, c, a.cols, g);
#pragma unroll
                for (int e = 0; e < N; e++) {
                    const Acc h = (wide_of<E>(x[i], e) - mean) * rstd;
                    o[e] = fma_of(rstd, wide_of<E>(d[i], e) * g[e] - fma_of(h, sc, sa), a.res ? wide_of<E>(r[i], e) : (Acc)0);
                }
                store_vec<E, Acc, EVEN>(xo, c, a.cols, o);
            }
        }
#pragma unroll
        for (int i = 0; i < V; i++) { x[i] = nx[i]; d[i] = nd[i]; if (a.res) r[i] = nr[i]; }
        mean = nmean;
        rstd = nrstd;
    }
    if (!a.part) return;
    Acc* pg = (Acc*)a.part + (uint64_t)blockIdx.x * 2 * a.cols;
    if constexpr (PER == 1) {
#pragma unroll
        for (int i = 0; i < V; i++) {
            const uint32_t c = (uint32_t)(t0 + i * T) * N;
            store_row<Acc, Acc, N>(pg, c, a.cols, sg[i]);
            store_row<Acc, Acc, N>(pg + a.cols, c, a.cols, sb[i]);
        }
    } else {
#pragma unroll
        for (int which = 0; which < 2; which++) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < V; i++)
#pragma unroll
                for (int e = 0; e < N; e++) join[threadIdx.x / T][(t0 + i * T) * N + e] = which ? sb[i][e] : sg[i][e];
            __syncthreads();
            for (uint32_t c = threadIdx.x; c < a.cols; c += 256) {
                Acc s = join[0][c];
#pragma unroll
                for (int w = 1; w < PER; w++) s += join[w][c];
                pg[(uint64_t)which * a.cols + c] = s;
            }
        }
    }
}

/* Rows too long for registers. First the two sums of each row ... */
template <int DT>
__global__ __launch_bounds__(1024)
void norm_back_sums_kernel(NormBackArgs a, typename Elem<DT>::Acc* sums) {
    typedef typename Elem<DT>::T E;
    typedef typename Elem<DT>::Acc Acc;
    constexpr int N = Vec16<E>::N, T = 1024;
    __shared__ Acc scratch[2][T / 64];
    for (uint64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const E* xr = (const E*)a.x + row * a.ldx;
        const E* dr = (const E*)a.dy + row * a.ld_dy;
        const Acc mean = ((const Acc*)a.mean)[row], rstd = ((const Acc*)a.rstd)[row];
        Acc sa = 0, sc = 0;
        for (uint64_t c = threadIdx.x * N; c < a.cols; c += T * N) {
            Acc x[N], d[N], g[N];
            load_row<E, Acc, N>(xr, (uint32_t)c, a.cols, x);
            load_row<E, Acc, N>(dr, (uint32_t)c, a.cols, d);
            load_param<E, Acc, N>(a.gamma, a.wide, (Acc)1, (uint32_t)c, a.cols, g);
#pragma unroll
            for (int e = 0; e < N; e++) {
                if (c + e >= a.cols) continue;
                const Acc tt = d[e] * g[e];
                sa += tt;
                sc = fma_of(tt, (x[e] - mean) * rstd, sc);
            }
        }
        sa = team_sum<T, Acc>(sa, scratch, 0);
        sc = team_sum<T, Acc>(sc, scratch, 1);
        if (threadIdx.x == 0) { sums[2 * row] = sa / (Acc)a.cols; sums[2 * row + 1] = sc / (Acc)a.cols; }
        __syncthreads();
    }
}

/* ... then grad_x and the partial column sums, a workgroup taking 256 vectors of
 * columns (grid y) and every gridDim.x-th row. */
template <int DT>
__global__ __launch_bounds__(256)
void norm_back_long_kernel(NormBackArgs a, const typename Elem<DT>::Acc* sums) {
    typedef typename Elem<DT>::T E;
    typedef typename Elem<DT>::Acc Acc;
    constexpr int N = Vec16<E>::N;
    const uint64_t c64 = ((uint64_t)blockIdx.y * 256 + threadIdx.x) * N;
    if (c64 >= a.cols) return;
    const uint32_t c = (uint32_t)c64;
    Acc g[N], sg[N], sb[N];
    load_param<E, Acc, N>(a.gamma, a.wide, (Acc)1, c, a.cols, g);
#pragma unroll
    for (int e = 0; e < N; e++) sg[e] = sb[e] = 0;
    for (uint64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const Acc mean = ((const Acc*)a.mean)[row], rstd = ((const Acc*)a.rstd)[row];
        Acc x[N], d[N], r[N];
        load_row<E, Acc, N>((const E*)a.x + row * a.ldx, c, a.cols, x);
        load_row<E, Acc, N>((const E*)a.dy + row * a.ld_dy, c, a.cols, d);
#pragma unroll
        for (int e = 0; e < N; e++) r[e] = 0;
        if (a.res) load_row<E, Acc, N>((const E*)a.res + row * a.ld_res, c, a.cols, r);
#pragma unroll
        for (int e = 0; e < N; e++) {
            const Acc h = (x[e] - mean) * rstd;
            sg[e] = fma_of(d[e], h, sg[e]);
            sb[e] += d[e];
            if (a.dx) r[e] = fma_of(rstd, d[e] * g[e] - fma_of(h, sums[2 * row + 1], sums[2 * row]), r[e]);
        }
        if (a.dx) store_row<E, Acc, N>((E*)a.dx + row * a.ld_dx, c, a.cols, r);
    }
    if (!a.part) return;
    Acc* pg = (Acc*)a.part + (uint64_t)blockIdx.x * 2 * a.cols;
    store_row<Acc, Acc, N>(pg, c, a.cols, sg);
    store_row<Acc, Acc, N>(pg + a.cols, c, a.cols, sb);
}

/* grad_gamma[c] and grad_beta[c]: the sums of the n partial rows. A workgroup
 * takes 32 columns of one of the two; 32 threads share a column, each the partial
 * rows s, s + 32, ..., and their sums are added in ascending order. */
template <class Acc>
__global__ __launch_bounds__(1024)
void norm_join_kernel(const Acc* __restrict__ part, uint32_t n, uint32_t cols, Acc* gg, Acc* gb) {
    __shared__ Acc tile[32][33];
    Acc* out = blockIdx.y ? gb : gg;
    if (!out) return;
    const uint32_t c = blockIdx.x * 32 + (threadIdx.x & 31);
    const uint32_t s = threadIdx.x >> 5;
    Acc sum = 0;
    if (c < cols)
#pragma unroll 16
        for (uint32_t p = s; p < n; p += 32) sum += part[((uint64_t)p * 2 + blockIdx.y) * cols + c];
    tile[s][threadIdx.x & 31] = sum;
    __syncthreads();
    if (s == 0 && c < cols) {
#pragma unroll
        for (int k = 1; k < 32; k++) sum += tile[k][threadIdx.x];
        out[c] = sum;
    }
}

/* vectors of 16 bytes in a row of `cols` elements */
uint64_t vectors(uint64_t cols, int dtype) {
    const uint64_t n = 16 / layer_dtype_size(dtype);
    return (cols + n - 1) / n;
}

int check_common(const char* name, uint64_t rows, uint64_t cols, int dtype, int param, const void* gamma) {
    if (dtype < 0 || dtype > 3) LAYER_REFUSE(name, "dtype %d", dtype);
    if (!layer_param_ok(dtype, param)) LAYER_REFUSE(name, "param_dtype %d beside dtype %d", param, dtype);
    if (cols == 0 || cols > (1ull << 24)) LAYER_REFUSE(name, "cols %llu", (unsigned long long)cols);
    if (rows > (1ull << 40)) LAYER_REFUSE(name, "rows %llu", (unsigned long long)rows);
    if (gamma && !layer_aligned(gamma, param)) LAYER_REFUSE(name, "gamma is not aligned to its elements");
    return 0;
}

/* a matrix of a call: there, aligned, with a pitch that holds a row */
int check_matrix(const char* name, const char* what, const void* p, int dtype, uint64_t cols, uint64_t* ld) {
    if (!p) LAYER_REFUSE(name, "%s is NULL", what);
    if (!layer_aligned(p, dtype)) LAYER_REFUSE(name, "%s is not aligned to its elements", what);
    if (*ld == 0) *ld = cols;
    if (*ld < cols || *ld > (1ull << 40)) LAYER_REFUSE(name, "the pitch of %s is %llu, a row has %llu", what, (unsigned long long)*ld, (unsigned long long)cols);
    return 0;
}

int check_norm(const HipLayerNormArgs* u, NormArgs* a) {
    const char* name = "hip_layernorm";
    if (!u) LAYER_REFUSE(name, "no arguments");
    if (check_common(name, u->rows, u->cols, u->dtype, u->param_dtype, u->gamma)) return -1;
    a->ldx = u->ldx;
    a->ldy = u->ldy;
    if (u->rows) {
        if (check_matrix(name, "x", u->x, u->dtype, u->cols, &a->ldx)) return -1;
        if (check_matrix(name, "y", u->y, u->dtype, u->cols, &a->ldy)) return -1;
        if (u->x == u->y && a->ldx != a->ldy) LAYER_REFUSE(name, "y is x with another pitch");
    }
    if (u->beta && !layer_aligned(u->beta, u->param_dtype)) LAYER_REFUSE(name, "beta is not aligned to its elements");
    const int acc = u->dtype == 0 ? 0 : 1;
    if (!layer_aligned(u->mean, acc) || !layer_aligned(u->rstd, acc)) LAYER_REFUSE(name, "mean or rstd is not aligned to its elements");
    if (!(u->epsilon >= 0) || !isfinite(u->epsilon)) LAYER_REFUSE(name, "epsilon %g", u->epsilon);
    a->x = u->x; a->gamma = u->gamma; a->beta = u->beta;
    a->y = u->y; a->mean = u->mean; a->rstd = u->rstd;
    a->rows = u->rows; a->cols = (uint32_t)u->cols;
    a->wide = u->param_dtype == 1 && u->dtype != 1;
    a->epsilon = u->epsilon;
    return 0;
}

template <int DT, int T, int V>
void launch_norm(const NormArgs& a, hipStream_t st) {
    constexpr int PER = T < 256 ? 256 / T : 1;
    const uint64_t most = (uint64_t)eshkol_hip_num_cus() * (T > 256 ? 2 : V >= 8 ? 4 : 8);
    const uint64_t grid = std::min<uint64_t>((a.rows + PER - 1) / PER, most);
    const dim3 g((unsigned)grid), b(T < 256 ? 256 : T);
    if (a.cols % Vec16<typename Elem<DT>::T>::N == 0) hipLaunchKernelGGL((norm_kernel<DT, T, V, true>), g, b, 0, st, a);
    else hipLaunchKernelGGL((norm_kernel<DT, T, V, false>), g, b, 0, st, a);
}

template <int DT>
void dispatch_norm(const NormArgs& a, hipStream_t st) {
    const uint64_t nv = vectors(a.cols, DT);
    /* a row per wave as long as it fits and there are rows enough to fill the device with waves */
    const bool many = a.rows >= 4 * (uint64_t)eshkol_hip_num_cus();
    if (nv <= 64) launch_norm<DT, 64, 1>(a, st);
    else if (nv <= 128) launch_norm<DT, 64, 2>(a, st);
    else if (many && nv <= 256) launch_norm<DT, 64, 4>(a, st);
    else if (many && nv <= 512) launch_norm<DT, 64, 8>(a, st);
    else if (nv <= 256) launch_norm<DT, 256, 1>(a, st);
    else if (nv <= 512) launch_norm<DT, 256, 2>(a, st);
    else if (nv <= 1024) launch_norm<DT, 256, 4>(a, st);
    else if (nv <= 2048) launch_norm<DT, 256, 8>(a, st);
    else if (nv <= 4096) launch_norm<DT, 1024, 4>(a, st);
    else {
        const uint64_t grid = std::min<uint64_t>(a.rows, (uint64_t)eshkol_hip_num_cus() * 4);
        hipLaunchKernelGGL((norm_long_kernel<DT>), dim3((unsigned)grid), dim3(1024), 0, st, a);
    }
}

/* How the backward pass is cut: the threads and vectors of a row, the workgroups
 * that walk the rows (each leaves one partial row of either sum), and where the
 * workspace's parts lie. threads == 0: the path for long rows. */
struct NormBackPlan {
    int threads, per;
    uint64_t grid;
    uint64_t sums_bytes, part_bytes;
};

NormBackPlan plan_back(uint64_t rows, uint64_t cols, int dtype, bool want_params) {
    NormBackPlan p;
    const uint64_t nv = vectors(cols, dtype), acc = dtype == 0 ? 8 : 4;
    /* a row per wave while the sums of its columns (twice V vectors, widened) leave registers for three waves */
    p.threads = nv <= (dtype >= 2 ? 128 : 256) ? 64 : nv <= 1024 ? 256 : nv <= 2048 ? 1024 : 0;
    p.per = p.threads == 64 ? 4 : 1;
    const uint64_t cus = (uint64_t)eshkol_hip_num_cus();
    uint64_t most = p.threads == 1024 ? cus : 4 * cus;
    if (p.threads == 0) {
        const uint64_t tiles = (nv + 255) / 256;
        most = std::max<uint64_t>(1, (8 * cus + tiles - 1) / tiles);
    }
    /* two rows at least for every thread's sums, so that the second launch has less to add up than the first to read */
    p.grid = std::min<uint64_t>((rows + 2 * p.per - 1) / (2 * p.per), most);
    p.sums_bytes = p.threads == 0 ? round_up_sz((size_t)(rows * 2 * acc), 256) : 0;
    p.part_bytes = want_params ? p.grid * 2 * cols * acc : 0;
    return p;
}

int check_back(const char* name, const HipLayerNormBackwardArgs* u, NormBackArgs* a) {
    if (!u) LAYER_REFUSE(name, "no arguments");
    if (check_common(name, u->rows, u->cols, u->dtype, u->param_dtype, u->gamma)) return -1;
    if (!u->grad_x && !u->grad_gamma && !u->grad_beta) LAYER_REFUSE(name, "no output is asked for");
    a->ld_dy = u->ld_grad_y; a->ldx = u->ldx; a->ld_res = u->ld_grad_residual; a->ld_dx = u->ld_grad_x;
    const int acc = u->dtype == 0 ? 0 : 1;
    if (u->rows) {
        if (check_matrix(name, "grad_y", u->grad_y, u->dtype, u->cols, &a->ld_dy)) return -1;
        if (check_matrix(name, "x", u->x, u->dtype, u->cols, &a->ldx)) return -1;
        if (u->grad_residual && check_matrix(name, "grad_residual", u->grad_residual, u->dtype, u->cols, &a->ld_res)) return -1;
        if (u->grad_x && check_matrix(name, "grad_x", u->grad_x, u->dtype, u->cols, &a->ld_dx)) return -1;
        if (!u->mean || !u->rstd || !layer_aligned(u->mean, acc) || !layer_aligned(u->rstd, acc)) LAYER_REFUSE(name, "mean or rstd is NULL or not aligned");
        if (u->grad_x && ((u->grad_x == u->grad_y && a->ld_dx != a->ld_dy) || (u->grad_x == u->x && a->ld_dx != a->ldx) ||
                          (u->grad_x == u->grad_residual && a->ld_dx != a->ld_res))) LAYER_REFUSE(name, "grad_x is an input with another pitch");
    }
    if (!layer_aligned(u->grad_gamma, acc) || !layer_aligned(u->grad_beta, acc)) LAYER_REFUSE(name, "grad_gamma or grad_beta is not aligned to its elements");
    if (u->grad_gamma && u->grad_gamma == u->grad_beta) LAYER_REFUSE(name, "grad_gamma is grad_beta");
    a->dy = u->grad_y; a->x = u->x; a->gamma = u->gamma; a->mean = u->mean; a->rstd = u->rstd; a->res = u->grad_residual;
    a->dx = u->grad_x; a->part = nullptr;
    a->rows = u->rows; a->cols = (uint32_t)u->cols;
    a->wide = u->param_dtype == 1 && u->dtype != 1;
    return 0;
}

template <int DT, int T, int V>
void launch_back(const NormBackArgs& a, uint64_t grid, hipStream_t st) {
    const dim3 g((unsigned)grid), b(T < 256 ? 256 : T);
    if (a.cols % Vec16<typename Elem<DT>::T>::N == 0) hipLaunchKernelGGL((norm_back_kernel<DT, T, V, true>), g, b, 0, st, a);
    else hipLaunchKernelGGL((norm_back_kernel<DT, T, V, false>), g, b, 0, st, a);
}

template <int DT>
void dispatch_back(const NormBackArgs& a, const NormBackPlan& p, void* sums, void* gg, void* gb, hipStream_t st) {
    typedef typename Elem<DT>::Acc Acc;
    const uint64_t nv = vectors(a.cols, DT);
    if (a.rows) {
        if (p.threads == 0) {
            const uint64_t g1 = std::min<uint64_t>(a.rows, (uint64_t)eshkol_hip_num_cus() * 4);
            if (a.dx) hipLaunchKernelGGL((norm_back_sums_kernel<DT>), dim3((unsigned)g1), dim3(1024), 0, st, a, (Acc*)sums);
            hipLaunchKernelGGL((norm_back_long_kernel<DT>), dim3((unsigned)p.grid, (unsigned)((nv + 255) / 256)), dim3(256), 0, st, a, (const Acc*)sums);
        } else if (nv <= 64) launch_back<DT, 64, 1>(a, p.grid, st);
        else if (nv <= 128) launch_back<DT, 64, 2>(a, p.grid, st);
        else if (nv <= 256) {
            if constexpr (DT >= 2) launch_back<DT, 256, 1>(a, p.grid, st);
            else launch_back<DT, 64, 4>(a, p.grid, st);
        }
        else if (nv <= 512) launch_back<DT, 256, 2>(a, p.grid, st);
        else if (nv <= 1024) launch_back<DT, 256, 4>(a, p.grid, st);
        else launch_back<DT, 1024, 2>(a, p.grid, st);
    }
    if (gg || gb)
        hipLaunchKernelGGL((norm_join_kernel<Acc>), dim3((unsigned)((a.cols + 31) / 32), 2), dim3(1024), 0, st,
                           (const Acc*)a.part, a.rows ? (uint32_t)p.grid : 0u, a.cols, (Acc*)gg, (Acc*)gb);
}

}  // namespace

extern "C" int hip_layernorm(const HipLayerNormArgs* args, void* stream) {
    NormArgs a;
    if (check_norm(args, &a)) return -1;
    if (a.rows == 0) return 0;
    hipStream_t st = (hipStream_t)stream;
    EshkolStreamDevice on(st);
    if (!on.ok) return -1;
    switch (args->dtype) {
    case 0: dispatch_norm<0>(a, st); break;
    case 1: dispatch_norm<1>(a, st); break;
    case 2: dispatch_norm<2>(a, st); break;
    default: dispatch_norm<3>(a, st); break;
    }
    return ESHKOL_HIP_OK(hipGetLastError()) ? 0 : -1;
}

extern "C" int64_t hip_layernorm_backward_workspace(const HipLayerNormBackwardArgs* args) {
    NormBackArgs a;
    if (check_back("hip_layernorm_backward_workspace", args, &a)) return -1;
    const NormBackPlan p = plan_back(a.rows, a.cols, args->dtype, args->grad_gamma || args->grad_beta);
    return (int64_t)(p.sums_bytes + p.part_bytes);
}

extern "C" int hip_layernorm_backward(const HipLayerNormBackwardArgs* args, void* stream) {
    const char* name = "hip_layernorm_backward";
    NormBackArgs a;
    if (check_back(name, args, &a)) return -1;
    const NormBackPlan p = plan_back(a.rows, a.cols, args->dtype, args->grad_gamma || args->grad_beta);
    const uint64_t need = p.sums_bytes + p.part_bytes;
    if (need && (!args->workspace || ((uintptr_t)args->workspace & 15) || args->workspace_bytes < need)) {
        GPU_LOG("%s: the workspace has to hold %llu bytes, 16-byte aligned", name, (unsigned long long)need);
        return -2;
    }
    if (a.rows == 0 && !args->grad_gamma && !args->grad_beta) return 0;
    if (p.part_bytes) a.part = (char*)args->workspace + p.sums_bytes;
    hipStream_t st = (hipStream_t)stream;
    EshkolStreamDevice on(st);
    if (!on.ok) return -1;
    switch (args->dtype) {
    case 0: dispatch_back<0>(a, p, args->workspace, args->grad_gamma, args->grad_beta, st); break;
    case 1: dispatch_back<1>(a, p, args->workspace, args->grad_gamma, args->grad_beta, st); break;
    case 2: dispatch_back<2>(a, p, args->workspace, args->grad_gamma, args->grad_beta, st); break;
    default: dispatch_back<3>(a, p, args->workspace, args->grad_gamma, args->grad_beta, st); break;
    }
    return ESHKOL_HIP_OK(hipGetLastError()) ? 0 : -1;
}
