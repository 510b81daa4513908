/*
 * The tiled 16-bit product behind the linear layer and the products by expert
 * (gpu_hip_layers.h): C[m][n] = sum_k A(m, k) B(n, k) with fp32 sums on the matrix
 * cores and the layer's epilogue, operands as the caller holds them.
 *
 * Forms. k contiguous in both (grad_x of a layer, and W held [N][K]), k contiguous
 * in A only (forward with W [K][N]), k contiguous in neither (grad_w). Operands go
 * from global memory straight into LDS, 16 bytes a lane (buffer_load ... lds), in
 * blocks of 64 k. An operand with k contiguous lies in LDS as rows of 128 bytes
 * and a fragment is one 16-byte read; one with its rows contiguous lies as 64 rows
 * of k, and ds_read_b64_tr_b16 hands every lane four k of its own row, so no
 * operand is ever transposed in memory. Both layouts are permuted inside a row
 * (16-byte chunks by row / 2 modulo 8, 32-byte units by k modulo 4) so that the
 * lanes served together fall into different banks; a load to LDS writes lanes in
 * order, so it is the global address that is permuted.
 *
 * Edges. Addresses outside an operand are moved to ones inside it; what they bring
 * only reaches outputs that are not stored, except along k, where the fragments of
 * the last block are masked element by element.
 */
#include "linear_args.h"
#include "gemm_pipe2.h"

#include <algorithm>
#include <mutex>

namespace {

using namespace linear;

constexpr int BK = 64;

__device__ __forceinline__ void wait_and_barrier() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

/* One operand of a tile: R rows (m or n) by 64 k, moved by NW waves. */
template <int FORM, int R, int NW> struct Operand {
    static constexpr int BYTES = R * BK * 2;
    static constexpr int CALLS = BYTES / 1024 / NW;
    static constexpr int SLOTS = FORM == ROWS_K ? 8 : R / 8;       /* 16-byte slots in a row of LDS */

    uint32_t voff[CALLS];
    uint64_t base;              /* of the next block to request            */
    uint64_t step;              /* bytes from one block of k to the next   */
    uint32_t ld2, extent;

    /* the element that slot (call, lane) holds: its row and its first k */
    static __device__ __forceinline__ void place(int call, int lane, uint32_t* r, uint32_t* k) {
        const int s = call * 64 + lane;
        const int line = s / SLOTS, at = s % SLOTS;
        if constexpr (FORM == ROWS_K) {
            *r = line;
            *k = (at ^ ((line >> 1) & 7)) * 8;
        } else {
            *k = line;
            *r = ((at >> 1) ^ ((line & 3) * 2)) * 16 + (at & 1) * 8;
        }
    }
    __device__ __forceinline__ uint32_t offset(uint32_t r, uint32_t k) const {
        if constexpr (FORM == ROWS_K) return min(r, extent - 1) * ld2 + k * 2;
        else return k * ld2 + min(r, extent - 8) * 2;
    }
    /* p: the tile's first element at the first k; rows: how many rows (FORM ROWS_K) or readable
     * row elements (K_ROWS, a multiple of 8) lie from there on */
    __device__ __forceinline__ void start(const uint16_t* p, uint64_t ld, uint32_t rows, int wave, int lane) {
        ld2 = (uint32_t)ld * 2;
        extent = rows;
        base = (uint64_t)p;
        step = FORM == ROWS_K ? BK * 2 : (uint64_t)BK * ld * 2;
#pragma unroll
        for (int i = 0; i < CALLS; i++) {
            uint32_t r, k;
            place(wave * CALLS + i, lane, &r, &k);
            voff[i] = offset(r, k);
        }
    }
    /* requests the next block into LDS at `lds`; klen < 64: only so many k are there */
    __device__ __forceinline__ void request(uint32_t lds, int klen, int wave, int lane) {
        const v4i_t rs = pipe2::rsrc_words((const void*)base);
        if (klen >= BK) {
#pragma unroll
            for (int i = 0; i < CALLS; i++)
                pipe2::load_to_lds<0>(lds + (uint32_t)(wave * CALLS + i) * 1024u, rs, voff[i], 0);
        } else {
#pragma unroll
            for (int i = 0; i < CALLS; i++) {
                uint32_t r, k;
                place(wave * CALLS + i, lane, &r, &k);
                pipe2::load_to_lds<0>(lds + (uint32_t)(wave * CALLS + i) * 1024u, rs, offset(r, (int)k < klen ? k : 0), 0);
            }
        }
        base += step;
    }
};

/* The fragments of T 32-row blocks from row `first` of the operand's tile: lane l holds row l % 32, k = 16 s + 8 (l / 32) + 0..7 */
template <int FORM, int R, int T>
struct Fragments {
    uint32_t at[FORM == ROWS_K ? 4 : T];
    __device__ __forceinline__ void start(int first, int lane) {
        if constexpr (FORM == ROWS_K) {
            const int r = first + (lane & 31);
#pragma unroll
            for (int s = 0; s < 4; s++) at[s] = (uint32_t)(r * 128 + (((2 * s + (lane >> 5)) ^ ((r >> 1) & 7)) * 16));
        } else {
            const int k = 8 * (lane >> 5) + ((lane & 15) >> 2);
#pragma unroll
            for (int t = 0; t < T; t++) {
                const int unit = first / 16 + 2 * t + ((lane >> 4) & 1);
                at[t] = (uint32_t)(k * R * 2 + (unit ^ ((k & 3) * 2)) * 32 + (lane & 3) * 8);
            }
        }
    }
    __device__ __forceinline__ v4i_t read(const int8_t* tile, int s, int t) const {
        if constexpr (FORM == ROWS_K) {
            return *(const v4i_t*)(tile + at[s] + t * 32 * 128);
        } else {
            typedef __attribute__((address_space(3))) v4s_t lds_v4s;
            const int8_t* p = tile + at[t] + s * 16 * R * 2;
            const v4s_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)p);
            const v4s_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(p + 4 * R * 2));
            v4i_t f;
            __builtin_memcpy(&f, &lo, 8);
            __builtin_memcpy((char*)&f + 8, &hi, 8);
            return f;
        }
    }
};

/* clears the elements of a fragment from the n-th on */
__device__ __forceinline__ void keep_first(v4i_t& f, int n) {
#pragma unroll
    for (int j = 0; j < 4; j++) f[j] = n >= 2 * j + 2 ? f[j] : n == 2 * j + 1 ? (f[j] & 0xffff) : 0;
}

template <bool BF16>
__device__ __forceinline__ void mfma32(const v4i_t& first, const v4i_t& second, v16f_t& acc) {
    if constexpr (BF16)
        acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8b_t, first), __builtin_bit_cast(v8b_t, second), acc, 0, 0, 0);
    else
        acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h_t, first), __builtin_bit_cast(v8h_t, second), acc, 0, 0, 0);
}

/* A wave's sums on their way out: blocks of 32 rows go through the wave's own LDS as fp32, so that a lane then holds
 * eight consecutive columns of a row and every store is one of 16 bytes, whole lines at a time. */
template <int TN> constexpr int park_pitch() { return TN * 128 + 16; }
template <int TM, int TN> constexpr int park_bytes() { return 32 * park_pitch<TN>(); }

template <bool BF16, int TM, int TN>
__device__ __forceinline__ void finish_tile(const LinearArgs& g, v16f_t (&acc)[TM][TN], int8_t* park, uint32_t row0, uint32_t rows_end, uint32_t col0,
                                            uint32_t expert, uint32_t split, void* y_at) {
    constexpr int PITCH = park_pitch<TN>();
    constexpr int LPR = TN * 4;                         /* lanes a row takes, eight columns each */
    const int lane = threadIdx.x & 63;
    const int li = lane & 31, lh = lane >> 5;
    const uint32_t c = col0 + (uint32_t)(lane % LPR) * 8;
    float bias[8];
    const bool whole = g.splits <= 1;
    if (whole && c < g.N) load_bias<BF16>(g.e, expert, c, g.N, bias);
#pragma unroll
    for (int t = 0; t < TM; t++) {
#pragma unroll
        for (int u = 0; u < TN; u++)
#pragma unroll
            for (int v = 0; v < 4; v++)
                *(v4f_t*)(park + li * PITCH + u * 128 + 32 * v + 16 * lh) = (v4f_t){acc[t][u][4 * v], acc[t][u][4 * v + 1], acc[t][u][4 * v + 2], acc[t][u][4 * v + 3]};
#pragma unroll 1
        for (int i = 0; i < 32 * LPR / 64; i++) {
            const int r = lane / LPR + i * (64 / LPR);
            const v4f_t lo = *(const v4f_t*)(park + r * PITCH + (lane % LPR) * 32);
            const v4f_t hi = *(const v4f_t*)(park + r * PITCH + (lane % LPR) * 32 + 16);
            const uint32_t row = row0 + t * 32 + r;
            if (row >= rows_end || c >= g.N) continue;
            float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
            if (whole) finish_row8<BF16>(g.e, y_at, row, c, g.N, v, bias);
            else store_row<float, float, 8>(g.part + ((uint64_t)split * g.M + row) * g.part_ld, c, g.part_ld, v);
        }
    }
}

/* The tile of a workgroup. XCD x (workgroups x, x + 8, ...) takes a contiguous run of the tiles, and the run walks 8 tile
 * rows at a time, so that what an XCD's CUs read together stays in its L2. */
__device__ __forceinline__ bool pick_tile(uint32_t wg, uint32_t total, uint32_t* L) {
    const uint32_t per = (total + 7) >> 3;
    const uint32_t seq = wg >> 3;
    if (seq >= per) return false;
    *L = (wg & 7) * per + seq;
    return *L < total;
}
__device__ __forceinline__ void walk(uint32_t L, uint32_t tiles_m, uint32_t tiles_n, uint32_t* tm, uint32_t* tn) {
    constexpr uint32_t GM = 8;
    const uint32_t width = GM * tiles_n;
    const uint32_t group = L / width, first = group * GM;
    const uint32_t size = min(GM, tiles_m - first), in = L - group * width;
    *tm = first + in % size;
    *tn = in / size;
}

/* Finds the expert whose tiles hold tile number L; per expert ceil(rows / BM) tile rows of tiles_n tiles. All lanes of a
 * wave work on it together: 64 experts at a time. */
template <int BM>
__device__ __forceinline__ bool find_expert(const LinearArgs& g, uint32_t wg, uint32_t* expert, uint32_t* lo, uint32_t* hi, uint32_t* tm, uint32_t* tn) {
    const int lane = threadIdx.x & 63;
    uint32_t total = 0;
    for (uint32_t e0 = 0; e0 < g.experts; e0 += 64) {
        uint32_t l = 0, h = 0;
        if (e0 + lane < g.experts) expert_range(g.offsets, e0 + lane, g.M, &l, &h);
        total += wave_sum<uint32_t>((h - l + BM - 1) / BM);
    }
    uint32_t L;
    if (!pick_tile(wg, total * g.tiles_n, &L)) return false;
    uint32_t before = 0;
    for (uint32_t e0 = 0; e0 < g.experts; e0 += 64) {
        uint32_t l = 0, h = 0;
        if (e0 + lane < g.experts) expert_range(g.offsets, e0 + lane, g.M, &l, &h);
        const uint32_t mine = (h - l + BM - 1) / BM * g.tiles_n;
        uint32_t upto = mine;                               /* inclusive sum over the lanes */
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const uint32_t o = __shfl_up(upto, off, 64);
            if (lane >= off) upto += o;
        }
        const uint64_t past = __ballot(before + upto > L);
        if (past) {
            const int who = __ffsll((unsigned long long)past) - 1;
            const uint32_t start = before + __shfl(upto - mine, who, 64);
            *expert = e0 + who;
            *lo = __builtin_amdgcn_readfirstlane(__shfl(l, who, 64));
            *hi = __builtin_amdgcn_readfirstlane(__shfl(h, who, 64));
            const uint32_t in = L - start, rows = (*hi - *lo + BM - 1) / BM;
            *tm = __builtin_amdgcn_readfirstlane(in % rows);
            *tn = __builtin_amdgcn_readfirstlane(in / rows);
            *expert = __builtin_amdgcn_readfirstlane(*expert);
            return true;
        }
        before += __shfl(upto, 63, 64);
    }
    return false;
}

template <int FA, int FB, int BM, int BN, int WM, int WN, bool BF16, int GROUP>
__global__ __launch_bounds__(WM * WN * 64)
void linear_tile_kernel(LinearArgs g) {
    constexpr int NW = WM * WN, TM = BM / WM / 32, TN = BN / WN / 32;
    typedef Operand<FA, BM, NW> OpA;
    typedef Operand<FB, BN, NW> OpB;
    constexpr int STAGE = OpA::BYTES + OpB::BYTES;
    extern __shared__ __align__(16) int8_t smem_l[];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

    uint32_t tm, tn, expert = 0, lo = 0, hi = g.M, k_first = 0, k_count = g.K;
    if constexpr (GROUP == GROUP_ROWS) {
        if (!find_expert<BM>(g, blockIdx.x, &expert, &lo, &hi, &tm, &tn)) return;
    } else {
        uint32_t L;
        const uint32_t per = g.tiles_m * g.tiles_n;
        if (!pick_tile(blockIdx.x, per * (GROUP == GROUP_K ? g.experts : 1u), &L)) return;
        if constexpr (GROUP == GROUP_K) {
            expert = L / per;
            L -= expert * per;
            uint32_t kl, kh;
            expert_range(g.offsets, expert, g.K, &kl, &kh);
            k_first = __builtin_amdgcn_readfirstlane(kl);
            k_count = __builtin_amdgcn_readfirstlane(kh - kl);
        }
        walk(L, g.tiles_m, g.tiles_n, &tm, &tn);
    }
    const uint32_t split = blockIdx.y;
    if (g.splits > 1) {
        k_first = split * g.part_k;
        k_count = min(g.part_k, g.K - k_first);
    }
    const uint32_t m0 = lo + tm * BM, n0 = tn * BN;

    OpA A;
    OpB B;
    if constexpr (FA == ROWS_K) A.start(g.a + (uint64_t)m0 * g.lda + k_first, g.lda, hi - m0, wave, lane);
    else A.start(g.a + (uint64_t)k_first * g.lda + m0, g.lda, g.a_extent - m0, wave, lane);
    const uint16_t* b = g.b + (GROUP == GROUP_ROWS ? (uint64_t)expert * g.b_stride : 0);
    if constexpr (FB == ROWS_K) B.start(b + (uint64_t)n0 * g.ldb + k_first, g.ldb, g.N - n0, wave, lane);
    else B.start(b + (uint64_t)k_first * g.ldb + n0, g.ldb, g.b_extent - n0, wave, lane);

    const int wm = wave / WN, wn = wave % WN;
    Fragments<FA, BM, TM> fa;
    Fragments<FB, BN, TN> fb;
    fa.start(wm * TM * 32, lane);
    fb.start(wn * TN * 32, lane);
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) int8_t*)smem_l;

    v16f_t acc[TM][TN];
#pragma unroll
    for (int t = 0; t < TM; t++)
#pragma unroll
        for (int u = 0; u < TN; u++)
#pragma unroll
            for (int r = 0; r < 16; r++) acc[t][u][r] = 0.0f;

    auto request = [&](int stage, int klen) {
        A.request(lds0 + (uint32_t)(stage * STAGE), klen, wave, lane);
        B.request(lds0 + (uint32_t)(stage * STAGE + OpA::BYTES), klen, wave, lane);
    };
    auto multiply = [&](int stage) {
        const int8_t* ta = smem_l + stage * STAGE;
        const int8_t* tb = ta + OpA::BYTES;
#pragma unroll
        for (int s = 0; s < 4; s++) {
            v4i_t a[TM], b[TN];
#pragma unroll
            for (int t = 0; t < TM; t++) a[t] = fa.read(ta, s, t);
#pragma unroll
            for (int u = 0; u < TN; u++) b[u] = fb.read(tb, s, u);
#pragma unroll
            for (int t = 0; t < TM; t++)
#pragma unroll
                for (int u = 0; u < TN; u++) mfma32<BF16>(b[u], a[t], acc[t][u]);
        }
    };
    auto multiply_tail = [&](int stage, int klen) {
        const int8_t* ta = smem_l + stage * STAGE;
        const int8_t* tb = ta + OpA::BYTES;
#pragma unroll
        for (int s = 0; s < 4; s++) {
            if (s * 16 >= klen) break;
            const int n = klen - s * 16 - 8 * (lane >> 5);
            v4i_t a[TM], b[TN];
#pragma unroll
            for (int t = 0; t < TM; t++) { a[t] = fa.read(ta, s, t); keep_first(a[t], n); }
#pragma unroll
            for (int u = 0; u < TN; u++) { b[u] = fb.read(tb, s, u); keep_first(b[u], n); }
#pragma unroll
            for (int t = 0; t < TM; t++)
#pragma unroll
                for (int u = 0; u < TN; u++) mfma32<BF16>(b[u], a[t], acc[t][u]);
        }
    };

    const int nkb = (int)((k_count + BK - 1) / BK);
    if (nkb) {
        request(0, (int)min(k_count, (uint32_t)BK));
        wait_and_barrier();
        int stage = 0;
        for (int kb = 0; kb < nkb - 1; kb++) {
            request(stage ^ 1, (int)min(k_count - (uint32_t)(kb + 1) * BK, (uint32_t)BK));
            multiply(stage);
            wait_and_barrier();
            stage ^= 1;
        }
        const int last = (int)(k_count - (uint32_t)(nkb - 1) * BK);
        if (last == BK) multiply(stage);
        else multiply_tail(stage, last);
        wait_and_barrier();
    }
    int8_t* park = smem_l + wave * park_bytes<TM, TN>();
    void* y_at = g.e.y;
    if constexpr (GROUP == GROUP_K) y_at = g.e.out32 ? (void*)((float*)y_at + expert * g.y_stride) : (void*)((uint16_t*)y_at + expert * g.y_stride);
    finish_tile<BF16, TM, TN>(g, acc, park, m0 + wm * TM * 32, GROUP == GROUP_ROWS ? hi : g.M, n0 + wn * TN * 32, expert, split, y_at);
}

/* ---- a few rows: B streamed once, from memory into the matrix cores ---------------------------------------------
 * C^T = B A^T on 16 x 16 x 32 MFMAs. A wave takes 128 columns and 32 k at a time: a lane loads 8 k of 8 columns, 128
 * bytes. With k contiguous those are the operands; with columns contiguous they are an 8 x 8 block in the lane's own
 * registers, transposed by 32 byte permutes. Position p of the MFMA's rows holds column 8 p + i in product i, so a lane
 * ends with 32 consecutive columns of one row. The four waves of a workgroup take every fourth 32 k of the part of k
 * their workgroup has; LDS joins them, and a second launch joins the parts. */
template <bool BF16>
__device__ __forceinline__ v4f_t mfma16(const v4i_t& first, const v4i_t& second, v4f_t acc) {
    if constexpr (BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8b_t, first), __builtin_bit_cast(v8b_t, second), acc, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h_t, first), __builtin_bit_cast(v8h_t, second), acc, 0, 0, 0);
}

/* eight 16-bit elements c .. c + 7 of a row of n, zeros beyond its end, as four words */
__device__ __forceinline__ v4i_t load8(const uint16_t* row, uint32_t c, uint32_t n) {
    typedef int v4iu_t __attribute__((ext_vector_type(4), aligned(2)));
    if (c + 8 <= n) return *(const v4iu_t*)(row + c);
    v4i_t v;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const uint32_t lo = c + 2 * j < n ? row[c + 2 * j] : 0u, hi = c + 2 * j + 1 < n ? row[c + 2 * j + 1] : 0u;
        v[j] = (int)(lo | (hi << 16));
    }
    return v;
}

template <int FB, int RT, bool BF16, bool GROUPED>
__global__ __launch_bounds__(256)
void linear_thin_kernel(LinearArgs g) {
    __shared__ __align__(16) v4f_t joined[4][8][64];
    const int lane = threadIdx.x & 63, li = lane & 15, lg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t n0 = blockIdx.x * 128, split = blockIdx.y, expert = blockIdx.z;
    uint32_t lo = 0, hi = g.M;
    const uint16_t* B = g.b;
    if constexpr (GROUPED) {
        expert_range(g.offsets, expert, g.M, &lo, &hi);
        lo = __builtin_amdgcn_readfirstlane(lo);
        hi = __builtin_amdgcn_readfirstlane(hi);
        B += (uint64_t)expert * g.b_stride;
    }
    const uint32_t k_first = split * g.part_k, k_end = min(g.K, k_first + g.part_k);
    for (uint32_t r0 = lo; r0 < hi; r0 += 16 * RT) {
        v4f_t acc[8][RT];
#pragma unroll
        for (int i = 0; i < 8; i++)
#pragma unroll
            for (int t = 0; t < RT; t++) acc[i][t] = (v4f_t){0.0f, 0.0f, 0.0f, 0.0f};
        for (uint32_t k0 = k_first + 32 * wave; k0 < k_end; k0 += 128) {
            const uint32_t k = k0 + 8 * lg;
            v4i_t w[8], x[RT], f[8];
            if constexpr (FB == ROWS_K) {
#pragma unroll
                for (int i = 0; i < 8; i++) f[i] = load8(B + (uint64_t)min(n0 + 8 * li + i, g.N - 1) * g.ldb, k, k_end);
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++) w[i] = k + i < k_end ? load8(B + (uint64_t)(k + i) * g.ldb, n0 + 8 * li, g.N) : (v4i_t){0, 0, 0, 0};
            }
#pragma unroll
            for (int t = 0; t < RT; t++) x[t] = load8(g.a + (uint64_t)min(r0 + 16 * t + li, hi - 1) * g.lda, k, k_end);
            if constexpr (FB == K_ROWS) {
#pragma unroll
                for (int i = 0; i < 8; i++)
#pragma unroll
                    for (int p = 0; p < 4; p++)
                        f[i][p] = (int)__builtin_amdgcn_perm((uint32_t)w[2 * p + 1][i / 2], (uint32_t)w[2 * p][i / 2], (i & 1) ? 0x07060302u : 0x05040100u);
            }
#pragma unroll
            for (int i = 0; i < 8; i++)
#pragma unroll
                for (int t = 0; t < RT; t++) acc[i][t] = mfma16<BF16>(f[i], x[t], acc[i][t]);
        }
        /* lane: row lane % 16, columns 32 (lane / 16) + 8 r + i in register r of product i */
#pragma unroll
        for (int t = 0; t < RT; t++) {
            if (t) __syncthreads();
#pragma unroll
            for (int r = 0; r < 4; r++) {
                joined[wave][2 * r][lane] = (v4f_t){acc[0][t][r], acc[1][t][r], acc[2][t][r], acc[3][t][r]};
                joined[wave][2 * r + 1][lane] = (v4f_t){acc[4][t][r], acc[5][t][r], acc[6][t][r], acc[7][t][r]};
            }
            __syncthreads();
            v4f_t lo4 = joined[0][2 * wave][lane], hi4 = joined[0][2 * wave + 1][lane];
#pragma unroll
            for (int o = 1; o < 4; o++) { lo4 += joined[o][2 * wave][lane]; hi4 += joined[o][2 * wave + 1][lane]; }
            const uint32_t row = r0 + 16 * t + li, c = n0 + 32 * lg + 8 * wave;
            if (row < hi && c < g.N) {
                float v[8] = {lo4[0], lo4[1], lo4[2], lo4[3], hi4[0], hi4[1], hi4[2], hi4[3]};
                if (g.splits > 1) store_row<float, float, 8>(g.part + ((uint64_t)split * g.M + row) * g.part_ld, c, g.part_ld, v);
                else {
                    float bias[8];
                    load_bias<BF16>(g.e, expert, c, g.N, bias);
                    finish_row8<BF16>(g.e, g.e.y, row, c, g.N, v, bias);
                }
            }
        }
        __syncthreads();
    }
}

/* The parts of k added in ascending order, and the epilogue: a thread takes eight columns of a row. */
template <bool BF16, bool GROUPED>
__global__ __launch_bounds__(256)
void linear_join_kernel(LinearArgs g) {
    const uint32_t per = g.part_ld / 8;
    const uint64_t id = (uint64_t)blockIdx.x * 256 + threadIdx.x;
    const uint32_t row = (uint32_t)(id / per), c = (uint32_t)(id % per) * 8;
    if (row >= g.M || c >= g.N) return;
    uint32_t expert = 0;
    if constexpr (GROUPED) {
        /* the last expert whose group starts at or before the row; its group may end before it */
        uint32_t a = 0, b = g.experts;
        while (b - a > 1) {
            const uint32_t mid = (a + b) / 2;
            if (g.offsets[mid] <= (int)row) a = mid; else b = mid;
        }
        uint32_t lo, hi;
        expert_range(g.offsets, a, g.M, &lo, &hi);
        if (row < lo || row >= hi) return;
        expert = a;
    }
    float v[8], bias[8];
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = 0.0f;
    for (uint32_t s = 0; s < g.splits; s++) {
        const v4f_t* p = (const v4f_t*)(g.part + ((uint64_t)s * g.M + row) * g.part_ld + c);
        const v4f_t a = p[0], b = p[1];
#pragma unroll
        for (int i = 0; i < 4; i++) { v[i] += a[i]; v[4 + i] += b[i]; }
    }
    load_bias<BF16>(g.e, expert, c, g.N, bias);
    finish_row8<BF16>(g.e, g.e.y, row, c, g.N, v, bias);
}

/* ---- around the products ---------------------------------------------------------------------------------------- */

/* Rows that do not start on 16-byte boundaries, or are no multiple of 16 bytes, copied to ones that do and are (zeros
 * behind their end): `count` matrices of rows x cols. */
__global__ __launch_bounds__(256)
void linear_align_kernel(const uint16_t* __restrict__ in, uint64_t ld, uint64_t stride, uint16_t* __restrict__ out, uint32_t out_ld,
                         uint64_t rows, uint32_t cols, uint64_t chunks) {
    const uint32_t per = out_ld / 8;
    for (uint64_t id = (uint64_t)blockIdx.x * 256 + threadIdx.x; id < chunks; id += (uint64_t)gridDim.x * 256) {
        const uint64_t line = id / per;
        const uint32_t c = (uint32_t)(id % per) * 8;
        const uint64_t matrix = line / rows, row = line - matrix * rows;
        *(v4i_t*)(out + line * out_ld + c) = load8(in + matrix * stride + row * ld, c, cols);
    }
}

/* dz = grad_y act'(pre), and the sums of dz's columns before it is rounded. A workgroup takes 256 columns (32 threads, eight
 * each) of every parts-th run of rows of its expert; its eight rows of threads are joined in LDS. Grid: column blocks, parts, experts. */
struct SlopeArgs {
    const uint16_t *dy, *pre;
    uint16_t* dz;               /* NULL: the sums alone (act 0, or no product wants dz) */
    float* part;                /* [experts][parts][N], or NULL                    */
    uint64_t ld_dy, ld_pre, ld_dz;
    uint32_t rows, N, parts, experts;
    const int32_t* offsets;
    int act;
};
template <bool BF16>
__global__ __launch_bounds__(256)
void linear_slope_kernel(SlopeArgs a) {
    typedef typename Half16<BF16>::T E;
    __shared__ __align__(16) float sums[8][32][9];
    const uint32_t t = threadIdx.x & 31, r = threadIdx.x >> 5;
    const uint32_t c = blockIdx.x * 256 + t * 8, part = blockIdx.y, expert = blockIdx.z;
    uint32_t lo = 0, hi = a.rows;
    if (a.offsets) expert_range(a.offsets, expert, a.rows, &lo, &hi);
    float s[8];
#pragma unroll
    for (int i = 0; i < 8; i++) s[i] = 0.0f;
    if (c < a.N)
        for (uint64_t row = (uint64_t)lo + part * 8 + r; row < hi; row += a.parts * 8) {
            float d[8];
            load_row<E, float, 8>((const E*)a.dy + row * a.ld_dy, c, a.N, d);
            if (a.act) {
                float z[8];
                load_row<E, float, 8>((const E*)a.pre + row * a.ld_pre, c, a.N, z);
#pragma unroll
                for (int i = 0; i < 8; i++) d[i] *= slope_of(z[i], a.act);
            }
            if (a.dz) store_row<E, float, 8>((E*)a.dz + row * a.ld_dz, c, (uint32_t)a.ld_dz, d);
#pragma unroll
            for (int i = 0; i < 8; i++) s[i] += d[i];
        }
    if (!a.part) return;
#pragma unroll
    for (int i = 0; i < 8; i++) sums[r][t][i] = s[i];
    __syncthreads();
    const uint32_t col = blockIdx.x * 256 + threadIdx.x;
    if (col >= a.N) return;
    float sum = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; k++) sum += sums[k][threadIdx.x >> 3][threadIdx.x & 7];
    a.part[((uint64_t)expert * a.parts + part) * a.N + col] = sum;
}

__global__ __launch_bounds__(256)
void linear_bias_join_kernel(const float* __restrict__ part, float* __restrict__ out, uint32_t N, uint32_t parts) {
    const uint32_t c = blockIdx.x * 256 + threadIdx.x;
    if (c >= N) return;
    const float* p = part + (uint64_t)blockIdx.y * parts * N + c;
    float s = 0.0f;
    for (uint32_t k = 0; k < parts; k++) s += p[(uint64_t)k * N];
    out[(uint64_t)blockIdx.y * N + c] = s;
}

/* ---- launches ---------------------------------------------------------------------------------------------------- */

bool lds_ready(const void* kern, int bytes) {
    /* once per kernel and device: attributes belong to the device a kernel runs on */
    static std::mutex m;
    static struct { const void* k; int dev; } done[256];
    static int n = 0;
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess) return false;
    std::lock_guard<std::mutex> lk(m);
    for (int i = 0; i < n; i++) if (done[i].k == kern && done[i].dev == dev) return true;
    if (!ESHKOL_HIP_OK(hipFuncSetAttribute(kern, hipFuncAttributeMaxDynamicSharedMemorySize, bytes))) return false;
    if (n < 256) { done[n].k = kern; done[n].dev = dev; n++; }
    return true;
}

uint32_t tiles_of(uint64_t n, uint32_t t) { return (uint32_t)((n + t - 1) / t); }

/* A matrix operand as the caller gave it, and where it has to be copied to before the tiled kernel may read it. */
struct Matrix {
    const uint16_t* p;
    uint64_t ld, stride, rows, cols, count;
    bool copy;
    uint64_t copy_bytes;
};
Matrix matrix_of(const void* p, uint64_t ld, uint64_t stride, uint64_t rows, uint64_t cols, uint64_t count) {
    Matrix m = {(const uint16_t*)p, ld, stride, rows, cols, count, false, 0};
    m.copy = ((uintptr_t)p & 15) || (ld & 7) || (cols & 7) || (count > 1 && (stride & 7)) || ld > (1u << 22);
    if (m.copy) m.copy_bytes = round_up_sz((size_t)(count * rows * round_up_sz(cols, 8) * 2), 256);
    return m;
}
void align_matrix(Matrix* m, uint16_t* room, hipStream_t st) {
    const uint64_t ld = round_up_sz(m->cols, 8), chunks = m->count * m->rows * (ld / 8);
    const uint64_t grid = std::min<uint64_t>((chunks + 255) / 256, (uint64_t)eshkol_hip_num_cus() * 16);
    if (chunks) hipLaunchKernelGGL(linear_align_kernel, dim3((unsigned)grid), dim3(256), 0, st, m->p, m->ld, m->stride, room, (uint32_t)ld, m->rows, (uint32_t)m->cols, chunks);
    m->p = room;
    m->ld = ld;
    m->stride = m->rows * ld;
    m->cols = ld;
    m->copy = false;
}

/* What a product is: C[M][N] over K; per expert where group says so. */
struct Shape {
    int fa, fb, group;
    uint64_t M, N, K, experts;
};
/* How it is run. */
struct Plan {
    bool thin;
    int rt;
    uint32_t splits, part_k, part_ld;
    uint64_t part_bytes;
};

Plan plan_product(const Shape& s) {
    Plan p = {false, 0, 1, 0, 0, 0};
    const uint64_t cus = (uint64_t)eshkol_hip_num_cus();
    const uint64_t k64 = round_up_sz((size_t)s.K, BK);
    p.part_k = (uint32_t)k64;
    uint64_t splits = 1;
    if (s.fa == ROWS_K && s.group != GROUP_K && (s.group == GROUP_ROWS ? s.M <= 16 * s.experts : s.M <= 64)) {
        p.thin = true;
        const uint64_t rows = s.group == GROUP_ROWS ? (s.M + s.experts - 1) / s.experts : s.M;
        p.rt = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
        const uint64_t have = (uint64_t)tiles_of(s.N, 128) * (s.group == GROUP_ROWS ? std::min(s.experts, s.M) : 1);
        const uint64_t want = (2 * cus + have - 1) / have;
        splits = std::max<uint64_t>(1, std::min<uint64_t>(want, k64 / 128));
    } else if (s.group == GROUP_NONE) {
        const uint64_t have = (uint64_t)tiles_of(s.M, 128) * tiles_of(s.N, 128);
        if (have < cus) splits = std::max<uint64_t>(1, std::min<uint64_t>(cus / have, k64 / 256));
    }
    if (splits > 1) {
        p.part_k = (uint32_t)round_up_sz((size_t)((k64 + splits - 1) / splits), p.thin ? 128 : BK);
        splits = (s.K + p.part_k - 1) / p.part_k;
    }
    if (splits > 1) {
        p.splits = (uint32_t)splits;
        p.part_ld = (uint32_t)round_up_sz((size_t)s.N, 8);
        p.part_bytes = round_up_sz((size_t)(splits * s.M * p.part_ld * 4), 256);
    } else p.part_k = (uint32_t)k64;
    return p;
}

template <int FA, int FB, int BM, int BN, int WM, int WN, bool BF16, int GROUP>
int launch_tile(LinearArgs g, hipStream_t st) {
    constexpr int NW = WM * WN, TM = BM / WM / 32, TN = BN / WN / 32;
    constexpr int SMEM = std::max(2 * (Operand<FA, BM, NW>::BYTES + Operand<FB, BN, NW>::BYTES), NW * park_bytes<TM, TN>());
    auto kern = linear_tile_kernel<FA, FB, BM, BN, WM, WN, BF16, GROUP>;
    if (!lds_ready((const void*)kern, SMEM)) return -1;
    g.tiles_n = tiles_of(g.N, BN);
    g.tiles_m = tiles_of(g.M, BM);
    uint64_t tiles = (uint64_t)g.tiles_m * g.tiles_n;
    if (GROUP == GROUP_ROWS) tiles = ((uint64_t)g.tiles_m + std::min(g.experts, g.M)) * g.tiles_n;      /* each group may end inside a tile */
    if (GROUP == GROUP_K) tiles *= g.experts;
    const uint64_t grid = (tiles + 7) / 8 * 8;
    if (grid > 0x7fffffffULL) return -1;
    hipLaunchKernelGGL(kern, dim3((unsigned)grid, g.splits), dim3(NW * 64), SMEM, st, g);
    return 0;
}

template <bool BF16>
int launch_product(const Shape& s, const Plan& p, LinearArgs g, hipStream_t st) {
    g.M = (uint32_t)s.M; g.N = (uint32_t)s.N; g.K = (uint32_t)s.K;
    g.experts = (uint32_t)s.experts;
    g.splits = p.splits; g.part_k = p.part_k; g.part_ld = p.part_ld;
    const bool rows = s.group == GROUP_ROWS;
    if (p.thin) {
        const dim3 grid(tiles_of(s.N, 128), p.splits, rows ? g.experts : 1);
#define THIN(FB, RT) do { if (rows) hipLaunchKernelGGL((linear_thin_kernel<FB, RT, BF16, true>), grid, dim3(256), 0, st, g); \
                          else hipLaunchKernelGGL((linear_thin_kernel<FB, RT, BF16, false>), grid, dim3(256), 0, st, g); } while (0)
        if (s.fb == ROWS_K) { if (p.rt == 1) THIN(ROWS_K, 1); else if (p.rt == 2) THIN(ROWS_K, 2); else THIN(ROWS_K, 4); }
        else { if (p.rt == 1) THIN(K_ROWS, 1); else if (p.rt == 2) THIN(K_ROWS, 2); else THIN(K_ROWS, 4); }
#undef THIN
    } else {
        int rc;
        if (s.fa == K_ROWS) rc = s.group == GROUP_K ? launch_tile<K_ROWS, K_ROWS, 128, 128, 2, 2, BF16, GROUP_K>(g, st)
                                                    : launch_tile<K_ROWS, K_ROWS, 128, 128, 2, 2, BF16, GROUP_NONE>(g, st);
        else if (s.fb == ROWS_K) rc = rows ? launch_tile<ROWS_K, ROWS_K, 128, 128, 2, 2, BF16, GROUP_ROWS>(g, st)
                                           : launch_tile<ROWS_K, ROWS_K, 128, 128, 2, 2, BF16, GROUP_NONE>(g, st);
        else rc = rows ? launch_tile<ROWS_K, K_ROWS, 128, 128, 2, 2, BF16, GROUP_ROWS>(g, st)
                       : launch_tile<ROWS_K, K_ROWS, 128, 128, 2, 2, BF16, GROUP_NONE>(g, st);
        if (rc) return rc;
    }
    if (p.splits > 1) {
        const uint64_t grid = (s.M * (p.part_ld / 8) + 255) / 256;
        if (grid > 0x7fffffffULL) return -1;
        if (rows) hipLaunchKernelGGL((linear_join_kernel<BF16, true>), dim3((unsigned)grid), dim3(256), 0, st, g);
        else hipLaunchKernelGGL((linear_join_kernel<BF16, false>), dim3((unsigned)grid), dim3(256), 0, st, g);
    }
    return 0;
}

/* Runs a product whose operands may have to be copied first: room for that and for the parts comes from *ws. */
struct Product {
    Shape s;
    Plan p;
    Matrix a, b;
    LinearArgs g;
    uint64_t bytes() const { return p.part_bytes + (p.thin ? 0 : a.copy_bytes + b.copy_bytes); }
};

Product make_product(const Shape& s, const Matrix& a, const Matrix& b) {
    Product q;
    q.s = s;
    q.p = plan_product(s);
    q.a = a;
    q.b = b;
    q.g = LinearArgs();
    return q;
}

int run_product(Product q, char* ws, bool bf16, hipStream_t st) {
    q.g.part = (float*)ws;
    ws += q.p.part_bytes;
    if (!q.p.thin) {
        if (q.a.copy) { const uint64_t n = q.a.copy_bytes; align_matrix(&q.a, (uint16_t*)ws, st); ws += n; }
        if (q.b.copy) { const uint64_t n = q.b.copy_bytes; align_matrix(&q.b, (uint16_t*)ws, st); ws += n; }
    }
    q.g.a = q.a.p; q.g.lda = q.a.ld;
    q.g.b = q.b.p; q.g.ldb = q.b.ld;
    q.g.b_stride = q.b.stride;
    q.g.a_extent = (uint32_t)q.a.cols;
    q.g.b_extent = (uint32_t)q.b.cols;
    return bf16 ? launch_product<true>(q.s, q.p, q.g, st) : launch_product<false>(q.s, q.p, q.g, st);
}

/* ---- checks -------------------------------------------------------------------------------------------------------- */

constexpr uint64_t MAX_KN = 1ull << 22;

int check_16(const char* name, const char* what, const void* p, int dtype, uint64_t cols, uint64_t* ld) {
    if (!p) LAYER_REFUSE(name, "%s is NULL", what);
    if (!layer_aligned(p, dtype)) LAYER_REFUSE(name, "%s is not aligned to its elements", what);
    if (*ld == 0) *ld = cols;
    if (*ld < cols || *ld > (1ull << 32)) LAYER_REFUSE(name, "the pitch of %s is %llu, a row has %llu", what, (unsigned long long)*ld, (unsigned long long)cols);
    return 0;
}
int check_sizes(const char* name, uint64_t rows, uint64_t K, uint64_t N, int dtype, int act, uint64_t experts, bool grouped) {
    if (dtype != 2 && dtype != 3) LAYER_REFUSE(name, "dtype %d is not a 16-bit type", dtype);
    if (act < 0 || act > HIP_ACT_SILU) LAYER_REFUSE(name, "act %d", act);
    if (rows > 0x7fffffffULL) LAYER_REFUSE(name, "%llu rows", (unsigned long long)rows);
    if (K == 0 || N == 0 || K > MAX_KN || N > MAX_KN) LAYER_REFUSE(name, "K %llu, N %llu", (unsigned long long)K, (unsigned long long)N);
    if (grouped && (experts == 0 || experts > 4096)) LAYER_REFUSE(name, "%llu experts", (unsigned long long)experts);
    return 0;
}
int check_stride(const char* name, const char* what, uint64_t rows, uint64_t ld, uint64_t cols, uint64_t* stride) {
    if (*stride == 0) *stride = rows * ld;
    if (*stride < (rows - 1) * ld + cols || *stride > (1ull << 48)) LAYER_REFUSE(name, "%s is %llu", what, (unsigned long long)*stride);
    return 0;
}
int check_room(const char* name, const void* ws, uint64_t have, uint64_t need) {
    if (!need) return 0;
    if (ws && !((uintptr_t)ws & 15) && have >= need) return 0;
    GPU_LOG("%s: the workspace has to hold %llu bytes, 16-byte aligned", name, (unsigned long long)need);
    return -2;
}

/* ---- forward -------------------------------------------------------------------------------------------------------- */

struct ForwardCall {
    Product q;
    bool none;                  /* no rows */
};

/* HipLinearArgs and HipExpertsArgs as one: a linear layer is one expert without offsets */
int plan_forward(const char* name, HipExpertsArgs u, const void* residual, uint64_t ld_res, bool grouped, ForwardCall* f) {
    if (check_sizes(name, u.rows, u.K, u.N, u.dtype, u.act, u.experts, grouped)) return -1;
    if (!layer_param_ok(u.dtype, u.param_dtype)) LAYER_REFUSE(name, "param_dtype %d beside dtype %d", u.param_dtype, u.dtype);
    const uint64_t wr = u.trans_w ? u.N : u.K, wc = u.trans_w ? u.K : u.N;
    if (u.bias && !layer_aligned(u.bias, u.param_dtype)) LAYER_REFUSE(name, "bias is not aligned to its elements");
    f->none = u.rows == 0;
    if (f->none) return 0;
    if (check_16(name, "x", u.x, u.dtype, u.K, &u.ldx) || check_16(name, "w", u.w, u.dtype, wc, &u.ldw) || check_16(name, "y", u.y, u.dtype, u.N, &u.ldy)) return -1;
    if (u.pre && check_16(name, "pre", u.pre, u.dtype, u.N, &u.ld_pre)) return -1;
    if (residual && check_16(name, "residual", residual, u.dtype, u.N, &ld_res)) return -1;
    if (grouped && check_stride(name, "w_stride", wr, u.ldw, wc, &u.w_stride)) return -1;
    if (grouped && (!u.offsets || ((uintptr_t)u.offsets & 3))) LAYER_REFUSE(name, "offsets is NULL or not aligned");
    if (u.y == u.x || u.y == u.w || u.pre == u.y || (u.pre && (u.pre == u.x || u.pre == u.w || u.pre == residual))) LAYER_REFUSE(name, "an output is an input or the other output");
    if (residual && u.y == residual && u.ldy != ld_res) LAYER_REFUSE(name, "y is residual with another pitch");
    const Shape s = {ROWS_K, u.trans_w ? ROWS_K : K_ROWS, grouped ? GROUP_ROWS : GROUP_NONE, u.rows, u.N, u.K, grouped ? u.experts : 1};
    f->q = make_product(s, matrix_of(u.x, u.ldx, 0, u.rows, u.K, 1), matrix_of(u.w, u.ldw, u.w_stride, wr, wc, s.experts));
    LinearEpilogue& e = f->q.g.e;
    e.bias = u.bias; e.bias_wide = u.param_dtype == 1; e.act = u.act;
    e.residual = (const uint16_t*)residual; e.ld_res = ld_res;
    e.y = u.y; e.ldy = u.ldy;
    e.pre = (uint16_t*)u.pre; e.ld_pre = u.ld_pre;
    f->q.g.offsets = grouped ? u.offsets : nullptr;
    return 0;
}
int64_t forward_workspace(const char* name, const HipExpertsArgs& u, const void* residual, uint64_t ld_res, bool grouped) {
    ForwardCall f;
    if (plan_forward(name, u, residual, ld_res, grouped, &f)) return -1;
    return f.none ? 0 : (int64_t)f.q.bytes();
}
int forward(const char* name, const HipExpertsArgs& u, const void* residual, uint64_t ld_res, bool grouped, void* stream) {
    ForwardCall f;
    if (plan_forward(name, u, residual, ld_res, grouped, &f)) return -1;
    if (f.none) return 0;
    if (check_room(name, u.workspace, u.workspace_bytes, f.q.bytes())) return -2;
    hipStream_t st = (hipStream_t)stream;
    EshkolStreamDevice on(st);
    if (!on.ok) return -1;
    if (run_product(f.q, (char*)u.workspace, u.dtype == 3, st)) return -1;
    return ESHKOL_HIP_OK(hipGetLastError()) ? 0 : -1;
}
HipExpertsArgs as_experts(const HipLinearArgs& u) {
    HipExpertsArgs a = {};
    a.x = u.x; a.w = u.w; a.bias = u.bias; a.y = u.y; a.pre = u.pre;
    a.rows = u.M; a.experts = 1; a.K = u.K; a.N = u.N;
    a.ldx = u.ldx; a.ldw = u.ldw; a.ldy = u.ldy; a.ld_pre = u.ld_pre;
    a.dtype = u.dtype; a.param_dtype = u.param_dtype; a.act = u.act; a.trans_w = u.trans_w;
    a.workspace = u.workspace; a.workspace_bytes = u.workspace_bytes;
    return a;
}

/* ---- backward ------------------------------------------------------------------------------------------------------- */

struct BackwardCall {
    bool want_x, want_w, want_b;
    SlopeArgs slope;
    bool run_slope;
    uint64_t dz_bytes, sum_bytes;
    Product x, w;
};

int plan_backward(const char* name, HipExpertsBackwardArgs u, bool grouped, BackwardCall* c) {
    if (check_sizes(name, u.rows, u.K, u.N, u.dtype, u.act, u.experts, grouped)) return -1;
    if (!layer_param_ok(u.dtype, u.grad_w_dtype)) LAYER_REFUSE(name, "grad_w_dtype %d beside dtype %d", u.grad_w_dtype, u.dtype);
    if (!u.grad_x && !u.grad_w && !u.grad_bias) LAYER_REFUSE(name, "no output is asked for");
    const uint64_t wr = u.trans_w ? u.N : u.K, wc = u.trans_w ? u.K : u.N;
    const bool some = u.rows != 0;
    c->want_x = u.grad_x && some;
    c->want_w = u.grad_w != nullptr;
    c->want_b = u.grad_bias != nullptr;
    if (some) {
        if (check_16(name, "grad_y", u.grad_y, u.dtype, u.N, &u.ld_grad_y)) return -1;
        if (u.act && check_16(name, "pre", u.pre, u.dtype, u.N, &u.ld_pre)) return -1;
        if (u.grad_w && check_16(name, "x", u.x, u.dtype, u.K, &u.ldx)) return -1;
        if (u.grad_x && check_16(name, "w", u.w, u.dtype, wc, &u.ldw)) return -1;
        if (u.grad_x && check_16(name, "grad_x", u.grad_x, u.dtype, u.K, &u.ld_grad_x)) return -1;
        if (grouped && u.grad_x && check_stride(name, "w_stride", wr, u.ldw, wc, &u.w_stride)) return -1;
        if (grouped && (!u.offsets || ((uintptr_t)u.offsets & 3))) LAYER_REFUSE(name, "offsets is NULL or not aligned");
    }
    if (u.grad_w && check_16(name, "grad_w", u.grad_w, u.grad_w_dtype, wc, &u.ld_grad_w)) return -1;
    if (grouped && u.grad_w && check_stride(name, "grad_w_stride", wr, u.ld_grad_w, wc, &u.grad_w_stride)) return -1;
    if (!layer_aligned(u.grad_bias, 1)) LAYER_REFUSE(name, "grad_bias is not aligned to its elements");
    const void* outs[3] = {u.grad_x, u.grad_w, u.grad_bias};
    const void* ins[4] = {u.grad_y, u.pre, u.x, u.w};
    for (int i = 0; i < 3; i++) {
        if (!outs[i]) continue;
        for (int j = 0; j < 4; j++) if (outs[i] == ins[j]) LAYER_REFUSE(name, "an output is an input");
        for (int j = 0; j < i; j++) if (outs[i] == outs[j]) LAYER_REFUSE(name, "two outputs are one");
    }

    const uint64_t experts = grouped ? u.experts : 1;
    const bool products = c->want_x || (c->want_w && some);
    const bool make_dz = some && u.act && products;
    c->run_slope = some && (make_dz || c->want_b);
    const uint64_t ld_dz = round_up_sz((size_t)u.N, 8);
    c->dz_bytes = make_dz ? round_up_sz((size_t)(u.rows * ld_dz * 2), 256) : 0;

    /* enough runs of rows to fill the device, none shorter than 32 rows on average */
    const uint64_t blocks = (uint64_t)tiles_of(u.N, 256) * experts, cus = (uint64_t)eshkol_hip_num_cus();
    const uint64_t parts = std::max<uint64_t>(1, std::min<uint64_t>((4 * cus + blocks - 1) / blocks, (u.rows / experts + 31) / 32));
    c->sum_bytes = c->want_b && some ? round_up_sz((size_t)(experts * parts * u.N * 4), 256) : 0;
    SlopeArgs& a = c->slope;
    a.dy = (const uint16_t*)u.grad_y; a.pre = (const uint16_t*)u.pre;
    a.dz = nullptr; a.part = nullptr;
    a.ld_dy = u.ld_grad_y; a.ld_pre = u.ld_pre; a.ld_dz = ld_dz;
    a.rows = (uint32_t)u.rows; a.N = (uint32_t)u.N; a.parts = (uint32_t)parts; a.experts = (uint32_t)experts;
    a.offsets = grouped ? u.offsets : nullptr;
    a.act = u.act;

    /* dz as the products see it: its own room when there is an activation (16-byte aligned rows, N of them read), grad_y itself otherwise */
    const Matrix dz = make_dz ? matrix_of((const void*)(uintptr_t)256, ld_dz, 0, u.rows, ld_dz, 1) : matrix_of(u.grad_y, u.ld_grad_y, 0, u.rows, u.N, 1);
    if (c->want_x) {
        const Shape s = {ROWS_K, u.trans_w ? K_ROWS : ROWS_K, grouped ? GROUP_ROWS : GROUP_NONE, u.rows, u.K, u.N, experts};
        c->x = make_product(s, dz, matrix_of(u.w, u.ldw, u.w_stride, wr, wc, experts));
        c->x.g.e.y = u.grad_x; c->x.g.e.ldy = u.ld_grad_x;
        c->x.g.offsets = a.offsets;
    }
    if (c->want_w) {
        const Shape s = {K_ROWS, K_ROWS, grouped ? GROUP_K : GROUP_NONE, wr, wc, u.rows, experts};
        const Matrix x = matrix_of(u.x, u.ldx, 0, u.rows, u.K, 1);
        c->w = u.trans_w ? make_product(s, dz, x) : make_product(s, x, dz);
        c->w.g.e.y = u.grad_w; c->w.g.e.ldy = u.ld_grad_w; c->w.g.e.out32 = u.grad_w_dtype == 1;
        c->w.g.y_stride = u.grad_w_stride;
        c->w.g.offsets = a.offsets;
    }
    return 0;
}
uint64_t backward_bytes(const BackwardCall& c) {
    /* the two products run one after the other and share their room */
    return c.dz_bytes + c.sum_bytes + std::max(c.want_x ? c.x.bytes() : 0, c.want_w ? c.w.bytes() : 0);
}
int backward(const char* name, const HipExpertsBackwardArgs& u, bool grouped, void* stream) {
    BackwardCall c;
    if (plan_backward(name, u, grouped, &c)) return -1;
    if (check_room(name, u.workspace, u.workspace_bytes, backward_bytes(c))) return -2;
    hipStream_t st = (hipStream_t)stream;
    EshkolStreamDevice on(st);
    if (!on.ok) return -1;
    char* ws = (char*)u.workspace;
    const bool bf16 = u.dtype == 3;
    const uint32_t experts = c.slope.experts;
    if (c.run_slope) {
        if (c.dz_bytes) { c.slope.dz = (uint16_t*)ws; ws += c.dz_bytes; }
        if (c.want_b) { c.slope.part = (float*)ws; ws += c.sum_bytes; }
        const dim3 grid(tiles_of(u.N, 256), c.slope.parts, experts);
        if (bf16) hipLaunchKernelGGL((linear_slope_kernel<true>), grid, dim3(256), 0, st, c.slope);
        else hipLaunchKernelGGL((linear_slope_kernel<false>), grid, dim3(256), 0, st, c.slope);
    }
    if (c.want_b)
        hipLaunchKernelGGL(linear_bias_join_kernel, dim3(tiles_of(u.N, 256), experts), dim3(256), 0, st, c.slope.part, (float*)u.grad_bias, (uint32_t)u.N,
                           c.run_slope ? c.slope.parts : 0u);
    for (int which = 0; which < 2; which++) {
        if (!(which ? c.want_w : c.want_x)) continue;
        Product& q = which ? c.w : c.x;
        if (c.dz_bytes) {
            Matrix& m = which && u.trans_w ? q.a : which ? q.b : q.a;
            m.p = c.slope.dz;
        }
        if (run_product(q, ws, bf16, st)) return -1;
    }
    return ESHKOL_HIP_OK(hipGetLastError()) ? 0 : -1;
}
HipExpertsBackwardArgs as_experts(const HipLinearBackwardArgs& u) {
    HipExpertsBackwardArgs a = {};
    a.grad_y = u.grad_y; a.pre = u.pre; a.x = u.x; a.w = u.w;
    a.grad_x = u.grad_x; a.grad_w = u.grad_w; a.grad_bias = u.grad_bias;
    a.rows = u.M; a.experts = 1; a.K = u.K; a.N = u.N;
    a.ld_grad_y = u.ld_grad_y; a.ld_pre = u.ld_pre; a.ldx = u.ldx; a.ldw = u.ldw; a.ld_grad_x = u.ld_grad_x; a.ld_grad_w = u.ld_grad_w;
    a.dtype = u.dtype; a.grad_w_dtype = u.grad_w_dtype; a.act = u.act; a.trans_w = u.trans_w;
    a.workspace = u.workspace; a.workspace_bytes = u.workspace_bytes;
    return a;
}
int64_t backward_workspace(const char* name, const HipExpertsBackwardArgs& u, bool grouped) {
    BackwardCall c;
    if (plan_backward(name, u, grouped, &c)) return -1;
    return (int64_t)backward_bytes(c);
}

}  // namespace

#define NEED_ARGS(name) if (!args) LAYER_REFUSE(name, "no arguments")

extern "C" int64_t hip_linear_16_workspace(const HipLinearArgs* args) {
    NEED_ARGS("hip_linear_16_workspace");
    return forward_workspace("hip_linear_16_workspace", as_experts(*args), args->residual, args->ld_residual, false);
}
extern "C" int hip_linear_16(const HipLinearArgs* args, void* stream) {
    NEED_ARGS("hip_linear_16");
    return forward("hip_linear_16", as_experts(*args), args->residual, args->ld_residual, false, stream);
}
extern "C" int64_t hip_linear_backward_16_workspace(const HipLinearBackwardArgs* args) {
    NEED_ARGS("hip_linear_backward_16_workspace");
    return backward_workspace("hip_linear_backward_16_workspace", as_experts(*args), false);
}
extern "C" int hip_linear_backward_16(const HipLinearBackwardArgs* args, void* stream) {
    NEED_ARGS("hip_linear_backward_16");
    return backward("hip_linear_backward_16", as_experts(*args), false, stream);
}
extern "C" int64_t hip_experts_16_workspace(const HipExpertsArgs* args) {
    NEED_ARGS("hip_experts_16_workspace");
    return forward_workspace("hip_experts_16_workspace", *args, nullptr, 0, true);
}
extern "C" int hip_experts_16(const HipExpertsArgs* args, void* stream) {
    NEED_ARGS("hip_experts_16");
    return forward("hip_experts_16", *args, nullptr, 0, true, stream);
}
extern "C" int64_t hip_experts_backward_16_workspace(const HipExpertsBackwardArgs* args) {
    NEED_ARGS("hip_experts_backward_16_workspace");
    return backward_workspace("hip_experts_backward_16_workspace", *args, true);
}
extern "C" int hip_experts_backward_16(const HipExpertsBackwardArgs* args, void* stream) {
    NEED_ARGS("hip_experts_backward_16");
    return backward("hip_experts_backward_16", *args, true, stream);
}
