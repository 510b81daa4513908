/*
 * The kernels behind the linear layer and the products by expert (gpu_hip_layers.h):
 * C[m][n] = sum_k A(m, k) B(n, k) of 16-bit operands as the caller holds them, with
 * fp32 sums on the matrix cores and the layer's epilogue; what a backward pass needs
 * before its two products and adds up behind them. Compiled once per element type.
 *
 * Forms. k contiguous in both (grad_x of a layer, and W held [N][K]), k contiguous
 * in A only (forward with W [K][N]), k contiguous in neither (grad_w). Operands go
 * from global memory straight into LDS, 16 bytes a lane (buffer_load ... lds), in
 * blocks of 32 or 64 k. An operand with k contiguous lies in LDS as rows of 64 or
 * 128 bytes and a fragment is one 16-byte read; one with its rows contiguous lies as
 * rows of k, and ds_read_b64_tr_b16 hands every lane four k of its own row, so no
 * operand is ever transposed in memory. Both layouts are permuted inside a row
 * (16-byte chunks by row / 2 modulo 8, or row / 4 modulo 4; 32-byte units by k modulo
 * 4) so that the lanes served together fall into different banks; a load to LDS
 * writes lanes in order, so it is the global address that is permuted. Measured: one
 * LDS cycle in a hundred is a conflict, all of them the epilogue's.
 *
 * What bounds the tiles. 8192^3 with the 256 x 256 tile, no epilogue: 820-860 us
 * (1.28-1.34 PFLOP/s; with bias, gelu and pre 865-920), the matrix pipe busy 67 per cent of the time; without its loads the loop
 * takes 670 us, without its multiplications 680: operand blocks arrive in the L2 from
 * behind it at the rate at which they are multiplied, and what is lost is where the
 * two wait for each other. More blocks in flight (four and five of 32 k) gained
 * nothing (880 us), and lines requested two blocks ahead into the L2 cost more
 * request slots than they saved time (925). Smaller tiles are bound by the same
 * stream sooner: about 55 GB/s per CU of operand blocks, whatever their shape.
 *
 * Edges. Addresses outside an operand are moved to ones inside it; what they bring
 * only reaches outputs that are not stored, except along k, where the fragments of
 * the last block are masked element by element.
 */
#ifndef ESHKOL_HIP_LINEAR_16_H
#define ESHKOL_HIP_LINEAR_16_H

#include "linear_args.h"
#include "gemm_pipe2.h"

#include <algorithm>
#include <mutex>

namespace linear {


using pipe2::IC;
using pipe2::static_for;

/* at most N of the wave's requests still on their way, its LDS reads done, and all waves as far */
template <int N>
__device__ __forceinline__ void wait_and_barrier() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" :: "n"(N) : "memory"); }

/* how the 16-byte chunks of row r of an operand with k contiguous are permuted in LDS */
template <int BK> __device__ __forceinline__ int turn_of(int r) { return BK == 64 ? (r >> 1) & 7 : (r >> 2) & 3; }

/* One operand of a tile: R rows (m or n) by BK k, moved by NW waves. */
template <int FORM, int R, int BK, int NW> struct Operand {
    static constexpr int BYTES = R * BK * 2;
    static constexpr int CALLS = BYTES / 1024 / NW;
    static constexpr int SLOTS = FORM == ROWS_K ? BK / 8 : R / 8;       /* 16-byte slots in a row of LDS */

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
            *k = (at ^ turn_of<BK>(line)) * 8;
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
    /* requests the next block into LDS at `lds`; klen < BK: only so many k are there */
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
    /* the same in pieces, a whole block: point() once, then each of CALLS */
    v4i_t rs;
    __device__ __forceinline__ void point() {
        rs = pipe2::rsrc_words((const void*)base);
        base += step;
    }
    template <int I>
    __device__ __forceinline__ void request_one(IC<I>, uint32_t lds, int wave) {
        pipe2::load_to_lds<0>(lds + (uint32_t)(wave * CALLS + I) * 1024u, rs, voff[I], 0);
    }
};

/* The fragments of T 32-row blocks from row `first` of the operand's tile: lane l holds row l % 32, k = 16 s + 8 (l / 32) + 0..7 */
template <int FORM, int R, int BK, int T>
struct Fragments {
    uint32_t at[FORM == ROWS_K ? BK / 16 : T];
    __device__ __forceinline__ void start(int first, int lane) {
        if constexpr (FORM == ROWS_K) {
            const int r = first + (lane & 31);
#pragma unroll
            for (int s = 0; s < BK / 16; s++) at[s] = (uint32_t)(r * BK * 2 + (((2 * s + (lane >> 5)) ^ turn_of<BK>(r)) * 16));
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
            return *(const v4i_t*)(tile + at[s] + t * 32 * BK * 2);
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
            if (whole) finish_row8<BF16, true>(g.e, y_at, row, c, g.N, v, bias);
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

/* S blocks of k are in LDS or on their way. The multiplications of a k-step (16 of k) are spread out with the next
 * step's LDS reads and the requests between them, in an order the compiler is not to change. The one barrier of a block
 * stands before its last step: behind it every wave holds that step's fragments, so the block's LDS is free for block
 * + S, and the next block, whose first fragments the last step reads, has landed. */
template <int BM_, int BN_, int BK_, int WM_, int WN_, int S_, bool GROUPS_ = false> struct TileShape {
    static constexpr bool GROUPS = GROUPS_;
    static constexpr int BM = BM_, BN = BN_, BK = BK_, WM = WM_, WN = WN_, S = S_;
    static constexpr int THREADS = WM * WN * 64;
    static constexpr int SMEM = S * (BM + BN) * BK * 2 > WM * WN * park_bytes<BM / WM / 32, BN / WN / 32>()
                                    ? S * (BM + BN) * BK * 2 : WM * WN * park_bytes<BM / WM / 32, BN / WN / 32>();
};

template <int FA, int FB, class C, bool BF16, int GROUP>
__device__ __forceinline__ void multiply_tile(const LinearArgs& g, uint32_t wg, int8_t* smem_l) {
    constexpr int BM = C::BM, BN = C::BN, BK = C::BK, WM = C::WM, WN = C::WN, S = C::S;
    constexpr int NW = WM * WN, TM = BM / WM / 32, TN = BN / WN / 32;
    typedef Operand<FA, BM, BK, NW> OpA;
    typedef Operand<FB, BN, BK, NW> OpB;
    constexpr int STAGE = OpA::BYTES + OpB::BYTES;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

    uint32_t tm, tn, expert = 0, lo = 0, hi = g.M, k_first = 0, k_count = g.K;
    const uint32_t split = wg / g.wg_tiles;              /* part of k; a part's workgroups are a multiple of 8 */
    wg -= split * g.wg_tiles;
    if constexpr (GROUP == GROUP_ROWS) {
        if (!find_expert<BM>(g, wg, &expert, &lo, &hi, &tm, &tn)) return;
    } else {
        uint32_t L;
        const uint32_t per = g.tiles_m * g.tiles_n;
        if (!pick_tile(wg, per * (GROUP == GROUP_K ? g.experts : 1u), &L)) return;
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
    Fragments<FA, BM, BK, TM> fa;
    Fragments<FB, BN, BK, TN> fb;
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

    constexpr int CALLS = OpA::CALLS + OpB::CALLS;
    auto request = [&](int stage, int klen) {
        A.request(lds0 + (uint32_t)(stage * STAGE), klen, wave, lane);
        B.request(lds0 + (uint32_t)(stage * STAGE + OpA::BYTES), klen, wave, lane);
    };
    auto multiply_tail = [&](int stage, int klen) {
        const int8_t* ta = smem_l + stage * STAGE;
        const int8_t* tb = ta + OpA::BYTES;
#pragma unroll
        for (int s = 0; s < BK / 16; s++) {
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

    const int nkb = (int)((k_count + BK - 1) / BK), whole = (int)(k_count / BK);
    const int last = (int)(k_count - (uint32_t)(nkb - 1) * BK);           /* k in the last block */
    if (nkb) {
#pragma unroll
        for (int i = 0; i < S; i++) if (i < nkb) request(i, i == nkb - 1 ? last : BK);
        if (nkb >= S) wait_and_barrier<(S - 1) * CALLS>();
        else wait_and_barrier<0>();
        v4i_t a[2][TM], b[2][TN];
        /* fragment i of the order they are needed in: a 0, all of b, the rest of a */
        auto read = [&](auto which, const int8_t* tile, auto step, auto idx) {
            constexpr int W = decltype(which)::value, KS = decltype(step)::value, I = decltype(idx)::value;
            if constexpr (I == 0) a[W][0] = fa.read(tile, KS, 0);
            else if constexpr (I <= TN) b[W][I - 1] = fb.read(tile + OpA::BYTES, KS, I - 1);
            else a[W][I - TN] = fa.read(tile, KS, I - TN);
        };
        static_for<TM + TN>([&](auto i) { read(IC<0>{}, smem_l, IC<0>{}, i); });
        /* one k-step: its multiplications, two reads of (tile, next step) behind each of the first of them (spread evenly
         * over all of them 8192^3 took 866 us instead of 856), mem(i) behind the i-th */
        auto kstep = [&](auto which, const int8_t* tile, auto next, auto mem) {
            constexpr int W = decltype(which)::value;
            constexpr int MF = TM * TN, RD = TM + TN;
            static_assert(RD <= 2 * MF, "every fragment has its multiplication");
            static_for<MF>([&](auto i) {
                constexpr int I = decltype(i)::value, T = I / TN, U_ = I % TN;
                mfma32<BF16>(b[W][U_], a[W][T], acc[T][U_]);
                static_for<RD>([&](auto r) {
                    if constexpr (decltype(r)::value / 2 == I) read(IC<1 - W>{}, tile, next, r);
                });
                mem(i);
                __builtin_amdgcn_sched_barrier(0);
            });
        };
        auto nothing = [](auto) {};
        int stage = 0;
        for (int kb = 0; kb < whole; kb++) {
            const int8_t* tile = smem_l + stage * STAGE;
            const int after = stage + 1 == S ? 0 : stage + 1;
            static_for<BK / 16 - 1>([&](auto s) { kstep(IC<decltype(s)::value & 1>{}, tile, IC<decltype(s)::value + 1>{}, nothing); });
            if (kb + S <= nkb) wait_and_barrier<(S - 2) * CALLS>();
            else wait_and_barrier<0>();
            const int left = nkb - 1 - (kb + S);                          /* blocks behind the one to request */
            const uint32_t lds = lds0 + (uint32_t)(stage * STAGE);
            const bool full = left > 0 || (left == 0 && last == BK);
            if (full) { A.point(); B.point(); }
            kstep(IC<1>{}, smem_l + after * STAGE, IC<0>{}, [&](auto i) {
                constexpr int I = decltype(i)::value, MF = TM * TN;
                if (full)
                    static_for<CALLS>([&](auto c) {
                        constexpr int Q = decltype(c)::value;
                        if constexpr (Q * MF / CALLS == I) {
                            if constexpr (Q < OpA::CALLS) A.request_one(IC<Q>{}, lds, wave);
                            else B.request_one(IC<Q - OpA::CALLS>{}, lds + OpA::BYTES, wave);
                        }
                    });
            });
            if (left == 0 && !full) request(stage, last);
            stage = after;
        }
        if (last != BK) multiply_tail(stage, last);
        wait_and_barrier<0>();
    }
    int8_t* park = smem_l + wave * park_bytes<TM, TN>();
    void* y_at = g.e.y;
    if constexpr (GROUP == GROUP_K) y_at = g.e.out32 ? (void*)((float*)y_at + expert * g.y_stride) : (void*)((uint16_t*)y_at + expert * g.y_stride);
    finish_tile<BF16, TM, TN>(g, acc, park, m0 + wm * TM * 32, GROUP == GROUP_ROWS ? hi : g.M, n0 + wn * TN * 32, expert, split, y_at);
}

template <int FA, int FB, class C, bool BF16, int GROUP>
__global__ __launch_bounds__(C::THREADS)
void linear_tile_kernel(LinearArgs g) {
    extern __shared__ __align__(16) int8_t smem_l[];
    multiply_tile<FA, FB, C, BF16, GROUP>(g, blockIdx.x, smem_l);
}

/* The two products of a backward pass, grad_x (the first `first` workgroups) and grad_w, in one launch: neither waits for
 * the other's last tiles, and two that would each leave CUs idle fill them together. */
struct LinearPair {
    LinearArgs x, w;
    uint32_t first, both;       /* workgroups of x, of x and w; the rest add up the bias gradient */
    BiasJoin bias;
};
/* a column of an expert: the bias gradient's parts, in ascending order */
__device__ __forceinline__ void join_bias(const BiasJoin& a, uint64_t id) {
    const uint32_t expert = (uint32_t)(id / a.N), c = (uint32_t)(id % a.N);
    if (expert >= a.experts) return;
    const float* p = a.part + (uint64_t)expert * a.parts * a.N + c;
    float s = 0.0f;
#pragma unroll 16
    for (uint32_t k = 0; k < a.parts; k++) s += p[(uint64_t)k * a.N];
    a.out[(uint64_t)expert * a.N + c] = s;
}
template <int FB, class C, bool BF16, bool GROUPED>
__global__ __launch_bounds__(C::THREADS)
void linear_pair_kernel(LinearPair p) {
    extern __shared__ __align__(16) int8_t smem_l[];
    if (blockIdx.x < p.first) multiply_tile<ROWS_K, FB, C, BF16, GROUPED ? GROUP_ROWS : GROUP_NONE>(p.x, blockIdx.x, smem_l);
    else if (blockIdx.x < p.both) multiply_tile<K_ROWS, K_ROWS, C, BF16, GROUPED ? GROUP_K : GROUP_NONE>(p.w, blockIdx.x - p.first, smem_l);
    else join_bias(p.bias, (uint64_t)(blockIdx.x - p.both) * C::THREADS + threadIdx.x);
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

/* eight 16-bit elements c .. c + 7 of a row of n, zeros beyond its end, as four words; THERE: all of them are */
template <bool THERE = false>
__device__ __forceinline__ v4i_t load8(const uint16_t* row, uint32_t c, uint32_t n) {
    typedef int v4iu_t __attribute__((ext_vector_type(4), aligned(2)));
    if (THERE || c + 8 <= n) return *(const v4iu_t*)(row + c);
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

/* ---- a few rows, K whole in a workgroup: no parts, no second launch ------------------------------------------------
 * Sixteen waves share K and join in LDS; a workgroup's columns are few, so that there are workgroups enough.
 *
 * k contiguous (W [N][K]), up to sixteen rows: 16 columns, a wave takes every sixteenth 64 k. K = N = 4096, bf16, the weights
 * of 44 layers in turn, so that they come from memory: one row 9.9 us, sixteen 12.2; the kernel above with its second launch
 * 15.4 and 16.4. */
template <bool BF16>
__global__ __launch_bounds__(1024)
void linear_few_rows_kernel(LinearArgs g) {
    __shared__ __align__(16) v4f_t joined[16][64];
    const int lane = threadIdx.x & 63, li = lane & 15, lg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t n0 = blockIdx.x * 16;
    const uint16_t* wr = g.b + (uint64_t)min(n0 + li, g.N - 1) * g.ldb;
    const uint16_t* xr = g.a + (uint64_t)min((uint32_t)li, g.M - 1) * g.lda;
    v4f_t acc = {0.0f, 0.0f, 0.0f, 0.0f};
    auto step = [&](uint32_t k0, auto full) {
        constexpr bool FULL = decltype(full)::value != 0;       /* all 64 k are there */
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const uint32_t k = k0 + 32 * h + 8 * lg;
            acc = mfma16<BF16>(load8<FULL>(wr, k, g.K), load8<FULL>(xr, k, g.K), acc);
        }
    };
    uint32_t k0 = 64 * wave;
    for (; k0 + 1088 <= g.K; k0 += 2048) { step(k0, IC<1>{}); step(k0 + 1024, IC<1>{}); }
    if (k0 + 64 <= g.K) { step(k0, IC<1>{}); k0 += 1024; }
    if (k0 < g.K) step(k0, IC<0>{});
    /* lane: row lane % 16, columns 4 (lane / 16) + 0..3; then a thread takes eight columns of a row, two lanes' four, over
     * the waves in ascending order */
    joined[wave][lane] = acc;
    __syncthreads();
    const uint32_t row = threadIdx.x & 15, pair = threadIdx.x >> 4, col = n0 + 8 * pair;
    if (threadIdx.x >= 32 || row >= g.M || col >= g.N) return;
    v4f_t lo = joined[0][32 * pair + row], hi = joined[0][32 * pair + 16 + row];
#pragma unroll 5
    for (int w = 1; w < 16; w++) { lo += joined[w][32 * pair + row]; hi += joined[w][32 * pair + 16 + row]; }
    float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]}, bias[8];
    load_bias<BF16>(g.e, 0, col, g.N, bias);
    finish_row8<BF16>(g.e, g.e.y, row, col, g.N, v, bias);
}

/* Columns contiguous (W [K][N]), up to four rows: 32 columns. One row, K = N = 4096, bf16: 10.7 us where the last-level cache
 * holds W (the kernel above with its second launch 12.4), but 17.9 against 14.0 with the weights of 44 layers in turn, which come
 * from memory. It is ahead there too up to K = 2048 (11.1 both; K = 1024: 7.5 against 9.0) and where N is no multiple of 128 (4160:
 * 14.3 against 21.9). A lane holds 8 k of 8 columns (transposed in its registers
 * as above), and of a wave's 128 k lane l holds the sixteenth l / 4. The MFMA wants one k for all of its sixteen positions,
 * so four of them, q = l / 4 % 4, carry the same columns at different k, and the other operand's sixteen positions are four
 * rows at each of those four k: the blocks where the two q agree are the sums, the others are not looked at. */
template <bool BF16>
__global__ __launch_bounds__(1024)
void linear_few_rows_strip_kernel(LinearArgs g) {
    __shared__ __align__(16) float joined[64][4][33];           /* [wave, q][row][column] */
    __shared__ float part[8][4][33];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    /* the two halves of a 128-byte line of W go to workgroups of one XCD, so that its L2 fetches the line once */
    const uint32_t strip = ((blockIdx.x >> 4) * 8 + (blockIdx.x & 7)) * 2 + ((blockIdx.x >> 3) & 1);
    const uint32_t n0 = strip * 32, c = n0 + 8 * (lane & 3);
    if (n0 >= g.N) return;
    v4f_t acc[8];
#pragma unroll
    for (int i = 0; i < 8; i++) acc[i] = (v4f_t){0.0f, 0.0f, 0.0f, 0.0f};
    const int q = (lane >> 2) & 3;
    auto step = [&](uint32_t k0, auto full) {
        constexpr bool FULL = decltype(full)::value != 0;       /* all 128 k and 32 columns are there */
        const uint32_t k = k0 + 8 * (lane >> 2);                /* of the columns' operand */
        v4i_t w[8];
#pragma unroll
        for (int j = 0; j < 8; j++) w[j] = FULL || k + j < g.K ? load8<FULL>(g.b + (uint64_t)(k + j) * g.ldb, c, g.N) : (v4i_t){0, 0, 0, 0};
        /* of the rows' operand: position 4 q + row at k group 4 (lane / 16) + q: the same k */
        const v4i_t x = load8<FULL>(g.a + (uint64_t)min((uint32_t)(lane & 3), g.M - 1) * g.lda, k, g.K);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            v4i_t f;
#pragma unroll
            for (int p = 0; p < 4; p++)
                f[p] = (int)__builtin_amdgcn_perm((uint32_t)w[2 * p + 1][i / 2], (uint32_t)w[2 * p][i / 2], (i & 1) ? 0x07060302u : 0x05040100u);
            acc[i] = mfma16<BF16>(f, x, acc[i]);
        }
    };
    uint32_t k0 = 128 * wave;
    if (n0 + 32 <= g.N) {
        for (; k0 + 2176 <= g.K; k0 += 4096) { step(k0, IC<1>{}); step(k0 + 2048, IC<1>{}); }
        if (k0 + 128 <= g.K) { step(k0, IC<1>{}); k0 += 2048; }
    }
    for (; k0 < g.K; k0 += 2048) step(k0, IC<0>{});
    /* lane: position 4 q + row of the rows' operand, positions 4 (lane / 16) + r, column group r, of the columns' */
    if (q == lane >> 4)
#pragma unroll
        for (int i = 0; i < 8; i++)
#pragma unroll
            for (int r = 0; r < 4; r++) joined[wave * 4 + q][lane & 3][8 * r + i] = acc[i][r];
    __syncthreads();
    {
        const int o = threadIdx.x & 127, p = threadIdx.x >> 7;
        float s = joined[8 * p][o >> 5][o & 31];
#pragma unroll
        for (int k = 1; k < 8; k++) s += joined[8 * p + k][o >> 5][o & 31];
        part[p][o >> 5][o & 31] = s;
    }
    __syncthreads();
    const int row = threadIdx.x >> 2, group = threadIdx.x & 3;
    const uint32_t col = n0 + 8 * group;
    if (threadIdx.x >= 16 || (uint32_t)row >= g.M || col >= g.N) return;
    float v[8], bias[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        v[i] = part[0][row][8 * group + i];
#pragma unroll
        for (int p = 1; p < 8; p++) v[i] += part[p][row][8 * group + i];
    }
    load_bias<BF16>(g.e, 0, col, g.N, bias);
    finish_row8<BF16>(g.e, g.e.y, row, col, g.N, v, bias);
}

/* ---- around the products ---------------------------------------------------------------------------------------- */

/* The parts of k added in ascending order, and the epilogue: a thread takes eight columns of a row. */
template <bool BF16, bool GROUPED>
__device__ __forceinline__ void join_parts(const LinearArgs& g, uint32_t block) {
    const uint32_t per = g.part_ld / 8;
    const uint64_t id = (uint64_t)block * 256 + threadIdx.x;
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
#pragma unroll 4
    for (uint32_t s = 0; s < g.splits; s++) {
        const v4f_t* p = (const v4f_t*)(g.part + ((uint64_t)s * g.M + row) * g.part_ld + c);
        const v4f_t a = p[0], b = p[1];
#pragma unroll
        for (int i = 0; i < 4; i++) { v[i] += a[i]; v[4 + i] += b[i]; }
    }
    load_bias<BF16>(g.e, expert, c, g.N, bias);
    finish_row8<BF16>(g.e, g.e.y, row, c, g.N, v, bias);
}


/* What is left to add up behind the products, in one launch: the parts of up to two products and of a bias gradient. */
struct JoinArgs {
    LinearArgs product[2];
    BiasJoin bias;
    uint32_t blocks[3];         /* of either product, of the bias                  */
};
template <bool BF16, bool GROUPED>
__global__ __launch_bounds__(256)
void linear_join_kernel(JoinArgs a) {
    uint32_t b = blockIdx.x;
    if (b < a.blocks[0]) { join_parts<BF16, GROUPED>(a.product[0], b); return; }
    b -= a.blocks[0];
    if (b < a.blocks[1]) { join_parts<BF16, false>(a.product[1], b); return; }
    join_bias(a.bias, (uint64_t)(b - a.blocks[1]) * 256 + threadIdx.x);
}

__device__ __forceinline__ void align_rows(const AlignArgs& a, uint32_t block) {
    const uint32_t per = a.out_ld / 8;
    for (uint64_t id = (uint64_t)block * 256 + threadIdx.x; id < a.chunks; id += (uint64_t)a.blocks * 256) {
        const uint64_t line = id / per;
        const uint32_t c = (uint32_t)(id % per) * 8;
        const uint64_t matrix = line / a.rows, row = line - matrix * a.rows;
        *(v4i_t*)(a.out + line * a.out_ld + c) = load8(a.in + matrix * a.stride + row * a.ld, c, a.cols);
    }
}

/* dz is rounded to the 16-bit type: it is an operand of the matrix cores. That adds its half step to the ones that x, w and the
 * outputs were rounded with: grad_x and grad_w are 2.3e-3 off the 64-bit formula in the 2-norm instead of 1.7e-3 (bf16; f16 2.9e-4
 * and 2.1e-4). A second operand for what the rounding leaves would double both products. The bias gradient needs no operand and
 * sums the unrounded values. */
template <bool BF16>
__device__ __forceinline__ void slope_rows(const SlopeArgs& a, uint32_t block, float (*sums)[32][9]) {
    typedef typename Half16<BF16>::T E;
    const uint32_t t = threadIdx.x & 31, r = threadIdx.x >> 5;
    const uint32_t across = block % a.across, part = block / a.across % a.parts, expert = block / a.across / a.parts;
    const uint32_t c = across * 256 + t * 8;
    uint32_t lo = 0, hi = a.rows;
    if (a.offsets) expert_range(a.offsets, expert, a.rows, &lo, &hi);
    float s[8];
#pragma unroll
    for (int i = 0; i < 8; i++) s[i] = 0.0f;
    if (c < a.N) {
        const uint64_t step = (uint64_t)a.parts * 8;
        for (uint64_t row = (uint64_t)lo + part * 8 + r; row < hi; row += 2 * step) {
            /* two rows' loads together */
            const bool more = row + step < hi;
            float d[2][8], z[2][8];
            load_row<E, float, 8>((const E*)a.dy + row * a.ld_dy, c, a.N, d[0]);
            if (a.act) load_row<E, float, 8>((const E*)a.pre + row * a.ld_pre, c, a.N, z[0]);
            if (more) {
                load_row<E, float, 8>((const E*)a.dy + (row + step) * a.ld_dy, c, a.N, d[1]);
                if (a.act) load_row<E, float, 8>((const E*)a.pre + (row + step) * a.ld_pre, c, a.N, z[1]);
            }
#pragma unroll
            for (int k = 0; k < 2; k++) {
                if (k && !more) break;
                slope8(d[k], z[k], a.act);
                if (a.dz) store_row<E, float, 8>((E*)a.dz + (row + k * step) * a.ld_dz, c, (uint32_t)a.ld_dz, d[k]);
#pragma unroll
                for (int i = 0; i < 8; i++) s[i] += d[k][i];
            }
        }
    }
    if (!a.part) return;
#pragma unroll
    for (int i = 0; i < 8; i++) sums[r][t][i] = s[i];
    __syncthreads();
    const uint32_t col = across * 256 + threadIdx.x;
    if (col >= a.N) return;
    float sum = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; k++) sum += sums[k][threadIdx.x >> 3][threadIdx.x & 7];
    a.part[((uint64_t)expert * a.parts + part) * a.N + col] = sum;
}

/* What the products need first, in one launch: dz and its sums, and aligned copies of up to two operands. */
struct PrepareArgs {
    SlopeArgs slope;
    AlignArgs copy[2];
};
template <bool BF16>
__global__ __launch_bounds__(256)
void linear_prepare_kernel(PrepareArgs a) {
    __shared__ __align__(16) float sums[8][32][9];
    uint32_t b = blockIdx.x;
    if (b < a.slope.blocks) { slope_rows<BF16>(a.slope, b, sums); return; }
    b -= a.slope.blocks;
    if (b < a.copy[0].blocks) { align_rows(a.copy[0], b); return; }
    align_rows(a.copy[1], b - a.copy[0].blocks);
}

/* ---- launches ---------------------------------------------------------------------------------------------------- */

inline bool lds_ready(const void* kern, int bytes) {
    /* once per kernel and device: attributes belong to the device a kernel runs on */
    static std::mutex m;
    static struct { const void* k; int dev; } done[512];
    static int n = 0;
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess) return false;
    std::lock_guard<std::mutex> lk(m);
    for (int i = 0; i < n; i++) if (done[i].k == kern && done[i].dev == dev) return true;
    if (!ESHKOL_HIP_OK(hipFuncSetAttribute(kern, hipFuncAttributeMaxDynamicSharedMemorySize, bytes))) return false;
    if (n < 512) { done[n].k = kern; done[n].dev = dev; n++; }
    return true;
}

typedef TileShape<256, 256, 64, 2, 4, 2> LargeTile;
typedef TileShape<128, 256, 32, 2, 4, 3, true> WideTile;
typedef TileShape<128, 128, 32, 2, 2, 3, true> SquareTile;
typedef TileShape<32, 128, 64, 1, 4, 3, true> Rows32Tile;
typedef TileShape<64, 128, 64, 2, 2, 4, true> Rows64Tile;
typedef TileShape<128, 256, 64, 2, 4, 3> WideAloneTile;
typedef TileShape<128, 128, 64, 2, 2, 4> SquareAloneTile;


/* the copy's work; the matrix is the copy from here on */
inline AlignArgs align_matrix(Matrix* m, uint16_t* room) {
    AlignArgs a = {};
    a.in = m->p; a.out = room;
    a.ld = m->ld; a.stride = m->stride; a.rows = m->rows; a.cols = (uint32_t)m->cols;
    const uint64_t ld = round_up_sz(m->cols, 8);
    a.out_ld = (uint32_t)ld;
    a.chunks = m->count * m->rows * (ld / 8);
    a.blocks = (uint32_t)std::min<uint64_t>((a.chunks + 255) / 256, (uint64_t)eshkol_hip_num_cus() * 16);
    m->p = room;
    m->ld = ld;
    m->stride = m->rows * ld;
    m->cols = ld;
    m->copy = false;
    return a;
}

/* the arguments of the kernels, and the workgroups of a product on a tile */
template <class C>
uint64_t fill_tiles(Product* q) {
    q->g.tiles_m = tiles_of(q->s.M, C::BM);
    q->g.tiles_n = tiles_of(q->s.N, C::BN);
    const uint64_t tiles = (tile_count(q->s, C::BM, C::BN) + 7) / 8 * 8;
    q->g.wg_tiles = (uint32_t)tiles;
    return tiles * q->splits;
}
inline void fill_args(Product* q, float* part) {
    LinearArgs& g = q->g;
    g.a = q->a.p; g.lda = q->a.ld;
    g.b = q->b.p; g.ldb = q->b.ld;
    g.b_stride = q->b.stride;
    g.a_extent = (uint32_t)q->a.cols;
    g.b_extent = (uint32_t)q->b.cols;
    g.M = (uint32_t)q->s.M; g.N = (uint32_t)q->s.N; g.K = (uint32_t)q->s.K;
    g.experts = (uint32_t)q->s.experts;
    g.splits = q->splits; g.part_k = q->part_k; g.part_ld = q->part_ld;
    g.part = part;
}

template <int FA, int FB, class C, bool BF16, int GROUP>
int launch_tile(Product* q, hipStream_t st) {
    auto kern = linear_tile_kernel<FA, FB, C, BF16, GROUP>;
    if (!lds_ready((const void*)kern, C::SMEM)) return -1;
    const uint64_t grid = fill_tiles<C>(q);
    if (grid > 0x7fffffffULL) return -1;
    hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(C::THREADS), C::SMEM, st, q->g);
    return 0;
}
/* the tiles that plan_products gives to products of one matrix alone have no kernels for groups */
template <class C, bool BF16>
int launch_tiles(Product* q, hipStream_t st) {
    const Shape& s = q->s;
    if constexpr (C::GROUPS) {
        if (s.group == GROUP_K) return launch_tile<K_ROWS, K_ROWS, C, BF16, GROUP_K>(q, st);
        if (s.group == GROUP_ROWS) return s.fb == ROWS_K ? launch_tile<ROWS_K, ROWS_K, C, BF16, GROUP_ROWS>(q, st) : launch_tile<ROWS_K, K_ROWS, C, BF16, GROUP_ROWS>(q, st);
    }
    if (s.group != GROUP_NONE) return -1;
    if (s.fa == K_ROWS) return launch_tile<K_ROWS, K_ROWS, C, BF16, GROUP_NONE>(q, st);
    return s.fb == ROWS_K ? launch_tile<ROWS_K, ROWS_K, C, BF16, GROUP_NONE>(q, st) : launch_tile<ROWS_K, K_ROWS, C, BF16, GROUP_NONE>(q, st);
}
template <int FB, class C, bool BF16, bool GROUPED>
int launch_pair(Product* x, Product* w, const BiasJoin& bias, hipStream_t st) {
    auto kern = linear_pair_kernel<FB, C, BF16, GROUPED>;
    if (!lds_ready((const void*)kern, C::SMEM)) return -1;
    LinearPair p;
    const uint64_t a = fill_tiles<C>(x), b = fill_tiles<C>(w);
    const uint64_t c = bias.out ? ((uint64_t)bias.N * bias.experts + C::THREADS - 1) / C::THREADS : 0;
    if (a + b + c > 0x7fffffffULL) return -1;
    p.x = x->g;
    p.w = w->g;
    p.first = (uint32_t)a;
    p.both = (uint32_t)(a + b);
    p.bias = bias;
    hipLaunchKernelGGL(kern, dim3((unsigned)(a + b + c)), dim3(C::THREADS), C::SMEM, st, p);
    return 0;
}
template <class C, bool BF16>
int launch_pairs(Product* x, Product* w, const BiasJoin& bias, hipStream_t st) {
    const bool rows_k = x->s.fb == ROWS_K;
    if (x->s.group == GROUP_ROWS) {
        if constexpr (C::GROUPS) return rows_k ? launch_pair<ROWS_K, C, BF16, true>(x, w, bias, st) : launch_pair<K_ROWS, C, BF16, true>(x, w, bias, st);
        else return -1;
    }
    return rows_k ? launch_pair<ROWS_K, C, BF16, false>(x, w, bias, st) : launch_pair<K_ROWS, C, BF16, false>(x, w, bias, st);
}
template <bool BF16>
int launch_pairs(int tile, Product* x, Product* w, const BiasJoin& bias, hipStream_t st) {
    switch (tile) {
    case TILE_LARGE: return launch_pairs<LargeTile, BF16>(x, w, bias, st);
    case TILE_WIDE: return launch_pairs<WideTile, BF16>(x, w, bias, st);
    case TILE_WIDE_ALONE: return launch_pairs<WideAloneTile, BF16>(x, w, bias, st);
    case TILE_SQUARE_ALONE: return launch_pairs<SquareAloneTile, BF16>(x, w, bias, st);
    default: return launch_pairs<SquareTile, BF16>(x, w, bias, st);
    }
}
/* tiles of 32 or 64 rows are for products whose first operand has k contiguous */
template <class C, bool BF16>
int launch_rows(Product* q, hipStream_t st) {
    const bool rows_k = q->s.fb == ROWS_K;
    if (q->s.fa != ROWS_K) return -1;
    if (q->s.group == GROUP_ROWS) return rows_k ? launch_tile<ROWS_K, ROWS_K, C, BF16, GROUP_ROWS>(q, st) : launch_tile<ROWS_K, K_ROWS, C, BF16, GROUP_ROWS>(q, st);
    return rows_k ? launch_tile<ROWS_K, ROWS_K, C, BF16, GROUP_NONE>(q, st) : launch_tile<ROWS_K, K_ROWS, C, BF16, GROUP_NONE>(q, st);
}
template <bool BF16>
int launch_tiles(int tile, Product* q, hipStream_t st) {
    if (q->kind == RUN_TILES_32) return launch_rows<Rows32Tile, BF16>(q, st);
    if (q->kind == RUN_TILES_64) return launch_rows<Rows64Tile, BF16>(q, st);
    switch (tile) {
    case TILE_LARGE: return launch_tiles<LargeTile, BF16>(q, st);
    case TILE_WIDE: return launch_tiles<WideTile, BF16>(q, st);
    case TILE_WIDE_ALONE: return launch_tiles<WideAloneTile, BF16>(q, st);
    case TILE_SQUARE_ALONE: return launch_tiles<SquareAloneTile, BF16>(q, st);
    default: return launch_tiles<SquareTile, BF16>(q, st);
    }
}
template <bool BF16>
int launch_thin(Product* q, hipStream_t st) {
    const bool rows = q->s.group == GROUP_ROWS;
    if (q->kind == RUN_STREAM_WHOLE) {
        if (q->s.fb == K_ROWS) hipLaunchKernelGGL((linear_few_rows_strip_kernel<BF16>), dim3((tiles_of(q->s.N, 32) + 15) / 16 * 16), dim3(1024), 0, st, q->g);
        else hipLaunchKernelGGL((linear_few_rows_kernel<BF16>), dim3(tiles_of(q->s.N, 16)), dim3(1024), 0, st, q->g);
        return 0;
    }
    const dim3 grid(tiles_of(q->s.N, 128), q->splits, rows ? q->g.experts : 1);
    /* more than sixteen rows by expert are tiles */
#define THIN(FB, RT) hipLaunchKernelGGL((linear_thin_kernel<FB, RT, BF16, false>), grid, dim3(256), 0, st, q->g)
    if (rows) {
        if (q->s.fb == ROWS_K) hipLaunchKernelGGL((linear_thin_kernel<ROWS_K, 1, BF16, true>), grid, dim3(256), 0, st, q->g);
        else hipLaunchKernelGGL((linear_thin_kernel<K_ROWS, 1, BF16, true>), grid, dim3(256), 0, st, q->g);
    } else if (q->s.fb == ROWS_K) { if (q->rt == 1) THIN(ROWS_K, 1); else if (q->rt == 2) THIN(ROWS_K, 2); else THIN(ROWS_K, 4); }
    else { if (q->rt == 1) THIN(K_ROWS, 1); else if (q->rt == 2) THIN(K_ROWS, 2); else THIN(K_ROWS, 4); }
#undef THIN
    return 0;
}

/* One or two products (grad_x and grad_w), their operands' copies and dz before them, their parts joined behind them. */
template <bool BF16>
int run_products(Product* q, int n, int tile, const SlopeArgs* slope, const BiasJoin* bias, char* ws, hipStream_t st) {
    /* one launch for everything the products need; dz, where it is made, is aligned by itself, and the two products
     * share no other operand */
    PrepareArgs pre = {};
    if (slope) pre.slope = *slope;
    int copies = 0;
    for (int i = 0; i < n; i++) {
        if (q[i].streams()) continue;
        for (Matrix* m : {&q[i].a, &q[i].b}) {
            if (!m->copy) continue;
            const uint64_t bytes = m->copy_bytes;
            pre.copy[copies++] = align_matrix(m, (uint16_t*)ws);
            ws += bytes;
        }
    }
    const uint64_t blocks = (uint64_t)pre.slope.blocks + pre.copy[0].blocks + pre.copy[1].blocks;
    if (blocks > 0x7fffffffULL) return -1;
    if (blocks) hipLaunchKernelGGL((linear_prepare_kernel<BF16>), dim3((unsigned)blocks), dim3(256), 0, st, pre);

    JoinArgs join = {};
    uint64_t joins = 0;
    for (int i = 0; i < n; i++) {
        fill_args(&q[i], (float*)ws);
        ws += q[i].part_bytes;
    }
    int rc = 0;
    bool bias_done = !bias || !bias->out;
    if (n == 2 && q[0].kind == RUN_TILES && q[1].kind == RUN_TILES) {
        /* without parts to join there is no launch behind the products: the bias gradient is added up beside them */
        const bool beside = !bias_done && q[0].splits <= 1 && q[1].splits <= 1;
        rc = launch_pairs<BF16>(tile, &q[0], &q[1], beside ? *bias : BiasJoin{}, st);
        bias_done |= beside;
    } else
        for (int i = 0; i < n && !rc; i++) rc = q[i].streams() ? launch_thin<BF16>(&q[i], st) : launch_tiles<BF16>(tile, &q[i], st);
    if (rc) return rc;
    bool grouped = false;
    for (int i = 0; i < n; i++) {
        if (q[i].splits <= 1) continue;
        /* the first place is for the product whose rows may be grouped */
        const int at = i == 0 && q[0].s.fa == ROWS_K ? 0 : 1;
        join.product[at] = q[i].g;
        const uint64_t b = (q[i].s.M * (q[i].part_ld / 8) + 255) / 256;
        if (b > 0x7fffffffULL) return -1;
        join.blocks[at] = (uint32_t)b;
        joins += b;
        grouped |= q[i].s.group == GROUP_ROWS;
    }
    if (!bias_done) {
        join.bias = *bias;
        const uint64_t b = ((uint64_t)bias->N * bias->experts + 255) / 256;
        if (b > 0x7fffffffULL) return -1;
        join.blocks[2] = (uint32_t)b;
        joins += b;
    }
    if (joins > 0x7fffffffULL) return -1;
    if (joins) {
        if (grouped) hipLaunchKernelGGL((linear_join_kernel<BF16, true>), dim3((unsigned)joins), dim3(256), 0, st, join);
        else hipLaunchKernelGGL((linear_join_kernel<BF16, false>), dim3((unsigned)joins), dim3(256), 0, st, join);
    }
    return 0;
}
}  // namespace linear
#endif
