/*
 * The linear layer and the products by expert (gpu_hip_layers.h), host side: the checks of a call, how its products
 * are cut, and what its workspace holds. The kernels are in linear_16.h, compiled once per element type.
 */
#include "linear_args.h"

namespace {

using namespace linear;

Matrix matrix_of(const void* p, uint64_t ld, uint64_t stride, uint64_t rows, uint64_t cols, uint64_t count) {
    Matrix m = {(const uint16_t*)p, ld, stride, rows, cols, count, false, 0};
    m.copy = rows && (((uintptr_t)p & 15) || (ld & 7) || (cols & 7) || (count > 1 && (stride & 7)) || ld > (1u << 22));
    if (m.copy) m.copy_bytes = round_up_sz((size_t)(count * rows * round_up_sz(cols, 8) * 2), 256);
    return m;
}
/* How a product is run. Up to sixteen rows (on average, by expert: the groups' sizes are on the device) B is streamed past them,
 * sixteen at a time, so an expert with many more is late: 1024 rows of 64 experts, 1024 x 4096, take 107 us at 16 each, 371 with 512
 * on one and 549 with all on one. Up to 64 rows in tiles of 32 or 64
 * rows: the streaming kernel's loads of more rows outgrow those of B (K = N = 4096, W [N][K], bf16, us without the second
 * launch: 32 rows 11.3 and 7.6, 64 rows 16.9 and 8.4; one row 6.6 and 7.6). The tiles want aligned operands, and a copy of
 * B would cost more than they gain. */
Product make_product(const Shape& s, const Matrix& a, const Matrix& b) {
    Product q = {};
    q.s = s;
    q.a = a;
    q.b = b;
    q.splits = 1;
    q.part_k = (uint32_t)round_up_sz((size_t)s.K, 64);
    q.kind = RUN_TILES;
    if (s.fa != ROWS_K || s.group == GROUP_K) return q;
    const bool grouped = s.group == GROUP_ROWS;
    const uint64_t rows = grouped ? (s.M + s.experts - 1) / s.experts : s.M;
    if (rows > 64) return q;
    q.rt = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
    if (rows > 16 && !a.copy && !b.copy) { q.kind = rows <= 32 && !grouped ? RUN_TILES_32 : RUN_TILES_64; return q; }
    if (rows > 16 && grouped) return q;
    /* K whole in a workgroup where the narrow strips of columns alone give a third of the CUs work */
    const uint64_t strips = tiles_of(s.N, s.fb == K_ROWS ? 32 : 16);
    const bool whole = !grouped && s.M <= (s.fb == K_ROWS ? 4 : 16) && strips * 3 >= (uint64_t)eshkol_hip_num_cus();
    q.kind = whole ? RUN_STREAM_WHOLE : RUN_STREAM;
    return q;
}
/* cuts K into about `want` parts of at least `least` */
void split_product(Product* q, uint64_t want, uint64_t least) {
    const uint64_t k64 = round_up_sz((size_t)q->s.K, 64);
    uint64_t splits = std::min<uint64_t>(want, k64 / least);
    if (splits <= 1) return;
    const uint64_t part = round_up_sz((size_t)((k64 + splits - 1) / splits), q->kind == RUN_STREAM ? 128 : 64);
    splits = (q->s.K + part - 1) / part;
    if (splits <= 1) return;
    q->part_k = (uint32_t)part;
    q->splits = (uint32_t)splits;
    q->part_ld = (uint32_t)round_up_sz((size_t)q->s.N, 8);
    q->part_bytes = round_up_sz((size_t)(splits * q->s.M * q->part_ld * 4), 256);
}
/* The tile of one or two products launched together, and how their K is cut. Times are of bf16 products without an epilogue, us,
 * those of one comparison from one run.
 * 256 x 256 where at least three quarters of the CUs get one (8192^3: 819; 128 x 256 921, 128 x 128 1170), products of one
 * matrix only: the last rows of a group leave half a tile empty on average.
 * 128 x 256 where that many of those there are (the two products of 4096 x 1024 x 4096: 74, 128 x 128 79; 16384 rows of 64
 * experts, 1024 x 4096: 236 and 279). Two fit on a CU; where no CU gets two, blocks of 64 k instead of 32 need half the
 * barriers (the same two: 65).
 * 128 x 128 otherwise, three on a CU, or alone with blocks of 64 k (4096 x 1024 x 4096: 41 and 47). */
int plan_products(Product* q, int n) {
    const uint64_t cus = (uint64_t)eshkol_hip_num_cus();
    uint64_t large = 0, wide = 0, square = 0, work = 0;
    bool any = false, grouped = false;
    for (int i = 0; i < n; i++) {
        const Shape& s = q[i].s;
        if (q[i].kind != RUN_TILES) {
            const uint64_t have = (uint64_t)tiles_of(s.N, 128) * (s.group == GROUP_ROWS ? std::min(s.experts, s.M) : 1);
            if (q[i].kind == RUN_STREAM) split_product(&q[i], (2 * cus + have - 1) / have, 128);
            else if (q[i].kind != RUN_STREAM_WHOLE && s.group == GROUP_NONE) split_product(&q[i], (cus + have - 1) / have, 256);
            continue;
        }
        any = true;
        grouped |= s.group != GROUP_NONE;
        large += tile_count(s, 256, 256);
        wide += tile_count(s, 128, 256);
        square += tile_count(s, 128, 128);
        work += tile_count(s, 128, 128) * ((s.K + 63) / 64);
    }
    if (!any) return TILE_SQUARE;
    if (grouped) return wide * 4 >= cus * 3 ? TILE_WIDE : TILE_SQUARE;
    if (large * 4 >= cus * 3) return TILE_LARGE;
    if (wide * 4 >= cus * 3) return wide <= cus ? TILE_WIDE_ALONE : TILE_WIDE;
    /* too few tiles for the CUs: K is cut so that every workgroup has about a CU's share of the blocks, at least 512 of K */
    const uint64_t share = std::max<uint64_t>(1, work / cus);
    uint64_t workgroups = 0;
    for (int i = 0; i < n; i++) {
        if (q[i].kind != RUN_TILES) continue;
        if (square < cus) split_product(&q[i], ((q[i].s.K + 63) / 64 + share / 2) / share, 512);
        workgroups += tile_count(q[i].s, 128, 128) * q[i].splits;
    }
    return workgroups <= cus + cus / 4 ? TILE_SQUARE_ALONE : TILE_SQUARE;
}

uint64_t products_bytes(const Product* q, int n) {
    uint64_t b = 0;
    for (int i = 0; i < n; i++) b += q[i].part_bytes + q[i].copy_bytes();
    return b;
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

/* a launch holds 2^31 - 1 workgroups; nothing is queued before this is known */
int check_tiles(const char* name, const Product* q, int n) {
    uint64_t total = 0;
    for (int i = 0; i < n; i++) {
        const uint64_t tiles = q[i].kind == RUN_TILES ? tile_count(q[i].s, 128, 128) : tile_count(q[i].s, 32, 128);
        total += (tiles + 8) * q[i].splits;
    }
    if (total > 0x3fffffffULL) LAYER_REFUSE(name, "%llu tiles", (unsigned long long)total);
    return 0;
}

/* ---- forward -------------------------------------------------------------------------------------------------------- */

struct ForwardCall {
    Product q;
    int tile;
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
    f->tile = plan_products(&f->q, 1);
    return check_tiles(name, &f->q, 1);
}
int64_t forward_workspace(const char* name, const HipExpertsArgs& u, const void* residual, uint64_t ld_res, bool grouped) {
    ForwardCall f;
    if (plan_forward(name, u, residual, ld_res, grouped, &f)) return -1;
    return f.none ? 0 : (int64_t)products_bytes(&f.q, 1);
}
int forward(const char* name, const HipExpertsArgs& u, const void* residual, uint64_t ld_res, bool grouped, void* stream) {
    ForwardCall f;
    if (plan_forward(name, u, residual, ld_res, grouped, &f)) return -1;
    if (f.none) return 0;
    if (check_room(name, u.workspace, u.workspace_bytes, products_bytes(&f.q, 1))) return -2;
    hipStream_t st = (hipStream_t)stream;
    EshkolStreamDevice on(st);
    if (!on.ok) return -1;
    char* ws = (char*)u.workspace;
    if (u.dtype == 3 ? run_bf16(&f.q, 1, f.tile, nullptr, nullptr, ws, st) : run_f16(&f.q, 1, f.tile, nullptr, nullptr, ws, st)) return -1;
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
    SlopeArgs slope;            /* blocks 0: not run */
    BiasJoin bias;
    uint64_t dz_bytes, sum_bytes;
    Product q[2];
    int n, tile;
};

int plan_backward(const char* name, HipExpertsBackwardArgs u, bool grouped, BackwardCall* c) {
    if (check_sizes(name, u.rows, u.K, u.N, u.dtype, u.act, u.experts, grouped)) return -1;
    if (!layer_param_ok(u.dtype, u.grad_w_dtype)) LAYER_REFUSE(name, "grad_w_dtype %d beside dtype %d", u.grad_w_dtype, u.dtype);
    if (!u.grad_x && !u.grad_w && !u.grad_bias) LAYER_REFUSE(name, "no output is asked for");
    const uint64_t wr = u.trans_w ? u.N : u.K, wc = u.trans_w ? u.K : u.N;
    const bool some = u.rows != 0;
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

    const uint64_t experts = grouped ? u.experts : 1, cus = (uint64_t)eshkol_hip_num_cus();
    const bool want_x = u.grad_x && some, want_w = u.grad_w != nullptr, want_b = u.grad_bias != nullptr;
    const Shape sx = {ROWS_K, u.trans_w ? K_ROWS : ROWS_K, grouped ? GROUP_ROWS : GROUP_NONE, u.rows, u.K, u.N, experts};
    const Shape sw = {K_ROWS, K_ROWS, grouped ? GROUP_K : GROUP_NONE, wr, wc, u.rows, experts};
    const Matrix w = matrix_of(u.w, u.ldw, u.w_stride, wr, wc, experts), x = matrix_of(u.x, u.ldx, 0, u.rows, u.K, 1);
    Matrix dz = matrix_of(u.grad_y, u.ld_grad_y, 0, u.rows, u.N, 1);
    /* dz has room of its own where there is an activation, or where grad_y is not as the tiled kernel wants it */
    const bool tiled = want_w || (want_x && !make_product(sx, dz, w).streams());
    const bool make_dz = some && ((u.act && (want_x || want_w)) || (tiled && dz.copy));
    const uint64_t ld_dz = round_up_sz((size_t)u.N, 8);
    if (make_dz) dz = matrix_of((const void*)(uintptr_t)256, ld_dz, 0, u.rows, ld_dz, 1);       /* its address is known later */
    c->dz_bytes = make_dz ? round_up_sz((size_t)(u.rows * ld_dz * 2), 256) : 0;

    /* enough runs of rows to fill the device, on average at least 16 rows long */
    SlopeArgs& a = c->slope;
    a = SlopeArgs();
    const uint64_t across = tiles_of(u.N, 256), have = across * experts;
    const uint64_t parts = std::max<uint64_t>(1, std::min<uint64_t>((8 * cus + have - 1) / have, (u.rows / experts + 15) / 16));
    c->sum_bytes = want_b && some ? round_up_sz((size_t)(experts * parts * u.N * 4), 256) : 0;
    a.dy = (const uint16_t*)u.grad_y; a.pre = (const uint16_t*)u.pre;
    a.ld_dy = u.ld_grad_y; a.ld_pre = u.ld_pre; a.ld_dz = ld_dz;
    a.rows = (uint32_t)u.rows; a.N = (uint32_t)u.N; a.parts = (uint32_t)parts; a.experts = (uint32_t)experts; a.across = (uint32_t)across;
    a.offsets = grouped ? u.offsets : nullptr;
    a.act = u.act;
    if (some && (make_dz || want_b)) {
        if (have * parts > 0x7fffffffULL) LAYER_REFUSE(name, "too many columns and experts");
        a.blocks = (uint32_t)(have * parts);
    }
    c->bias = {nullptr, (float*)u.grad_bias, (uint32_t)u.N, a.blocks ? a.parts : 0u, (uint32_t)experts};

    c->n = 0;
    if (want_x) {
        Product& q = c->q[c->n++];
        q = make_product(sx, dz, w);
        q.g.e.y = u.grad_x; q.g.e.ldy = u.ld_grad_x;
        q.g.offsets = a.offsets;
    }
    if (want_w) {
        Product& q = c->q[c->n++];
        q = u.trans_w ? make_product(sw, dz, x) : make_product(sw, x, dz);
        q.g.e.y = u.grad_w; q.g.e.ldy = u.ld_grad_w; q.g.e.out32 = u.grad_w_dtype == 1;
        q.g.y_stride = u.grad_w_stride;
        q.g.offsets = a.offsets;
    }
    c->tile = plan_products(c->q, c->n);
    return check_tiles(name, c->q, c->n);
}
uint64_t backward_bytes(const BackwardCall& c) { return c.dz_bytes + c.sum_bytes + products_bytes(c.q, c.n); }

int backward(const char* name, const HipExpertsBackwardArgs& u, bool grouped, void* stream) {
    BackwardCall c;
    if (plan_backward(name, u, grouped, &c)) return -1;
    if (check_room(name, u.workspace, u.workspace_bytes, backward_bytes(c))) return -2;
    hipStream_t st = (hipStream_t)stream;
    EshkolStreamDevice on(st);
    if (!on.ok) return -1;
    char* ws = (char*)u.workspace;
    if (c.dz_bytes) {
        c.slope.dz = (uint16_t*)ws;
        ws += c.dz_bytes;
        /* dz is the first operand of grad_x, and of grad_w where W is held [N][K] */
        for (int i = 0; i < c.n; i++) (c.q[i].s.fa == ROWS_K || u.trans_w ? c.q[i].a : c.q[i].b).p = c.slope.dz;
    }
    if (c.sum_bytes) {
        c.slope.part = (float*)ws;
        c.bias.part = (const float*)ws;
        ws += c.sum_bytes;
    }
    if (u.dtype == 3 ? run_bf16(c.q, c.n, c.tile, &c.slope, &c.bias, ws, st) : run_f16(c.q, c.n, c.tile, &c.slope, &c.bias, ws, st)) return -1;
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
