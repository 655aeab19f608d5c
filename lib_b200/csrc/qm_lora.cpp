// qm_lora.cpp — host side of the low-rank adapters beside a stored projection (include/qmatmul.h).
#include <math.h>
#include <string.h>

#include <algorithm>
#include <new>

#include "qm_internal.h"

#define QM_LORA_MAGIC 0x514D4C52u  // "QMLR"

struct qm_lora {
    uint32_t magic;
    qm_ctx *ctx;
    int64_t rows, cols, np;
    int32_t slots, max_rank, rpad, max_tokens;
    CUdeviceptr a, b;            // [slots][rpad][cols], [slots][rpad][np] bf16
    CUdeviceptr at, bt;          // [slots][cols][rpad], [slots][rows][rpad] bf16
    CUdeviceptr scale, rank;     // [slots]
    CUdeviceptr low[2];          // [low_rows][pitch] bf16, three parts of rpad ranks: u, v
    int64_t low_rows;
    int32_t at_once[4];          // clusters of 1, 2, 4, 8 CTAs that run at once with one CTA per SM
    int32_t few_at_once;         // clusters of qm_lora_few_*
    CUstream side;               // the backward pass: dx beside the gradients of A and B
    CUevent fork, join;
    CUtensorMap w_map[2], low_map[2];
    CUdeviceptr list, offsets, tiles;
    CUdeviceptr aligned;         // [max_tokens][np] bf16, from the first backward pass on whose dy no tensor map takes
};

static int32_t lora_check(qm_ctx *c, const qm_lora *l) { return l && l->magic == QM_LORA_MAGIC && l->ctx == c ? QM_OK : QM_ERR_ARG; }

// The most tiles that `tokens` tokens make: whole ones, and one that ends early for every group that has any.
static int64_t lora_tiles(const qm_lora *l, int64_t tokens, bool listed) {
    const int64_t whole = (tokens + QM_LORA_TILE - 1) / QM_LORA_TILE;
    return listed ? whole + std::min<int64_t>(tokens, l->slots + 1) : whole;
}

static void lora_release(qm_ctx *c, qm_lora *l) {
    CUdeviceptr all[] = {l->a, l->b, l->at, l->bt, l->scale, l->rank, l->low[0], l->low[1], l->list, l->offsets, l->tiles, l->aligned};
    for (CUdeviceptr p : all)
        if (p) c->drv->cuMemFree_v2(p);
    if (l->fork) c->drv->cuEventDestroy_v2(l->fork);
    if (l->join) c->drv->cuEventDestroy_v2(l->join);
    if (l->side) c->drv->cuStreamDestroy_v2(l->side);
    l->magic = 0;
    delete l;
}

// A bf16 matrix [rows][pitch] of `cols` columns, read in boxes of 64 columns x `box` rows.
static CUresult tensor_map(qm_ctx *c, CUtensorMap *map, uint64_t p, int64_t cols, int64_t rows, int64_t pitch, int box) {
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)pitch * 2};
    const cuuint32_t boxes[2] = {64, (cuuint32_t)box}, one[2] = {1, 1};
    return c->drv->cuTensorMapEncodeTiled(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, (void *)(uintptr_t)p, dims, strides, boxes, one,
                                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
}

static int rank_kernel(const qm_lora *l) { return l->rpad == 16 ? 0 : l->rpad == 32 ? 1 : l->rpad == 64 ? 2 : 3; }
// Shared memory of the kernels.
static int64_t rows_smem(const qm_lora *l) {
    const int64_t ks = ((l->cols + QM_LORA_CLUSTER - 1) / QM_LORA_CLUSTER + 7) & ~(int64_t)7;
    const int64_t chunk = (int64_t)l->rpad * QM_LORA_CHUNK * 2;
    return 16ll * l->rpad * 4 + 8 * 4 + chunk + std::max<int64_t>(8 * ks * 4, 32 * QM_LORA_CHUNK * 4 + chunk);
}
static int64_t few_smem(const qm_lora *l) {
    return 8 * 16 * (l->rpad + 4) * 4 + 16 * QM_LORA_EXPAND_ROW(l->rpad / 16) + (3 * QM_LORA_FEW + 24) * 4;
}
static int64_t shrink_smem(const qm_lora *l) { return 1024 + QM_LORA_SHRINK_STAGES(l->rpad / 16) * (16384 + l->rpad * 128ll) + 128; }
static int64_t outer_smem(const qm_lora *l) {
    const int rp = l->rpad / 16;
    return 1024 + QM_LORA_OUTER_STAGES(rp) * 8192ll * (QM_LORA_PITCH(rp) / 64 + QM_LORA_OUTER_COLS(rp) / 64) + 128;
}

extern "C" int32_t qm_lora_create(qm_ctx *c, int64_t rows, int64_t cols, int32_t adapters, int32_t max_rank, int32_t max_tokens,
                                  qm_lora **out) {
    CHECK_CTX(c);
    if (!out) return QM_ERR_ARG;
    *out = nullptr;
    if (rows < 1 || cols < 32 || cols % 32 != 0 || adapters < 1 || max_rank < 1 || max_tokens < 1) return QM_ERR_SHAPE;
    // (cols: eight staged rows of x and a chunk of B fit in the shared memory of qm_lora_rows)
    if (rows > (1 << 22) || cols > 32768 || adapters > 256 || max_rank > 128 || max_tokens > (1 << 20)) return QM_ERR_LIMIT;
    CtxGuard g(c);
    DRV(g.rc);
    if (int32_t rc = qm_refuse_capture(c)) return rc;   // (the clear below would run again with the graph)
    qm_lora *l = new (std::nothrow) qm_lora();
    if (!l) return QM_ERR_NOMEM;
    l->magic = QM_LORA_MAGIC;
    l->ctx = c;
    l->rows = rows;
    l->cols = cols;
    l->np = (rows + 7) & ~(int64_t)7;
    l->slots = adapters;
    l->max_rank = max_rank;
    l->rpad = max_rank <= 16 ? 16 : max_rank <= 32 ? 32 : max_rank <= 64 ? 64 : 128;
    l->max_tokens = max_tokens;
    const int64_t pitch = QM_LORA_PITCH(l->rpad / 16);
    l->low_rows = ((int64_t)max_tokens + QM_LORA_TILE - 1) / QM_LORA_TILE * QM_LORA_TILE + (std::min(adapters, max_tokens) + 1) * (int64_t)QM_LORA_BLOCK;
    CUresult r = CUDA_SUCCESS;
    const int64_t low = l->low_rows * pitch * 2;
    struct {
        CUdeviceptr *p;
        int64_t bytes;
    } need[] = {{&l->a, (int64_t)adapters * l->rpad * cols * 2}, {&l->b, (int64_t)adapters * l->rpad * l->np * 2},
                {&l->at, (int64_t)adapters * l->rpad * cols * 2}, {&l->bt, (int64_t)adapters * l->rpad * rows * 2},
                {&l->scale, adapters * 4ll}, {&l->rank, adapters * 4ll}, {&l->low[0], low}, {&l->low[1], low},
                {&l->list, max_tokens * 4ll}, {&l->offsets, (adapters + 2) * 8ll},
                {&l->tiles, 32 * lora_tiles(l, max_tokens, true)}};
    for (auto &n : need)
        if (r == CUDA_SUCCESS) r = c->drv->cuMemAlloc_v2(n.p, (size_t)n.bytes);
    if (r == CUDA_SUCCESS) r = c->drv->cuMemsetD8Async(l->rank, 0, (size_t)adapters * 4, c->stream);
    if (r == CUDA_SUCCESS) r = c->drv->cuStreamSynchronize(c->stream);   // the next call may be on another stream
    if (r == CUDA_SUCCESS) r = c->drv->cuStreamCreate(&l->side, CU_STREAM_NON_BLOCKING);
    if (r == CUDA_SUCCESS) r = c->drv->cuEventCreate(&l->fork, CU_EVENT_DISABLE_TIMING);
    if (r == CUDA_SUCCESS) r = c->drv->cuEventCreate(&l->join, CU_EVENT_DISABLE_TIMING);
    const int64_t wide[2] = {cols, rows}, w_pitch[2] = {cols, l->np};
    const CUdeviceptr w[2] = {l->a, l->b};
    for (int i = 0; i < 2; i++) {
        if (r == CUDA_SUCCESS) r = tensor_map(c, &l->w_map[i], w[i], wide[i], (int64_t)adapters * l->rpad, w_pitch[i], l->rpad);
        if (r == CUDA_SUCCESS) r = tensor_map(c, &l->low_map[i], l->low[i], pitch, l->low_rows, pitch, QM_LORA_BLOCK);
    }
    if (r != CUDA_SUCCESS) {
        lora_release(c, l);
        return (int32_t)r;
    }
    for (int i = 0; i < 4; i++)
        l->at_once[i] = qm_max_clusters(c, QM_K_LORA_OUTER_R16 + rank_kernel(l), 1 << i, (QM_LORA_OUTER_READERS(l->rpad / 16) + 2) * 32, (unsigned)outer_smem(l));
    l->few_at_once = qm_max_clusters(c, QM_K_LORA_FEW_R16 + rank_kernel(l), QM_LORA_CLUSTER, 256, (unsigned)few_smem(l));
    *out = l;
    return QM_OK;
}

extern "C" int32_t qm_lora_destroy(qm_ctx *c, qm_lora *l) {
    CHECK_CTX(c);
    if (int32_t rc = lora_check(c, l)) return rc;
    CtxGuard g(c);
    DRV(g.rc);
    c->drv->cuStreamSynchronize(c->stream);
    lora_release(c, l);
    return QM_OK;
}

extern "C" int32_t qm_lora_set(qm_ctx *c, qm_lora *l, int32_t slot, int32_t rank, float scale, uint64_t a_dev, uint64_t b_dev,
                               int32_t type) {
    CHECK_CTX(c);
    if (int32_t rc = lora_check(c, l)) return rc;
    if (slot < 0 || slot >= l->slots || rank < 0 || rank > l->max_rank) return QM_ERR_SHAPE;
    if (type != QM_TYPE_F32 && type != QM_TYPE_F16 && type != QM_TYPE_BF16) return QM_ERR_FORMAT;
    const uint64_t part = type == QM_TYPE_F32 ? 3 : 1;
    if (!isfinite(scale) || (rank && (!a_dev || !b_dev || ((a_dev | b_dev) & part)))) return QM_ERR_ARG;
    CtxGuard g(c);
    DRV(g.rc);
    QmLoraSetArgs a;
    memset(&a, 0, sizeof a);
    a.a = (const void *)(uintptr_t)a_dev;
    a.b = (const void *)(uintptr_t)b_dev;
    a.da = (uint16_t *)(uintptr_t)l->a + (int64_t)slot * l->rpad * l->cols;
    a.db = (uint16_t *)(uintptr_t)l->b + (int64_t)slot * l->rpad * l->np;
    a.dat = (uint16_t *)(uintptr_t)l->at + (int64_t)slot * l->rpad * l->cols;
    a.dbt = (uint16_t *)(uintptr_t)l->bt + (int64_t)slot * l->rpad * l->rows;
    a.scale_out = (float *)(uintptr_t)l->scale + slot;
    a.rank_out = (int32_t *)(uintptr_t)l->rank + slot;
    a.rows = (int32_t)l->rows;
    a.cols = (int32_t)l->cols;
    a.np = (int32_t)l->np;
    a.rpad = l->rpad;
    a.rank = rank;
    a.type = type;
    a.scale = scale;
    const int64_t tiles = rank ? (l->rpad + 31) / 32 * ((l->cols + 63) / 64 + (l->np + 63) / 64) : 1;
    return qm_launch(c, QM_K_LORA_SET, (unsigned)std::min<int64_t>(tiles, 8ll * c->sm_count), 1, 256, 0, &a, true);
}

// Rows of `width` bytes, `pitch` bytes apart: do two such sets of bytes (by their hulls) meet?
static bool rows_meet(uint64_t p, int64_t pitch_p, int64_t width_p, uint64_t q, int64_t pitch_q, int64_t width_q, int64_t rows) {
    return p && q && p < q + (uint64_t)((rows - 1) * pitch_q + width_q) && q < p + (uint64_t)((rows - 1) * pitch_p + width_p);
}
// base onto y: absent, the very same rows, or apart
static bool base_ok(uint64_t base, int64_t ldb, uint64_t y, int64_t ldy, int64_t cols, int64_t rows) {
    return !base || (base == y && ldb == ldy) || !rows_meet(base, ldb * 4, cols * 4, y, ldy * 4, cols * 4, rows);
}

static int32_t rows_check(const qm_lora *l, uint64_t x_dev, uint64_t x2_dev, int32_t m, int64_t ldx, uint64_t ids_dev,
                          uint64_t base_dev, int64_t ldb, uint64_t y_dev, int64_t ldy, uint32_t flags) {
    const uint32_t xop = flags & 0xFu;
    if (m < 1 || m > 8 || ldx < l->cols || ldy < l->rows || (base_dev && ldb < l->rows)) return QM_ERR_SHAPE;
    if (ldx > (1 << 30) || ldy > (1 << 30) || ldb > (1 << 30)) return QM_ERR_SHAPE;
    if (xop > QM_XOP_SWIGLU || (flags & ~(0xFu | QM_FLAG_PDL))) return QM_ERR_ARG;
    if (!x_dev || !y_dev || (x_dev & 15) || (ldx & 3) || ((ids_dev | base_dev | y_dev) & 3)) return QM_ERR_ARG;
    const bool two = xop == QM_XOP_ADD_RMSNORM || xop == QM_XOP_SWIGLU;
    if (two && (!x2_dev || (x2_dev & 15))) return QM_ERR_ARG;
    if (!base_ok(base_dev, ldb, y_dev, ldy, l->rows, m) || rows_meet(x_dev, ldx * 4, l->cols * 4, y_dev, ldy * 4, l->rows * 4, m) ||
        (two && rows_meet(x2_dev, ldx * 4, l->cols * 4, y_dev, ldy * 4, l->rows * 4, m)) ||
        rows_meet(ids_dev, 4, 4, y_dev, ldy * 4, l->rows * 4, m))
        return QM_ERR_ARG;
    return QM_OK;
}

static int32_t rows_launch(qm_ctx *c, const qm_lora *l, uint64_t x_dev, uint64_t x2_dev, int32_t m, int64_t ldx, uint64_t ids_dev,
                           uint64_t base_dev, int64_t ldb, uint64_t y_dev, int64_t ldy, uint32_t flags) {
    QmLoraRowsArgs a;
    memset(&a, 0, sizeof a);
    a.x = (const float *)(uintptr_t)x_dev;
    a.x2 = (const float *)(uintptr_t)x2_dev;
    a.ids = (const int32_t *)(uintptr_t)ids_dev;
    a.base = (const float *)(uintptr_t)base_dev;
    a.y = (float *)(uintptr_t)y_dev;
    a.a = (const uint16_t *)(uintptr_t)l->a;
    a.b = (const uint16_t *)(uintptr_t)l->b;
    a.scale = (const float *)(uintptr_t)l->scale;
    a.rank = (const int32_t *)(uintptr_t)l->rank;
    a.ldx = ldx;
    a.ldb = ldb;
    a.ldy = ldy;
    a.rows = (int32_t)l->rows;
    a.cols = (int32_t)l->cols;
    a.np = (int32_t)l->np;
    a.rpad = l->rpad;
    a.slots = l->slots;
    a.m = m;
    a.xop = (int32_t)(flags & 0xFu);
    a.eps = 1e-6f;
    // As many clusters as run at once (one CTA per SM), and none with less than a chunk of columns per CTA. (Eight rows on
    // eight adapters, 6144 columns: 9.2 us; with sixteen clusters, of which one has to wait, 13.6.)
    const int64_t pieces = (l->np + QM_LORA_CLUSTER * QM_LORA_CHUNK - 1) / (QM_LORA_CLUSTER * QM_LORA_CHUNK);
    int64_t clusters = m;
    for (int i = 1; i <= 8; i++) {
        const int64_t parts = std::max<int64_t>(1, std::min<int64_t>(pieces, l->at_once[3] / i));
        a.parts[i - 1] = (int32_t)parts;
        a.width[i - 1] = (int32_t)(((l->np + parts * QM_LORA_CLUSTER - 1) / (parts * QM_LORA_CLUSTER) + 7) & ~(int64_t)7);
        if (i <= m) clusters = std::max(clusters, i * parts);
    }
    return qm_launch_ex(c, QM_K_LORA_ROWS, (unsigned)(clusters * QM_LORA_CLUSTER), 512, (unsigned)rows_smem(l), &a, true, false, QM_LORA_CLUSTER);
}

extern "C" int32_t qm_lora_matvec(qm_ctx *c, qm_lora *l, uint64_t x_dev, uint64_t x2_dev, int32_t m, int64_t ldx, uint64_t ids_dev,
                                  uint64_t base_dev, int64_t ldb, uint64_t y_dev, int64_t ldy, uint32_t flags) {
    CHECK_CTX(c);
    int32_t rc = lora_check(c, l);
    if (!base_dev) ldb = 0;   // (the pitch of nothing: neither refused nor a reason for another kernel)
    if (!rc) rc = rows_check(l, x_dev, x2_dev, m, ldx, ids_dev, base_dev, ldb, y_dev, ldy, flags);
    if (rc) return rc;
    CtxGuard g(c);
    DRV(g.rc);
    return rows_launch(c, l, x_dev, x2_dev, m, ldx, ids_dev, base_dev, ldb, y_dev, ldy, flags);
}

extern "C" int32_t qm_matvec_lora(qm_ctx *c, qm_weight h, qm_lora *l, uint64_t x_dev, uint64_t x2_dev, int32_t m, int64_t ldx,
                                  uint64_t ids_dev, uint64_t y_dev, int64_t ldy, uint32_t flags) {
    CHECK_CTX(c);
    QmWeight *w = qm_weight_from_handle(h);
    int32_t rc = w ? lora_check(c, l) : QM_ERR_ARG;
    if (!rc && (w->rows != l->rows || w->cols != l->cols)) rc = QM_ERR_SHAPE;
    if (!rc) rc = rows_check(l, x_dev, x2_dev, m, ldx, ids_dev, y_dev, ldy, y_dev, ldy, flags);
    if (rc) return rc;
    CtxGuard g(c);
    DRV(g.rc);
    rc = qm_matvec_launch(c, w, x_dev, x2_dev, m, ldx, y_dev, ldy, flags, c->partials_dev, c->tickets_dev);
    if (rc) return rc;
    return rows_launch(c, l, x_dev, x2_dev, m, ldx, ids_dev, y_dev, ldy, y_dev, ldy, flags);
}

// ---- bf16 batches ----------------------------------------------------------------------------------
static int32_t lists_launch(qm_ctx *c, const qm_lora *l, uint64_t ids_dev, int32_t tokens) {
    QmLoraListsArgs a;
    memset(&a, 0, sizeof a);
    a.ids = (const int32_t *)(uintptr_t)ids_dev;
    a.rank = (const int32_t *)(uintptr_t)l->rank;
    a.list = (int32_t *)(uintptr_t)l->list;
    a.offsets = (int32_t *)(uintptr_t)l->offsets;
    a.tiles = (int32_t *)(uintptr_t)l->tiles;
    a.tokens = tokens;
    a.slots = l->slots;
    a.tiles_max = (int32_t)lora_tiles(l, tokens, true);
    return qm_launch(c, QM_K_LORA_LISTS, 1, 1, 1024, (unsigned)((32 * (l->slots + 1) + 1536) * 4 + 256), &a, true);
}

static int32_t batch_args(qm_ctx *c, QmLoraTcArgs *ta, const qm_lora *l, uint64_t x, int64_t ldx, uint64_t dy, int64_t lddy, uint64_t ids_dev,
                          int32_t tokens) {
    memset(ta, 0, sizeof *ta);
    QmLoraBatchArgs *a = &ta->b;
    const uint64_t in[2] = {x, dy}, wt[2] = {l->at, l->bt};
    const int64_t ld[2] = {ldx, lddy}, cols[2] = {l->cols, l->rows};
    for (int i = 0; i < 2; i++) {
        QmLoraSide &s = a->side[i];
        s.wt = (const uint16_t *)(uintptr_t)wt[i];
        s.low = (uint16_t *)(uintptr_t)l->low[i];
        s.cols = (int32_t)cols[i];
        ta->w[i] = l->w_map[i];
        ta->low[i] = l->low_map[i];
        if (in[i]) {
            DRV(tensor_map(c, &ta->gather[i], in[i], cols[i], tokens, ld[i], 1));
            DRV(tensor_map(c, &ta->rows[i], in[i], cols[i], tokens, ld[i], 32));
        }
    }
    a->list = ids_dev ? (const int32_t *)(uintptr_t)l->list : nullptr;
    a->offsets = (const int32_t *)(uintptr_t)l->offsets;
    a->tiles = (const int32_t *)(uintptr_t)l->tiles;
    a->scale = (const float *)(uintptr_t)l->scale;
    a->rank = (const int32_t *)(uintptr_t)l->rank;
    a->status = (unsigned int *)(uintptr_t)c->status_dev;
    a->tokens = tokens;
    a->tiles_max = (int32_t)lora_tiles(l, tokens, ids_dev != 0);
    a->rpad = l->rpad;
    a->slots = l->slots;
    a->max_rank = l->max_rank;
    return QM_OK;
}

// CTAs that share one piece of work of `steps` steps, `per_sm` CTAs on an SM: 1, 2, 4 or 8, whichever takes the fewest steps
// in all, a CTA's start and end counted as ten. (Clusters of eight leave 28 of the 148 SMs idle.)
static int32_t share(const qm_lora *l, int64_t units, int64_t steps, int per_sm) {
    int32_t best = 1;
    int64_t least = INT64_MAX;
    for (int i = 0; i < 4; i++) {
        const int32_t s = 1 << i;
        const int64_t clusters = (int64_t)per_sm * std::max(1, l->at_once[i]);
        const int64_t cost = (units + clusters - 1) / clusters * ((steps + s - 1) / s + 10);
        if (cost < least) {
            least = cost;
            best = s;
        }
    }
    return best;
}

// Clusters of `split` CTAs that run at once, `per_sm` CTAs on an SM.
static int64_t at_once(const qm_lora *l, int32_t split, int per_sm) {
    return (int64_t)per_sm * std::max(1, l->at_once[split == 1 ? 0 : split == 2 ? 1 : split == 4 ? 2 : 3]);
}
// How many tiles there are only the device knows, so the grids are made for every adapter having tokens. A CTA without a tile
// costs about 1 ns of the whole (4 ns where it asks for tensor memory): thousands of them are a loss with hundreds of slots of
// which few are in use, and then _m kernels with a grid that fills the GPU a few times take one tile after another. 256 slots,
// four in use: 391 tokens, 28672 x 4096, rank 32: 39 us instead of 96; 2048 tokens, 4096 x 4096, rank 16: 31 instead of 43. With
// all 256 in use they take 247 instead of 261 and 104 instead of 102. For every grid they would cost 5 % (2048 tokens, four
// slots: 28.5 instead of 26.6), and for both sides of a backward pass, whose next kernel starts while the last tiles are worked
// on, 5 % too (2048 tokens, four of 256 slots: 357 us instead of 341).
constexpr int64_t IDLE_SHRINK = 1024, IDLE_EXPAND = 8192;

static int32_t shrink_launch(qm_ctx *c, const qm_lora *l, QmLoraTcArgs *ta, int sides) {
    QmLoraBatchArgs *a = &ta->b;
    const int64_t cols = sides == 2 ? std::max(l->cols, l->rows) : l->cols;
    const int64_t whole = sides * (((int64_t)a->tokens + QM_LORA_TILE - 1) / QM_LORA_TILE);
    a->first_side = sides == 2 && l->rows > l->cols;   // the longer one first, the shorter one fills its last wave
    // (the tiles that are there for certain; those that short lists add come on top)
    a->split = share(l, whole, (cols + 63) / 64, 2);
    int64_t clusters = sides * (int64_t)a->tiles_max;
    const bool many = sides == 1 && (clusters - whole) * a->split > IDLE_SHRINK;
    if (many) clusters = std::min(clusters, std::max(whole, 2 * at_once(l, a->split, 2)));
    return qm_launch_ex(c, (many ? QM_K_LORA_SHRINK_R16_M : QM_K_LORA_SHRINK_R16) + rank_kernel(l), (unsigned)(clusters * a->split), 192,
                        (unsigned)shrink_smem(l), ta, true, false, a->split);
}

static int32_t expand_launch(qm_ctx *c, const qm_lora *l, QmLoraBatchArgs *a, int out_side, uint64_t base, int64_t ldb, uint64_t y,
                             int64_t ldy) {
    a->out_side = out_side;
    a->base = (const float *)(uintptr_t)base;
    a->ldb = ldb;
    a->y = (float *)(uintptr_t)y;
    a->ldy = ldy;
    const bool vec = !((base | y) & 15) && !((ldb | ldy) & 3) && a->side[out_side].cols % 4 == 0;
    const int rp = l->rpad / 16, threads = QM_LORA_EXPAND_WARPS(rp) * 32, across = (a->side[out_side].cols + threads - 1) / threads;
    const int64_t whole = ((int64_t)a->tokens + 63) / 64;
    int64_t halves = 2 * (int64_t)a->tiles_max;
    const bool many = vec && (halves - whole) * across > IDLE_EXPAND;
    // (an odd number: the halves of a CTA are first and second ones in turn, second ones are often empty)
    if (many) halves = std::min(halves, std::max<int64_t>(whole, 8ll * c->sm_count / across) | 1);
    return qm_launch(c, (many ? QM_K_LORA_EXPAND_R16_M : vec ? QM_K_LORA_EXPAND_R16 : QM_K_LORA_EXPAND_R16_S) + rank_kernel(l), (unsigned)halves,
                     (unsigned)across, (unsigned)threads,
                     (unsigned)(threads * 256 + 64 * QM_LORA_EXPAND_ROW(rp)), a, true);
}

static int32_t outer_launch(qm_ctx *c, const qm_lora *l, QmLoraTcArgs *ta, bool listed, uint64_t da, uint64_t db) {
    QmLoraBatchArgs *a = &ta->b;
    a->side[0].grad = (float *)(uintptr_t)da;
    a->side[0].grad_slot = (int64_t)l->max_rank * l->cols;
    a->side[0].grad_rank = l->cols;
    a->side[0].grad_col = 1;
    a->side[1].grad = (float *)(uintptr_t)db;
    a->side[1].grad_slot = (int64_t)l->max_rank * l->rows;
    a->side[1].grad_rank = 1;
    a->side[1].grad_col = l->max_rank;
    const int rp = l->rpad / 16, bn = QM_LORA_OUTER_COLS(rp);
    const int64_t ba = (l->cols + bn - 1) / bn, bb = (l->rows + bn - 1) / bn;
    const int64_t slots = listed ? std::min(l->slots, a->tokens) : 1;
    a->outer_units = (int32_t)(std::max(ba, bb) * l->slots);
    a->split = share(l, ((da ? ba : 0) + (db ? bb : 0)) * slots, (a->tokens / slots + 63) / 64, 1);
    return qm_launch_ex(c, QM_K_LORA_OUTER_R16 + rank_kernel(l), (unsigned)(2 * a->outer_units * a->split), (QM_LORA_OUTER_READERS(rp) + 2) * 32,
                        (unsigned)outer_smem(l), ta, true, false, a->split);
}

static int32_t batch_check(const qm_lora *l, uint64_t x, int64_t ldx, int32_t tokens, uint64_t ids_dev, uint64_t base, int64_t ldb,
                           uint64_t y, int64_t ldy, int64_t in_cols, int64_t out_cols) {
    if (tokens < 0 || ldx < in_cols || ldy < out_cols || (base && ldb < out_cols)) return QM_ERR_SHAPE;
    if (ldx > (1 << 30) || ldy > (1 << 30) || ldb > (1 << 30)) return QM_ERR_SHAPE;
    if (tokens > l->max_tokens) return QM_ERR_LIMIT;
    if (tokens == 0) return QM_OK;
    if (!x || !y || (x & 15) || (ldx & 7) || ((ids_dev | base | y) & 3)) return QM_ERR_ARG;
    if (!base_ok(base, ldb, y, ldy, out_cols, tokens) || rows_meet(x, ldx * 2, in_cols * 2, y, ldy * 4, out_cols * 4, tokens) ||
        rows_meet(ids_dev, 4, 4, y, ldy * 4, out_cols * 4, tokens))
        return QM_ERR_ARG;
    return QM_OK;
}

// Up to QM_LORA_FEW tokens: one launch.
static int32_t few_launch(qm_ctx *c, const qm_lora *l, uint64_t x, int32_t tokens, int64_t ldx, uint64_t ids_dev, uint64_t base, int64_t ldb,
                          uint64_t y, int64_t ldy) {
    QmLoraFewArgs a;
    memset(&a, 0, sizeof a);
    a.x = (const uint16_t *)(uintptr_t)x;
    a.ids = (const int32_t *)(uintptr_t)ids_dev;
    a.base = (const float *)(uintptr_t)base;
    a.y = (float *)(uintptr_t)y;
    a.a = (const uint16_t *)(uintptr_t)l->a;
    a.bt = (const uint16_t *)(uintptr_t)l->bt;
    a.scale = (const float *)(uintptr_t)l->scale;
    a.rank = (const int32_t *)(uintptr_t)l->rank;
    a.ldx = ldx;
    a.ldb = ldb;
    a.ldy = ldy;
    a.rows = (int32_t)l->rows;
    a.cols = (int32_t)l->cols;
    a.np = (int32_t)l->np;
    a.slots = l->slots;
    a.tokens = tokens;
    a.pieces = (int32_t)((l->np + QM_LORA_CLUSTER * 256 - 1) / (QM_LORA_CLUSTER * 256));
    const int64_t most = ids_dev ? tokens : (tokens + 15) / 16;   // items
    a.at_once = l->few_at_once;
    const int64_t clusters = std::max(most, std::min<int64_t>(l->few_at_once, most * a.pieces));
    const bool vec = !((base | y) & 7) && !((ldb | ldy) & 1);
    return qm_launch_ex(c, (vec ? QM_K_LORA_FEW_R16 : QM_K_LORA_FEW_R16_S) + rank_kernel(l), (unsigned)(clusters * QM_LORA_CLUSTER), 256,
                        (unsigned)few_smem(l), &a, true, false, QM_LORA_CLUSTER);
}

static int32_t batch_launch(qm_ctx *c, const qm_lora *l, uint64_t x, int32_t tokens, int64_t ldx, uint64_t ids_dev, uint64_t base,
                            int64_t ldb, uint64_t y, int64_t ldy) {
    if (tokens <= QM_LORA_FEW) return few_launch(c, l, x, tokens, ldx, ids_dev, base, ldb, y, ldy);
    if (ids_dev) {
        int32_t rc = lists_launch(c, l, ids_dev, tokens);
        if (rc) return rc;
    }
    QmLoraTcArgs a;
    int32_t rc = batch_args(c, &a, l, x, ldx, 0, 0, ids_dev, tokens);
    if (!rc) rc = shrink_launch(c, l, &a, 1);
    if (rc) return rc;
    return expand_launch(c, l, &a.b, 1, base, ldb, y, ldy);
}

extern "C" int32_t qm_lora_matmul_bf16(qm_ctx *c, qm_lora *l, uint64_t x_bf16_dev, int32_t tokens, int64_t ldx, uint64_t ids_dev,
                                       uint64_t base_dev, int64_t ldb, uint64_t y_dev, int64_t ldy) {
    CHECK_CTX(c);
    int32_t rc = lora_check(c, l);
    if (!base_dev) ldb = 0;
    if (!rc) rc = batch_check(l, x_bf16_dev, ldx, tokens, ids_dev, base_dev, ldb, y_dev, ldy, l->cols, l->rows);
    if (rc || tokens == 0) return rc;
    CtxGuard g(c);
    DRV(g.rc);
    return batch_launch(c, l, x_bf16_dev, tokens, ldx, ids_dev, base_dev, ldb, y_dev, ldy);
}

extern "C" int32_t qm_matmul_bf16_lora(qm_ctx *c, qm_weight h, qm_lora *l, uint64_t a_dev, int32_t m, int64_t lda, uint64_t ids_dev,
                                       uint64_t c_dev, int64_t ldc) {
    CHECK_CTX(c);
    QmWeight *w = qm_weight_from_handle(h);
    int32_t rc = w ? lora_check(c, l) : QM_ERR_ARG;
    if (!rc && (w->rows != l->rows || w->cols != l->cols)) rc = QM_ERR_SHAPE;
    if (!rc) rc = batch_check(l, a_dev, lda, m, ids_dev, c_dev, ldc, c_dev, ldc, l->cols, l->rows);
    if (!rc) rc = qm_matmul_bf16(c, h, a_dev, m, lda, c_dev, ldc);   // (no tokens: refused there)
    if (rc) return rc;
    CtxGuard g(c);
    DRV(g.rc);
    return batch_launch(c, l, a_dev, m, lda, ids_dev, c_dev, ldc, c_dev, ldc);
}

// dy where a tensor map takes it: itself, or a copy in the handle (of its full size at once, so that no later call moves it).
static int32_t align_dy(qm_ctx *c, qm_lora *l, uint64_t *dy, int64_t *lddy, int32_t tokens) {
    if (!(*dy & 15) && !(*lddy & 7)) return QM_OK;
    if (!l->aligned) {
        if (int32_t rc = qm_refuse_capture(c)) return rc;
        DRV(c->drv->cuMemAlloc_v2(&l->aligned, (size_t)l->max_tokens * l->np * 2));
    }
    QmLoraAlignArgs a;
    memset(&a, 0, sizeof a);
    a.src = (const uint16_t *)(uintptr_t)*dy;
    a.dst = (uint16_t *)(uintptr_t)l->aligned;
    a.ld = *lddy;
    a.pitch = l->np;
    a.rows = tokens;
    a.cols = (int32_t)l->rows;
    *dy = l->aligned;
    *lddy = l->np;
    const int64_t work = ((int64_t)tokens * l->np / 8 + 255) / 256;
    return qm_launch(c, QM_K_LORA_ALIGN, (unsigned)std::min<int64_t>(work, 8ll * c->sm_count), 1, 256, 0, &a, true);
}

extern "C" int32_t qm_lora_backward(qm_ctx *c, qm_lora *l, uint64_t x_bf16_dev, int64_t ldx, uint64_t dy_bf16_dev, int64_t lddy,
                                    int32_t tokens, uint64_t ids_dev, uint64_t base_dev, int64_t ldb, uint64_t dx_dev, int64_t lddx,
                                    uint64_t da_dev, uint64_t db_dev) {
    CHECK_CTX(c);
    int32_t rc = lora_check(c, l);
    if (rc) return rc;
    if (!dx_dev && !da_dev && !db_dev) return QM_ERR_ARG;
    if (!dx_dev) base_dev = 0, lddx = 0;
    if (!base_dev) ldb = 0;
    if (tokens < 0 || ldx < l->cols || lddy < l->rows || ldx > (1 << 30) || lddy > (1 << 30)) return QM_ERR_SHAPE;
    if (tokens > l->max_tokens) return QM_ERR_LIMIT;
    if (tokens && (!x_bf16_dev || !dy_bf16_dev)) return QM_ERR_ARG;
    if ((x_bf16_dev & 15) || (ldx & 7) || (dy_bf16_dev & 1) || ((ids_dev | da_dev | db_dev) & 3)) return QM_ERR_ARG;
    const int64_t na = (int64_t)l->slots * l->max_rank * l->cols, nb = (int64_t)l->slots * l->max_rank * l->rows;
    if (dx_dev) {
        rc = batch_check(l, x_bf16_dev, ldx, tokens, ids_dev, base_dev, ldb, dx_dev, lddx, l->cols, l->cols);
        if (rc) return rc;
        if (tokens && rows_meet(dy_bf16_dev, lddy * 2, l->rows * 2, dx_dev, lddx * 4, l->cols * 4, tokens)) return QM_ERR_ARG;
    }
    // a gradient of A or B on nothing else
    const struct {
        uint64_t p;
        int64_t bytes;
    } span[] = {{da_dev, na * 4}, {db_dev, nb * 4}, {dx_dev, ((tokens - 1) * lddx + l->cols) * 4}, {base_dev, ((tokens - 1) * ldb + l->cols) * 4},
                {x_bf16_dev, ((tokens - 1) * ldx + l->cols) * 2}, {dy_bf16_dev, ((tokens - 1) * lddy + l->rows) * 2}, {ids_dev, tokens * 4ll}};
    for (int i = 0; i < 2; i++)
        for (int k = i + 1; k < 7 && tokens; k++)
            if (span[i].p && span[k].p && span[i].p < span[k].p + (uint64_t)span[k].bytes && span[k].p < span[i].p + (uint64_t)span[i].bytes) return QM_ERR_ARG;
    CtxGuard g(c);
    DRV(g.rc);
    if (tokens == 0) {
        if (da_dev) DRV(c->drv->cuMemsetD8Async(da_dev, 0, (size_t)na * 4, c->stream));
        if (db_dev) DRV(c->drv->cuMemsetD8Async(db_dev, 0, (size_t)nb * 4, c->stream));
        return QM_OK;
    }
    if (ids_dev) {
        rc = lists_launch(c, l, ids_dev, tokens);
        if (rc) return rc;
    }
    rc = align_dy(c, l, &dy_bf16_dev, &lddy, tokens);
    if (rc) return rc;
    QmLoraTcArgs ta;
    rc = batch_args(c, &ta, l, x_bf16_dev, ldx, dy_bf16_dev, lddy, ids_dev, tokens);
    if (!rc) rc = shrink_launch(c, l, &ta, 2);
    if (rc) return rc;
    QmLoraBatchArgs &a = ta.b;
    // dx and the gradients of A and B need nothing of each other: with both wanted dx goes beside the others, on a stream of
    // the handle (777 tokens, 6144 x 4096, rank 8: 53 -> 44 us)
    const bool grads = da_dev || db_dev, both = dx_dev && grads;
    CUstream main = c->stream;
    if (both) {
        DRV(c->drv->cuEventRecord(l->fork, main));
        DRV(c->drv->cuStreamWaitEvent(l->side, l->fork, 0));
    }
    // (first, so that its CTAs, one to an SM, find their place)
    if (grads) rc = outer_launch(c, l, &ta, ids_dev != 0, da_dev, db_dev);
    if (both) c->stream = l->side;
    if (dx_dev && !rc) rc = expand_launch(c, l, &ta.b, 0, base_dev, ldb, dx_dev, lddx);
    c->stream = main;
    if (both) {   // whatever became of the launches
        DRV(c->drv->cuEventRecord(l->join, l->side));
        DRV(c->drv->cuStreamWaitEvent(main, l->join, 0));
    }
    return rc;
}
