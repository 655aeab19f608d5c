// qm_rope.cpp — host side of the norm and rotation of query and key heads (include/qmatmul.h): the handle with the
// rotation's frequencies, the forward pass and its gradient.
#include <math.h>
#include <string.h>

#include <algorithm>
#include <new>
#include <vector>

#include "qm_internal.h"

#define QM_ROPE_MAGIC 0x514D5250u  // "QMRP"
#define QM_ROPE_MAX_DIM 512

struct qm_rope {
    uint32_t magic;
    qm_ctx *ctx;
    int32_t dim, rot, interleaved;
    CUdeviceptr freq;       // [rot/2]: turns per position, in units of 2^-64, whole turns dropped
    CUdeviceptr partial;    // backward: [grad_ctas][dim]
    int32_t grad_ctas;
};

extern "C" int32_t qm_rope_create(qm_ctx *c, int32_t head_dim, int32_t rot_dim, float theta, const float *factors,
                                  uint32_t flags, qm_rope **out) {
    CHECK_CTX(c);
    if (!out) return QM_ERR_ARG;
    *out = nullptr;
    if (head_dim < 2 || (head_dim & 1) || rot_dim < 0 || (rot_dim & 1) || rot_dim > head_dim) return QM_ERR_SHAPE;
    if (head_dim > QM_ROPE_MAX_DIM) return QM_ERR_LIMIT;
    if ((flags & ~QM_ROPE_INTERLEAVED) || !(theta > 0.f) || isinf(theta)) return QM_ERR_ARG;
    std::vector<uint64_t> freq;
    try {
        freq.resize(rot_dim / 2 + 1);
    } catch (const std::bad_alloc &) {
        return QM_ERR_NOMEM;
    }
    for (int i = 0; i < rot_dim / 2; i++) {
        const double f = factors ? (double)factors[i] : 1.0;
        if (!(f > 0.0) || isinf(f)) return QM_ERR_ARG;
        const long double turns = powl((long double)theta, -2.0l * i / rot_dim) / (long double)f / (2.0l * acosl(-1.0l));
        if (!isfinite(turns)) return QM_ERR_ARG;
        freq[i] = (uint64_t)ldexpl(turns - floorl(turns), 64);
    }
    CtxGuard g(c);
    DRV(g.rc);
    if (int32_t rc = qm_refuse_capture(c)) return rc;   // (the copy below would run again with the graph, from this frame)
    qm_rope *r = new (std::nothrow) qm_rope();
    if (!r) return QM_ERR_NOMEM;
    r->magic = QM_ROPE_MAGIC;
    r->ctx = c;
    r->dim = head_dim;
    r->rot = rot_dim;
    r->interleaved = (flags & QM_ROPE_INTERLEAVED) ? 1 : 0;
    r->grad_ctas = 3 * c->sm_count;   // the most that qm_qk_norm_rope_backward launches
    CUresult e = c->drv->cuMemAlloc_v2(&r->freq, freq.size() * sizeof(uint64_t));
    if (e == CUDA_SUCCESS) e = c->drv->cuMemAlloc_v2(&r->partial, (size_t)r->grad_ctas * head_dim * sizeof(float));
    // (a copy on the default stream may return before it has arrived, and nothing orders the context's streams behind it)
    if (e == CUDA_SUCCESS) e = c->drv->cuMemcpyHtoDAsync_v2(r->freq, freq.data(), freq.size() * sizeof(uint64_t), c->stream);
    if (e == CUDA_SUCCESS) e = c->drv->cuStreamSynchronize(c->stream);
    if (e != CUDA_SUCCESS) {
        if (r->freq) c->drv->cuMemFree_v2(r->freq);
        if (r->partial) c->drv->cuMemFree_v2(r->partial);
        delete r;
        return (int32_t)e;
    }
    *out = r;
    return QM_OK;
}

extern "C" int32_t qm_rope_destroy(qm_ctx *c, qm_rope *r) {
    CHECK_CTX(c);
    if (!r || r->magic != QM_ROPE_MAGIC || r->ctx != c) return QM_ERR_ARG;
    CtxGuard g(c);
    DRV(g.rc);
    c->drv->cuStreamSynchronize(c->stream);
    c->drv->cuMemFree_v2(r->freq);
    c->drv->cuMemFree_v2(r->partial);
    r->magic = 0;
    delete r;
    return QM_OK;
}

// Bytes [lo, hi) of `rows` rows of `width` bytes, `pitch` bytes apart.
struct Span {
    uint64_t lo, hi;
};
static Span span_of(uint64_t base, int64_t rows, int64_t pitch, int64_t width) {
    return {base, base + (uint64_t)((rows - 1) * pitch + width)};
}
static bool overlap(const Span &a, const Span &b) { return a.lo < b.hi && b.lo < a.hi; }
// A result on the positions or a gain.
static bool on_small(const Span &out, uint64_t pos, int64_t tokens, uint64_t gq, uint64_t gk, int64_t dim) {
    return (pos && overlap(out, span_of(pos, tokens, 4, 4))) || (gq && overlap(out, span_of(gq, 1, 0, dim * 4))) ||
           (gk && overlap(out, span_of(gk, 1, 0, dim * 4)));
}

// Without the norm gains and eps do not count, whatever they are.
static void drop_unused(uint64_t *gq, uint64_t *gk, float *eps, uint32_t flags) {
    if (!(flags & QM_QK_NO_NORM)) return;
    *gq = *gk = 0;
    *eps = 0.f;
}

// What both directions ask of their arguments. `out`: dx of the backward pass (0 forward); q and k are results or their
// gradients. Results may lie on the raw heads they come from, place for place; any other overlap of a result is refused.
static int32_t check(qm_ctx *c, const qm_rope *r, uint64_t x, int64_t ldx, int32_t tokens, int32_t hq, int32_t hk, uint64_t gq,
                     uint64_t gk, float eps, uint64_t pos, uint64_t q, int64_t ldq, uint64_t k, int64_t ldk, uint32_t flags) {
    if (!r || r->magic != QM_ROPE_MAGIC || r->ctx != c) return QM_ERR_ARG;
    if (flags & ~(QM_QK_NO_NORM | QM_QK_BF16)) return QM_ERR_ARG;
    if (tokens < 0 || hq < 0 || hk < 0 || (int64_t)hq + hk < 1 || (int64_t)hq + hk > (1 << 20)) return QM_ERR_SHAPE;
    // (the backward pass steps a token number past the last one, and spans of rows are counted in 64-bit bytes)
    if (tokens > (1 << 30)) return QM_ERR_LIMIT;
    const int64_t dim = r->dim;
    if (ldx < (hq + (int64_t)hk) * dim || ldq < hq * dim || ldk < hk * dim) return QM_ERR_SHAPE;
    if (ldx > (1 << 30) || ldq > (1 << 30) || ldk > (1 << 30)) return QM_ERR_SHAPE;
    if (!(eps >= 0.f) || isinf(eps)) return QM_ERR_SHAPE;
    if (tokens == 0) return QM_OK;
    const uint64_t part = (flags & QM_QK_BF16) ? 1 : 3;
    if (!x || !pos || (hq && !q) || (hk && !k)) return QM_ERR_ARG;
    if (((x | pos | gq | gk) & 3) || (hq && (q & part)) || (hk && (k & part))) return QM_ERR_ARG;
    return QM_OK;
}

static void fill(QmQkArgs *a, const qm_rope *r, uint64_t x, int64_t ldx, int32_t tokens, int32_t hq, int32_t hk, uint64_t gq,
                 uint64_t gk, float eps, uint64_t pos, uint64_t q, int64_t ldq, uint64_t k, int64_t ldk, uint32_t flags) {
    memset(a, 0, sizeof *a);
    a->x = (const float *)(uintptr_t)x;
    a->gain_q = (const float *)(uintptr_t)gq;
    a->gain_k = (const float *)(uintptr_t)gk;
    a->pos = (const int32_t *)(uintptr_t)pos;
    a->freq = (const uint64_t *)(uintptr_t)r->freq;
    a->q = (void *)(uintptr_t)q;
    a->k = (void *)(uintptr_t)k;
    a->ldx = ldx;
    a->ldq = ldq;
    a->ldk = ldk;
    a->tokens = tokens;
    a->hq = hq;
    a->hk = hk;
    a->dim = r->dim;
    a->rot = r->rot;
    a->interleaved = r->interleaved;
    a->norm = (flags & QM_QK_NO_NORM) ? 0 : 1;
    a->eps = eps;
    a->inv_dim = 1.f / (float)r->dim;
}

// Two neighbouring pairs per lane: whole vectors of two elements everywhere. Otherwise one.
static bool vectors(const QmQkArgs &a, bool bf16, uint64_t f32_ptrs, int64_t f32_lds) {
    const uint64_t part = bf16 ? 3 : 7;
    const uint64_t qk = (a.hq ? (uint64_t)(uintptr_t)a.q : 0) | (a.hk ? (uint64_t)(uintptr_t)a.k : 0);
    const int64_t lds = f32_lds | (a.hq ? a.ldq : 0) | (a.hk ? a.ldk : 0);
    return a.dim % 4 == 0 && a.rot % 4 == 0 && !(f32_ptrs & 7) && !(qk & part) && !(lds & 1);
}

// The slots of a lane, and with them the kernel: 0, 1, 2 for vectors of two, 3 for single elements.
static int form(const QmQkArgs &a, bool vec) { return !vec ? 3 : a.dim <= 128 ? 0 : a.dim <= 256 ? 1 : 2; }

// As many warps as the device holds before a warp gets a second head of its token; then up to `most` heads share the angles.
// The groups of heads of a token (grid y, which holds 65535).
static int64_t deal(const qm_ctx *c, QmQkArgs *a, int64_t most, int64_t groups_max) {
    const int64_t heads = (int64_t)a->hq + a->hk;
    const int64_t least = (heads + groups_max - 2) / (groups_max - 1);
    a->chunk = (int32_t)std::max(least, std::min(std::min(most, heads), a->tokens * heads / (64 * (int64_t)c->sm_count)));
    a->q_chunks = (a->hq + a->chunk - 1) / a->chunk;
    return a->q_chunks + (a->hk + a->chunk - 1) / a->chunk;
}

extern "C" int32_t qm_qk_norm_rope(qm_ctx *c, qm_rope *r, uint64_t x_dev, int64_t ldx, int32_t tokens, int32_t q_heads,
                                   int32_t k_heads, uint64_t q_gain_dev, uint64_t k_gain_dev, float eps, uint64_t pos_dev,
                                   uint64_t q_out, int64_t ldq, uint64_t k_out, int64_t ldk, uint32_t flags) {
    CHECK_CTX(c);
    drop_unused(&q_gain_dev, &k_gain_dev, &eps, flags);
    int32_t rc = check(c, r, x_dev, ldx, tokens, q_heads, k_heads, q_gain_dev, k_gain_dev, eps, pos_dev, q_out, ldq, k_out, ldk, flags);
    if (rc || tokens == 0) return rc;
    QmQkArgs a;
    fill(&a, r, x_dev, ldx, tokens, q_heads, k_heads, q_gain_dev, k_gain_dev, eps, pos_dev, q_out, ldq, k_out, ldk, flags);
    const bool bf16 = (flags & QM_QK_BF16) != 0;
    const int64_t dim = r->dim, size = bf16 ? 2 : 4;
    const Span x = span_of(x_dev, tokens, ldx * 4, (q_heads + (int64_t)k_heads) * dim * 4);
    const Span q = q_heads ? span_of(q_out, tokens, ldq * size, q_heads * dim * size) : Span{0, 0};
    const Span k = k_heads ? span_of(k_out, tokens, ldk * size, k_heads * dim * size) : Span{0, 0};
    const bool q_on = !bf16 && q_out == x_dev && ldq == ldx;
    const bool k_on = !bf16 && k_out == x_dev + (uint64_t)q_heads * dim * 4 && ldk == ldx;
    if ((q_heads && on_small(q, pos_dev, tokens, q_gain_dev, k_gain_dev, dim)) || (k_heads && on_small(k, pos_dev, tokens, q_gain_dev, k_gain_dev, dim)))
        return QM_ERR_ARG;
    if (q_heads && overlap(q, x) && !q_on) return QM_ERR_ARG;
    if (k_heads && overlap(k, x) && !k_on) return QM_ERR_ARG;
    // side by side in one buffer of rows (q_on and k_on among them) the two do not meet
    if (q_heads && k_heads && overlap(q, k)) {
        const int64_t gap = (int64_t)(k_out - q_out), row = ldq * size;
        const int64_t in = ((gap % row) + row) % row;
        if (ldq != ldk || in < q_heads * dim * size || in + k_heads * dim * size > row) return QM_ERR_ARG;
    }
    const int64_t groups = deal(c, &a, 16, 65535);
    const int kernel = QM_K_QK_NORM_W1 + (bf16 ? 4 : 0) + form(a, vectors(a, bf16, x_dev | q_gain_dev | k_gain_dev, ldx));
    CtxGuard g(c);
    DRV(g.rc);
    return qm_launch(c, kernel, (unsigned)(((int64_t)tokens + 7) / 8), (unsigned)groups, 256, 0, &a, true);
}

extern "C" int32_t qm_qk_norm_rope_backward(qm_ctx *c, qm_rope *r, uint64_t x_dev, int64_t ldx, int32_t tokens, int32_t q_heads,
                                            int32_t k_heads, uint64_t q_gain_dev, uint64_t k_gain_dev, float eps,
                                            uint64_t pos_dev, uint64_t dq_dev, int64_t lddq, uint64_t dk_dev, int64_t lddk,
                                            uint64_t dx_dev, int64_t lddx, uint64_t dq_gain_dev, uint64_t dk_gain_dev,
                                            uint32_t flags) {
    CHECK_CTX(c);
    drop_unused(&q_gain_dev, &k_gain_dev, &eps, flags);
    int32_t rc = check(c, r, x_dev, ldx, tokens, q_heads, k_heads, q_gain_dev, k_gain_dev, eps, pos_dev, dq_dev, lddq, dk_dev, lddk, flags);
    if (rc) return rc;
    const int64_t dim = r->dim, heads = (int64_t)q_heads + k_heads;
    const bool gains = dq_gain_dev || dk_gain_dev;
    if (lddx < heads * dim || lddx > (1 << 30)) return QM_ERR_SHAPE;
    if ((tokens && !dx_dev) || ((dx_dev | dq_gain_dev | dk_gain_dev) & 3)) return QM_ERR_ARG;
    if (gains && (flags & QM_QK_NO_NORM)) return QM_ERR_ARG;   // there is no gain without the norm
    CtxGuard g(c);
    DRV(g.rc);
    if (tokens == 0) {
        if (dq_gain_dev) DRV(c->drv->cuMemsetD8Async(dq_gain_dev, 0, (size_t)dim * 4, c->stream));
        if (dk_gain_dev) DRV(c->drv->cuMemsetD8Async(dk_gain_dev, 0, (size_t)dim * 4, c->stream));
        return QM_OK;
    }
    QmQkArgs a;
    fill(&a, r, x_dev, ldx, tokens, q_heads, k_heads, q_gain_dev, k_gain_dev, eps, pos_dev, dq_dev, lddq, dk_dev, lddk, flags);
    const bool bf16 = (flags & QM_QK_BF16) != 0;
    const int64_t size = bf16 ? 2 : 4;
    const Span dx = span_of(dx_dev, tokens, lddx * 4, heads * dim * 4);
    if (overlap(dx, span_of(x_dev, tokens, ldx * 4, heads * dim * 4)) && !(dx_dev == x_dev && lddx == ldx)) return QM_ERR_ARG;
    if (q_heads && overlap(dx, span_of(dq_dev, tokens, lddq * size, q_heads * dim * size)) && !(size == 4 && dq_dev == dx_dev && lddq == lddx))
        return QM_ERR_ARG;
    if (k_heads && overlap(dx, span_of(dk_dev, tokens, lddk * size, k_heads * dim * size)) &&
        !(size == 4 && dk_dev == dx_dev + (uint64_t)q_heads * dim * 4 && lddk == lddx))
        return QM_ERR_ARG;
    if (on_small(dx, pos_dev, tokens, q_gain_dev, k_gain_dev, dim) || on_small(dx, 0, 1, dq_gain_dev, dk_gain_dev, dim)) return QM_ERR_ARG;
    if (dq_gain_dev && dk_gain_dev && overlap(span_of(dq_gain_dev, 1, 0, dim * 4), span_of(dk_gain_dev, 1, 0, dim * 4))) return QM_ERR_ARG;
    a.dx = (float *)(uintptr_t)dx_dev;
    a.lddx = lddx;
    a.partial = gains ? (float *)(uintptr_t)r->partial : nullptr;
    // As many CTAs as run at once (registers: three per SM, two, one and one by form), dealt evenly to the groups of heads; a
    // group's CTAs share its tokens. Groups of at most eight heads, so that few tokens more or less per warp weigh little.
    const int f = form(a, vectors(a, bf16, x_dev | q_gain_dev | k_gain_dev | dx_dev, ldx | lddx));
    const int64_t at_once = (f == 0 ? 3 : f == 1 ? 2 : 1) * c->sm_count;
    const int64_t groups = deal(c, &a, 8, at_once);
    const int64_t gx = std::min<int64_t>(((int64_t)tokens + 7) / 8, at_once / groups);
    rc = qm_launch(c, QM_K_QK_GRAD_W1 + (bf16 ? 4 : 0) + f, (unsigned)gx, (unsigned)groups, 256, gains ? (unsigned)(8 * dim * 4) : 0, &a, true);
    if (rc || !gains) return rc;
    QmGainSumArgs s;
    memset(&s, 0, sizeof s);
    s.partial = a.partial;
    s.dq = (float *)(uintptr_t)dq_gain_dev;
    s.dk = (float *)(uintptr_t)dk_gain_dev;
    s.q_ctas = (int32_t)(a.q_chunks * gx);
    s.ctas = (int32_t)(groups * gx);
    s.dim = (int32_t)dim;
    return qm_launch(c, QM_K_QK_GAIN_SUM, (unsigned)((dim + 31) / 32), 2, 1024, 0, &s, true);
}
