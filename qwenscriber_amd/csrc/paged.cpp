// C ABI entry points of the paged key/value cache.
#include <cmath>
#include <new>
#include <vector>

#include "common.h"
#include "paged.h"

using namespace qwh;

namespace {

int32_t refused(qwh_ctx *ctx, const paged::Refusal &r) { return fail(ctx, r.status, "%s", r.why); }

#define QWH_REFUSE(expr)                                             \
    do {                                                             \
        const paged::Refusal qwh_refusal_ = (expr);                  \
        if (qwh_refusal_.status != QWH_OK) return refused(ctx, qwh_refusal_); \
    } while (0)

}  // namespace

extern "C" {

int32_t qwh_paged_append(qwh_ctx *ctx, const qwh_paged_cache *cache, uint32_t layer, const qwh_paged_batch *batch,
                         const float *qkv_dev, uint32_t qkv_stride, uint32_t heads, const float *q_norm_dev,
                         const float *k_norm_dev, float eps, const float *rope_cos_dev, const float *rope_sin_dev,
                         uint32_t rope_positions, float *query_dev, uint32_t query_stride) {
    if (!ctx) return QWH_E_INVALID_ARGUMENT;
    QWH_REFUSE(paged::check_cache(cache));
    QWH_REFUSE(paged::check_layer(*cache, layer));
    QWH_REFUSE(paged::check_batch(batch));
    QWH_REFUSE(paged::check_heads(*cache, heads));
    QWH_REFUSE(paged::check_positions(*cache, *batch));
    QWH_REFUSE(paged::check_row_heads(*batch, heads));
    if (!(eps >= 0.0f)) return fail(ctx, QWH_E_INVALID_ARGUMENT, "eps is not a number from 0 on");
    if (paged::nothing_to_do(*batch)) return QWH_OK;
    const uint64_t D = cache->head_dim;
    QWH_REFUSE(paged::check_rows(qkv_dev, qkv_stride, (heads + 2ull * cache->kv_heads) * D, "qkv is null",
                                 "qkv_stride is smaller than a row"));
    QWH_REFUSE(paged::check_rows(query_dev, query_stride, heads * D, "query is null", "query_stride is smaller than a row"));
    if (query_dev == qkv_dev && query_stride != qkv_stride)
        return fail(ctx, QWH_E_INVALID_ARGUMENT, "a query written in place takes qkv's stride");
    QWH_REFUSE(paged::check_floats(q_norm_dev, k_norm_dev, rope_cos_dev, rope_sin_dev));
    OnDevice device(ctx->device);
    QWH_TRY(on_device(ctx, device));
    PagedAppendArgs a{};
    a.cache = paged_layer(*cache, layer);
    a.batch = *batch;
    a.qkv = qkv_dev;
    a.qkv_stride = qkv_stride;
    a.heads = heads;
    a.q_norm = q_norm_dev;
    a.k_norm = k_norm_dev;
    a.rope_cos = rope_cos_dev;
    a.rope_sin = rope_sin_dev;
    a.eps = eps;
    const uint64_t held = (uint64_t)batch->table_pages * cache->page_size;
    a.positions = held < rope_positions ? held : rope_positions;
    a.query = query_dev;
    a.query_stride = query_stride;
    return check_hip(ctx, launch_paged_append(ctx->stream, a), "paged append");
}

int32_t qwh_paged_attention(qwh_ctx *ctx, const qwh_paged_cache *cache, uint32_t layer, const qwh_paged_batch *batch,
                            float *out_dev, const float *query_dev, uint32_t query_stride, uint32_t heads) {
    if (!ctx) return QWH_E_INVALID_ARGUMENT;
    QWH_REFUSE(paged::check_cache(cache));
    QWH_REFUSE(paged::check_layer(*cache, layer));
    QWH_REFUSE(paged::check_batch(batch));
    QWH_REFUSE(paged::check_heads(*cache, heads));
    QWH_REFUSE(paged::check_positions(*cache, *batch));
    QWH_REFUSE(paged::check_row_heads(*batch, heads));
    if (paged::nothing_to_do(*batch)) return QWH_OK;
    QWH_REFUSE(paged::check_units(*cache, *batch, heads));
    const uint64_t width = (uint64_t)heads * cache->head_dim;
    QWH_REFUSE(paged::check_rows(query_dev, query_stride, width, "query is null", "query_stride is smaller than a row"));
    QWH_REFUSE(paged::check_rows(out_dev, (uint32_t)width, width, "out is null", ""));
    OnDevice device(ctx->device);
    QWH_TRY(on_device(ctx, device));
    PagedAttentionArgs a{};
    a.cache = paged_layer(*cache, layer);
    a.batch = *batch;
    a.out = out_dev;
    a.query = query_dev;
    a.query_stride = query_stride;
    a.heads = heads;
    QWH_TRY(ensure_workspace(ctx, ctx->scratch, paged_attention_scratch_bytes(ctx->cus, a)));
    return check_hip(ctx, launch_paged_attention(ctx->stream, ctx->cus, a, ctx->scratch.ptr, ctx->scratch.bytes),
                     "paged attention");
}

int32_t qwh_paged_copy(qwh_ctx *ctx, const qwh_paged_cache *cache, const uint32_t *src_pages, const uint32_t *dst_pages,
                       uint32_t count) {
    if (!ctx) return QWH_E_INVALID_ARGUMENT;
    QWH_REFUSE(paged::check_cache(cache));
    if (count == 0) return QWH_OK;
    if (!src_pages || !dst_pages) return fail(ctx, QWH_E_INVALID_ARGUMENT, "src_pages or dst_pages is null");
    QWH_REFUSE(paged::check_page(*cache));
    paged::CopyLaunches plan(cache->pages <= paged::kShortPages);
    try {
        paged::CopyPairs pairs;
        QWH_REFUSE(paged::check_copies(src_pages, dst_pages, count, cache->pages, pairs));
        paged::order_copies(pairs, plan);
    } catch (const std::bad_alloc &) {
        return fail(ctx, QWH_E_OUT_OF_MEMORY, "no host memory to order %u copies", count);
    }
    OnDevice device(ctx->device);
    QWH_TRY(on_device(ctx, device));
    for (const paged::CopyLaunch &launch : plan.launches)
        QWH_TRY(check_hip(ctx, launch_paged_copy(ctx->stream, *cache, launch, plan.is_short), "paged copy"));
    return QWH_OK;
}

int32_t qwh_rope_tables(qwh_ctx *ctx, uint32_t head_dim, uint32_t positions, float theta, float *cos_dev, float *sin_dev) {
    if (!ctx) return QWH_E_INVALID_ARGUMENT;
    if (head_dim < 2 || head_dim % 2 != 0) return fail(ctx, QWH_E_SHAPE_MISMATCH, "head_dim %u is not even", head_dim);
    if (!(theta > 0.0f)) return fail(ctx, QWH_E_INVALID_ARGUMENT, "theta is not above 0");
    if (positions == 0) return QWH_OK;
    if (!cos_dev || !sin_dev) return fail(ctx, QWH_E_INVALID_ARGUMENT, "cos or sin is null");
    if ((uint64_t)positions * (head_dim / 2) > (1ull << 32))
        return fail(ctx, QWH_E_LIMIT_EXCEEDED, "rotation tables of more than 2^32 values");
    std::vector<float> cos_t, sin_t;
    try {
        build_rope_tables(cos_t, sin_t, head_dim / 2, theta, positions);
    } catch (const std::bad_alloc &) {
        return fail(ctx, QWH_E_OUT_OF_MEMORY, "no host memory for the rotation tables");
    }
    OnDevice device(ctx->device);
    QWH_TRY(on_device(ctx, device));
    QWH_TRY(check_hip(ctx, hipMemcpyAsync(cos_dev, cos_t.data(), cos_t.size() * 4, hipMemcpyHostToDevice, ctx->stream), "rope"));
    const int32_t st =
        check_hip(ctx, hipMemcpyAsync(sin_dev, sin_t.data(), sin_t.size() * 4, hipMemcpyHostToDevice, ctx->stream), "rope");
    // (Also after a failure: the tables leave with this call.)
    const int32_t sync = check_hip(ctx, hipStreamSynchronize(ctx->stream), "rope sync");
    return st != QWH_OK ? st : sync;
}

}  // extern "C"
