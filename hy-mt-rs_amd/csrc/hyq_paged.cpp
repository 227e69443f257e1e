// Entry points of the paged KV cache and of the sampler: checks of arguments
// and launches (kernels in hyq_paged_*.hip, hyq_pages.hip, hyq_sample.hip).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "hyq_abi.hpp"
#include "hyq_paged.hpp"
#include "hyq_paged_attn.hpp"

using namespace hyq;

namespace {

bool aligned(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int type_of(const hyq_kv_layout *kl)
{
    return kl->dtype == HYQ_KV_Q8 ? KV_T_Q8 : kl->dtype == HYQ_F16 ? KV_T_F16 : KV_T_F32;
}

bool dtype_ok(const hyq_kv_layout *kl)
{
    return kl->dtype == HYQ_F32 || kl->dtype == HYQ_F16 || kl->dtype == HYQ_KV_Q8;
}

size_t page_bytes(const hyq_kv_layout *kl)
{
    return (size_t)2 * kl->kv_heads * kl->page_tokens * kv_row_bytes(type_of(kl));
}

bool layout_ok(const hyq_kv_layout *kl)
{
    if (!kl || !dtype_ok(kl)) return false;
    const int pt = kl->page_tokens;
    if (pt < 16 || pt > 256 || (pt & (pt - 1))) return false;
    if (kl->layers < 1 || kl->layers > 65536 || kl->kv_heads < 1 || kl->kv_heads > 256 ||
        kl->head_dim != KV_D || kl->pages < 1 || kl->pages > (1 << 24) || kl->seqs < 1 ||
        kl->seqs > KV_MAX_SEQS || kl->stride < 1 || (long long)kl->stride * pt > (1 << 24))
        return false;
    // (a pool whose bytes would not fit: layers * pages may be 2^40, a page 2^26)
    return (size_t)kl->layers * kl->pages <= (((size_t)1 << 62) / page_bytes(kl));
}

int check_layout(hyq_ctx *ctx, const hyq_kv_layout *kl, const char *who)
{
    if (!ctx) return fail(HYQ_EINVAL, "%s: null context", who);
    if (!kl) return fail(HYQ_EINVAL, "%s: null argument", who);
    if (!dtype_ok(kl))
        return fail(HYQ_EDTYPE, "%s: pages of type %d", who, kl->dtype);
    if (!layout_ok(kl))
        return fail(HYQ_EINVAL,
                    "%s: layout of %d layers, %d heads of dim %d, %d pages of %d tokens, %d slots "
                    "of %d entries",
                    who, kl->layers, kl->kv_heads, kl->head_dim, kl->pages, kl->page_tokens,
                    kl->seqs, kl->stride);
    return HYQ_OK;
}

int shift_of(const hyq_kv_layout *kl)
{
    int s = 4;
    while ((1 << s) < kl->page_tokens) ++s;
    return s;
}

bool heads_ok(const hyq_kv_layout *kl, size_t heads)
{
    return heads >= 1 && heads % kl->kv_heads == 0 && heads / kl->kv_heads <= (size_t)KV_MAX_REP;
}

PagedKv view(const hyq_kv_layout *kl, const void *pool, int layer, const int32_t *table,
             const int32_t *len, const int32_t *start, size_t rows, size_t heads)
{
    PagedKv v{};
    v.pages = (const char *)pool + (size_t)layer * kl->pages * page_bytes(kl);
    v.table = table;
    v.len = len;
    v.start = start;
    v.type = type_of(kl);
    v.seqs = kl->seqs;
    v.stride = kl->stride;
    v.npages = kl->pages;
    v.shift = shift_of(kl);
    v.kvh = kl->kv_heads;
    v.heads = (int)heads;
    v.rows = (int)rows;
    return v;
}

PagesArgs pages_args(const hyq_kv_layout *kl)
{
    PagesArgs a{};
    a.type = type_of(kl);
    a.layers = kl->layers;
    a.kvh = kl->kv_heads;
    a.shift = shift_of(kl);
    a.npages = kl->pages;
    a.seqs = kl->seqs;
    a.stride = kl->stride;
    return a;
}

// rows and heads of one call: their products index device buffers with 64
// bits, the counts themselves are ints
constexpr size_t MAX_ROWS = 1 << 20;

// Whether the attention's launches of these rows fit a grid (2^32 threads).
bool grid_ok(const hyq_kv_layout *kl, size_t rows, size_t heads)
{
    const int rep = (int)heads / kl->kv_heads;
    const int cap = max_blocks(kl->seqs, (int)rows, PR_ROWS / rep);
    return merge_groups(kl->seqs, kl->kv_heads, paged_few_rows(rep) * rep, cap) < (1 << 24);
}

// (served_len_d: null where the caller wants none)
int extend(hyq_ctx *ctx, const hyq_kv_layout *kl, void *pool_d, const int32_t *add_d,
           const int32_t *table_d, const int32_t *len_d, const int32_t *refs_d,
           int32_t *table_out_d, int32_t *len_out_d, int32_t *refs_out_d, int32_t *status_d,
           int32_t *served_len_d, void *scratch_d, size_t scratch_bytes)
{
    int rc = check_layout(ctx, kl, "pages_extend");
    if (rc) return rc;
    if (!pool_d || !add_d || !table_d || !len_d || !refs_d || !table_out_d || !len_out_d ||
        !refs_out_d || !status_d || !scratch_d)
        return fail(HYQ_EINVAL, "pages_extend: null argument");
    for (const int32_t *other : {add_d, table_d, len_d, refs_d, (const int32_t *)table_out_d,
                                 (const int32_t *)len_out_d, (const int32_t *)refs_out_d,
                                 (const int32_t *)status_d})
        if (other == served_len_d)
            return fail(HYQ_EINVAL, "pages_extend: the served lengths must be an array of their "
                                    "own");
    if (!aligned(pool_d) || !aligned(scratch_d))
        return fail(HYQ_EINVAL, "pages_extend: a buffer is not 16-byte aligned");
    if (scratch_bytes < hyq_pages_scratch_bytes(kl))
        return fail(HYQ_EINVAL, "pages_extend: scratch of %zu bytes, %zu needed", scratch_bytes,
                    hyq_pages_scratch_bytes(kl));
    DeviceGuard g(ctx->device);
    HYQ_LAUNCH(launch_pages_extend(pages_args(kl), pool_d, add_d, table_d, len_d, refs_d,
                                   table_out_d, len_out_d, refs_out_d, status_d, served_len_d,
                                   scratch_d, ctx->stream),
               "pages_extend");
    return HYQ_OK;
}

int shared_plan(hyq_ctx *ctx, const hyq_kv_layout *kl, const int32_t *group_d,
                const int32_t *table_d, const int32_t *len_d, const int32_t *start_d, size_t rows,
                size_t heads, long long least, void *plan_d, size_t plan_bytes)
{
    int rc = check_layout(ctx, kl, "paged_shared_plan");
    if (rc) return rc;
    if (!table_d || !len_d || !start_d || !plan_d)
        return fail(HYQ_EINVAL, "paged_shared_plan: null argument");
    if (!heads_ok(kl, heads) || rows == 0 || rows > MAX_ROWS)
        return fail(HYQ_EINVAL, "paged_shared_plan: %zu rows, heads %zu/%d", rows, heads,
                    kl->kv_heads);
    if (!aligned(plan_d)) return fail(HYQ_EINVAL, "paged_shared_plan: the plan is not 16-byte aligned");
    const size_t need = hyq_paged_shared_plan_bytes(kl, rows, heads);
    if (plan_bytes < need)
        return fail(HYQ_EINVAL, "paged_shared_plan: a plan of %zu bytes, %zu needed", plan_bytes,
                    need);
    DeviceGuard g(ctx->device);
    HYQ_LAUNCH(launch_shared_plan(view(kl, nullptr, 0, table_d, len_d, start_d, rows, heads),
                                  group_d, least, plan_d, ctx->stream),
               "paged_shared_plan");
    return HYQ_OK;
}

} // namespace

extern "C" {

size_t hyq_kv_pool_bytes(const hyq_kv_layout *kl)
{
    return layout_ok(kl) ? (size_t)kl->layers * kl->pages * page_bytes(kl) : 0;
}

int hyq_paged_rope_norm_append_d(hyq_ctx *ctx, const hyq_kv_layout *kl, void *pool_d, int layer,
                                 const int32_t *table_d, const int32_t *len_d,
                                 const int32_t *start_d, size_t rows, size_t heads,
                                 const float *q_d, const float *k_d, const float *v_d,
                                 const float *q_norm_d, const float *k_norm_d,
                                 const float *freq_d, float eps, int norm_first, float *q_out_d)
{
    int rc = check_layout(ctx, kl, "paged_rope_norm_append");
    if (rc) return rc;
    if (!pool_d || !table_d || !len_d || !start_d || !q_d || !k_d || !v_d || !q_norm_d ||
        !k_norm_d || !freq_d || !q_out_d)
        return fail(HYQ_EINVAL, "paged_rope_norm_append: null argument");
    if (layer < 0 || layer >= kl->layers)
        return fail(HYQ_EINVAL, "paged_rope_norm_append: layer %d of %d", layer, kl->layers);
    if (!heads_ok(kl, heads) || rows > MAX_ROWS)
        return fail(HYQ_EINVAL, "paged_rope_norm_append: %zu rows, heads %zu/%d", rows, heads,
                    kl->kv_heads);
    if (!aligned(pool_d) || !aligned(q_d) || !aligned(k_d) || !aligned(v_d) ||
        !aligned(q_norm_d) || !aligned(k_norm_d) || !aligned(freq_d) || !aligned(q_out_d))
        return fail(HYQ_EINVAL, "paged_rope_norm_append: a buffer is not 16-byte aligned");
    DeviceGuard g(ctx->device);
    HYQ_LAUNCH(launch_paged_append(view(kl, pool_d, layer, table_d, len_d, start_d, rows, heads),
                                   q_d, k_d, v_d, q_norm_d, k_norm_d, freq_d, eps, norm_first != 0,
                                   q_out_d, ctx->stream),
               "paged_rope_norm_append");
    return HYQ_OK;
}

int hyq_paged_read_d(hyq_ctx *ctx, const hyq_kv_layout *kl, const void *pool_d, int layer,
                     const int32_t *table_d, const int32_t *len_d, const int32_t *start_d,
                     size_t rows, float *k_d, float *v_d)
{
    int rc = check_layout(ctx, kl, "paged_read");
    if (rc) return rc;
    if (!pool_d || !table_d || !len_d || !start_d || !k_d || !v_d)
        return fail(HYQ_EINVAL, "paged_read: null argument");
    if (layer < 0 || layer >= kl->layers)
        return fail(HYQ_EINVAL, "paged_read: layer %d of %d", layer, kl->layers);
    if (rows > MAX_ROWS) return fail(HYQ_EINVAL, "paged_read: %zu rows", rows);
    if (!aligned(pool_d) || !aligned(k_d) || !aligned(v_d))
        return fail(HYQ_EINVAL, "paged_read: a buffer is not 16-byte aligned");
    if (k_d == v_d) return fail(HYQ_EINVAL, "paged_read: keys and values to one place");
    DeviceGuard g(ctx->device);
    HYQ_LAUNCH(launch_paged_read(view(kl, pool_d, layer, table_d, len_d, start_d, rows, 0), k_d,
                                 v_d, ctx->stream),
               "paged_read");
    return HYQ_OK;
}

size_t hyq_paged_attention_scratch_bytes(const hyq_kv_layout *kl, size_t rows, size_t max_rows,
                                         size_t heads)
{
    if (!layout_ok(kl) || !heads_ok(kl, heads) || rows == 0 || rows > MAX_ROWS || max_rows == 0 ||
        !grid_ok(kl, rows, heads))
        return 0;
    return paged_attention_scratch(type_of(kl), false, kl->seqs, kl->kv_heads, (int)heads,
                                   (int)rows, (int)std::min(rows, max_rows));
}

int hyq_paged_attention_d(hyq_ctx *ctx, const hyq_kv_layout *kl, const void *pool_d, int layer,
                          const int32_t *table_d, const int32_t *len_d, const int32_t *start_d,
                          size_t rows, size_t max_rows, size_t heads, const float *q_d,
                          void *scratch_d, size_t scratch_bytes, float *out_d)
{
    int rc = check_layout(ctx, kl, "paged_attention");
    if (rc) return rc;
    if (!pool_d || !table_d || !len_d || !start_d || !q_d || !scratch_d || !out_d)
        return fail(HYQ_EINVAL, "paged_attention: null argument");
    if (layer < 0 || layer >= kl->layers)
        return fail(HYQ_EINVAL, "paged_attention: layer %d of %d", layer, kl->layers);
    if (!heads_ok(kl, heads) || rows == 0 || rows > MAX_ROWS || max_rows == 0 ||
        !grid_ok(kl, rows, heads))
        return fail(HYQ_EINVAL, "paged_attention: %zu rows (at most %zu of a slot), heads %zu/%d",
                    rows, max_rows, heads, kl->kv_heads);
    if (!aligned(pool_d) || !aligned(q_d) || !aligned(scratch_d) || !aligned(out_d))
        return fail(HYQ_EINVAL, "paged_attention: a buffer is not 16-byte aligned");
    const size_t need = hyq_paged_attention_scratch_bytes(kl, rows, max_rows, heads);
    if (scratch_bytes < need)
        return fail(HYQ_EINVAL, "paged_attention: scratch of %zu bytes, %zu needed", scratch_bytes,
                    need);
    if (out_d == q_d) return fail(HYQ_EINVAL, "paged_attention: the output must not be q");
    DeviceGuard g(ctx->device);
    HYQ_LAUNCH(launch_paged_attention(view(kl, pool_d, layer, table_d, len_d, start_d, rows, heads),
                                      (int)std::min(rows, max_rows), q_d, scratch_d, nullptr,
                                      out_d, ctx->stream),
               "paged_attention");
    return HYQ_OK;
}

size_t hyq_paged_shared_plan_bytes(const hyq_kv_layout *kl, size_t rows, size_t heads)
{
    if (!layout_ok(kl) || !heads_ok(kl, heads) || rows == 0 || rows > MAX_ROWS) return 0;
    return shared_plan_bytes(kl->seqs, kl->kv_heads, (int)heads);
}

int hyq_paged_shared_plan_d(hyq_ctx *ctx, const hyq_kv_layout *kl, const int32_t *group_d,
                            const int32_t *table_d, const int32_t *len_d, const int32_t *start_d,
                            size_t rows, size_t heads, void *plan_d, size_t plan_bytes)
{
    // What sharing has to save to be worth its parts, in positions times KV heads. One
    // group of slots before 600 to 6000 common positions and some 60 of their own, 16
    // heads over 4, us a layer, shared and not: 8-bit pages 12.8 and 12.4 at 16,800, 13.8
    // and 14.5 at 42,000, 14.9 and 16.2 at 60,000; f16 13.5 and 13.4, 16.9 and 18.4, 17.1
    // and 19.0; f32 13.3 and 13.9, 17.0 and 17.0, 17.0 and 19.3. (The plan, 15 us a step,
    // is spent before it is known, and pays over the layers or not: four layers of the
    // f32 pages at 42,000 take 76 us with it and 70 without.)
    constexpr long long least = 25000;
    return shared_plan(ctx, kl, group_d, table_d, len_d, start_d, rows, heads, least, plan_d,
                       plan_bytes);
}

int hyq_paged_shared_plan_least_d(hyq_ctx *ctx, const hyq_kv_layout *kl, const int32_t *group_d,
                                  const int32_t *table_d, const int32_t *len_d,
                                  const int32_t *start_d, size_t rows, size_t heads, size_t least,
                                  void *plan_d, size_t plan_bytes)
{
    if (least > ((size_t)1 << 62)) least = (size_t)1 << 62;
    return shared_plan(ctx, kl, group_d, table_d, len_d, start_d, rows, heads, (long long)least,
                       plan_d, plan_bytes);
}

size_t hyq_paged_shared_attention_scratch_bytes(const hyq_kv_layout *kl, size_t rows,
                                                size_t max_rows, size_t heads)
{
    if (!hyq_paged_attention_scratch_bytes(kl, rows, max_rows, heads)) return 0;
    return shared_attention_scratch(type_of(kl), kl->seqs, kl->kv_heads, (int)heads, (int)rows,
                                    (int)std::min(rows, max_rows));
}

int hyq_paged_shared_attention_d(hyq_ctx *ctx, const hyq_kv_layout *kl, const void *pool_d,
                                 int layer, const int32_t *table_d, const int32_t *len_d,
                                 const int32_t *start_d, size_t rows, size_t max_rows, size_t heads,
                                 const void *plan_d, size_t plan_bytes, const float *q_d,
                                 void *scratch_d, size_t scratch_bytes, float *out_d)
{
    int rc = check_layout(ctx, kl, "paged_shared_attention");
    if (rc) return rc;
    if (!pool_d || !table_d || !len_d || !start_d || !plan_d || !q_d || !scratch_d || !out_d)
        return fail(HYQ_EINVAL, "paged_shared_attention: null argument");
    if (layer < 0 || layer >= kl->layers)
        return fail(HYQ_EINVAL, "paged_shared_attention: layer %d of %d", layer, kl->layers);
    if (!heads_ok(kl, heads) || rows == 0 || rows > MAX_ROWS || max_rows == 0 ||
        !grid_ok(kl, rows, heads))
        return fail(HYQ_EINVAL,
                    "paged_shared_attention: %zu rows (at most %zu of a slot), heads %zu/%d", rows,
                    max_rows, heads, kl->kv_heads);
    if (!aligned(pool_d) || !aligned(plan_d) || !aligned(q_d) || !aligned(scratch_d) ||
        !aligned(out_d))
        return fail(HYQ_EINVAL, "paged_shared_attention: a buffer is not 16-byte aligned");
    if (plan_bytes < hyq_paged_shared_plan_bytes(kl, rows, heads))
        return fail(HYQ_EINVAL, "paged_shared_attention: a plan of %zu bytes, %zu needed",
                    plan_bytes, hyq_paged_shared_plan_bytes(kl, rows, heads));
    const size_t need = hyq_paged_shared_attention_scratch_bytes(kl, rows, max_rows, heads);
    if (scratch_bytes < need)
        return fail(HYQ_EINVAL, "paged_shared_attention: scratch of %zu bytes, %zu needed",
                    scratch_bytes, need);
    if (out_d == q_d) return fail(HYQ_EINVAL, "paged_shared_attention: the output must not be q");
    DeviceGuard g(ctx->device);
    HYQ_LAUNCH(launch_paged_attention(view(kl, pool_d, layer, table_d, len_d, start_d, rows, heads),
                                      (int)std::min(rows, max_rows), q_d, scratch_d, plan_d, out_d,
                                      ctx->stream),
               "paged_shared_attention");
    return HYQ_OK;
}

int hyq_pages_fork_d(hyq_ctx *ctx, const hyq_kv_layout *kl, const int32_t *parent_d,
                     const int32_t *keep_d, const int32_t *table_d, const int32_t *len_d,
                     int32_t *table_out_d, int32_t *len_out_d, int32_t *refs_out_d)
{
    int rc = check_layout(ctx, kl, "pages_fork");
    if (rc) return rc;
    if (!parent_d || !table_d || !len_d || !table_out_d || !len_out_d || !refs_out_d)
        return fail(HYQ_EINVAL, "pages_fork: null argument");
    if (table_out_d == table_d || len_out_d == len_d)
        return fail(HYQ_EINVAL, "pages_fork: the new table must not be the old one");
    DeviceGuard g(ctx->device);
    HYQ_LAUNCH(launch_pages_fork(pages_args(kl), parent_d, keep_d, table_d, len_d, table_out_d,
                                 len_out_d, refs_out_d, ctx->stream),
               "pages_fork");
    return HYQ_OK;
}

size_t hyq_pages_scratch_bytes(const hyq_kv_layout *kl)
{
    return layout_ok(kl) ? pages_scratch(kl->pages, kl->seqs) : 0;
}

int hyq_pages_extend_d(hyq_ctx *ctx, const hyq_kv_layout *kl, void *pool_d, const int32_t *add_d,
                       const int32_t *table_d, const int32_t *len_d, const int32_t *refs_d,
                       int32_t *table_out_d, int32_t *len_out_d, int32_t *refs_out_d,
                       int32_t *status_d, void *scratch_d, size_t scratch_bytes)
{
    return extend(ctx, kl, pool_d, add_d, table_d, len_d, refs_d, table_out_d, len_out_d,
                  refs_out_d, status_d, nullptr, scratch_d, scratch_bytes);
}

int hyq_pages_extend_served_d(hyq_ctx *ctx, const hyq_kv_layout *kl, void *pool_d,
                              const int32_t *add_d, const int32_t *table_d, const int32_t *len_d,
                              const int32_t *refs_d, int32_t *table_out_d, int32_t *len_out_d,
                              int32_t *refs_out_d, int32_t *status_d, int32_t *served_len_d,
                              void *scratch_d, size_t scratch_bytes)
{
    if (!served_len_d) return fail(HYQ_EINVAL, "pages_extend: null argument");
    return extend(ctx, kl, pool_d, add_d, table_d, len_d, refs_d, table_out_d, len_out_d,
                  refs_out_d, status_d, served_len_d, scratch_d, scratch_bytes);
}

int hyq_pages_compact_d(hyq_ctx *ctx, const hyq_kv_layout *kl, void *pool_d,
                        const int32_t *table_d, const int32_t *refs_d, int32_t *table_out_d,
                        int32_t *refs_out_d, int32_t *live_d, void *scratch_d,
                        size_t scratch_bytes)
{
    int rc = check_layout(ctx, kl, "pages_compact");
    if (rc) return rc;
    if (!pool_d || !table_d || !refs_d || !table_out_d || !refs_out_d || !live_d || !scratch_d)
        return fail(HYQ_EINVAL, "pages_compact: null argument");
    if (!aligned(pool_d) || !aligned(scratch_d))
        return fail(HYQ_EINVAL, "pages_compact: a buffer is not 16-byte aligned");
    if (scratch_bytes < hyq_pages_scratch_bytes(kl))
        return fail(HYQ_EINVAL, "pages_compact: scratch of %zu bytes, %zu needed", scratch_bytes,
                    hyq_pages_scratch_bytes(kl));
    DeviceGuard g(ctx->device);
    HYQ_LAUNCH(launch_pages_compact(pages_args(kl), pool_d, table_d, refs_d, table_out_d,
                                    refs_out_d, live_d, scratch_d, ctx->stream),
               "pages_compact");
    return HYQ_OK;
}

int hyq_logits_adjust_d(hyq_ctx *ctx, const float *logits_d, size_t rows, size_t vocab,
                        const hyq_logit_rules *r, float *out_d)
{
    if (!ctx) return fail(HYQ_EINVAL, "logits_adjust: null context");
    if (!logits_d || !r || !out_d) return fail(HYQ_EINVAL, "logits_adjust: null argument");
    if (rows == 0 || rows > 65535 || vocab == 0 || vocab > (1 << 24))
        return fail(HYQ_EINVAL, "logits_adjust: %zu rows of %zu logits", rows, vocab);
    if (r->history_d && !r->history_len_d)
        return fail(HYQ_EINVAL, "logits_adjust: a history without lengths");
    if (r->history_d && (r->history_stride == 0 || r->history_stride > (1 << 24)))
        return fail(HYQ_EINVAL, "logits_adjust: a history of %zu tokens a row", r->history_stride);
    if ((r->bias_start_d || r->bias_token_d || r->bias_d) &&
        !(r->bias_start_d && r->bias_token_d && r->bias_d))
        return fail(HYQ_EINVAL, "logits_adjust: biases without starts, tokens or values");
    if (r->bias_d && r->biases > (1 << 30))
        return fail(HYQ_EINVAL, "logits_adjust: %zu biases", r->biases);
    if ((r->mask_d || r->mask_row_d) && !(r->mask_d && r->mask_row_d))
        return fail(HYQ_EINVAL, "logits_adjust: masks without the rows' choice, or that alone");
    if (r->mask_d && r->masks > (1 << 24))
        return fail(HYQ_EINVAL, "logits_adjust: %zu masks", r->masks);
    const uintptr_t from = reinterpret_cast<uintptr_t>(logits_d),
                    to = reinterpret_cast<uintptr_t>(out_d), bytes = rows * vocab * 4;
    if (from != to && from < to + bytes && to < from + bytes)
        return fail(HYQ_EINVAL, "logits_adjust: the output overlaps the logits in part");
    LogitRulesArgs a{};
    if (r->history_d) {
        a.history = r->history_d;
        a.history_len = r->history_len_d;
        a.prompt_len = r->prompt_len_d;
        a.history_stride = (int)r->history_stride;
        a.repetition = r->repetition_d;
        a.presence = r->presence_d;
        a.frequency = r->frequency_d;
    }
    a.bias_start = r->bias_start_d;
    a.bias_token = r->bias_token_d;
    a.bias = r->bias_d;
    a.biases = (int)r->biases;
    a.mask = r->mask_d;
    a.mask_row = r->mask_row_d;
    a.masks = (int)r->masks;
    DeviceGuard g(ctx->device);
    HYQ_LAUNCH(launch_logits_adjust(logits_d, (int)rows, (int)vocab, a, out_d, ctx->stream),
               "logits_adjust");
    return HYQ_OK;
}

size_t hyq_sample_scratch_bytes(size_t rows, size_t vocab)
{
    if (rows == 0 || rows > 65535 || vocab == 0 || vocab > (1 << 24)) return 0;
    return sample_scratch((int)rows, (int)vocab);
}

int hyq_sample_d(hyq_ctx *ctx, const float *logits_d, size_t rows, size_t vocab,
                 const float *temperature_d, const int32_t *top_k_d, const float *top_p_d,
                 const float *min_p_d, const float *random_d, void *scratch_d,
                 size_t scratch_bytes, int32_t *token_d, float *prob_d)
{
    if (!ctx) return fail(HYQ_EINVAL, "sample: null context");
    if (!logits_d || !temperature_d || !top_k_d || !top_p_d || !min_p_d || !random_d ||
        !scratch_d || !token_d)
        return fail(HYQ_EINVAL, "sample: null argument");
    if (rows == 0 || rows > 65535 || vocab == 0 || vocab > (1 << 24))
        return fail(HYQ_EINVAL, "sample: %zu rows of %zu logits", rows, vocab);
    if (!aligned(scratch_d)) return fail(HYQ_EINVAL, "sample: scratch is not 16-byte aligned");
    if (scratch_bytes < hyq_sample_scratch_bytes(rows, vocab))
        return fail(HYQ_EINVAL, "sample: scratch of %zu bytes, %zu needed", scratch_bytes,
                    hyq_sample_scratch_bytes(rows, vocab));
    DeviceGuard g(ctx->device);
    HYQ_LAUNCH(launch_sample(logits_d, (int)rows, (int)vocab, temperature_d, top_k_d, top_p_d,
                             min_p_d, random_d, scratch_d, token_d, prob_d, ctx->stream),
               "sample");
    return HYQ_OK;
}

} // extern "C"

// ---------------------------------------------------------------------------
// the attention's two forms
// ---------------------------------------------------------------------------

namespace hyq {

// Scratch: the few-row form's parts, then the tile form's plan and parts.
size_t paged_attention_scratch(int type, bool shared, int seqs, int kvh, int heads, int rows,
                               int max_rows)
{
    const int few = std::min(paged_few_rows(heads / kvh), max_rows);
    size_t n = paged_few_scratch(type, shared, seqs, kvh, heads, few);
    if (max_rows > few) n += rows_layout(seqs, kvh, heads, rows).bytes;
    return n;
}

// Behind them, in whole 256 bytes, the prefixes' parts.
size_t shared_attention_scratch(int type, int seqs, int kvh, int heads, int rows, int max_rows)
{
    const size_t n = paged_attention_scratch(type, true, seqs, kvh, heads, rows, max_rows);
    return (n + 255) / 256 * 256 + shared_parts_bytes(seqs, kvh, heads);
}

size_t shared_plan_bytes(int seqs, int kvh, int heads)
{
    return shared_layout(seqs, kvh, heads).bytes;
}

int launch_paged_attention(const PagedKv &kv, int max_rows, const float *q, void *scratch,
                           const void *plan, float *out, void *stream)
{
    SharedPlan sp{};
    float *prefix = nullptr;
    if (plan) {
        sp = shared_plan(plan, kv.seqs, kv.kvh, kv.heads);
        const size_t n =
            paged_attention_scratch(kv.type, true, kv.seqs, kv.kvh, kv.heads, kv.rows, max_rows);
        prefix = (float *)((char *)scratch + (n + 255) / 256 * 256);
        const int rc = launch_paged_prefix(kv, sp, q, prefix, stream);
        if (rc) return rc;
    }
    const int few = std::min(paged_few_rows(kv.heads / kv.kvh), max_rows);
    float *part = (float *)scratch;
    RowsScratch rs{};
    if (max_rows > few) {
        const RowsLayout l = rows_layout(kv.seqs, kv.kvh, kv.heads, kv.rows);
        char *base = (char *)scratch + paged_few_scratch(kv.type, plan, kv.seqs, kv.kvh, kv.heads, few);
        rs.plan = (Plan *)base;
        rs.blocks = (Block *)(base + l.blocks);
        rs.pieces = (Piece *)(base + l.pieces);
        rs.groups = (int *)(base + l.groups);
        rs.parts = (float *)(base + l.parts);
        rs.tq = PR_ROWS / (kv.heads / kv.kvh);
        rs.cap = max_blocks(kv.seqs, kv.rows, rs.tq);
        rs.most = max_rows;
    }
    int rc = launch_paged_few(kv, few, rs, plan ? &sp : nullptr, q, part, out, stream);
    if (rc == 0 && rs.cap) rc = launch_paged_rows(kv, rs, q, out, stream);
    if (rc == 0)
        rc = launch_paged_merge(kv, few, rs, plan ? &sp : nullptr, part, prefix, out, stream);
    return rc;
}

} // namespace hyq
