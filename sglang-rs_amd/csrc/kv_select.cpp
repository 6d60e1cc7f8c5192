// kv_select.cpp -- host side of page selection: the plan, the checks and the
// launches of page_bounds, select_pages and selected_attention (kernels in
// kv_select.hip). Nothing here allocates or waits, and everything that a launch
// relies on is derived again from the plan's configuration at each call, so an
// edited plan is checked like a new one.
#include <hip/hip_runtime.h>

#include <string.h>

#include "kv_attention_route.h"
#include "kv_internal.h"

using namespace sglkv;

namespace {

constexpr uint64_t kMaxPageSize = 1ull << 24;
constexpr uint64_t kMaxListed = 1ull << 31;
constexpr uint64_t kMaxQueryElements = 76ull << 10;  // of one KV head's query heads: 152 KiB of LDS

uint64_t ceil_div(uint64_t a, uint64_t b) { return a / b + (a % b != 0); }

int32_t null_argument(const char *name) {
    return fail(SGL_KV_INVALID_ARGUMENT, name, 0, 0, 0, "null argument");
}

int32_t misaligned(const char *name) {
    return fail(SGL_KV_INVALID_ARGUMENT, "alignment", 0, 0, 0, "%s must be aligned to its element size", name);
}

// The launch shapes of a plan's two calls.
struct SelectionShape {
    uint64_t max_length, sequence_pages, items;  // items: (query, KV head)s
    uint64_t chunk_pages, chunks, near_queries;  // of the scores
    uint64_t key_bytes;
    uint64_t split_pages, splits;                // of the attention
    uint64_t record_bytes;
};

// Chunks of pages that the scores are cut into, 16 pages or more each: a wave to
// each where the KV heads come in fours. A wave waits some 4 us for its length, slots
// and first rows, which short shares do not hide; long ones leave CUs idle at the end
// of ragged batches. Rows of 64 dims are half as long and want half the chunks: 120
// drafted queries of 24 sequences of up to 20,000 tokens on 2 heads took 24.7, 26.7
// and 27.6 us with 2,048, 4,096 and 8,192 of them; 64 of up to 32,768 on 8 heads of
// 128 dims 107 and 77 us with 2,048 and 4,096.
uint64_t score_chunks(uint64_t dk) { return dk <= 64 ? 2048 : 4096; }
// Waves of the attention that stay resident at once, each with 64 tokens or
// more: what the staged body's LDS leaves room for on 256 CUs (its registers, at
// dims 64), or the generic one's LDS.
uint64_t attend_waves(const sgl_kv_attention_plan_config &c) {
    return 256 * (c.value_head_dim > 128 ? 2 : c.value_head_dim > 64 ? 5 : 8);
}

// The staged body's shapes (its alignments are the call's to see).
bool staged_shape(const sgl_kv_attention_plan_config &c) {
    const uint64_t d = c.query_key_head_dim, page = c.layout.page_size;
    return d == c.value_head_dim && (d == 64 || d == 128 || d == 256) && page >= 8 && (page & (page - 1)) == 0 &&
           c.query_head_count / c.kv_head_count <= SGLKV_ATTN_HEADS && c.slot_count < (1ull << 32) &&
           c.layout.page_stride_bytes <= UINT32_MAX;
}

int32_t selection_shape(const sgl_kv_attention_plan_config &c, const sgl_kv_page_selection_config &s,
                        SelectionShape *out) {
    SelectionShape &h = *out;
    const uint64_t page = c.layout.page_size;
    h.max_length = s.max_sequence_length && s.max_sequence_length < c.sequence_slot_count ? s.max_sequence_length
                                                                                         : c.sequence_slot_count;
    h.sequence_pages = ceil_div(h.max_length, page);
    const uint64_t group = c.query_head_count / c.kv_head_count;
    const struct {
        const char *name;
        uint64_t value, maximum;
    } limits[] = {{"page_size", page, kMaxPageSize},
                  {"max_pages", s.max_pages, kMaxListed},
                  {"sequence_pages", h.sequence_pages, kMaxListed},
                  {"query_key_head_dim", c.query_key_head_dim, SGLKV_ATTN_MAX_DK},
                  {"value_head_dim", c.value_head_dim, UINT32_MAX / 4},
                  {"query_heads_per_kv_head", group, kMaxQueryElements / SGLKV_SELECT_QSTRIDE(c.query_key_head_dim)}};
    for (const auto &l : limits)
        if (l.value > l.maximum) return too_large_dim(l.name, l.value, l.maximum);
    if (mul_ovf(c.query_count, c.kv_head_count, &h.items)) return attention_overflow();
    // Scores.
    uint64_t pages;
    if (mul_ovf(h.items, h.sequence_pages, &pages) || mul_ovf(pages, 8, &h.key_bytes)) return attention_overflow();
    if (h.sequence_pages <= s.max_pages) h.key_bytes = 0;
    const uint64_t share = ceil_div(pages, score_chunks(c.query_key_head_dim));
    h.chunk_pages = ceil_div(share < h.sequence_pages ? share : h.sequence_pages, 16) * 16;
    h.chunks = ceil_div(h.sequence_pages, h.chunk_pages);
    // Attention.
    const uint64_t list = s.max_pages < h.sequence_pages ? s.max_pages : h.sequence_pages;
    const uint64_t head_groups = ceil_div(group, SGLKV_ATTN_HEADS), dv_blocks = ceil_div(c.value_head_dim, SGLKV_ATTN_DV);
    uint64_t base;
    if (mul_ovf(h.items, head_groups, &base) || mul_ovf(base, dv_blocks, &base)) return attention_overflow();
    const uint64_t waves = attend_waves(c), shared = staged_shape(c) ? h.items : base;
    h.split_pages = ceil_div(list, shared < waves ? waves / shared : 1);
    const uint64_t least = ceil_div(64, page);
    if (h.split_pages < least) h.split_pages = least;
    if (h.split_pages > SGLKV_SELECT_CHUNK_PAGES) h.split_pages = SGLKV_SELECT_CHUNK_PAGES;
    h.splits = ceil_div(list, h.split_pages);
    if (h.splits > 65535) return too_large_dim("max_pages", list, 65535 * h.split_pages);  // grid y
    h.record_bytes = 0;
    uint64_t heads;
    if (mul_ovf(c.query_count, c.query_head_count, &heads)) return attention_overflow();
    if (h.splits > 1 && (mul_ovf(heads, h.splits, &h.record_bytes) ||
                         mul_ovf(h.record_bytes, 4ull * (SGLKV_ATTN_OPAD(c.value_head_dim) + 2), &h.record_bytes)))
        return attention_overflow();
    // A dispatch counts its work-items in 32 bits.
    // (The scores' workgroups are placed eight (near queries, chunk)s at a time: 64 or
    // more of them, or all queries of one prompt would share one XCD.)
    h.near_queries = ceil_div(c.query_count, c.request_count);
    uint64_t placed;
    if (mul_ovf(c.query_count, h.chunks, &placed)) return attention_overflow();
    if (h.near_queries > placed / 64) h.near_queries = placed < 64 ? 1 : placed / 64;
    if (mul_ovf(ceil_div(c.query_count, h.near_queries), h.chunks, &placed) || placed > UINT64_MAX - 7 ||
        mul_ovf(ceil_div(placed, 8) * 8, h.near_queries, &placed) || mul_ovf(placed, c.kv_head_count, &placed))
        return attention_overflow();
    if (placed > UINT32_MAX / SGLKV_SELECT_THREADS)
        return too_large_dim("workgroups", placed, UINT32_MAX / SGLKV_SELECT_THREADS);
    if (base > UINT32_MAX / 64) return too_large_dim("workgroups", base, UINT32_MAX / 64);
    if (heads > UINT32_MAX / 64) return too_large_dim("workgroups", heads, UINT32_MAX / 64);
    return SGL_KV_OK;
}

// The checked parameters of a call; `attends`: selected_attention, else
// select_pages.
int32_t selection_params(sgl_rocm_kv_ctx *ctx, const sgl_kv_page_selection_plan *plan,
                         const sgl_kv_page_selection_buffers *b, bool attends, sglkv_select_params *params,
                         SelectionShape *shape) {
    if (!ctx || !plan || !b) return null_argument("ctx/plan/buffers");
    sgl_kv_page_selection_plan fresh;
    int32_t rc = sgl_kv_page_selection_plan_new(&plan->attention, &plan->config, &fresh);
    if (!rc) rc = selection_shape(fresh.attention.config, fresh.config, shape);
    if (rc) return rc;
    const sgl_kv_attention_plan &a = fresh.attention;
    const sgl_kv_attention_plan_config &c = a.config;
    const uint64_t scratch = attends ? shape->record_bytes : shape->key_bytes;
    sglkv_select_params &p = *params;
    memset(&p, 0, sizeof p);
    uint64_t queries, requests, lengths, offsets, slots, pool = 0, output = 0, bounds = 0, selected, workspace = 0;
    const struct {
        const char *name;
        const sgl_kv_device_buffer *buffer;
        uint64_t offset, need;
        uint64_t *address;
        uint64_t align;
        bool used;
    } all[] = {
        {"queries", &b->attention.queries, b->attention.queries_offset, a.query_required_bytes, &queries, 2, true},
        {"query_request_indices", &b->attention.query_request_indices, b->attention.query_request_indices_offset,
         a.query_request_indices_required_bytes, &requests, 4, true},
        {"query_sequence_lengths", &b->attention.query_sequence_lengths, b->attention.query_sequence_lengths_offset,
         a.query_sequence_lengths_required_bytes, &lengths, 8, true},
        {"request_slot_offsets", &b->attention.request_slot_offsets, b->attention.request_slot_offsets_offset,
         a.request_slot_offsets_required_bytes, &offsets, 8, true},
        {"sequence_slots", &b->attention.sequence_slots, b->attention.sequence_slots_offset,
         a.sequence_slots_required_bytes, &slots, 8, true},
        {"pool", &b->attention.pool, b->attention.pool_offset, a.pool_required_bytes, &pool, 2, attends},
        {"output", &b->attention.output, b->attention.output_offset, a.output_required_bytes, &output, 2, attends},
        {"bounds", &b->bounds, b->bounds_offset, fresh.bounds_required_bytes, &bounds, 2, !attends},
        {"selected", &b->selected, b->selected_offset, fresh.selected_required_bytes, &selected, 4, true},
        {"workspace", &b->workspace, b->workspace_offset, scratch, &workspace, 16, scratch > 0}};
    for (const auto &x : all)
        if (x.used && (rc = check_device(ctx, x.name, *x.buffer))) return rc;
    for (const auto &x : all)
        if (x.used && (rc = attention_ptr(x.name, *x.buffer, x.offset, x.need, x.address))) return rc;
    for (const auto &x : all)
        if (x.used && *x.address % x.align) return misaligned(x.name);
    if (attends && ((c.layout.key_in_page_offset | c.layout.value_in_page_offset | c.layout.page_stride_bytes) & 1))
        return misaligned("pool rows");
    p.a.queries = reinterpret_cast<const uint16_t *>(queries);
    p.a.query_request_indices = reinterpret_cast<const uint32_t *>(requests);
    p.a.query_sequence_lengths = reinterpret_cast<const uint64_t *>(lengths);
    p.a.request_slot_offsets = reinterpret_cast<const uint64_t *>(offsets);
    p.a.sequence_slots = reinterpret_cast<const uint64_t *>(slots);
    p.a.pool = reinterpret_cast<const uint8_t *>(pool);
    p.a.output = reinterpret_cast<uint16_t *>(output);
    p.a.partial = attends ? reinterpret_cast<float *>(workspace) : nullptr;
    p.a.flag = ctx->attn_flag;
    attention_geometry(c, &p.a);
    p.a.zero_row = ctx->zero_row;
    p.a.splits = (uint32_t)shape->splits;
    p.bounds = reinterpret_cast<const uint16_t *>(bounds);
    p.selected = reinterpret_cast<uint32_t *>(selected);
    p.keys = attends ? nullptr : reinterpret_cast<uint64_t *>(workspace);
    p.max_length = shape->max_length;
    p.max_pages = (uint32_t)fresh.config.max_pages;
    p.first_pages = (uint32_t)fresh.config.first_pages;
    p.last_pages = (uint32_t)fresh.config.last_pages;
    p.sequence_pages = (uint32_t)shape->sequence_pages;
    return SGL_KV_OK;
}

// The function for rows of `dims` dims that 16-byte accesses read (vector) or
// not: 8, 16, 32 or 64 lanes to a row, or the element-wise one.
int row_lanes(uint64_t dims, bool vector) { return !vector ? 4 : dims <= 64 ? 0 : dims <= 128 ? 1 : dims <= 256 ? 2 : 3; }

}  // namespace

extern "C" int32_t sgl_kv_page_selection_plan_new(const sgl_kv_attention_plan *attention,
                                                  const sgl_kv_page_selection_config *config,
                                                  sgl_kv_page_selection_plan *out) {
    if (!attention || !config || !out) return null_argument("attention/config/out");
    sgl_kv_page_selection_plan p;
    memset(&p, 0, sizeof p);
    int32_t rc = sgl_kv_attention_plan_new(&attention->config, &p.attention);
    if (rc) return rc;
    const sgl_kv_attention_plan_config &c = p.attention.config;
    if (!config->max_pages)
        return fail(SGL_KV_ZERO_DIMENSION, "max_pages", 0, 0, 0, "page selection dimension max_pages must be non-zero");
    if (config->first_pages > config->max_pages || config->last_pages > config->max_pages - config->first_pages)
        return fail(SGL_KV_INVALID_ARGUMENT, "first_pages", config->first_pages, config->last_pages, config->max_pages,
                    "%llu first and %llu last pages do not fit a list of %llu", (unsigned long long)config->first_pages,
                    (unsigned long long)config->last_pages, (unsigned long long)config->max_pages);
    p.config = *config;
    SelectionShape shape;
    if ((rc = selection_shape(c, *config, &shape))) return rc;
    uint64_t row;
    if (mul_ovf(c.kv_head_count, 4 * c.query_key_head_dim, &row) ||
        mul_ovf(ceil_div(c.slot_count, c.layout.page_size), row, &p.bounds_required_bytes) ||
        mul_ovf(shape.items, 4 * config->max_pages, &p.selected_required_bytes))
        return attention_overflow();
    p.workspace_required_bytes = shape.key_bytes > shape.record_bytes ? shape.key_bytes : shape.record_bytes;
    *out = p;
    return ok();
}

extern "C" int32_t sgl_rocm_kv_page_bounds(sgl_rocm_kv_ctx *ctx, const sgl_kv_pool_view *keys,
                                           const sgl_kv_device_buffer *pages, const sgl_kv_device_buffer *counts,
                                           uint64_t count, const sgl_kv_device_buffer *bounds, void *stream) {
    if (!ctx || !keys || !keys->base || !pages || !counts || !bounds)
        return null_argument("ctx/keys/pages/counts/bounds");
    const sgl_kv_pool_view &v = *keys;
    int32_t rc = check_pool_view(keys);
    if (rc) return rc;
    if (v.row_bytes % (2ull * v.heads))
        return fail(SGL_KV_INVALID_ARGUMENT, "heads", v.heads, v.row_bytes, 0,
                    "a %llu-byte key row does not split into %u heads of bf16 elements", (unsigned long long)v.row_bytes,
                    v.heads);
    const uint64_t head = v.row_bytes / v.heads, dims = head / 2;
    if (dims > SGLKV_ATTN_MAX_DK) return too_large_dim("query_key_head_dim", dims, SGLKV_ATTN_MAX_DK);
    if (v.page_count > UINT32_MAX) return too_large_dim("page_count", v.page_count, UINT32_MAX);
    if (count == 0) return ok();
    uint64_t items, list_bytes, bound_bytes;
    if (mul_ovf(count, v.heads, &items) || mul_ovf(count, 4, &list_bytes) ||
        mul_ovf(v.page_count, 2 * v.row_bytes, &bound_bytes))
        return attention_overflow();
    if (items > UINT32_MAX / 64 - 4) return too_large_dim("workgroups", items, UINT32_MAX / 64 - 4);
    uint64_t page_at, count_at, bound_at;
    const sgl_kv_device_buffer pool = {v.base, v.byte_len};
    if ((rc = check_device(ctx, "pool", pool)) || (rc = check_device(ctx, "pages", *pages)) ||
        (rc = check_device(ctx, "counts", *counts)) || (rc = check_device(ctx, "bounds", *bounds)) ||
        (rc = attention_ptr("pages", *pages, 0, list_bytes, &page_at)) ||
        (rc = attention_ptr("counts", *counts, 0, list_bytes, &count_at)) ||
        (rc = attention_ptr("bounds", *bounds, 0, bound_bytes, &bound_at)))
        return rc;
    sglkv_bounds_params p;
    memset(&p, 0, sizeof p);
    const uint64_t base = (uint64_t)(uintptr_t)v.base;
    p.pool = static_cast<const uint8_t *>(v.base);
    p.pages = reinterpret_cast<const uint32_t *>(page_at);
    p.counts = reinterpret_cast<const uint32_t *>(count_at);
    p.bounds = reinterpret_cast<uint16_t *>(bound_at);
    p.flag = ctx->flag;
    p.count = count;
    p.page_count = v.page_count;
    p.page_stride = v.page_stride_bytes;
    p.key_offset = v.tensor_offset[0];
    p.key_head_stride = v.head_layout == SGL_KV_HND ? v.page_size * head : head;
    p.key_token_stride = v.head_layout == SGL_KV_HND ? head : v.row_bytes;
    p.page_size = (uint32_t)v.page_size;
    p.heads = v.heads;
    p.dk = (uint32_t)dims;
    if (page_at % 4 || count_at % 4 || bound_at % 2 || ((base | p.key_offset | p.page_stride) & 1))
        return misaligned("pages, counts, bounds or pool rows");
    const bool vector = dims % 8 == 0 && bound_at % 16 == 0 &&
                        ((base + p.key_offset) | p.page_stride | p.key_head_stride | p.key_token_stride) % 16 == 0;
    DeviceScope scope(ctx->device);
    if (scope.status() != hipSuccess) return hip_fail(scope.status(), "hipSetDevice");
    rc = launch_kernel(ctx->page_bounds[row_lanes(dims, vector)], ceil_div(items, 4), 1, 1, 256, 0, static_cast<hipStream_t>(stream),
                &p, "page bounds launch");
    return rc ? rc : ok();
}

extern "C" int32_t sgl_rocm_kv_select_pages(sgl_rocm_kv_ctx *ctx, const sgl_kv_page_selection_plan *plan,
                                            const sgl_kv_page_selection_buffers *b, void *stream) {
    sglkv_select_params p;
    SelectionShape shape;
    int32_t rc = selection_params(ctx, plan, b, false, &p, &shape);
    if (rc) return rc;
    DeviceScope scope(ctx->device);
    if (scope.status() != hipSuccess) return hip_fail(scope.status(), "hipSetDevice");
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (shape.key_bytes) {
        const bool vector = p.a.dk % 8 == 0 && reinterpret_cast<uint64_t>(p.bounds) % 16 == 0;
        p.chunk_pages = (uint32_t)shape.chunk_pages;
        p.heads = p.a.kv_heads * (uint32_t)shape.chunks;
        const int dims = p.a.dk == 64 ? 0 : p.a.dk == 128 ? 1 : p.a.dk == 256 ? 2 : -1;
        if (vector && dims >= 0 && reinterpret_cast<uint64_t>(p.a.queries) % 16 == 0 &&
            shape.chunk_pages <= SGLKV_SELECT_LDS_PAGES) {
            // 4, 8 or 16 query heads a turn; past that several, whose maxima wait in LDS.
            const int heads = p.a.group <= 4 ? 0 : p.a.group <= 8 || dims == 2 ? 1 : 2;
            p.block_heads = p.a.kv_heads % 4 == 0 ? 4 : p.a.kv_heads % 2 == 0 ? 2 : 1;
            p.near_queries = (uint32_t)shape.near_queries;
            const uint64_t groups = ceil_div(ceil_div(p.a.query_count, shape.near_queries) * shape.chunks, 8) * 8 *
                                    shape.near_queries * (p.a.kv_heads / p.block_heads);
            rc = launch_kernel(ctx->page_scores_fast[dims][heads], groups, 1, 1, SGLKV_SELECT_THREADS,
                               p.a.group > (4u << heads) ? (unsigned)(8 * shape.chunk_pages * p.block_heads) : 0, s, &p,
                               "page scores launch");
        } else {
            rc = launch_kernel(ctx->page_scores[row_lanes(p.a.dk, vector)], shape.items * shape.chunks, 1, 1,
                               SGLKV_SELECT_THREADS, 2 * p.a.group * SGLKV_SELECT_QSTRIDE(p.a.dk), s, &p,
                               "page scores launch");
        }
        if (rc) return rc;
    }
    rc = launch_kernel(ctx->pick_pages, shape.items, 1, 1, SGLKV_SELECT_THREADS, 0, s, &p, "page pick launch");
    return rc ? rc : ok();
}

extern "C" int32_t sgl_rocm_kv_selected_attention(sgl_rocm_kv_ctx *ctx, const sgl_kv_page_selection_plan *plan,
                                                  const sgl_kv_page_selection_buffers *b, void *stream) {
    sglkv_select_params p;
    SelectionShape shape;
    int32_t rc = selection_params(ctx, plan, b, true, &p, &shape);
    if (rc) return rc;
    DeviceScope scope(ctx->device);
    if (scope.status() != hipSuccess) return hip_fail(scope.status(), "hipSetDevice");
    hipStream_t s = static_cast<hipStream_t>(stream);
    const sgl_kv_attention_layout &lay = plan->attention.config.layout;
    const uint64_t pool = reinterpret_cast<uint64_t>(p.a.pool);
    const bool vector = p.a.dk % 8 == 0 && p.a.dv % 8 == 0 &&
                        ((pool + lay.key_in_page_offset) | (pool + lay.value_in_page_offset) | lay.page_stride_bytes |
                         p.a.key_head_stride | p.a.key_token_stride | p.a.value_head_stride | p.a.value_token_stride) %
                                16 == 0;
    p.chunk_pages = (uint32_t)shape.split_pages;
    const bool staged = vector && staged_shape(plan->attention.config) && reinterpret_cast<uint64_t>(p.a.queries) % 16 == 0 &&
                        p.a.key_token_stride == p.a.value_token_stride && p.a.key_token_stride < (1u << 24);
    if (staged) {
        p.a.dv_blocks = 1;
        p.a.page_stride32 = (uint32_t)p.a.page_stride;
        p.a.key_token_stride32 = p.a.value_token_stride32 = (uint32_t)p.a.key_token_stride;
        rc = launch_kernel(ctx->selected_staged[p.a.dk == 64 ? 0 : p.a.dk == 128 ? 1 : 2], shape.items, p.a.splits, 1, 64,
                           256 * p.a.dk, s, &p, "selected attention launch");
    } else {
        const unsigned lds = 2 * (SGLKV_ATTN_HEADS * (p.a.dk_pad + 8) + SGLKV_ATTN_DV * SGLKV_ATTN_VT_STRIDE);
        rc = launch_kernel(ctx->selected_attention[vector ? 0 : 1], shape.items * p.a.head_groups * p.a.dv_blocks, p.a.splits,
                           1, 64, lds, s, &p, "selected attention launch");
    }
    if (!rc && p.a.splits > 1)
        rc = launch_kernel(ctx->selected_combine, p.a.query_count * p.a.query_heads, 1, 1, 64, 0, s, &p,
                    "selected attention combine launch");
    return rc ? rc : ok();
}
