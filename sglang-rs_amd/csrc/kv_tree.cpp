// kv_tree.cpp -- host side of tree attention: the plan, the checks and the
// launches (kernels in kv_tree.hip). Nothing here allocates or waits, and what a
// launch relies on is derived again from the plan's configuration at each call.
#include <hip/hip_runtime.h>

#include <string.h>

#include "kv_call.h"

using namespace sglkv;

namespace {

constexpr uint64_t kMaxTokens = 1ull << 31;

// The launch of the generic body: a wave to each (query, KV head, 16 query heads,
// block of value dims) and split.
struct TreeShape {
    uint64_t max_length, base, chunk, splits, record_bytes, combine_grid;
};

int32_t tree_shape(const sgl_kv_attention_plan_config &c, const sgl_kv_tree_attention_config &t, TreeShape *out) {
    TreeShape &h = *out;
    h.max_length = t.max_sequence_length && t.max_sequence_length < c.sequence_slot_count ? t.max_sequence_length
                                                                                         : c.sequence_slot_count;
    const uint64_t group = c.query_head_count / c.kv_head_count;
    const struct {
        const char *name;
        uint64_t value, maximum;
    } limits[] = {{"mask_words", t.mask_words, SGL_KV_TREE_MASK_WORDS_MAX},
                  {"max_sequence_length", h.max_length, kMaxTokens},
                  {"query_key_head_dim", c.query_key_head_dim, SGLKV_ATTN_MAX_DK},
                  {"value_head_dim", c.value_head_dim, UINT32_MAX / 4}};
    for (const auto &l : limits)
        if (l.value > l.maximum) return too_large_dim(l.name, l.value, l.maximum);
    uint64_t heads;
    if (mul_ovf(c.query_count, c.kv_head_count, &h.base) || mul_ovf(h.base, divide_up(group, SGLKV_ATTN_HEADS), &h.base) ||
        mul_ovf(h.base, divide_up(c.value_head_dim, SGLKV_ATTN_DV), &h.base) ||
        mul_ovf(c.query_count, c.query_head_count, &heads))
        return attention_overflow();
    // About 2,048 waves, each with 128 tokens or more.
    const uint64_t wanted = h.base < 2048 ? 2048 / h.base : 1;
    h.chunk = divide_up(h.max_length, wanted);
    if (h.chunk < 128) h.chunk = 128;
    h.chunk = divide_up(h.chunk, SGLKV_ATTN_TOKENS) * SGLKV_ATTN_TOKENS;
    h.splits = divide_up(h.max_length, h.chunk);
    h.record_bytes = h.combine_grid = 0;
    if (h.splits > 1) {
        if (mul_ovf(heads, h.splits, &h.record_bytes) ||
            mul_ovf(h.record_bytes, 4ull * (SGLKV_ATTN_OPAD(c.value_head_dim) + 2), &h.record_bytes))
            return attention_overflow();
        const uint32_t dv = (uint32_t)c.value_head_dim;
        h.combine_grid = divide_up(heads, SGLKV_ATTN_COMBINE_SETS(dv) / SGLKV_ATTN_COMBINE_PER(dv, (uint32_t)h.splits));
    }
    // A dispatch counts its work-items in 32 bits.
    const uint64_t limit = UINT32_MAX / SGLKV_ATTN_COMBINE_THREADS;
    if (h.base > limit) return too_large_dim("workgroups", h.base, limit);
    if (h.combine_grid > limit) return too_large_dim("workgroups", h.combine_grid, limit);
    return SGL_KV_OK;
}

}  // namespace

extern "C" int32_t sgl_kv_tree_attention_plan_new(const sgl_kv_attention_plan *attention,
                                                  const sgl_kv_tree_attention_config *config,
                                                  sgl_kv_tree_attention_plan *out) {
    if (!attention || !config || !out) return null_arguments("attention/config/out");
    sgl_kv_tree_attention_plan p;
    memset(&p, 0, sizeof p);
    int32_t rc = sgl_kv_attention_plan_new(&attention->config, &p.attention);
    if (rc) return rc;
    if (!config->mask_words)
        return fail(SGL_KV_ZERO_DIMENSION, "mask_words", 0, 0, 0, "tree attention dimension mask_words must be non-zero");
    p.config = *config;
    TreeShape shape;
    if ((rc = tree_shape(p.attention.config, *config, &shape))) return rc;
    if (mul_ovf(p.attention.config.query_count, 8 * config->mask_words, &p.masks_required_bytes)) return attention_overflow();
    p.workspace_required_bytes = shape.record_bytes;
    *out = p;
    return ok();
}

extern "C" int32_t sgl_rocm_kv_tree_attention(sgl_rocm_kv_ctx *ctx, const sgl_kv_tree_attention_plan *plan,
                                              const sgl_kv_tree_attention_buffers *b, void *stream) {
    if (!ctx || !plan || !b) return null_arguments("ctx/plan/buffers");
    sgl_kv_tree_attention_plan fresh;
    TreeShape shape;
    int32_t rc = sgl_kv_tree_attention_plan_new(&plan->attention, &plan->config, &fresh);
    if (!rc) rc = tree_shape(fresh.attention.config, fresh.config, &shape);
    if (rc) return rc;
    const sgl_kv_attention_plan &a = fresh.attention;
    const sgl_kv_attention_plan_config &c = a.config;
    const sgl_kv_attention_layout &lay = c.layout;
    uint64_t queries, requests, lengths, offsets, slots, pool, output, masks, workspace = 0;
    const sgl_kv_attention_buffers &ab = b->attention;
    const CallBuffer all[] = {
        {"queries", &ab.queries, ab.queries_offset, a.query_required_bytes, &queries, 2, true},
        {"query_request_indices", &ab.query_request_indices, ab.query_request_indices_offset,
         a.query_request_indices_required_bytes, &requests, 4, true},
        {"query_sequence_lengths", &ab.query_sequence_lengths, ab.query_sequence_lengths_offset,
         a.query_sequence_lengths_required_bytes, &lengths, 8, true},
        {"request_slot_offsets", &ab.request_slot_offsets, ab.request_slot_offsets_offset,
         a.request_slot_offsets_required_bytes, &offsets, 8, true},
        {"sequence_slots", &ab.sequence_slots, ab.sequence_slots_offset, a.sequence_slots_required_bytes, &slots, 8, true},
        {"pool", &ab.pool, ab.pool_offset, a.pool_required_bytes, &pool, 2, true},
        {"output", &ab.output, ab.output_offset, a.output_required_bytes, &output, 2, true},
        {"masks", &b->masks, b->masks_offset, fresh.masks_required_bytes, &masks, 8, true},
        {"workspace", &b->workspace, b->workspace_offset, shape.record_bytes, &workspace, 16, shape.record_bytes > 0}};
    if ((rc = resolve_buffers(ctx, all))) return rc;
    if ((lay.key_in_page_offset | lay.value_in_page_offset | lay.page_stride_bytes) & 1)
        return fail(SGL_KV_INVALID_ARGUMENT, "alignment", 0, 0, 0, "pool rows must be aligned to their element size");
    sglkv_tree_params p;
    memset(&p, 0, sizeof p);
    p.a.queries = reinterpret_cast<const uint16_t *>(queries);
    p.a.query_request_indices = reinterpret_cast<const uint32_t *>(requests);
    p.a.query_sequence_lengths = reinterpret_cast<const uint64_t *>(lengths);
    p.a.request_slot_offsets = reinterpret_cast<const uint64_t *>(offsets);
    p.a.sequence_slots = reinterpret_cast<const uint64_t *>(slots);
    p.a.pool = reinterpret_cast<const uint8_t *>(pool);
    p.a.output = reinterpret_cast<uint16_t *>(output);
    p.a.partial = reinterpret_cast<float *>(workspace);
    p.a.flag = ctx->attn_flag;
    attention_geometry(c, &p.a);
    p.a.zero_row = ctx->zero_row;
    p.a.chunk_tokens = shape.chunk;
    p.a.splits = (uint32_t)shape.splits;
    p.masks = reinterpret_cast<const uint64_t *>(masks);
    p.mask_words = (uint32_t)fresh.config.mask_words;
    p.max_length = shape.max_length;
    const bool vector = p.a.dk % 8 == 0 && p.a.dv % 8 == 0 &&
                        ((pool + lay.key_in_page_offset) | (pool + lay.value_in_page_offset) | lay.page_stride_bytes |
                         p.a.key_head_stride | p.a.key_token_stride | p.a.value_head_stride | p.a.value_token_stride) %
                                16 == 0;
    DeviceScope scope(ctx->device);
    if (scope.status() != hipSuccess) return hip_fail(scope.status(), "hipSetDevice");
    hipStream_t s = static_cast<hipStream_t>(stream);
    const unsigned lds = 2 * (SGLKV_ATTN_HEADS * (p.a.dk_pad + 8) + SGLKV_ATTN_DV * SGLKV_ATTN_VT_STRIDE);
    rc = launch_kernel(ctx->tree_attention[vector ? 0 : 1], shape.base, shape.splits, 1, 64, lds, s, &p, "tree attention launch");
    if (!rc && shape.splits > 1)
        rc = launch_kernel(ctx->tree_combine, shape.combine_grid, 1, 1, SGLKV_ATTN_COMBINE_THREADS, 0, s, &p,
                           "tree attention combine launch");
    return rc ? rc : ok();
}
