// kv_tree.cpp -- host side of tree attention: the plan, the checks and the
// launches (kernels in kv_tree.hip). Nothing here allocates or waits, and what a
// launch relies on is derived again from the plan's configuration at each call.
#include <hip/hip_runtime.h>

#include <string.h>

#include "kv_call.h"

using namespace sglkv;

namespace {

constexpr uint64_t kMaxTokens = 1ull << 31;

// A body's launch: `base` workgroups to a split for the generic one (a wave to
// each (query, KV head, 16 query heads, block of value dims)), a number of all for
// the tiles.
struct TreeWay {
    uint64_t base, chunk, splits, record_bytes, combine_grid;
};

struct TreeShape {
    uint64_t max_length;
    TreeWay any;
    // Tiles: head dims 64, 128 or 256 on rows that the buffers' alignment, which is the call's to see, lets 16-byte
    // accesses read.
    bool tiles;
    uint32_t row_waves, tile_queries, tile_slots, unit, least;
    bool balanced;
    uint64_t pairs, used_at;
    TreeWay tile;
};

// The records of a query head's `splits` splits, and their merge.
int32_t split_records(const sgl_kv_attention_plan_config &c, TreeWay *w) {
    uint64_t heads;
    if (mul_ovf(c.query_count, c.query_head_count, &heads)) return attention_overflow();
    w->record_bytes = w->combine_grid = 0;
    if (w->splits > 1) {
        if (mul_ovf(heads, w->splits, &w->record_bytes) ||
            mul_ovf(w->record_bytes, 4ull * (SGLKV_ATTN_OPAD(c.value_head_dim) + 2), &w->record_bytes))
            return attention_overflow();
        const uint32_t dv = (uint32_t)c.value_head_dim;
        w->combine_grid = divide_up(heads, SGLKV_ATTN_COMBINE_SETS(dv) / SGLKV_ATTN_COMBINE_PER(dv, (uint32_t)w->splits));
    }
    // A dispatch counts its work-items in 32 bits.
    const uint64_t limit = UINT32_MAX / SGLKV_ATTN_COMBINE_THREADS;
    if (w->combine_grid > limit) return too_large_dim("workgroups", w->combine_grid, limit);
    return SGL_KV_OK;
}

int32_t tile_shape(const sgl_kv_attention_plan_config &c, const sgl_kv_tree_attention_config &t, TreeShape *out) {
    TreeShape &h = *out;
    const uint64_t group = c.query_head_count / c.kv_head_count, d = c.query_key_head_dim, page = c.layout.page_size;
    const uint32_t most = d > 128 ? 2 : 4;
    h.tiles = d == c.value_head_dim && (d == 64 || d == 128 || d == 256) && (page & (page - 1)) == 0 && page <= 1u << 24 &&
              group <= 32 * most && c.slot_count < 1ull << 32 && c.layout.page_stride_bytes <= UINT32_MAX &&
              c.layout.key_row_bytes < 1u << 24 && c.query_count < 1ull << 31;
    if (!h.tiles) return SGL_KV_OK;
    // Row waves: one, with four (at head dim 256 two) token groups, where the launch has few tiles anyway and each is to
    // be done sooner (one request of up to 4,096 tokens with up to 16 drafts, head dims 64, 128 and 256: 15.4, 19.8 and
    // 26.5 us, with two 16.6, 22.1 and 30.6; 16 such with 4: 27.7, 41.5 and 87.8, with two 26.2, 38.2 and 65.6). Else two
    // or four by the rows that a request has on average (64 requests with up to 12 drafts of 4 heads: 76 and 156 us with
    // two, 82 and 159 with four; with up to 24: 103 and 185 with two, 91 and 171 with four).
    const uint64_t mean = divide_up(c.query_count, c.request_count), rows = mean * group;
    uint64_t few;
    h.row_waves = rows <= 32 || most == 2 ? 2 : 4;
    if (!mul_ovf(c.request_count, divide_up(rows, 32) * c.kv_head_count, &few) && few <= (d > 128 ? 16 : 64)) h.row_waves = 1;
    while (group > 32 * h.row_waves) h.row_waves *= 2;
    h.tile_queries = 32 * h.row_waves / (uint32_t)group;
    // (Request, split, tile)s: as many as make the workgroups that stay resident at once, or a multiple of that (40
    // requests of 300 to 4,096 tokens: 107 us with 64 a KV head, 128 with 80). A request has at most twice its even share
    // of splits and two more, which bounds the records.
    const uint64_t groups = 4 / (h.row_waves * SGLKV_TREE_SHARE(d)), count = c.request_count;
    const uint64_t resident = 256 * (d == 128 && h.row_waves == 1 ? 1 : d == 256 && h.row_waves == 1 ? 1 : 2);
    const uint64_t tiles = divide_up(mean, h.tile_queries), most_tiles = c.query_count / h.tile_queries + count;
    h.unit = (uint32_t)(groups * SGLKV_TREE_BLOCK(d, h.row_waves));
    h.least = 2;
    h.tile_slots = 0;
    h.balanced = count <= SGLKV_TREE_BALANCED && c.query_count <= SGLKV_TREE_LISTED;
    TreeWay &w = h.tile;
    h.pairs = resident / c.kv_head_count > 1 ? resident / c.kv_head_count : 1;
    uint64_t pieces = 2 * divide_up(h.pairs, count * tiles) + 2, numbers = divide_up(most_tiles, h.pairs) * h.pairs;
    if (2 * most_tiles > h.pairs) numbers += h.pairs;
    if (!h.balanced) {
        // One length of splits for all, twice the average request's and an eighth of the longest's at least; workgroups
        // for the tiles of twice the average one.
        const uint64_t drafts = 64 * t.mask_words < 2 * mean ? 64 * t.mask_words : 2 * mean;
        h.tile_slots = (uint32_t)divide_up(drafts < c.query_count ? drafts : c.query_count, h.tile_queries);
        w.chunk = 2 * divide_up(c.sequence_slot_count, count);
        if (w.chunk > h.max_length) w.chunk = h.max_length;
        if (w.chunk < divide_up(h.max_length, 8)) w.chunk = divide_up(h.max_length, 8);
        if (w.chunk < h.unit * h.least) w.chunk = h.unit * h.least;
        pieces = divide_up(h.max_length, w.chunk);
        if (mul_ovf(count, pieces, &numbers) || mul_ovf(numbers, h.tile_slots, &numbers)) return attention_overflow();
    }
    w.splits = divide_up(h.max_length, h.unit * h.least);
    if (w.splits > pieces) w.splits = pieces;
    int32_t rc = split_records(c, &w);
    if (rc) return rc;
    if (h.pairs > UINT32_MAX / 2 || w.splits > UINT32_MAX || mul_ovf(numbers, c.kv_head_count, &w.base)) {
        h.tiles = false;
        return SGL_KV_OK;
    }
    h.used_at = w.record_bytes;  // (whole records: a multiple of 4)
    if (add_ovf(w.record_bytes, 4 * c.query_count, &w.record_bytes)) return attention_overflow();
    h.tiles = w.base <= UINT32_MAX / 256;
    return SGL_KV_OK;
}

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
    TreeWay &w = h.any;
    if (mul_ovf(c.query_count, c.kv_head_count, &w.base) || mul_ovf(w.base, divide_up(group, SGLKV_ATTN_HEADS), &w.base) ||
        mul_ovf(w.base, divide_up(c.value_head_dim, SGLKV_ATTN_DV), &w.base))
        return attention_overflow();
    // About 2,048 waves, each with 128 tokens or more.
    const uint64_t wanted = w.base < 2048 ? 2048 / w.base : 1;
    w.chunk = divide_up(h.max_length, wanted);
    if (w.chunk < 128) w.chunk = 128;
    w.chunk = divide_up(w.chunk, SGLKV_ATTN_TOKENS) * SGLKV_ATTN_TOKENS;
    const uint64_t limit = UINT32_MAX / 64;  // a dispatch counts its work-items in 32 bits
    if (w.base > limit) return too_large_dim("workgroups", w.base, limit);
    w.splits = divide_up(h.max_length, w.chunk);
    int32_t rc = split_records(c, &w);
    return rc ? rc : tile_shape(c, t, out);
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
    p.workspace_required_bytes = shape.any.record_bytes;
    if (shape.tiles && shape.tile.record_bytes > shape.any.record_bytes) p.workspace_required_bytes = shape.tile.record_bytes;
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
        {"workspace", &b->workspace, b->workspace_offset, fresh.workspace_required_bytes, &workspace, 16,
         fresh.workspace_required_bytes > 0}};
    if ((rc = resolve_buffers(ctx, all))) return rc;
    // (A query's row is read by a workgroup of its own for every 128 value dims, in the generic body.)
    if ((rc = refuse_overlaps(all, 6)) || (rc = refuse_overlaps(all, 8))) return rc;
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
    p.masks = reinterpret_cast<const uint64_t *>(masks);
    p.mask_words = (uint32_t)fresh.config.mask_words;
    p.max_length = shape.max_length;
    const bool vector = p.a.dk % 8 == 0 && p.a.dv % 8 == 0 &&
                        ((pool + lay.key_in_page_offset) | (pool + lay.value_in_page_offset) | lay.page_stride_bytes |
                         p.a.key_head_stride | p.a.key_token_stride | p.a.value_head_stride | p.a.value_token_stride) %
                                16 == 0;
    const bool tiles = vector && shape.tiles && queries % 16 == 0 && output % 8 == 0;
    const TreeWay &way = tiles ? shape.tile : shape.any;
    p.a.chunk_tokens = way.chunk;
    p.a.splits = (uint32_t)way.splits;
    DeviceScope scope(ctx->device);
    if (scope.status() != hipSuccess) return hip_fail(scope.status(), "hipSetDevice");
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (tiles) {
        p.a.page_stride32 = (uint32_t)p.a.page_stride;
        p.a.key_token_stride32 = p.a.value_token_stride32 = (uint32_t)p.a.key_token_stride;
        p.tile_queries = shape.tile_queries;
        p.tile_slots = shape.tile_slots;
        p.pairs = (uint32_t)shape.pairs;
        p.balanced = shape.balanced;
        p.unit = shape.unit;
        p.least = shape.least;
        p.used = reinterpret_cast<uint32_t *>(workspace + shape.used_at);
        const int dims = p.a.dk == 64 ? 0 : p.a.dk == 128 ? 1 : 2, rows = shape.row_waves == 1 ? 0 : shape.row_waves == 2 ? 1 : 2;
        rc = launch_kernel(ctx->tree_tile[dims][rows], way.base, 1, 1, 256, SGLKV_TREE_LDS_BYTES(p.a.dk, shape.row_waves), s, &p,
                           "tree attention launch");
    } else {
        const unsigned lds = 2 * (SGLKV_ATTN_HEADS * (p.a.dk_pad + 8) + SGLKV_ATTN_DV * SGLKV_ATTN_VT_STRIDE);
        rc = launch_kernel(ctx->tree_attention[vector ? 0 : 1], way.base, way.splits, 1, 64, lds, s, &p, "tree attention launch");
    }
    if (!rc && way.splits > 1)
        rc = launch_kernel(ctx->tree_combine, way.combine_grid, 1, 1, SGLKV_ATTN_COMBINE_THREADS, 0, s, &p,
                           "tree attention combine launch");
    return rc ? rc : ok();
}
