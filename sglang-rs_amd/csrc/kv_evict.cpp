// kv_evict.cpp -- host side of eviction by accumulated attention weight: the
// plans, the checks and the launches of accumulate_weights, select_tokens and
// compact_tokens (kernels in kv_evict.hip). Nothing here allocates or waits, and
// everything that a launch relies on is derived again at each call.
#include <hip/hip_runtime.h>

#include <string.h>

#include "kv_attention_route.h"
#include "kv_internal.h"

using namespace sglkv;

namespace {

constexpr uint64_t kMaxTokens = 1ull << 31;

uint64_t ceil_div(uint64_t a, uint64_t b) { return a / b + (a % b != 0); }

int32_t null_argument(const char *name) {
    return fail(SGL_KV_INVALID_ARGUMENT, name, 0, 0, 0, "null argument");
}

// A named buffer of a call and what it has to hold.
struct Want {
    const char *name;
    const sgl_kv_device_buffer *buffer;
    uint64_t offset, need;
    uint64_t *address;
    uint64_t align;
    bool used;
};

template <size_t N>
int32_t resolve(const sgl_rocm_kv_ctx *ctx, const Want (&all)[N]) {
    int32_t rc;
    for (const Want &x : all)
        if (x.used && (rc = check_device(ctx, x.name, *x.buffer))) return rc;
    for (const Want &x : all)
        if (x.used && (rc = attention_ptr(x.name, *x.buffer, x.offset, x.need, x.address))) return rc;
    for (const Want &x : all)
        if (x.used && *x.address % x.align)
            return fail(SGL_KV_INVALID_ARGUMENT, "alignment", 0, 0, 0, "%s must be aligned to %llu bytes", x.name,
                        (unsigned long long)x.align);
    return SGL_KV_OK;
}

// The launch shape of accumulate_weights. `rows`: the bodies for 16-byte rows of
// 64, 128 or 256 dims can take it; whether the buffers let them is the call's to
// see, so the workspace holds what either way needs.
struct WeightShape {
    uint64_t max_length;
    struct Way {
        uint64_t base, chunk, splits;  // statistics: workgroups of a split, its tokens
        uint64_t tiles, groups;        // accumulation: token tiles of a sequence, workgroups
        uint64_t bytes;                // workspace
    } any, rows;
    bool fits;                // `rows` is a way
    int body;                 // of ctx->weight_rows[dims]: 0 many rows, 1 few, 2 few with their scores
    uint64_t row_tiles, tile_queries, head_groups, segments;
    uint64_t stats_bytes, joined_bytes, score_stride;
};

constexpr uint64_t kMaxWorkgroups = UINT32_MAX / 64;  // of one wave: a dispatch counts its work-items in 32 bits

// Splits of `tokens` that give `waves` waves where `base` are those of one
// split, each of `least` tokens or more and a multiple of 64.
void split_tokens(uint64_t tokens, uint64_t base, uint64_t waves, uint64_t least, WeightShape::Way *w) {
    uint64_t chunk = ceil_div(tokens, base < waves ? waves / base : 1);
    if (chunk < least) chunk = least;
    if (chunk < ceil_div(tokens, 65535)) chunk = ceil_div(tokens, 65535);  // grid y
    w->chunk = ceil_div(chunk, 64) * 64;
    w->splits = ceil_div(tokens, w->chunk);
}

int32_t weight_shape(const sgl_kv_attention_plan_config &c, uint64_t max_sequence_length, WeightShape *out) {
    WeightShape &h = *out;
    memset(&h, 0, sizeof h);
    const uint64_t dk = c.query_key_head_dim, group = c.query_head_count / c.kv_head_count;
    if (dk > SGLKV_ATTN_MAX_DK) return too_large_dim("query_key_head_dim", dk, SGLKV_ATTN_MAX_DK);
    h.max_length =
        max_sequence_length && max_sequence_length < c.sequence_slot_count ? max_sequence_length : c.sequence_slot_count;
    uint64_t pairs;
    if (mul_ovf(c.query_count, c.query_head_count, &pairs)) return attention_overflow();

    // Any rows: a wave to a (query, KV head, 16 heads), and to 64 tokens.
    if (mul_ovf(c.query_count, c.kv_head_count, &h.any.base) ||
        mul_ovf(h.any.base, ceil_div(group, SGLKV_ATTN_HEADS), &h.any.base))
        return attention_overflow();
    if (h.any.base > kMaxWorkgroups) return too_large_dim("workgroups", h.any.base, kMaxWorkgroups);
    split_tokens(h.max_length, h.any.base, 2048, 128, &h.any);
    h.any.tiles = ceil_div(h.max_length, SGLKV_WEIGHTS_TILE);
    if (mul_ovf(h.any.tiles, c.kv_head_count, &h.any.groups) || mul_ovf(h.any.groups, c.request_count, &h.any.groups))
        return attention_overflow();
    if (h.any.groups > kMaxWorkgroups) return too_large_dim("workgroups", h.any.groups, kMaxWorkgroups);
    if (mul_ovf(pairs, h.any.splits, &h.any.bytes) || mul_ovf(h.any.bytes, 8, &h.any.bytes)) return attention_overflow();

    // 16-byte rows of 64, 128 or 256 dims; rows and tokens are counted in 32 bits.
    h.fits = (dk == 64 || dk == 128 || dk == 256) && pairs < (1ull << 27) && h.max_length <= (1ull << 31);
    if (!h.fits) return SGL_KV_OK;
    const uint64_t per = ceil_div(c.query_count, c.request_count);  // queries of a request
    // Kept scores cost 8 bytes a (query head, token), written and read, K rows read
    // a second time 2 dk bytes a token; 256 MiB of them at most.
    h.score_stride = ceil_div(h.max_length, 64) * 64;
    uint64_t score_bytes = 0;
    const bool keeps = 8 * group * per < 2 * dk && !mul_ovf(pairs, 4 * h.score_stride, &score_bytes) &&
                       score_bytes <= (256ull << 20);
    h.body = keeps ? 2 : per * group >= 32 ? 0 : 1;
    const uint64_t tile_rows = h.body == 0 ? (dk == 256 ? 128 : 256) : 16;
    h.head_groups = group > tile_rows ? ceil_div(group, tile_rows) : 1;
    h.tile_queries = group > tile_rows ? 1 : tile_rows / group;
    if (h.tile_queries > per) h.tile_queries = per;
    h.row_tiles = ceil_div(c.query_count, h.tile_queries);
    h.rows.base = h.row_tiles * h.head_groups * c.kv_head_count;
    // (Workgroups of four waves are placed eight items at a time.)
    auto placed = [&](uint64_t items) { return ceil_div(items, 8) * 8 * c.kv_head_count; };
    if (h.body == 0) h.rows.base = placed(h.row_tiles * h.head_groups);
    if (h.rows.base > kMaxWorkgroups / 4) {
        h.fits = false;
        return SGL_KV_OK;
    }
    // (Ragged sequences: as many workgroups have tokens as equal ones of the mean would.)
    // Many rows: four workgroups a CU. A split reads all queries again and starts for 5
    // us: four prompts of up to 2,048 tokens, 8 KV heads of 4, dims 128, took 80, 86 and
    // 107 us with 1,024, 2,048 and 4,096; one of 2,048 tokens 40 and 50 with the first two.
    const uint64_t mean = ceil_div(c.sequence_slot_count, c.request_count), base = h.row_tiles * h.head_groups * c.kv_head_count,
                   live = ceil_div(base * (mean < h.max_length ? mean : h.max_length), h.max_length);
    split_tokens(h.max_length, live, h.body == 0 ? 1024 : 4096, h.body == 0 ? 256 : 64, &h.rows);
    const uint64_t tile = keeps ? SGLKV_WEIGHTS_APPLY : dk == 256 ? 2 * SGLKV_WEIGHTS_TILE : 4 * SGLKV_WEIGHTS_TILE;
    h.rows.tiles = ceil_div(h.max_length, tile);
    // A prompt's first tokens are attended by all of its queries, its last by a
    // few: parts of 512 rows or more even the workgroups out. Short prompts leave CUs
    // idle while a few workgroups go through all rows, 32 in 0.8 us: their parts may be
    // as small as 64 rows where 384 or more are saved the joining launch's 6 us.
    const uint64_t rows = per * group, alone = h.rows.tiles * c.kv_head_count * c.request_count;
    h.segments = rows / 512;
    if (rows >= 384 && alone * h.segments < 1024) {
        const uint64_t fill = ceil_div(1024, alone);
        h.segments = fill < rows / 64 ? fill : rows / 64;
    }
    if (keeps || h.segments < 1) h.segments = 1;
    if (h.segments > 16) h.segments = 16;
    // (At most 16 times `any`'s.)
    h.rows.groups = keeps ? h.rows.tiles * c.kv_head_count * c.request_count : placed(h.rows.tiles * c.request_count * h.segments);
    if (h.rows.groups > kMaxWorkgroups / 4 || mul_ovf(pairs, 8 * h.rows.splits, &h.stats_bytes)) {
        h.fits = false;
        return SGL_KV_OK;
    }
    h.stats_bytes = ceil_div(h.stats_bytes, 256) * 256;
    h.joined_bytes = keeps || h.rows.splits == 1 ? 0 : ceil_div(8 * pairs, 256) * 256;
    uint64_t sums = 0;
    if (h.segments > 1 && (mul_ovf(h.segments * 4, c.kv_head_count, &sums) || mul_ovf(sums, c.sequence_slot_count, &sums) ||
                           sums >> 40)) {
        h.fits = false;
        return SGL_KV_OK;
    }
    h.rows.bytes = h.stats_bytes + (keeps ? score_bytes : h.joined_bytes + sums);
    return SGL_KV_OK;
}

}  // namespace

extern "C" int32_t sgl_kv_weight_plan_new(const sgl_kv_attention_plan *attention, uint64_t max_sequence_length,
                                          sgl_kv_weight_plan *out) {
    if (!attention || !out) return null_argument("attention/out");
    sgl_kv_weight_plan p;
    memset(&p, 0, sizeof p);
    int32_t rc = sgl_kv_attention_plan_new(&attention->config, &p.attention);
    WeightShape shape;
    if (!rc) rc = weight_shape(p.attention.config, max_sequence_length, &shape);
    if (rc) return rc;
    const sgl_kv_attention_plan_config &c = p.attention.config;
    p.max_sequence_length = max_sequence_length;
    if (mul_ovf(c.kv_head_count, c.sequence_slot_count, &p.weights_required_bytes) ||
        mul_ovf(p.weights_required_bytes, 4, &p.weights_required_bytes))
        return attention_overflow();
    p.workspace_required_bytes = shape.fits && shape.rows.bytes > shape.any.bytes ? shape.rows.bytes : shape.any.bytes;
    *out = p;
    return ok();
}

extern "C" int32_t sgl_rocm_kv_accumulate_weights(sgl_rocm_kv_ctx *ctx, const sgl_kv_weight_plan *plan,
                                                  const sgl_kv_weight_buffers *b, void *stream) {
    if (!ctx || !plan || !b) return null_argument("ctx/plan/buffers");
    sgl_kv_weight_plan fresh;
    WeightShape shape;
    int32_t rc = sgl_kv_weight_plan_new(&plan->attention, plan->max_sequence_length, &fresh);
    if (!rc) rc = weight_shape(fresh.attention.config, fresh.max_sequence_length, &shape);
    if (rc) return rc;
    const sgl_kv_attention_plan &a = fresh.attention;
    const sgl_kv_attention_plan_config &c = a.config;
    const sgl_kv_attention_layout &lay = c.layout;
    uint64_t queries, requests, lengths, offsets, slots, pool, weights, workspace;
    const sgl_kv_attention_buffers &ab = b->attention;
    const Want all[] = {
        {"queries", &ab.queries, ab.queries_offset, a.query_required_bytes, &queries, 2, true},
        {"query_request_indices", &ab.query_request_indices, ab.query_request_indices_offset,
         a.query_request_indices_required_bytes, &requests, 4, true},
        {"query_sequence_lengths", &ab.query_sequence_lengths, ab.query_sequence_lengths_offset,
         a.query_sequence_lengths_required_bytes, &lengths, 8, true},
        {"request_slot_offsets", &ab.request_slot_offsets, ab.request_slot_offsets_offset,
         a.request_slot_offsets_required_bytes, &offsets, 8, true},
        {"sequence_slots", &ab.sequence_slots, ab.sequence_slots_offset, a.sequence_slots_required_bytes, &slots, 8, true},
        {"pool", &ab.pool, ab.pool_offset, a.pool_required_bytes, &pool, 2, true},
        {"weights", &b->weights, b->weights_offset, fresh.weights_required_bytes, &weights, 4, true},
        {"workspace", &b->workspace, b->workspace_offset, fresh.workspace_required_bytes, &workspace, 16, true}};
    if ((rc = resolve(ctx, all))) return rc;
    if ((lay.key_in_page_offset | lay.page_stride_bytes) & 1)
        return fail(SGL_KV_INVALID_ARGUMENT, "alignment", 0, 0, 0, "pool rows must be aligned to their element size");
    sglkv_weights_params p;
    memset(&p, 0, sizeof p);
    p.a.queries = reinterpret_cast<const uint16_t *>(queries);
    p.a.query_request_indices = reinterpret_cast<const uint32_t *>(requests);
    p.a.query_sequence_lengths = reinterpret_cast<const uint64_t *>(lengths);
    p.a.request_slot_offsets = reinterpret_cast<const uint64_t *>(offsets);
    p.a.sequence_slots = reinterpret_cast<const uint64_t *>(slots);
    p.a.pool = reinterpret_cast<const uint8_t *>(pool);
    p.a.partial = reinterpret_cast<float *>(workspace);
    p.a.flag = ctx->attn_flag;
    attention_geometry(c, &p.a);
    p.a.zero_row = ctx->zero_row;
    p.weights = reinterpret_cast<float *>(weights);
    p.max_length = shape.max_length;
    const bool vector = p.a.dk % 8 == 0 && queries % 16 == 0 &&
                        ((pool + lay.key_in_page_offset) | lay.page_stride_bytes | p.a.key_head_stride |
                         p.a.key_token_stride) % 16 == 0;
    const bool rows = vector && shape.fits;
    const WeightShape::Way &way = rows ? shape.rows : shape.any;
    p.a.splits = (uint32_t)way.splits;
    p.a.chunk_tokens = way.chunk;
    p.tiles = (uint32_t)way.tiles;
    DeviceScope scope(ctx->device);
    if (scope.status() != hipSuccess) return hip_fail(scope.status(), "hipSetDevice");
    hipStream_t s = static_cast<hipStream_t>(stream);
    const char *const stats = "weight statistics launch", *const sums = "weight accumulation launch";
    if (!rows) {
        rc = launch_kernel(ctx->weight_stats[vector ? 0 : 1], way.base, way.splits, 1, 64,
                           2 * SGLKV_ATTN_HEADS * (p.a.dk_pad + 8), s, &p, stats);
        if (!rc) rc = launch_kernel(ctx->accumulate_weights[vector ? 0 : 1], way.groups, 1, 1, 64, 0, s, &p, sums);
        return rc ? rc : ok();
    }
    p.row_tiles = (uint32_t)shape.row_tiles;
    p.tile_queries = (uint32_t)shape.tile_queries;
    p.tile_head_groups = (uint32_t)shape.head_groups;
    p.score_stride = shape.score_stride;
    const bool keeps = shape.body == 2;
    if (keeps) p.scores = reinterpret_cast<float *>(workspace + shape.stats_bytes);
    p.joined = reinterpret_cast<float *>(way.splits > 1 ? workspace + shape.stats_bytes : workspace);
    p.segments = (uint32_t)shape.segments;
    if (shape.segments > 1) p.partial_sums = reinterpret_cast<float *>(workspace + shape.stats_bytes + shape.joined_bytes);
    const auto &body = ctx->weight_rows[p.a.dk == 64 ? 0 : p.a.dk == 128 ? 1 : 2];
    rc = launch_kernel(body[shape.body], way.base, way.splits, 1, shape.body == 0 ? 256 : 64,
                       keeps ? SGLKV_WEIGHTS_LDS_BYTES(p.a.dk) : 0, s, &p, stats);
    for (p.join_lanes = 1; p.join_lanes < way.splits && p.join_lanes < 16;) p.join_lanes *= 2;
    if (!rc && !keeps && way.splits > 1)
        rc = launch_kernel(ctx->join_statistics,
                           ceil_div(c.query_count * c.query_head_count, SGLKV_WEIGHTS_THREADS / p.join_lanes), 1, 1,
                           SGLKV_WEIGHTS_THREADS, 0, s, &p, "weight statistics join launch");
    if (!rc && keeps) rc = launch_kernel(ctx->apply_scores, way.groups, 1, 1, SGLKV_WEIGHTS_THREADS, 0, s, &p, sums);
    if (!rc && !keeps) rc = launch_kernel(body[3], way.groups, 1, 1, 256, 0, s, &p, sums);
    if (!rc && shape.segments > 1)
        rc = launch_kernel(ctx->add_segments,
                           ceil_div(shape.max_length, SGLKV_WEIGHTS_THREADS) * c.kv_head_count * c.request_count, 1, 1,
                           SGLKV_WEIGHTS_THREADS, 0, s, &p, "weight segments launch");
    return rc ? rc : ok();
}

extern "C" int32_t sgl_kv_eviction_plan_new(const sgl_kv_eviction_config *config, sgl_kv_eviction_plan *out) {
    if (!config || !out) return null_argument("config/out");
    const sgl_kv_eviction_config &c = *config;
    const struct {
        const char *name;
        uint64_t value;
    } dims[] = {{"request_count", c.request_count},
                {"kv_head_count", c.kv_head_count},
                {"sequence_slot_count", c.sequence_slot_count},
                {"max_kept", c.max_kept}};
    for (const auto &d : dims)
        if (d.value == 0)
            return fail(SGL_KV_ZERO_DIMENSION, d.name, 0, 0, 0, "eviction dimension %s must be non-zero", d.name);
    if (c.first_tokens > c.max_kept || c.last_tokens > c.max_kept - c.first_tokens)
        return fail(SGL_KV_INVALID_ARGUMENT, "first_tokens", c.first_tokens, c.last_tokens, c.max_kept,
                    "%llu first and %llu last tokens do not fit a list of %llu", (unsigned long long)c.first_tokens,
                    (unsigned long long)c.last_tokens, (unsigned long long)c.max_kept);
    const uint64_t longest =
        c.max_sequence_length && c.max_sequence_length < c.sequence_slot_count ? c.max_sequence_length : c.sequence_slot_count;
    if (c.max_kept > kMaxTokens) return too_large_dim("max_kept", c.max_kept, kMaxTokens);
    if (longest > kMaxTokens) return too_large_dim("max_sequence_length", longest, kMaxTokens);
    sgl_kv_eviction_plan p;
    memset(&p, 0, sizeof p);
    p.config = c;
    uint64_t lists, offsets;
    if (mul_ovf(c.request_count, c.kv_head_count, &lists) || add_ovf(c.request_count, 1, &offsets) ||
        mul_ovf(c.request_count, 8, &p.request_lengths_required_bytes) ||
        mul_ovf(offsets, 8, &p.request_slot_offsets_required_bytes) ||
        mul_ovf(c.sequence_slot_count, 8, &p.sequence_slots_required_bytes) ||
        mul_ovf(c.destination_slot_count, 8, &p.destination_slots_required_bytes) ||
        mul_ovf(c.kv_head_count, c.sequence_slot_count, &p.weights_required_bytes) ||
        mul_ovf(p.weights_required_bytes, 4, &p.weights_required_bytes) ||
        mul_ovf(c.kv_head_count, c.destination_slot_count, &p.destination_weights_required_bytes) ||
        mul_ovf(p.destination_weights_required_bytes, 4, &p.destination_weights_required_bytes) ||
        mul_ovf(lists, c.max_kept, &p.kept_required_bytes) || mul_ovf(p.kept_required_bytes, 4, &p.kept_required_bytes))
        return attention_overflow();
    const uint64_t limit = UINT32_MAX / SGLKV_EVICT_THREADS;  // a dispatch counts its work-items in 32 bits
    if (lists > limit) return too_large_dim("workgroups", lists, limit);
    *out = p;
    return ok();
}

namespace {

// What both calls have in common.
int32_t eviction_params(sgl_rocm_kv_ctx *ctx, const sgl_kv_eviction_plan *plan, const sgl_kv_eviction_buffers *b,
                        bool copies, sglkv_evict_params *params) {
    if (!ctx || !plan || !b) return null_argument("ctx/plan/buffers");
    sgl_kv_eviction_plan fresh;
    int32_t rc = sgl_kv_eviction_plan_new(&plan->config, &fresh);
    if (rc) return rc;
    const sgl_kv_eviction_config &c = fresh.config;
    const bool moves = copies && (b->weights.ptr || b->destination_weights.ptr);
    uint64_t lengths, offsets, slots = 0, weights = 0, kept, to_offsets = 0, to_slots = 0, to_weights = 0;
    const Want all[] = {
        {"request_lengths", &b->request_lengths, b->request_lengths_offset, fresh.request_lengths_required_bytes, &lengths, 8,
         true},
        {"request_slot_offsets", &b->request_slot_offsets, b->request_slot_offsets_offset,
         fresh.request_slot_offsets_required_bytes, &offsets, 8, true},
        {"sequence_slots", &b->sequence_slots, b->sequence_slots_offset, fresh.sequence_slots_required_bytes, &slots, 8,
         copies},
        {"weights", &b->weights, b->weights_offset, fresh.weights_required_bytes, &weights, 4, !copies || moves},
        {"kept", &b->kept, b->kept_offset, fresh.kept_required_bytes, &kept, 4, true},
        {"destination_slot_offsets", &b->destination_slot_offsets, b->destination_slot_offsets_offset,
         fresh.request_slot_offsets_required_bytes, &to_offsets, 8, copies},
        {"destination_slots", &b->destination_slots, b->destination_slots_offset, fresh.destination_slots_required_bytes,
         &to_slots, 8, copies && c.destination_slot_count > 0},
        {"destination_weights", &b->destination_weights, b->destination_weights_offset,
         fresh.destination_weights_required_bytes, &to_weights, 4, moves && c.destination_slot_count > 0}};
    if ((rc = resolve(ctx, all))) return rc;
    sglkv_evict_params &p = *params;
    memset(&p, 0, sizeof p);
    p.request_lengths = reinterpret_cast<const uint64_t *>(lengths);
    p.request_slot_offsets = reinterpret_cast<const uint64_t *>(offsets);
    p.sequence_slots = reinterpret_cast<const uint64_t *>(slots);
    p.weights = reinterpret_cast<const float *>(weights);
    p.kept = reinterpret_cast<uint32_t *>(kept);
    p.to_offsets = reinterpret_cast<const uint64_t *>(to_offsets);
    p.to_slots = reinterpret_cast<const uint64_t *>(to_slots);
    p.to_weights = reinterpret_cast<float *>(to_weights);
    p.flag = ctx->attn_flag;
    p.request_count = c.request_count;
    p.sequence_slot_count = c.sequence_slot_count;
    p.to_slot_count = c.destination_slot_count;
    p.max_length = c.max_sequence_length && c.max_sequence_length < c.sequence_slot_count ? c.max_sequence_length
                                                                                          : c.sequence_slot_count;
    p.heads = (uint32_t)c.kv_head_count;
    p.max_kept = (uint32_t)c.max_kept;
    p.first_tokens = (uint32_t)c.first_tokens;
    p.last_tokens = (uint32_t)c.last_tokens;
    return SGL_KV_OK;
}

}  // namespace

extern "C" int32_t sgl_rocm_kv_select_tokens(sgl_rocm_kv_ctx *ctx, const sgl_kv_eviction_plan *plan,
                                             const sgl_kv_eviction_buffers *b, void *stream) {
    sglkv_evict_params p;
    int32_t rc = eviction_params(ctx, plan, b, false, &p);
    if (rc) return rc;
    DeviceScope scope(ctx->device);
    if (scope.status() != hipSuccess) return hip_fail(scope.status(), "hipSetDevice");
    rc = launch_kernel(ctx->select_tokens, p.request_count * p.heads, 1, 1, SGLKV_EVICT_THREADS, 0,
                       static_cast<hipStream_t>(stream), &p, "token selection launch");
    return rc ? rc : ok();
}

extern "C" int32_t sgl_rocm_kv_compact_tokens(sgl_rocm_kv_ctx *ctx, const sgl_kv_eviction_plan *plan,
                                              const sgl_kv_eviction_buffers *b, const sgl_kv_pool_view *source,
                                              const sgl_kv_pool_view *destination, void *stream) {
    if (!source || !destination) return null_argument("source/destination");
    sglkv_evict_params p;
    int32_t rc = eviction_params(ctx, plan, b, true, &p);
    if (rc || (rc = pool_heads_side(source, &p.src)) || (rc = pool_heads_side(destination, &p.dst))) return rc;
    if (source->heads != p.heads || destination->heads != p.heads ||
        source->tensor_count != destination->tensor_count || source->row_bytes != destination->row_bytes ||
        (source->tensor_count == 2 && view_row_bytes(*source, 1) != view_row_bytes(*destination, 1)))
        return fail(SGL_KV_INVALID_ARGUMENT, "views", source->heads, destination->heads, p.heads,
                    "the views' heads (%u, %u, plan %u), tensors or row widths differ", source->heads, destination->heads,
                    p.heads);
    const sgl_kv_device_buffer from = {source->base, source->byte_len}, to = {destination->base, destination->byte_len};
    if ((rc = check_device(ctx, "source", from)) || (rc = check_device(ctx, "destination", to))) return rc;
    if (p.sequence_slots == p.to_slots && p.src.plane[0] == p.dst.plane[0])
        return fail(SGL_KV_INVALID_ARGUMENT, "in place", 0, 0, 0, "rows cannot be compacted onto their own slots");
    if (p.to_weights && p.to_weights == p.weights)
        return fail(SGL_KV_INVALID_ARGUMENT, "in place", 0, 0, 0, "sums cannot be compacted onto their own columns");
    if (source->scale && destination->scale) {
        const sgl_kv_device_buffer scales[2] = {{source->scale, 4ull * source->tensor_count},
                                                {destination->scale, 4ull * source->tensor_count}};
        if ((rc = check_device(ctx, "source scale", scales[0])) || (rc = check_device(ctx, "destination scale", scales[1])))
            return rc;
        p.scale_src = source->scale;
        p.scale_dst = destination->scale;
    }
    // The widest of 16, 4, 2 and 1 bytes that divides every address and chunk.
    p.tensors = source->tensor_count;
    uint64_t bits = 0, chunk[2];
    for (uint32_t t = 0; t < p.tensors; ++t) {
        chunk[t] = view_row_bytes(*source, t) / p.heads;
        bits |= chunk[t];
        for (const sglkv_side *x : {&p.src, &p.dst})
            bits |= x->plane[t] | x->stride[t] | x->pos_mult[t] | x->head_stride[t];
    }
    const int width = bits % 16 == 0 ? 0 : bits % 4 == 0 ? 1 : bits % 2 == 0 ? 2 : 3;
    const uint64_t bytes = width == 0 ? 16 : width == 1 ? 4 : width == 2 ? 2 : 1;
    for (uint32_t t = 0; t < p.tensors; ++t) {
        const uint64_t pieces = chunk[t] / bytes;
        if (pieces > UINT32_MAX / 2) return too_large_dim("row_bytes", chunk[t], UINT32_MAX / 2 * bytes);
        p.vectors[t] = (uint32_t)pieces;
        p.lanes[t] = 1;
        while (p.lanes[t] < pieces && p.lanes[t] < SGLKV_COMPACT_THREADS) p.lanes[t] *= 2;
    }
    p.block_heads = p.heads < SGLKV_COMPACT_HEADS ? p.heads : SGLKV_COMPACT_HEADS;
    p.rows = SGLKV_COMPACT_ROWS;
    const uint64_t tiles = ceil_div(p.max_kept, p.rows), blocks = ceil_div(p.heads, p.block_heads);
    uint64_t grid;
    if (mul_ovf(tiles, p.request_count, &grid)) return attention_overflow();
    const uint64_t limit = UINT32_MAX / SGLKV_COMPACT_THREADS;  // a dispatch counts its work-items in 32 bits
    if (grid > limit) return too_large_dim("workgroups", grid, limit);
    if (blocks > 65535) return too_large_dim("kv_head_count", p.heads, 65535ull * p.block_heads);
    p.row_tiles = (uint32_t)tiles;
    DeviceScope scope(ctx->device);
    if (scope.status() != hipSuccess) return hip_fail(scope.status(), "hipSetDevice");
    rc = launch_kernel(ctx->compact_tokens[width], grid, blocks, p.tensors, SGLKV_COMPACT_THREADS, 0,
                       static_cast<hipStream_t>(stream), &p, "token compaction launch");
    return rc ? rc : ok();
}
