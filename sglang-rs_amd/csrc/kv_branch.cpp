// kv_branch.cpp -- host side of keep_drafts and fork_sequences: the plans, the
// checks and the launches (kernels in kv_branch.hip). Nothing here allocates or
// waits, and what a launch relies on is derived again at each call.
#include <hip/hip_runtime.h>

#include <string.h>

#include "kv_call.h"

using namespace sglkv;

namespace {

constexpr uint64_t kMaxSequences = 1ull << 24;
constexpr uint64_t kMaxReservedRow = 1ull << 20;  // a thread may walk over a row's reserved pages

int32_t zero_dimension(const char *what, const char *name) {
    return fail(SGL_KV_ZERO_DIMENSION, name, 0, 0, 0, "%s dimension %s must be non-zero", what, name);
}

struct Named {
    const char *name;
    uint64_t value, maximum;
};
template <size_t N>
int32_t check_dims(const char *what, const Named (&dims)[N]) {
    for (const Named &d : dims)
        if (d.value == 0) return zero_dimension(what, d.name);
    for (const Named &d : dims)
        if (d.value > d.maximum) return too_large_dim(d.name, d.value, d.maximum);
    return SGL_KV_OK;
}

}  // namespace

extern "C" int32_t sgl_kv_draft_plan_new(const sgl_kv_draft_config *config, sgl_kv_draft_plan *out) {
    if (!config || !out) return null_arguments("config/out");
    const sgl_kv_draft_config &c = *config;
    const Named dims[] = {{"request_count", c.request_count, UINT64_MAX},
                          {"sequence_slot_count", c.sequence_slot_count, UINT64_MAX},
                          {"max_kept", c.max_kept, 1ull << 31}};
    int32_t rc = check_dims("draft", dims);
    if (rc) return rc;
    sgl_kv_draft_plan p;
    memset(&p, 0, sizeof p);
    p.config = c;
    uint64_t offsets;
    if (add_ovf(c.request_count, 1, &offsets) || mul_ovf(c.request_count, 8, &p.request_lengths_required_bytes) ||
        mul_ovf(offsets, 8, &p.request_slot_offsets_required_bytes) ||
        mul_ovf(c.sequence_slot_count, 8, &p.sequence_slots_required_bytes) ||
        mul_ovf(c.request_count, 4 * c.max_kept, &p.kept_required_bytes))
        return attention_overflow();
    *out = p;
    return ok();
}

extern "C" int32_t sgl_rocm_kv_keep_drafts(sgl_rocm_kv_ctx *ctx, const sgl_kv_draft_plan *plan,
                                           const sgl_kv_draft_buffers *b, const sgl_kv_pool_view *pool,
                                           uint32_t layer_count, uint64_t layer_stride, void *stream) {
    if (!ctx || !plan || !b) return null_arguments("ctx/plan/buffers");
    sgl_kv_draft_plan fresh;
    int32_t rc = sgl_kv_draft_plan_new(&plan->config, &fresh);
    if (rc) return rc;
    const sgl_kv_draft_config &c = fresh.config;
    uint64_t lengths, offsets, slots, kept;
    const CallBuffer all[] = {
        {"request_lengths", &b->request_lengths, b->request_lengths_offset, fresh.request_lengths_required_bytes, &lengths, 8,
         true},
        {"request_slot_offsets", &b->request_slot_offsets, b->request_slot_offsets_offset,
         fresh.request_slot_offsets_required_bytes, &offsets, 8, true},
        {"sequence_slots", &b->sequence_slots, b->sequence_slots_offset, fresh.sequence_slots_required_bytes, &slots, 8, true},
        {"kept", &b->kept, b->kept_offset, fresh.kept_required_bytes, &kept, 4, true}};
    if ((rc = resolve_buffers(ctx, all))) return rc;
    sglkv_keep_params p;
    memset(&p, 0, sizeof p);
    if ((rc = pool_layers(ctx, pool, layer_count, layer_stride, &p.pool, &p.heads))) return rc;
    if (p.pool.slot_count > UINT32_MAX) return too_large_dim("slot_count", p.pool.slot_count, UINT32_MAX);
    p.request_lengths = reinterpret_cast<const uint64_t *>(lengths);
    p.request_slot_offsets = reinterpret_cast<const uint64_t *>(offsets);
    p.sequence_slots = reinterpret_cast<const uint64_t *>(slots);
    p.kept = reinterpret_cast<const uint32_t *>(kept);
    p.flag = ctx->attn_flag;
    p.sequence_slot_count = c.sequence_slot_count;
    p.max_kept = (uint32_t)c.max_kept;
    p.tensors = pool->tensor_count;
    // The widest of 16, 4 and 1 bytes that divides every address and chunk.
    uint64_t bits = layer_count > 1 ? layer_stride : 0, chunk[2] = {0, 0};
    for (uint32_t t = 0; t < p.tensors; ++t) {
        chunk[t] = view_row_bytes(*pool, t) / p.heads;
        bits |= chunk[t] | p.pool.plane[t] | p.pool.stride[t] | p.pool.pos_mult[t] | p.pool.head_stride[t];
    }
    const int width = bits % 16 == 0 ? 0 : bits % 4 == 0 ? 1 : 2;
    const uint64_t bytes = width == 0 ? 16 : width == 1 ? 4 : 1;
    uint64_t pieces = 0;
    for (uint32_t t = 0; t < p.tensors; ++t) {
        if (chunk[t] / bytes * p.heads > UINT32_MAX / 4) return too_large_dim("row_bytes", chunk[t] * p.heads, UINT32_MAX / 4 * bytes);
        p.chunk_pieces[t] = (uint32_t)(chunk[t] / bytes);
        pieces += chunk[t] / bytes * p.heads;
    }
    p.pieces = (uint32_t)pieces;
    p.groups = (uint32_t)divide_up(pieces, SGLKV_KEEP_THREADS);
    uint64_t grid;
    const uint64_t limit = UINT32_MAX / SGLKV_KEEP_THREADS;  // a dispatch counts its work-items in 32 bits
    if (mul_ovf(c.request_count, p.groups, &grid)) return attention_overflow();
    if (grid > limit) return too_large_dim("workgroups", grid, limit);
    DeviceScope scope(ctx->device);
    if (scope.status() != hipSuccess) return hip_fail(scope.status(), "hipSetDevice");
    rc = launch_kernel(ctx->keep_drafts[width], grid, layer_count, 1, SGLKV_KEEP_THREADS, 0, static_cast<hipStream_t>(stream),
                       &p, "draft compaction launch");
    return rc ? rc : ok();
}

namespace {

// The workspace's parts, each a multiple of 64 bytes.
struct ForkParts {
    uint64_t first, children, held, before, copies, freed, bytes;
};

ForkParts fork_parts(const sgl_kv_fork_config &c) {
    auto lines = [](uint64_t words) { return divide_up(4 * words, 64) * 64; };
    ForkParts f;
    f.first = 4 * SGLKV_FORK_HEAD_WORDS;
    f.children = f.first + lines(c.parent_count);
    f.held = f.children + lines(c.parent_count);
    f.before = f.held + lines(c.keep_reserved ? c.parent_count : 0);
    f.copies = f.before + lines(c.sequence_count);
    f.freed = f.copies + sizeof(sglkv_page_copy) / 4 * lines(c.sequence_count);
    f.bytes = f.freed + lines(divide_up(c.page_count, 32));
    return f;
}

}  // namespace

extern "C" int32_t sgl_kv_fork_plan_new(const sgl_kv_fork_config *config, sgl_kv_fork_plan *out) {
    if (!config || !out) return null_arguments("config/out");
    const sgl_kv_fork_config &c = *config;
    const Named dims[] = {{"sequence_count", c.sequence_count, kMaxSequences},
                          {"parent_count", c.parent_count, kMaxSequences},
                          {"table_pages", c.table_pages, 1ull << 31},
                          {"page_size", c.page_size, UINT32_MAX},
                          {"page_count", c.page_count, INT32_MAX}};
    int32_t rc = check_dims("fork", dims);
    if (rc) return rc;
    if (c.append_tokens > UINT32_MAX) return too_large_dim("append_tokens", c.append_tokens, UINT32_MAX);
    if (c.keep_reserved > 1)
        return fail(SGL_KV_INVALID_ARGUMENT, "keep_reserved", c.keep_reserved, 1, 0, "keep_reserved is 0 or 1, not %llu",
                    (unsigned long long)c.keep_reserved);
    if (c.keep_reserved && c.table_pages > kMaxReservedRow) return too_large_dim("table_pages", c.table_pages, kMaxReservedRow);
    // A workgroup to each sequence, old and new.
    const uint64_t limit = UINT32_MAX / SGLKV_FORK_THREADS;
    if (c.sequence_count + c.parent_count > limit) return too_large_dim("workgroups", c.sequence_count + c.parent_count, limit);
    sgl_kv_fork_plan p;
    memset(&p, 0, sizeof p);
    p.config = c;
    const ForkParts parts = fork_parts(c);
    p.parents_required_bytes = 4 * c.sequence_count;
    p.lengths_required_bytes = 8 * c.parent_count;
    p.forked_lengths_required_bytes = 8 * c.sequence_count;
    p.page_tables_required_bytes = 4 * c.parent_count * c.table_pages;
    p.forked_tables_required_bytes = 4 * c.sequence_count * c.table_pages;
    p.page_references_required_bytes = p.free_pages_required_bytes = 4 * c.page_count;
    p.free_count_required_bytes = 8;
    p.workspace_required_bytes = parts.bytes;
    *out = p;
    return ok();
}

extern "C" int32_t sgl_rocm_kv_fork_sequences(sgl_rocm_kv_ctx *ctx, const sgl_kv_fork_plan *plan,
                                              const sgl_kv_fork_buffers *b, const sgl_kv_pool_view *pool,
                                              uint32_t layer_count, uint64_t layer_stride, void *stream) {
    if (!ctx || !plan || !b) return null_arguments("ctx/plan/buffers");
    sgl_kv_fork_plan f;
    int32_t rc = sgl_kv_fork_plan_new(&plan->config, &f);
    if (rc) return rc;
    const sgl_kv_fork_config &c = f.config;
    uint64_t parents, lengths, tables, forked_lengths, forked_tables, references, free_pages, free_count, workspace;
    const CallBuffer all[] = {
        {"parents", &b->parents, b->parents_offset, f.parents_required_bytes, &parents, 4, true},
        {"lengths", &b->lengths, b->lengths_offset, f.lengths_required_bytes, &lengths, 8, true},
        {"page_tables", &b->page_tables, b->page_tables_offset, f.page_tables_required_bytes, &tables, 4, true},
        {"forked_lengths", &b->forked_lengths, b->forked_lengths_offset, f.forked_lengths_required_bytes, &forked_lengths, 8,
         true},
        {"forked_tables", &b->forked_tables, b->forked_tables_offset, f.forked_tables_required_bytes, &forked_tables, 4, true},
        {"page_references", &b->page_references, b->page_references_offset, f.page_references_required_bytes, &references, 4,
         true},
        {"free_pages", &b->free_pages, b->free_pages_offset, f.free_pages_required_bytes, &free_pages, 4, true},
        {"free_count", &b->free_count, b->free_count_offset, f.free_count_required_bytes, &free_count, 8, true},
        {"workspace", &b->workspace, b->workspace_offset, f.workspace_required_bytes, &workspace, 16, true}};
    if ((rc = resolve_buffers(ctx, all))) return rc;
    // The new lengths and tables are written while the old ones are read.
    if ((rc = refuse_overlaps(all, 3)) || (rc = refuse_overlaps(all, 4))) return rc;
    sglkv_fork_params p;
    memset(&p, 0, sizeof p);
    if ((rc = pool_layers(ctx, pool, layer_count, layer_stride, &p.pool, &p.heads))) return rc;
    if (pool->page_size != c.page_size || pool->page_count != c.page_count)
        return fail(SGL_KV_INVALID_ARGUMENT, "pool", pool->page_size, pool->page_count, 0,
                    "the pool has %llu pages of %llu tokens, the plan %llu of %llu", (unsigned long long)pool->page_count,
                    (unsigned long long)pool->page_size, (unsigned long long)c.page_count, (unsigned long long)c.page_size);
    // The pool's pages, from the first byte of the first to the last of the last, are copied from and to all the while.
    uint64_t begin = UINT64_MAX, end = 0;
    for (uint32_t t = 0; t < pool->tensor_count; ++t) {
        const uint64_t last = p.pool.plane[t] + (c.page_count - 1) * pool->page_stride_bytes +
                              (uint64_t)(layer_count - 1) * layer_stride + c.page_size * view_row_bytes(*pool, t);
        begin = p.pool.plane[t] < begin ? p.pool.plane[t] : begin;
        end = last > end ? last : end;
    }
    for (const CallBuffer *x : {&all[3], &all[4]})
        if (overlap(*x->address, x->need, begin, end - begin))
            return fail(SGL_KV_INVALID_ARGUMENT, "in place", 0, 0, 0, "%s overlaps the pool", x->name);
    const ForkParts parts = fork_parts(c);
    p.parents = reinterpret_cast<const uint32_t *>(parents);
    p.lengths = reinterpret_cast<const uint64_t *>(lengths);
    p.tables = reinterpret_cast<const int32_t *>(tables);
    p.forked_lengths = reinterpret_cast<uint64_t *>(forked_lengths);
    p.forked_tables = reinterpret_cast<int32_t *>(forked_tables);
    p.references = reinterpret_cast<uint32_t *>(references);
    p.free_pages = reinterpret_cast<int32_t *>(free_pages);
    p.free_count = reinterpret_cast<uint64_t *>(free_count);
    p.head = reinterpret_cast<uint32_t *>(workspace);
    p.first = reinterpret_cast<uint32_t *>(workspace + parts.first);
    p.children = reinterpret_cast<uint32_t *>(workspace + parts.children);
    p.held = reinterpret_cast<uint32_t *>(workspace + parts.held);
    p.before = reinterpret_cast<uint32_t *>(workspace + parts.before);
    p.copies = reinterpret_cast<sglkv_page_copy *>(workspace + parts.copies);
    p.freed = reinterpret_cast<uint32_t *>(workspace + parts.freed);
    p.flag = ctx->flag;
    p.table_pages = c.table_pages;
    p.sequences = (uint32_t)c.sequence_count;
    p.old_sequences = (uint32_t)c.parent_count;
    p.page_count = (uint32_t)c.page_count;
    p.append = (uint32_t)c.append_tokens;
    p.keep_reserved = (uint32_t)c.keep_reserved;
    p.tensors = pool->tensor_count;
    p.layers = layer_count;
    uint64_t bits = layer_count > 1 ? layer_stride : 0, most = 0;
    for (uint32_t t = 0; t < p.tensors; ++t) {
        const uint64_t chunk = view_row_bytes(*pool, t) / p.heads;
        if (chunk > UINT32_MAX) return too_large_dim("row_bytes", chunk * p.heads, UINT32_MAX * (uint64_t)p.heads);
        p.chunk[t] = (uint32_t)chunk;
        bits |= chunk | p.pool.plane[t] | p.pool.head_stride[t];
        if (view_row_bytes(*pool, t) > most) most = view_row_bytes(*pool, t);
    }
    uint64_t region;
    p.wide = p.pool.stride[0] % 16 != 0 ? 0 : bits % 16 != 0 || mul_ovf(most, c.page_size, &region) || region > UINT32_MAX ? 1 : 2;
    const uint64_t groups = (uint64_t)p.sequences * p.layers * p.tensors, limit = UINT32_MAX / SGLKV_FORK_THREADS;
    if (groups > limit) return too_large_dim("workgroups", groups, limit);
    // One workgroup takes as long as the other way's three launches where it goes through some 8,000 entries (256
    // sequences with their copies, 4,352 entries: 48 us, with three launches 54; 8,192: 53 and 54; 16,384: 67 and 54;
    // 65,536: 133 and 54).
    const bool small = c.sequence_count <= SGLKV_FORK_SMALL_SEQUENCES && c.parent_count <= SGLKV_FORK_SMALL_SEQUENCES &&
                       c.table_pages <= SGLKV_FORK_SMALL_ENTRIES && c.page_count <= SGLKV_FORK_SMALL_PAGES &&
                       c.sequence_count * c.table_pages <= SGLKV_FORK_SMALL_ENTRIES &&
                       c.parent_count * c.table_pages <= SGLKV_FORK_SMALL_ENTRIES && c.table_pages * c.page_size < 1ull << 31;
    DeviceScope scope(ctx->device);
    if (scope.status() != hipSuccess) return hip_fail(scope.status(), "hipSetDevice");
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (small) {
        rc = launch_kernel(ctx->fork_small, 1, 1, 1, SGLKV_FORK_PLAN_THREADS, 4 * (unsigned)divide_up(c.page_count, 32), s, &p,
                           "fork plan launch");
    } else {
        rc = launch_kernel(ctx->fork_plan, 1, 1, 1, SGLKV_FORK_PLAN_THREADS, 0, s, &p, "fork plan launch");
        if (!rc)
            rc = launch_kernel(ctx->fork_tables, p.sequences + p.old_sequences, 1, 1, SGLKV_FORK_THREADS, 0, s, &p,
                               "fork tables launch");
        if (!rc) rc = launch_kernel(ctx->fork_free, 1, 1, 1, SGLKV_FORK_PLAN_THREADS, 0, s, &p, "fork free pages launch");
    }
    if (!rc)
        rc = launch_kernel(ctx->fork_copy, groups, 1, 1, SGLKV_FORK_THREADS, 0, s, &p, "fork copy launch");
    return rc ? rc : ok();
}
