// kv_beam.cpp -- host side of beam selection: the plan, the checks and the
// launches (kernels in kv_beam.hip). Nothing here allocates or waits, and what a
// launch relies on is derived again at each call.
#include <hip/hip_runtime.h>

#include <string.h>

#include "kv_call.h"

using namespace sglkv;

namespace {

struct BeamShape {
    uint64_t rows, stride, rounds, splits;
    uint64_t partial_bytes, candidate_bytes, list_bytes;
};

int32_t beam_shape(const sgl_kv_beam_config &c, BeamShape *out) {
    const struct {
        const char *name;
        uint64_t value, maximum;
    } dims[] = {{"request_count", c.request_count, UINT32_MAX},
                {"beam_count", c.beam_count, SGLKV_BEAM_MAX_BEAMS},
                {"vocab_size", c.vocab_size, (uint64_t)SGLKV_BEAM_CHUNK * SGLKV_BEAM_MAX_SPLITS},
                {"max_kept", c.max_kept, SGL_KV_BEAM_MAX_KEPT}};
    for (const auto &d : dims)
        if (d.value == 0)
            return fail(SGL_KV_ZERO_DIMENSION, d.name, 0, 0, 0, "beam dimension %s must be non-zero", d.name);
    if (c.dtype != SGL_KV_DTYPE_BFLOAT16 && c.dtype != SGL_KV_DTYPE_FLOAT32)
        return fail(SGL_KV_INVALID_ARGUMENT, "dtype", (uint64_t)(int64_t)c.dtype, 0, 0, "logits of type %d are not supported",
                    c.dtype);
    if (c.row_stride && c.row_stride < c.vocab_size)
        return fail(SGL_KV_INVALID_ARGUMENT, "row_stride", c.row_stride, c.vocab_size, 0,
                    "rows of %llu logits do not lie %llu apart", (unsigned long long)c.vocab_size,
                    (unsigned long long)c.row_stride);
    for (const auto &d : dims)
        if (d.value > d.maximum) return too_large_dim(d.name, d.value, d.maximum);
    BeamShape &h = *out;
    h.rows = c.request_count * c.beam_count;  // (below 2^42)
    h.stride = c.row_stride ? c.row_stride : c.vocab_size;
    // Several rounds a workgroup where there are more than fill the card: what a workgroup does once is shared by them (64
    // requests of 4 beams, 128,256 tokens: 28.8 us at a round each, 24.6 at 2,048 workgroups, 24.0 at 1,024 and 25.0 at 512;
    // 256 requests of 50,257 tokens: 35.9, 34.7, 35.0 and 34.9).
    const uint64_t chunks = divide_up(c.vocab_size, SGLKV_BEAM_CHUNK);
    h.rounds = h.rows * chunks / 2048;
    h.rounds = h.rounds < 1 ? 1 : h.rounds > chunks ? chunks : h.rounds;
    h.splits = divide_up(chunks, h.rounds);
    // A dispatch counts its work-items in 32 bits; parents are numbered in 32 bits, too.
    const uint64_t limit = UINT32_MAX / SGLKV_BEAM_THREADS;
    if (h.rows * h.splits > limit) return too_large_dim("workgroups", h.rows * h.splits, limit);
    const uint64_t joins = UINT32_MAX / SGLKV_BEAM_JOIN_THREADS;
    if (c.request_count > joins) return too_large_dim("workgroups", c.request_count, joins);
    h.partial_bytes = divide_up(8 * h.rows * h.splits, 64) * 64;
    h.candidate_bytes = 8 * h.rows * h.splits * c.max_kept;
    h.list_bytes = 8 * h.rows * c.max_kept;
    return SGL_KV_OK;
}

}  // namespace

extern "C" int32_t sgl_kv_beam_plan_new(const sgl_kv_beam_config *config, sgl_kv_beam_plan *out) {
    if (!config || !out) return null_arguments("config/out");
    BeamShape h;
    int32_t rc = beam_shape(*config, &h);
    if (rc) return rc;
    sgl_kv_beam_plan p;
    memset(&p, 0, sizeof p);
    p.config = *config;
    uint64_t elements;
    if (mul_ovf(h.rows - 1, h.stride, &elements) || add_ovf(elements, config->vocab_size, &elements) ||
        mul_ovf(elements, config->dtype == SGL_KV_DTYPE_FLOAT32 ? 4 : 2, &p.logits_required_bytes))
        return fail(SGL_KV_SHAPE_OVERFLOW, nullptr, 0, 0, 0, "beam selection shape overflowed");
    p.scores_required_bytes = 4 * h.rows;
    p.best_scores_required_bytes = p.best_parents_required_bytes = p.best_tokens_required_bytes =
        4 * config->request_count * config->max_kept;
    p.workspace_required_bytes = h.partial_bytes + h.candidate_bytes + h.list_bytes;
    *out = p;
    return ok();
}

extern "C" int32_t sgl_rocm_kv_select_beams(sgl_rocm_kv_ctx *ctx, const sgl_kv_beam_plan *plan,
                                            const sgl_kv_beam_buffers *b, void *stream) {
    if (!ctx || !plan || !b) return null_arguments("ctx/plan/buffers");
    sgl_kv_beam_plan f;
    BeamShape h;
    int32_t rc = sgl_kv_beam_plan_new(&plan->config, &f);
    if (!rc) rc = beam_shape(f.config, &h);
    if (rc) return rc;
    const sgl_kv_beam_config &c = f.config;
    const bool f32 = c.dtype == SGL_KV_DTYPE_FLOAT32;
    uint64_t logits, scores, best_scores, best_parents, best_tokens, workspace;
    const CallBuffer all[] = {
        {"logits", &b->logits, b->logits_offset, f.logits_required_bytes, &logits, f32 ? 4u : 2u, true},
        {"scores", &b->scores, b->scores_offset, f.scores_required_bytes, &scores, 4, true},
        {"best_scores", &b->best_scores, b->best_scores_offset, f.best_scores_required_bytes, &best_scores, 4, true},
        {"best_parents", &b->best_parents, b->best_parents_offset, f.best_parents_required_bytes, &best_parents, 4, true},
        {"best_tokens", &b->best_tokens, b->best_tokens_offset, f.best_tokens_required_bytes, &best_tokens, 4, true},
        {"workspace", &b->workspace, b->workspace_offset, f.workspace_required_bytes, &workspace, 16, true}};
    if ((rc = resolve_buffers(ctx, all))) return rc;
    // In place: a workgroup has read its request's scores before it writes the best ones to the same places.
    const bool in_place = best_scores == scores && c.max_kept == c.beam_count;
    if ((rc = refuse_overlaps(all, 2, in_place ? 1 : 2)) || (rc = refuse_overlaps(all, 3)) || (rc = refuse_overlaps(all, 4)) ||
        (rc = refuse_overlaps(all, 5)))
        return rc;
    sglkv_beam_params p;
    memset(&p, 0, sizeof p);
    p.logits = reinterpret_cast<const void *>(logits);
    p.scores = reinterpret_cast<const float *>(scores);
    p.best_scores = reinterpret_cast<float *>(best_scores);
    p.best_parents = reinterpret_cast<uint32_t *>(best_parents);
    p.best_tokens = reinterpret_cast<uint32_t *>(best_tokens);
    p.partial = reinterpret_cast<float *>(workspace);
    p.candidates = reinterpret_cast<uint64_t *>(workspace + h.partial_bytes);
    p.lists = reinterpret_cast<uint64_t *>(workspace + h.partial_bytes + h.candidate_bytes);
    p.row_stride = h.stride;
    p.beams = (uint32_t)c.beam_count;
    p.vocab = (uint32_t)c.vocab_size;
    p.kept = (uint32_t)c.max_kept;
    p.splits = (uint32_t)h.splits;
    p.rounds = (uint32_t)h.rounds;
    DeviceScope scope(ctx->device);
    if (scope.status() != hipSuccess) return hip_fail(scope.status(), "hipSetDevice");
    hipStream_t s = static_cast<hipStream_t>(stream);
    rc = launch_kernel(ctx->beam_rows[f32 ? 1 : 0], h.rows * h.splits, 1, 1, SGLKV_BEAM_THREADS, 0, s, &p, "beam rows launch");
    if (!rc)
        rc = launch_kernel(ctx->beam_join, c.request_count, 1, 1, SGLKV_BEAM_JOIN_THREADS, 0, s, &p, "beam join launch");
    return rc ? rc : ok();
}
