// kv_call.h -- what the entry points of several files check alike: named buffers
// of a call, and a pool of several layers.
#ifndef SGLKV_CALL_H
#define SGLKV_CALL_H

#include "kv_attention_route.h"
#include "kv_internal.h"

namespace sglkv {

inline uint64_t divide_up(uint64_t a, uint64_t b) { return a / b + (a % b != 0); }

inline int32_t null_arguments(const char *name) {
    return fail(SGL_KV_INVALID_ARGUMENT, name, 0, 0, 0, "null argument");
}

// A named buffer of a call and what it has to hold.
struct CallBuffer {
    const char *name;
    const sgl_kv_device_buffer *buffer;
    uint64_t offset, need;
    uint64_t *address;
    uint64_t align;
    bool used;
};

// Devices first, then ranges, then alignments: the order of the other calls.
template <size_t N>
int32_t resolve_buffers(const sgl_rocm_kv_ctx *ctx, const CallBuffer (&all)[N]) {
    int32_t rc;
    for (const CallBuffer &x : all)
        if (x.used && (rc = check_device(ctx, x.name, *x.buffer))) return rc;
    for (const CallBuffer &x : all)
        if (x.used && (rc = attention_ptr(x.name, *x.buffer, x.offset, x.need, x.address))) return rc;
    for (const CallBuffer &x : all)
        if (x.used && *x.address % x.align)
            return fail(SGL_KV_INVALID_ARGUMENT, "alignment", 0, 0, 0, "%s must be aligned to %llu bytes", x.name,
                        (unsigned long long)x.align);
    return SGL_KV_OK;
}

inline bool overlap(uint64_t a, uint64_t an, uint64_t b, uint64_t bn) { return an && bn && a < b + bn && b < a + an; }

// Buffer `written` of a call against all others but `same`, if any: it is written while these are read, or written, too.
template <size_t N>
int32_t refuse_overlaps(const CallBuffer (&all)[N], size_t written, size_t same = N) {
    const CallBuffer &x = all[written];
    for (const CallBuffer &y : all)
        if (&x != &y && &y != all + same && x.used && y.used && overlap(*x.address, x.need, *y.address, y.need))
            return fail(SGL_KV_INVALID_ARGUMENT, "in place", 0, 0, 0, "%s overlaps %s", x.name, y.name);
    return SGL_KV_OK;
}

// Whether two of the regions of `layer_count` layers, each `stride` bytes behind the
// one before, overlap inside a page: tensor t's has bytes[t] from offset[t] on.
inline bool layers_overlap(uint32_t tensors, const uint64_t (&offset)[2], const uint64_t (&bytes)[2], uint64_t layer_count,
                           uint64_t stride) {
    for (uint32_t t = 0; t < tensors; ++t)
        if (layer_count > 1 && stride < bytes[t]) return true;
    if (tensors < 2) return false;
    // The later tensor of a layer lies `apart` behind the earlier: behind, or inside, that of layer apart / stride after
    // it, and before that of the layer after.
    const uint32_t a = offset[0] <= offset[1] ? 0 : 1, b = 1 - a;
    const uint64_t apart = offset[b] - offset[a], at = layer_count > 1 ? apart / stride : 0, rest = apart - at * stride;
    return (at < layer_count && rest < bytes[a]) || (layer_count > 1 && at < layer_count - 1 && stride - rest < bytes[b]);
}

// The kernel side of `layer_count` layers of a pool, of which `pool` describes
// the first; `chunks` are a row's parts that lie apart: the heads of head-major
// pages, else one.
inline int32_t pool_layers(const sgl_rocm_kv_ctx *ctx, const sgl_kv_pool_view *pool, uint32_t layer_count,
                           uint64_t layer_stride, sglkv_side *side, uint32_t *chunks) {
    if (!pool) return null_arguments("pool");
    if (!layer_count)
        return fail(SGL_KV_ZERO_DIMENSION, "layer_count", 0, 0, 0, "KV copy dimension layer_count must be non-zero");
    if (layer_count > 65535) return too_large_dim("layer_count", layer_count, 65535);
    // The first layer and the last: those between lie between.
    sgl_kv_pool_view last = *pool;
    last.scale = nullptr;
    if (pool->head_layout == SGL_KV_NHD) last.heads = 1;
    int32_t rc = pool_heads_side(&last, side);
    for (uint32_t t = 0; t < 2; ++t) {
        uint64_t far;
        if (mul_ovf(layer_count - 1, layer_stride, &far) || add_ovf(last.tensor_offset[t], far, &last.tensor_offset[t]))
            return fail(SGL_KV_SHAPE_OVERFLOW, nullptr, 0, 0, 0, "KV copy layers overflowed");
    }
    if (rc || (rc = check_pool_view(&last))) return rc;
    // (A page's part of a layer lies inside the page, so that these multiply.)
    const uint64_t bytes[2] = {pool->page_size * view_row_bytes(*pool, 0), pool->page_size * view_row_bytes(*pool, 1)};
    if (layers_overlap(pool->tensor_count, pool->tensor_offset, bytes, layer_count, layer_stride))
        return fail(SGL_KV_INVALID_ARGUMENT, "layer_stride", layer_stride, layer_count, 0,
                    "the regions of %u layers that lie %llu bytes apart overlap", layer_count, (unsigned long long)layer_stride);
    const sgl_kv_device_buffer whole = {pool->base, pool->byte_len};
    if ((rc = check_device(ctx, "pool", whole))) return rc;
    side->layer_stride = layer_stride;
    *chunks = last.heads;
    return SGL_KV_OK;
}

}  // namespace sglkv

#endif
