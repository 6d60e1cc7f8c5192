// kv_tree.hip -- attention of a tree of drafted tokens over a paged cache.
//
// Query q (a drafted token) attends A = {t < L} and {L + j : bit j of its mask},
// L = query_sequence_lengths[q]: its request's tokens, its ancestors among the
// drafts and itself. o = sum_{t in A} softmax(scale q.k_t) v_t; an empty A gives
// zeros. The rows of tokens outside A may hold anything: they are not loaded, or
// where several queries share what is loaded, what they hold does not reach o.

namespace {

// A query's request, and how far it reaches: `context` tokens attended whole,
// `reach` tokens up to its mask's last bit. False: it attends nothing, by itself
// or because its metadata does not hold (reported).
struct tree_query {
    uint64_t start, context, reach;
};
__device__ __forceinline__ bool tree_metadata(const sglkv_tree_params &p, uint64_t q, bool report, tree_query *t) {
    const sglkv_attn_params &a = p.a;
    const uint64_t *mask = p.masks + q * p.mask_words;
    uint64_t drafts = 0;
    for (uint32_t w = 0; w < p.mask_words; ++w) {
        const uint64_t m = mask[w];
        if (m) drafts = 64 * w + 64 - static_cast<uint64_t>(__builtin_clzll(m));
    }
    t->context = a.query_sequence_lengths[q];
    t->reach = t->context + drafts;
    if ((t->context | drafts) == 0) return false;
    const uint32_t req = a.query_request_indices[q];
    if (req >= a.request_count) {
        if (report) atomicOr(a.flag, SGLKV_FLAG_ATTN_REQUEST);
        return false;
    }
    const uint64_t s = a.request_slot_offsets[req], e = a.request_slot_offsets[req + 1];
    if (s > e || e > a.sequence_slot_count || t->context > e - s || t->reach > e - s || t->reach > p.max_length) {
        if (report) atomicOr(a.flag, SGLKV_FLAG_ATTN_SEQUENCE);
        return false;
    }
    t->start = s;
    return true;
}

// Any head dims, page size and alignment: a wave to 16 query heads and
// SGLKV_ATTN_DV value dims of one query, 32 tokens a step, as the generic body of
// paged attention (attn_body), whose layouts of the matrix products it shares.
template <bool VEC>
__device__ __forceinline__ void tree_body(const sglkv_tree_params &p) {
    extern __shared__ __attribute__((aligned(16))) uint16_t tree_lds[];
    const sglkv_attn_params &a = p.a;
    const uint32_t lane = threadIdx.x, g = lane >> 4, r = lane & 15;
    uint32_t bx = blockIdx.x;
    attn_work w;
    w.dblk = bx % a.dv_blocks;
    bx /= a.dv_blocks;
    const uint32_t hg = bx % a.head_groups;
    bx /= a.head_groups;
    w.kvh = bx % a.kv_heads;
    w.q = bx / a.kv_heads;
    w.split = blockIdx.y;
    w.h0 = w.kvh * a.group + hg * SGLKV_ATTN_HEADS;
    const uint32_t heads = a.group - hg * SGLKV_ATTN_HEADS;
    w.nh = heads < SGLKV_ATTN_HEADS ? heads : SGLKV_ATTN_HEADS;
    w.d0 = w.dblk * SGLKV_ATTN_DV;
    tree_query t;
    const bool report = lane == 0 && w.split == 0 && hg == 0 && w.dblk == 0 && w.kvh == 0;
    if (report && w.q > 0 && a.query_request_indices[w.q - 1] > a.query_request_indices[w.q])
        atomicOr(a.flag, SGLKV_FLAG_ATTN_REQUEST);
    const bool any = tree_metadata(p, w.q, report, &t);
    w.t0 = w.split * a.chunk_tokens;
    if (!any) {
        // (With several splits the merge writes the zeros.)
        if (a.splits == 1)
            for (uint32_t i = lane; i < w.nh * SGLKV_ATTN_DV; i += 64) {
                const uint32_t h = i / SGLKV_ATTN_DV, d = w.d0 + i % SGLKV_ATTN_DV;
                if (d < a.dv) a.output[(w.q * a.query_heads + w.h0 + h) * a.dv + d] = 0;
            }
        return;
    }
    if (w.t0 >= t.reach) return;
    w.start = t.start;
    w.t1 = t.reach - w.t0 < a.chunk_tokens ? t.reach : w.t0 + a.chunk_tokens;
    const uint32_t qstride = a.dk_pad + 8;
    uint16_t *qs = tree_lds, *vt = tree_lds + SGLKV_ATTN_HEADS * qstride;
    attn_stage_queries(a, w, lane, qs, qstride);
    const uint64_t pool = reinterpret_cast<uint64_t>(a.pool);
    const uint64_t kbase = pool + a.key_offset + w.kvh * a.key_head_stride;
    const uint64_t vbase = pool + a.value_offset + w.kvh * a.value_head_stride;
    const uint64_t *mask = p.masks + w.q * p.mask_words;
    attn_state st;
    attn_state_init(st);
    for (uint64_t tb = w.t0; tb < w.t1; tb += SGLKV_ATTN_TOKENS) {
        uint64_t krow[2], vrow[2];
        bool valid[2];
#pragma unroll
        for (uint32_t b = 0; b < 2; ++b) {
            const uint64_t tok = tb + 8 * (r >> 2) + 4 * b + (r & 3);
            bool ok = tok < w.t1;
            if (ok && tok >= t.context) {
                const uint64_t j = tok - t.context;
                ok = (mask[j >> 6] >> (j & 63)) & 1;
            }
            uint64_t slot = 0;
            if (ok) {
                slot = a.sequence_slots[w.start + tok];
                if (slot >= a.slot_count) {
                    atomicOr(a.flag, SGLKV_FLAG_ATTN_SLOT);
                    ok = false;
                    slot = 0;
                }
            }
            uint64_t page, pos;
            attn_split_slot(a, slot, &page, &pos);
            krow[b] = kbase + page * a.page_stride + pos * a.key_token_stride;
            vrow[b] = vbase + page * a.page_stride + pos * a.value_token_stride;
            valid[b] = ok;
        }
        sglkv_f32x4 sc[2] = {sglkv_f32x4{0.f, 0.f, 0.f, 0.f}, sglkv_f32x4{0.f, 0.f, 0.f, 0.f}};
        for (uint32_t kk = 0; kk < a.dk_pad; kk += 32) {
            const sglkv_u16x8 qv = *reinterpret_cast<const sglkv_u16x8 *>(qs + r * qstride + kk + 8 * g);
#pragma unroll
            for (uint32_t b = 0; b < 2; ++b)
                sc[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                    attn_as_bf16(attn_load8<VEC>(krow[b], kk + 8 * g, a.dk, valid[b])), attn_as_bf16(qv), sc[b], 0, 0, 0);
        }
#pragma unroll
        for (uint32_t b = 0; b < 2; ++b) {
            const uint32_t tl = 8 * (r >> 2) + 4 * b + (r & 3);
#pragma unroll
            for (uint32_t n = 0; n < 4; ++n) {
                const sglkv_u16x8 v = attn_load8<VEC>(vrow[b], w.d0 + 8 * (g + 4 * n), a.dv, valid[b]);
#pragma unroll
                for (uint32_t e = 0; e < 8; ++e) vt[(8 * (g + 4 * n) + e) * SGLKV_ATTN_VT_STRIDE + tl] = v[e];
            }
        }
        attn_softmax_pv(a, g, sc, __ballot(valid[0]), __ballot(valid[1]), vt, r, st);
    }
    attn_finish(a, w, g, r, st);
}

}  // namespace

extern "C" __global__ __launch_bounds__(64) void sglkv_tree_attention_v16(sglkv_tree_params p) { tree_body<true>(p); }
extern "C" __global__ __launch_bounds__(64) __attribute__((amdgpu_waves_per_eu(2))) void sglkv_tree_attention_v2(
    sglkv_tree_params p) {
    tree_body<false>(p);
}

// Merges the split records of each (query, head), as
// sglkv_paged_attention_combine does for queries that attend all tokens up to
// their length; one that attends nothing gives zeros.
extern "C" __global__ __launch_bounds__(SGLKV_ATTN_COMBINE_THREADS) void sglkv_tree_attention_combine(sglkv_tree_params p) {
    __shared__ float part[SGLKV_ATTN_COMBINE_THREADS][6];  // m, l, o[4] of each thread
    const sglkv_attn_params &a = p.a;
    const sglkv_combine_place place = sglkv_combine_place_of(threadIdx.x, a.dv, a.splits);
    const uint32_t lanes = place.lanes, per = place.per, sub = place.sub;
    const uint64_t item = static_cast<uint64_t>(blockIdx.x) * place.items + place.own;
    const bool inside = place.own < place.items && item < a.query_count * a.query_heads;
    tree_query t;
    const bool any = inside && tree_metadata(p, item / a.query_heads, false, &t);
    const uint32_t used = any ? static_cast<uint32_t>((t.reach + a.chunk_tokens - 1) / a.chunk_tokens) : 0;
    const uint64_t i0 = inside ? item * a.splits : 0;
    const float2 *ml = reinterpret_cast<const float2 *>(attn_rec_ml(a, i0));
    const float *o = attn_rec_o(a, i0);
    const uint32_t opad = SGLKV_ATTN_OPAD(a.dv);
    for (uint32_t d0 = 0; d0 < a.dv; d0 += 4 * lanes) {  // (one pass where lanes cover dv: always if sets > 1)
        const uint32_t d = d0 + 4 * (threadIdx.x % lanes);
        float m = -3.402823466e+38f, l = 0.0f, acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (used && d < a.dv) attn_combine_groups(ml, o, opad, d, used, 8 * sub, 8 * per, m, l, acc);
        if (per > 1) {  // (uniform)
            float *pw = part[threadIdx.x];
            if (sub > 0) {
                pw[0] = m;
                pw[1] = l;
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e) pw[2 + e] = acc[e];
            }
            __syncthreads();
            if (place.merges) {
                for (uint32_t k = 1; k < per; ++k) {
                    const float *pk = pw + 6 * k * lanes;
                    const float m_new = fmaxf(m, pk[0]);
                    const float x = exp2f(m - m_new), y = exp2f(pk[0] - m_new);
                    l = l * x + pk[1] * y;
#pragma unroll
                    for (uint32_t e = 0; e < 4; ++e) acc[e] = acc[e] * x + pk[2 + e] * y;
                    m = m_new;
                }
            }
            __syncthreads();  // (the shares are read before the next dims' are written)
        }
        if (!inside || !place.merges) continue;
        const float linv = any ? 1.0f / l : 0.0f;
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e)
            if (d + e < a.dv) a.output[item * a.dv + d + e] = attn_to_bf16(acc[e] * linv);
    }
}
