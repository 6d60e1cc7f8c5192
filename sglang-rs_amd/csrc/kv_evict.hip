// kv_evict.hip -- eviction from a paged KV cache by accumulated attention
// weight, for gfx950: the softmax weights that each position of a sequence gets
// from the queries, added to a running sum per KV head; the positions with the
// largest sums; and the copy of their K/V rows (and sums) to other slots.
//
// For query head i of KV head h at query q, with scores s_t = scale q_i . k_t
// over the query's first len tokens,
//     weights[h][t] += sum_{q, i} exp(s_t - m) / l,  m = max s, l = sum exp(s - m).
// The values are not read. The first kernel finds (m, l) of each (query, head);
// the second computes the scores again, with the tokens as the outer loop, so
// that each position's sum is added up by one wave in one order: no atomics,
// and the same result every time.

namespace {

// A query's metadata; false, and nothing to weigh, for a query of no tokens or
// whose metadata does not hold (which sets the error word when `report`).
__device__ __forceinline__ bool wgt_query(const sglkv_weights_params &p, uint64_t q, bool report, uint64_t *start,
                                          uint64_t *len) {
    sel_sequence(p.a, p.max_length, q, report, start, len);
    // The second kernel finds a request's queries by halving: they come request by request.
    if (report && q > 0 && p.a.query_request_indices[q - 1] > p.a.query_request_indices[q])
        atomicOr(p.a.flag, SGLKV_FLAG_ATTN_REQUEST);
    return *len > 0;
}

// The (maximum, sum) pair of (query, head, split). A split without tokens
// leaves (-inf, 0); one with tokens has a finite maximum.
__device__ __forceinline__ float2 *wgt_stats(const sglkv_weights_params &p, uint64_t q, uint64_t head) {
    return reinterpret_cast<float2 *>(p.a.partial) + (q * p.a.query_heads + head) * p.a.splits;
}

// K row address of a sequence's token; false where its slot lies outside the
// pool (the address is slot 0's).
__device__ __forceinline__ bool wgt_row(const sglkv_attn_params &p, uint64_t kbase, uint64_t start, uint64_t tok,
                                        bool inside, bool report, uint64_t *row) {
    uint64_t slot = inside ? p.sequence_slots[start + tok] : 0;
    const bool ok = inside && slot < p.slot_count;
    if (inside && !ok) {
        if (report) atomicOr(p.flag, SGLKV_FLAG_ATTN_SLOT);
        slot = 0;
    }
    uint64_t page, pos;
    attn_split_slot(p, slot, &page, &pos);
    *row = kbase + page * p.page_stride + pos * p.key_token_stride;
    return ok;
}

// ---- Statistics -------------------------------------------------------------
//
// One wave per (query, KV head, 16 query heads, split); 32 tokens a step, K
// rows as the A operand of the matrix product, queries (from LDS) as B, so lane
// (g, r) gets tokens 4g .. 4g+3 of each 16 for head r and keeps a running
// (maximum, sum) of its own; the four lanes of a head join at the end.
template <bool VEC>
__device__ __forceinline__ void wgt_stats_body(const sglkv_weights_params &p) {
    extern __shared__ __attribute__((aligned(16))) uint16_t wgt_lds[];
    const sglkv_attn_params &a = p.a;
    const uint32_t lane = threadIdx.x, g = lane >> 4, r = lane & 15;
    uint32_t bx = blockIdx.x;
    const uint32_t hg = bx % a.head_groups;
    bx /= a.head_groups;
    attn_work w;
    w.kvh = bx % a.kv_heads;
    w.q = bx / a.kv_heads;
    w.h0 = w.kvh * a.group + hg * SGLKV_ATTN_HEADS;
    w.nh = a.group - hg * SGLKV_ATTN_HEADS < SGLKV_ATTN_HEADS ? a.group - hg * SGLKV_ATTN_HEADS : SGLKV_ATTN_HEADS;
    uint64_t start, len;
    const bool live =
        wgt_query(p, w.q, lane == 0 && hg == 0 && w.kvh == 0 && blockIdx.y == 0, &start, &len);
    const uint64_t t0 = static_cast<uint64_t>(blockIdx.y) * a.chunk_tokens;
    float m = -INFINITY, l = 0.0f;
    if (live && t0 < len) {
        const uint64_t t1 = len < t0 + a.chunk_tokens ? len : t0 + a.chunk_tokens;
        const uint32_t qstride = a.dk_pad + 8;
        attn_stage_queries(a, w, lane, wgt_lds, qstride);
        const uint64_t kbase = reinterpret_cast<uint64_t>(a.pool) + a.key_offset + w.kvh * a.key_head_stride;
        m = -3.402823466e+38f;
        for (uint64_t tb = t0; tb < t1; tb += 32) {
            uint64_t row[2];
            bool ok[2];
#pragma unroll
            for (uint32_t b = 0; b < 2; ++b)
                ok[b] = wgt_row(a, kbase, start, tb + 16 * b + r, tb + 16 * b + r < t1, w.kvh == 0, &row[b]);
            sglkv_f32x4 sc[2] = {sglkv_f32x4{0.f, 0.f, 0.f, 0.f}, sglkv_f32x4{0.f, 0.f, 0.f, 0.f}};
            for (uint32_t kk = 0; kk < a.dk_pad; kk += 32) {
                const sglkv_u16x8 qv = *reinterpret_cast<const sglkv_u16x8 *>(wgt_lds + r * qstride + kk + 8 * g);
#pragma unroll
                for (uint32_t b = 0; b < 2; ++b)
                    sc[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                        attn_as_bf16(attn_load8<VEC>(row[b], kk + 8 * g, a.dk, ok[b])), attn_as_bf16(qv), sc[b], 0, 0, 0);
            }
#pragma unroll
            for (uint32_t b = 0; b < 2; ++b) {
                const uint64_t valid = __ballot(ok[b]);
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e) {
                    const float x = (valid >> (4 * g + e)) & 1 ? sc[b][e] * a.scale_log2 : -INFINITY;
                    const float m_new = fmaxf(m, x);
                    l = l * exp2f(m - m_new) + exp2f(x - m_new);
                    m = m_new;
                }
            }
        }
#pragma unroll
        for (uint32_t s = 16; s < 64; s <<= 1) {
            const float mo = __shfl_xor(m, s), lo = __shfl_xor(l, s), m_new = fmaxf(m, mo);
            l = l * exp2f(m - m_new) + lo * exp2f(mo - m_new);
            m = m_new;
        }
    }
    if (g == 0 && r < w.nh) wgt_stats(p, w.q, w.h0 + r)[blockIdx.y] = make_float2(m, l);
}

// ---- Accumulation -----------------------------------------------------------
//
// One wave per (request, KV head, 64 tokens): for each of the request's
// queries, 16 heads at a time, the scores again, and their weights added to the
// lane's tokens; the 16 lanes of a token join at the end.
template <bool VEC>
__device__ __forceinline__ void wgt_accumulate_body(const sglkv_weights_params &p) {
    const sglkv_attn_params &a = p.a;
    const uint32_t lane = threadIdx.x, g = lane >> 4, r = lane & 15;
    const uint32_t tile = blockIdx.x % p.tiles;
    const uint32_t item = blockIdx.x / p.tiles, kvh = item % a.kv_heads, req = item / a.kv_heads;
    const uint64_t start = a.request_slot_offsets[req], end = a.request_slot_offsets[req + 1];
    const uint64_t tb = static_cast<uint64_t>(tile) * SGLKV_WEIGHTS_TILE;
    if (start > end || end > a.sequence_slot_count || tb >= end - start) return;
    // The request's queries.
    auto first_of = [&](uint32_t key) {
        uint64_t low = 0, high = a.query_count;
        while (low < high) {
            const uint64_t mid = low + (high - low) / 2;
            if (a.query_request_indices[mid] < key)
                low = mid + 1;
            else
                high = mid;
        }
        return low;
    };
    const uint64_t q0 = first_of(req), q1 = first_of(req + 1);
    // The tokens that any of them attends.
    auto length_of = [&](uint64_t q) {
        const uint64_t n = a.query_sequence_lengths[q];
        return n <= end - start && n <= p.max_length && a.query_request_indices[q] == req ? n : 0;
    };
    uint64_t longest = 0;
    for (uint64_t q = q0 + lane; q < q1; q += 64) {
        const uint64_t n = length_of(q);
        longest = n > longest ? n : longest;
    }
#pragma unroll
    for (uint32_t s = 1; s < 64; s <<= 1) {
        const uint64_t n = __shfl_xor(longest, s);
        longest = n > longest ? n : longest;
    }
    if (tb >= longest) return;
    const uint64_t kbase = reinterpret_cast<uint64_t>(a.pool) + a.key_offset + kvh * a.key_head_stride;
    // Lane (g, r) loads token 16 b + r's row and weighs tokens 16 b + 4 g .. + 3.
    // (A token whose slot is no slot of the pool has been reported.)
    uint64_t row[4];
    uint32_t ok = 0;
#pragma unroll
    for (uint32_t b = 0; b < 4; ++b) {
        const uint64_t tok = tb + 16 * b + r;
        ok |= (wgt_row(a, kbase, start, tok, tok < longest, false, &row[b]) ? 1u : 0u) << b;
    }
    float sum[4][4] = {};
    for (uint64_t q = q0; q < q1; ++q) {
        const uint64_t len = length_of(q);
        if (len <= tb) continue;
        for (uint32_t h0 = 0; h0 < a.group; h0 += 16) {
            const bool head = h0 + r < a.group;
            const uint64_t hi = static_cast<uint64_t>(kvh) * a.group + (head ? h0 + r : 0);
            // This lane's head: the softmax statistics of its splits joined.
            const float2 *stats = wgt_stats(p, q, hi);
            float m = -INFINITY, l = 0.0f;
            for (uint32_t s = 0; s < a.splits; ++s) m = fmaxf(m, stats[s].x);
            for (uint32_t s = 0; s < a.splits; ++s)
                if (stats[s].x != -INFINITY) l += stats[s].y * exp2f(stats[s].x - m);
            const bool weighs = head && m != -INFINITY;
            const float inv = weighs ? 1.0f / l : 0.0f;
            const uint32_t limit = !weighs ? 0 : len - tb < 64 ? static_cast<uint32_t>(len - tb) : 64;
            const uint64_t qrow = reinterpret_cast<uint64_t>(a.queries + (q * a.query_heads + hi) * a.dk);
            sglkv_f32x4 sc[4];
#pragma unroll
            for (uint32_t b = 0; b < 4; ++b) sc[b] = sglkv_f32x4{0.f, 0.f, 0.f, 0.f};
            for (uint32_t kk = 0; kk < a.dk_pad; kk += 32) {
                const sglkv_u16x8 qv = attn_load8<VEC>(qrow, kk + 8 * g, a.dk, head);
#pragma unroll
                for (uint32_t b = 0; b < 4; ++b)
                    sc[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                        attn_as_bf16(attn_load8<VEC>(row[b], kk + 8 * g, a.dk, (ok >> b) & 1)), attn_as_bf16(qv), sc[b], 0, 0,
                        0);
            }
#pragma unroll
            for (uint32_t b = 0; b < 4; ++b)
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e) {
                    const bool in = 16 * b + 4 * g + e < limit;
                    const float x = in ? fmaf(sc[b][e], a.scale_log2, -m) : -INFINITY;
                    sum[b][e] = fmaf(exp2f(x), in ? inv : 0.0f, sum[b][e]);
                }
        }
    }
#pragma unroll
    for (uint32_t b = 0; b < 4; ++b)
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) {
            float x = sum[b][e];
#pragma unroll
            for (uint32_t s = 1; s < 16; s <<= 1) x += __shfl_xor(x, s);
            const uint64_t t = tb + 16 * b + 4 * g + e;
            if (r == 0 && t < longest) p.weights[kvh * a.sequence_slot_count + start + t] += x;
        }
}

// ---- Rows bodies: 16-byte rows of 64, 128 or 256 dims ------------------------
//
// The same two steps for the shapes that models have, with the operands in
// registers. A row is a (query, query head) of one KV head; a tile of rows is
// `tile_queries` consecutive queries (or a group of one query's heads where those
// alone pass a tile), so a prompt's K rows are read once for NR * 16 rows.

// K rows of 64 tokens from t0 as addresses, lane l token t0 + l; the zero row
// past `end` and where a slot lies outside the pool (reported where `report`).
__device__ __forceinline__ uint64_t wgt_rows_at(const sglkv_attn_params &p, uint64_t kbase, uint64_t start, uint32_t t0,
                                                uint32_t end, bool report) {
    const uint32_t t = t0 + (threadIdx.x & 63);
    uint64_t row;
    return wgt_row(p, kbase, start, t, t < end, report, &row) ? row : reinterpret_cast<uint64_t>(p.zero_row);
}

// The 16-byte pieces of token `16 b + r`'s row (addresses in lanes as above)
// that lane (g, r) feeds to the matrix product: dims 32 c + 8 g.
template <uint32_t DKC>
__device__ __forceinline__ void wgt_load_rows(uint64_t rows, uint32_t b, uint32_t g, uint32_t r, sglkv_u16x8 (&k)[DKC]) {
    const uint64_t at = __shfl(rows, 16 * b + r) + 16 * g;
#pragma unroll
    for (uint32_t c = 0; c < DKC; ++c) k[c] = sel_load(at + 64 * c);
}

// The NR * 16 rows of a wave (lane (g, r) has rows 16 n + r): queries, running
// (maximum, sum) and metadata.
template <uint32_t NR, uint32_t DKC>
struct wgt_row_set {
    sglkv_u16x8 q[NR][DKC];
    float m[NR], l[NR];
    uint32_t len[NR], req[NR], row[NR];  // row: query * query_heads + head, ~0 where there is none
};

// Rows `from` + 16 n + r of the tile of queries qa .., whose heads h0 .. h0 +
// heads - 1 of a KV head are its rows. The loads of a kind go out at once (a lane
// without a row takes the first query's).
template <uint32_t DKC, uint32_t NR>
__device__ __forceinline__ void wgt_load_row_set(const sglkv_weights_params &p, uint32_t qa, uint32_t h0, uint32_t heads,
                                                 uint32_t from, uint32_t kvh, wgt_row_set<NR, DKC> &w) {
    const sglkv_attn_params &a = p.a;
    const uint32_t lane = threadIdx.x & 63, g = lane >> 4, r = lane & 15;
    uint64_t lengths[NR], starts[NR], ends[NR];
    uint32_t previous[NR];
    bool reports[NR];
#pragma unroll
    for (uint32_t n = 0; n < NR; ++n) {
        const uint32_t rho = from + 16 * n + r, qi = rho / heads, hi = h0 + rho - qi * heads;
        const uint32_t q = qa + qi;
        const bool own = qi < p.tile_queries && q < a.query_count && hi < a.group;
        const uint32_t query = own ? q : 0;
        w.row[n] = own ? q * a.query_heads + kvh * a.group + hi : ~0u;
        reports[n] = own && g == 0 && hi == 0 && kvh == 0 && blockIdx.y == 0;
        lengths[n] = a.query_sequence_lengths[query];
        w.req[n] = a.query_request_indices[query];
        previous[n] = a.query_request_indices[query > 0 ? query - 1 : 0];
        const uint64_t at = reinterpret_cast<uint64_t>(a.queries) + 2ull * (own ? w.row[n] : 0) * (32 * DKC) + 16 * g;
#pragma unroll
        for (uint32_t c = 0; c < DKC; ++c) w.q[n][c] = sel_load(at + 64 * c);
    }
#pragma unroll
    for (uint32_t n = 0; n < NR; ++n) {
        const uint32_t known = w.req[n] < a.request_count ? w.req[n] : 0;
        starts[n] = a.request_slot_offsets[known];
        ends[n] = a.request_slot_offsets[known + 1];
    }
#pragma unroll
    for (uint32_t n = 0; n < NR; ++n) {
        const bool known = w.req[n] < a.request_count;
        const bool holds = known && starts[n] <= ends[n] && ends[n] <= a.sequence_slot_count &&
                           lengths[n] <= ends[n] - starts[n] && lengths[n] <= p.max_length;
        if (reports[n]) {
            if (previous[n] > w.req[n] || (lengths[n] > 0 && !known))
                atomicOr(a.flag, SGLKV_FLAG_ATTN_REQUEST);
            else if (lengths[n] > 0 && !holds)
                atomicOr(a.flag, SGLKV_FLAG_ATTN_SEQUENCE);
        }
        w.len[n] = w.row[n] != ~0u && holds ? static_cast<uint32_t>(lengths[n]) : 0;  // (the host bounds it)
        if (w.len[n] == 0) w.req[n] = ~0u;
        w.m[n] = -3.402823466e+38f;
        w.l[n] = 0.0f;
    }
}

// The lowest request of the wave's rows whose bit is not in `seen`; ~0: none.
template <uint32_t NR>
__device__ __forceinline__ uint32_t wgt_next_request(const uint32_t (&req)[NR], uint32_t seen) {
    uint32_t now = ~0u;
#pragma unroll
    for (uint32_t n = 0; n < NR; ++n)
        if (!(seen >> n & 1) && req[n] < now) now = req[n];
#pragma unroll
    for (uint32_t s = 1; s < 64; s <<= 1) {
        const uint32_t o = __shfl_xor(now, s);
        now = o < now ? o : now;
    }
    return now;
}

// Marks request `now`'s rows seen; their lengths (0 for the others), and the
// longest and shortest in the wave.
template <uint32_t NR, uint32_t DKC>
__device__ __forceinline__ void wgt_take_request(const wgt_row_set<NR, DKC> &w, uint32_t now, uint32_t &seen,
                                                 uint32_t (&limit)[NR], uint32_t *longest, uint32_t *whole) {
    uint32_t most = 0, least = ~0u;
#pragma unroll
    for (uint32_t n = 0; n < NR; ++n) {
        const bool in = w.req[n] == now;
        limit[n] = in ? w.len[n] : 0;
        if (in) seen |= 1u << n;
        most = limit[n] > most ? limit[n] : most;
        if (w.row[n] != ~0u && limit[n] < least) least = limit[n];  // (a row of no query may hold anything)
    }
#pragma unroll
    for (uint32_t s = 1; s < 64; s <<= 1) {
        const uint32_t x = __shfl_xor(most, s), y = __shfl_xor(least, s);
        most = x > most ? x : most;
        least = y < least ? y : least;
    }
    *longest = __builtin_amdgcn_readfirstlane(most);
    *whole = __builtin_amdgcn_readfirstlane(least);
}

// 16 tokens from `t` (their K rows in kf) for all rows: scores and the running
// maximum and sum. `whole`: the rows' shortest length.
template <uint32_t DKC, uint32_t NR>
__device__ __forceinline__ void wgt_weigh_tile(const sglkv_weights_params &p, const sglkv_u16x8 (&kf)[DKC],
                                               wgt_row_set<NR, DKC> &w, const uint32_t (&limit)[NR], uint32_t t,
                                               uint32_t whole, uint32_t g) {
    const float scale = p.a.scale_log2;
    const uint32_t tt = t + 4 * g;  // this lane's tokens
    sglkv_f32x4 sc[NR];
#pragma unroll
    for (uint32_t n = 0; n < NR; ++n) sc[n] = sglkv_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (uint32_t c = 0; c < DKC; ++c)
#pragma unroll
        for (uint32_t n = 0; n < NR; ++n)
            sc[n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(attn_as_bf16(kf[c]), attn_as_bf16(w.q[n][c]), sc[n], 0, 0, 0);
    if (t + 16 > whole) {
#pragma unroll
        for (uint32_t n = 0; n < NR; ++n)
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e)
                if (tt + e >= limit[n]) sc[n][e] = -INFINITY;
    }
    // The reference moves only where a score passes it by more than 8 log2 units:
    // terms stay below 2^8 and most steps rescale nothing.
    float top[NR];
    bool moves = false;
#pragma unroll
    for (uint32_t n = 0; n < NR; ++n) {
        top[n] = fmaxf(fmaxf(sc[n][0], sc[n][1]), fmaxf(sc[n][2], sc[n][3])) * scale;
        moves |= top[n] > w.m[n] + 8.0f;
    }
    if (__ballot(moves)) {
#pragma unroll
        for (uint32_t n = 0; n < NR; ++n) {
            const float up = fmaxf(w.m[n], top[n]);
            w.l[n] *= __builtin_amdgcn_exp2f(w.m[n] - up);
            w.m[n] = up;
        }
    }
#pragma unroll
    for (uint32_t n = 0; n < NR; ++n)
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) w.l[n] += __builtin_amdgcn_exp2f(fmaf(sc[n][e], scale, -w.m[n]));
}

// The rows' statistics for the split whose tokens start at t0: the four lanes of
// a row join. One split's leave joined (wgt_joined).
template <uint32_t DKC, uint32_t NR>
__device__ __forceinline__ void wgt_leave_stats(const sglkv_weights_params &p, const wgt_row_set<NR, DKC> &w, uint32_t t0,
                                                uint32_t g) {
    const sglkv_attn_params &a = p.a;
#pragma unroll
    for (uint32_t n = 0; n < NR; ++n) {
        float m = w.m[n], l = w.l[n];
#pragma unroll
        for (uint32_t s = 16; s < 64; s <<= 1) {
            const float mo = __shfl_xor(m, s), lo = __shfl_xor(l, s), up = fmaxf(m, mo);
            l = l * exp2f(m - up) + lo * exp2f(mo - up);
            m = up;
        }
        if (g == 0 && w.row[n] != ~0u) {
            const bool some = t0 < w.len[n];
            float2 pair = some ? make_float2(m, l) : make_float2(-INFINITY, 0.0f);
            if (a.splits == 1) pair = some ? make_float2(m, 1.0f / l) : make_float2(INFINITY, 0.0f);
            reinterpret_cast<float2 *>(a.partial)[static_cast<uint64_t>(w.row[n]) * a.splits + blockIdx.y] = pair;
        }
    }
}

// Statistics of 16 rows, a wave each, over the tokens of split blockIdx.y; TB
// tiles of 16 tokens are weighed while the next TB are loading.
template <uint32_t DKC, uint32_t TB>
__device__ __forceinline__ void wgt_rows_body(const sglkv_weights_params &p) {
    const sglkv_attn_params &a = p.a;
    const uint32_t lane = threadIdx.x, g = lane >> 4, r = lane & 15;
    uint32_t bx = blockIdx.x;
    const uint32_t kvh = bx % a.kv_heads;
    bx /= a.kv_heads;
    const uint32_t hg = bx % p.tile_head_groups;
    const uint32_t tile = p.row_tiles - 1 - bx / p.tile_head_groups;
    wgt_row_set<1, DKC> w;
    wgt_load_row_set<DKC, 1>(p, tile * p.tile_queries, hg * 16, p.tile_head_groups > 1 ? 16 : a.group, 0, kvh, w);
    const uint64_t kbase = reinterpret_cast<uint64_t>(a.pool) + a.key_offset + kvh * a.key_head_stride;
    const uint32_t t0 = blockIdx.y * static_cast<uint32_t>(a.chunk_tokens);
    uint32_t seen = 0;
    for (;;) {  // one request after another (nearly always there is one)
        const uint32_t now = wgt_next_request<1>(w.req, seen);
        if (now == ~0u) break;
        uint32_t limit[1], longest, whole;
        wgt_take_request<1>(w, now, seen, limit, &longest, &whole);
        const uint64_t first = a.request_slot_offsets[__builtin_amdgcn_readfirstlane(now)];
        const uint32_t most = t0 + static_cast<uint32_t>(a.chunk_tokens), t1 = longest < most ? longest : most;
        if (t0 >= t1) continue;
        uint64_t rows = wgt_rows_at(a, kbase, first, t0, t1, kvh == 0);
        sglkv_u16x8 kf[2][TB][DKC];
#pragma unroll
        for (uint32_t b = 0; b < TB; ++b) wgt_load_rows<DKC>(rows, b, g, r, kf[0][b]);
        for (uint32_t t = t0; t < t1; t += 64) {
            const uint64_t next = t + 64 < t1 ? wgt_rows_at(a, kbase, first, t + 64, t1, kvh == 0)
                                              : reinterpret_cast<uint64_t>(p.a.zero_row);
#pragma unroll
            for (uint32_t part = 0; part < 4 / TB; ++part) {
                static_assert(TB == 1 || TB == 2, "the buffers come round with every 64 tokens");
#pragma unroll
                for (uint32_t b = 0; b < TB; ++b) {
                    const uint32_t ahead = part * TB + TB + b;
                    wgt_load_rows<DKC>(ahead < 4 ? rows : next, ahead & 3, g, r, kf[1 - part % 2][b]);
                }
                __builtin_amdgcn_sched_barrier(0);
                if (t + 16 * TB * part >= t1) continue;
#pragma unroll
                for (uint32_t b = 0; b < TB; ++b)
                    wgt_weigh_tile<DKC, 1>(p, kf[part % 2][b], w, limit, t + 16 * (part * TB + b), whole, g);
            }
            rows = next;
        }
    }
    wgt_leave_stats<DKC, 1>(p, w, t0, g);
}

// The same where the scores are kept in the workspace for the second step, so that K
// is read once: a decode step, which the bytes of K bound. K goes from the pool into
// LDS in blocks of 32 tokens, one in flight while another is weighed, laid out as in
// paged attention's staged body (attn_stg): a lane gets the scores of eight tokens in a
// row, and the four lanes of a row write 128 bytes. 64 sequences of up to 4,096 tokens,
// 8 KV heads of 4 query heads, dims 128 (266 MB of K, 17 MB of scores): 66 us, 4.3
// TB/s, and 13 for the second step; with K straight to registers, 64 bytes of 16 rows
// at a time, 76 and 17. The writes in between bound it: without them K alone goes at
// 5.9 TB/s (128 sequences of 4,096: 183 us of 232). Three or four stages, scores in
// blocks of 32 tokens, and stores past the caches take as long or longer.
template <uint32_t D>
__device__ __forceinline__ void wgt_scores_body(const sglkv_weights_params &p) {
    typedef attn_stg<D> S;
    constexpr uint32_t SECTION = SGLKV_WEIGHTS_SECTION;
    extern __shared__ __attribute__((aligned(16))) uint8_t wgt_stages[];
    uint64_t *const table = reinterpret_cast<uint64_t *>(wgt_stages + 2 * S::V);
    const sglkv_attn_params &a = p.a;
    const float scale = a.scale_log2;
    const uint32_t lane = threadIdx.x, g = lane >> 4, r = lane & 15;
    uint32_t bx = blockIdx.x;
    const uint32_t kvh = bx % a.kv_heads;
    bx /= a.kv_heads;
    const uint32_t hg = bx % p.tile_head_groups;
    const uint32_t tile = p.row_tiles - 1 - bx / p.tile_head_groups;
    wgt_row_set<1, S::KC> w;
    wgt_load_row_set<S::KC, 1>(p, tile * p.tile_queries, hg * 16, p.tile_head_groups > 1 ? 16 : a.group, 0, kvh, w);
    const uint64_t kbase = reinterpret_cast<uint64_t>(a.pool) + a.key_offset + kvh * a.key_head_stride;
    const uint32_t t0 = blockIdx.y * static_cast<uint32_t>(a.chunk_tokens);
    const uint32_t c = lane / S::PIECES, pc = lane % S::PIECES;
    auto issue = [&](uint32_t b) {
        const uint64_t *rows = table + kLatB * b + S::LOADS * c;  // tokens c, TPL + c, ..
        const uint32_t at = attn_lat_lds_at(wgt_stages) + (b & 1) * S::V;
#pragma unroll
        for (uint32_t h = 0; h < S::LOADS / 4; ++h) {
            uint64_t x[4];
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) x[i] = rows[4 * h + i] + 16 * S::kpos(S::TPL * (4 * h + i) + c, pc);
            attn_lat_load4v<1024>(x, at + 4096 * h);
        }
    };
    float *const scores = p.scores + static_cast<uint64_t>(w.row[0] == ~0u ? 0 : w.row[0]) * p.score_stride;
    uint32_t seen = 0;
    for (;;) {  // one request after another (nearly always there is one)
        const uint32_t now = wgt_next_request<1>(w.req, seen);
        if (now == ~0u) break;
        uint32_t limit[1], longest, whole;
        wgt_take_request<1>(w, now, seen, limit, &longest, &whole);
        const uint64_t first = a.request_slot_offsets[__builtin_amdgcn_readfirstlane(now)];
        const uint32_t most = t0 + static_cast<uint32_t>(a.chunk_tokens), t1 = longest < most ? longest : most;
        for (uint32_t s0 = t0; s0 < t1; s0 += SECTION) {
            uint64_t found[SECTION / 64];
#pragma unroll
            for (uint32_t i = 0; i < SECTION / 64; ++i)
                found[i] = wgt_rows_at(a, kbase, first, s0 + 64 * i, t1, kvh == 0);
            // (The last section's reads of the table are done: a wave's LDS accesses keep their order.)
#pragma unroll
            for (uint32_t i = 0; i < SECTION / 64; ++i) {
                const uint32_t at = 64 * i + lane;
                table[(at & ~31u) + S::entry(at & 31)] = found[i];
            }
            const uint32_t nb = ((t1 - s0 < SECTION ? t1 - s0 : SECTION) + kLatB - 1) / kLatB;
            // The last section's stages have been read, and nothing but the rows' loads and
            // the scores' stores counts from here on.
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
            issue(0);
            for (uint32_t k = 0; k < nb; ++k) {
                // Block k - 1's reads are done before block k + 1 takes its stage; then block
                // k has landed once no more is outstanding than block k + 1 (the stores
                // between make the wait longer, which costs nothing: counting them in took
                // as long).
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                if (k + 1 < nb) {
                    issue(k + 1);
                    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(S::LOADS) : "memory");
                } else {
                    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                }
                const uint8_t *kst = wgt_stages + (k & 1) * S::V;
                const uint32_t t = s0 + kLatB * k, tt = t + 8 * g;  // this lane's eight tokens
                sglkv_f32x4 sc[2] = {sglkv_f32x4{0.f, 0.f, 0.f, 0.f}, sglkv_f32x4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
                for (uint32_t q = 0; q < S::KC; ++q)
#pragma unroll
                    for (uint32_t b = 0; b < 2; ++b) {
                        const uint32_t j = 8 * (r >> 2) + 4 * b + (r & 3);
                        const sglkv_u16x8 kf = *reinterpret_cast<const sglkv_u16x8 *>(kst + S::ROW * j + 16 * S::kpos(j, 4 * q + g));
                        sc[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(attn_as_bf16(kf), attn_as_bf16(w.q[0][q]), sc[b], 0, 0, 0);
                    }
                float x[8];
#pragma unroll
                for (uint32_t e = 0; e < 8; ++e) x[e] = sc[e / 4][e % 4] * scale;
                if (tt < limit[0]) {
                    sglkv_f32x4 *to = reinterpret_cast<sglkv_f32x4 *>(scores + tt);
                    to[0] = sglkv_f32x4{x[0], x[1], x[2], x[3]};
                    to[1] = sglkv_f32x4{x[4], x[5], x[6], x[7]};
                }
                if (t + kLatB > whole) {
#pragma unroll
                    for (uint32_t e = 0; e < 8; ++e)
                        if (tt + e >= limit[0]) x[e] = -INFINITY;
                }
                // (As wgt_weigh_tile: the reference moves where a score passes it by 8.)
                float top = x[0];
#pragma unroll
                for (uint32_t e = 1; e < 8; ++e) top = fmaxf(top, x[e]);
                if (__ballot(top > w.m[0] + 8.0f)) {
                    const float up = fmaxf(w.m[0], top);
                    w.l[0] *= __builtin_amdgcn_exp2f(w.m[0] - up);
                    w.m[0] = up;
                }
#pragma unroll
                for (uint32_t e = 0; e < 8; ++e) w.l[0] += __builtin_amdgcn_exp2f(x[e] - w.m[0]);
            }
        }
    }
    wgt_leave_stats<S::KC, 1>(p, w, t0, g);
}

// The queries [*q0, *q1) of request `req`, whose indices never fall: 32 places
// probed at once for either end, so three loads in a row up to 32,768 queries.
__device__ __forceinline__ void wgt_queries_of(const sglkv_attn_params &p, uint32_t req, uint32_t *q0, uint32_t *q1) {
    const uint32_t lane = threadIdx.x & 63, side = lane >> 5, place = lane & 31;
    uint32_t low = 0, high = static_cast<uint32_t>(p.query_count);  // the first index >= req + side lies in [low, high]
    while (__ballot(low < high)) {
        const uint32_t step = (high - low + 31) / 32, at = low + place * step;
        const bool less = at < high && p.query_request_indices[at] < req + side;
        const uint64_t all = __ballot(less);
        const uint32_t below = __popc(static_cast<uint32_t>(side ? all >> 32 : all));
        if (below == 0) {
            high = low;  // (at low itself)
        } else {
            const uint32_t to = low + below * step;
            low += (below - 1) * step + 1;
            high = to < high ? to : high;
        }
    }
    *q0 = __builtin_amdgcn_readlane(low, 0);
    const uint32_t end = __builtin_amdgcn_readlane(low, 32);
    *q1 = end > *q0 ? end : *q0;  // (indices that fall have been reported)
}

// The splits' statistics of a row joined: the reference m and 1 / l, or (inf, 0)
// where the row weighs nothing. `lanes` lanes to a row (a power of two up to 16),
// this one lane v of them. (One split's statistics leave the first kernel like
// this.)
__device__ __forceinline__ float2 wgt_joined(const sglkv_attn_params &a, uint64_t row, uint32_t v, uint32_t lanes) {
    const float2 *stats = reinterpret_cast<const float2 *>(a.partial) + row * a.splits;
    float top = -INFINITY, l = 0.0f;
    auto join = [&](float m, float x) {
        const float up = fmaxf(top, m);
        if (up != -INFINITY) l = l * __builtin_amdgcn_exp2f(top - up) + x * __builtin_amdgcn_exp2f(m - up);
        top = up;
    };
    for (uint32_t s = v; s < a.splits; s += lanes) join(stats[s].x, stats[s].y);
    for (uint32_t s = 1; s < lanes; s <<= 1) join(__shfl_xor(top, s), __shfl_xor(l, s));
    return top == -INFINITY ? make_float2(INFINITY, 0.0f) : make_float2(top, 1.0f / l);
}

// Each row's statistics joined into p.joined, p.join_lanes lanes to a row.
__device__ __forceinline__ void wgt_join_body(const sglkv_weights_params &p) {
    const uint32_t lanes = p.join_lanes, v = threadIdx.x % lanes;
    const uint64_t row = (static_cast<uint64_t>(blockIdx.x) * SGLKV_WEIGHTS_THREADS + threadIdx.x) / lanes;
    if (row >= p.a.query_count * p.a.query_heads) return;
    const float2 x = wgt_joined(p.a, row, v, lanes);
    if (v == 0) reinterpret_cast<float2 *>(p.joined)[row] = x;
}

// Row pitch in LDS: 16 rows' pieces land in all banks once.
template <uint32_t DKC>
constexpr uint32_t kWgtPitch = 64 * DKC + 16;

// Statistics of many rows: four waves of NR * 16 rows each share the K rows of 64
// tokens through LDS, two stages deep, so K is read once for 64 NR rows. Four prompts
// of up to 2,048 tokens, 8 KV heads of 4 query heads, dims 128 (33 GFLOP): 77 us, 430
// TFLOP/s; 16 of 2,048 tokens 660, four of 8,192 840. With few workgroups the wait for
// the next stage's rows bounds it: half the rows a wave, four waves a SIMD or a fifth
// fewer vector instructions leave it where it is.
template <uint32_t DKC, uint32_t NR>
__device__ __forceinline__ void wgt_tile_stats_body(const sglkv_weights_params &p) {
    constexpr uint32_t PIECES = 4 * DKC, SIDE = 256 / PIECES, LOADS = 64 / SIDE, PITCH = kWgtPitch<DKC>;
    __shared__ __attribute__((aligned(16))) uint8_t stages[2][64 * PITCH];
    __shared__ uint32_t shared_words[4];
    const sglkv_attn_params &a = p.a;
    const uint32_t tid = threadIdx.x, lane = tid & 63, g = lane >> 4, r = lane & 15;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid / 64);
    uint32_t item, kvh;
    sel_place(a.kv_heads, &item, &kvh);  // (whole token and query rows in an XCD's L2)
    if (item >= p.row_tiles * p.tile_head_groups) return;
    const uint32_t hg = item % p.tile_head_groups;
    // (A prompt's last queries attend the most: they start first.)
    const uint32_t tile = p.row_tiles - 1 - item / p.tile_head_groups;
    const uint32_t heads = p.tile_head_groups > 1 ? 64 * NR : a.group;  // rows of a query in this tile
    wgt_row_set<NR, DKC> w;
    wgt_load_row_set<DKC, NR>(p, tile * p.tile_queries, hg * 64 * NR, heads, wave * 16 * NR, kvh, w);
    const uint64_t kbase = reinterpret_cast<uint64_t>(a.pool) + a.key_offset + kvh * a.key_head_stride;
    const uint32_t t0 = blockIdx.y * static_cast<uint32_t>(a.chunk_tokens);
    const uint32_t piece = 16 * (tid % PIECES), own = tid / PIECES;  // of a row; the first token it loads
    uint32_t seen = 0;
    for (;;) {  // one request after another (nearly always there is one)
        uint32_t now = wgt_next_request<NR>(w.req, seen);
        if (lane == 0) shared_words[wave] = now;
        __syncthreads();
        for (uint32_t i = 0; i < 4; ++i) now = shared_words[i] < now ? shared_words[i] : now;
        __syncthreads();
        if (now == ~0u) break;
        uint32_t limit[NR], longest, whole;
        wgt_take_request<NR>(w, now, seen, limit, &longest, &whole);
        const uint64_t first = a.request_slot_offsets[__builtin_amdgcn_readfirstlane(now)];
        if (lane == 0) shared_words[wave] = longest;
        __syncthreads();
        uint32_t t1 = 0;
        for (uint32_t i = 0; i < 4; ++i) t1 = shared_words[i] > t1 ? shared_words[i] : t1;
        __syncthreads();
        t1 = __builtin_amdgcn_readfirstlane(t1);
        const uint32_t most = t0 + static_cast<uint32_t>(a.chunk_tokens);
        t1 = t1 < most ? t1 : most;
        if (t0 >= t1) continue;
        sglkv_u16x8 ahead[LOADS];
        auto load = [&](uint64_t rows) {
#pragma unroll
            for (uint32_t i = 0; i < LOADS; ++i) ahead[i] = sel_load(__shfl(rows, own + SIDE * i) + piece);
        };
        auto put = [&](uint32_t stage) {
#pragma unroll
            for (uint32_t i = 0; i < LOADS; ++i)
                *reinterpret_cast<sglkv_u16x8 *>(stages[stage] + (own + SIDE * i) * PITCH + piece) = ahead[i];
        };
        const bool report = kvh == 0 && wave == 0;
        load(wgt_rows_at(a, kbase, first, t0, t1, report));
        uint64_t rows = wgt_rows_at(a, kbase, first, t0 + 64, t1, report);
        put(0);
        __syncthreads();
        uint32_t stage = 0;
        for (uint32_t t = t0; t < t1; t += 64, stage ^= 1) {
            const bool more = t + 64 < t1;
            if (more) {
                load(rows);
                rows = wgt_rows_at(a, kbase, first, t + 128, t1, report);
            }
            if (t < longest) {
                const uint32_t tiles = longest - t < 64 ? (longest - t + 15) / 16 : 4;
                for (uint32_t b = 0; b < tiles; ++b) {
                    const uint8_t *at = stages[stage] + (16 * b + r) * PITCH + 16 * g;
                    sglkv_u16x8 kf[DKC];
#pragma unroll
                    for (uint32_t c = 0; c < DKC; ++c) kf[c] = *reinterpret_cast<const sglkv_u16x8 *>(at + 64 * c);
                    wgt_weigh_tile<DKC, NR>(p, kf, w, limit, t + 16 * b, whole, g);
                }
            }
            if (more) {
                put(stage ^ 1);
                __syncthreads();
            }
        }
        __syncthreads();  // (the next request's first stage)
    }
    wgt_leave_stats<DKC, NR>(p, w, t0, g);
}

// Accumulation of many rows: a wave has TT tiles of 16 tokens of a (request, KV
// head) in registers, a workgroup four waves' side by side; the request's rows
// (or a segment's) pass through LDS, 32 at a time and two stages deep. The prompts
// above: 100 us, 330 TFLOP/s; 16 of 2,048 tokens 520, four of 8,192 730. Bound as the
// statistics are; half the tokens a wave took as long.
template <uint32_t DKC, uint32_t TT>
__device__ __forceinline__ void wgt_tile_accumulate_body(const sglkv_weights_params &p) {
    constexpr uint32_t ROWS = 32, PIECES = 4 * DKC, SIDE = 256 / PIECES, LOADS = ROWS / SIDE, PITCH = kWgtPitch<DKC>;
    struct info {
        float m, inv;
        uint64_t length;
    };
    __shared__ __attribute__((aligned(16))) uint8_t stages[2][ROWS * PITCH];
    __shared__ info infos[2][ROWS];
    __shared__ uint32_t extents[2][4];
    const sglkv_attn_params &a = p.a;
    const uint32_t tid = threadIdx.x, lane = tid & 63, g = lane >> 4, r = lane & 15;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid / 64);
    uint32_t item, kvh;
    sel_place(a.kv_heads, &item, &kvh);  // (whole token and query rows in an XCD's L2)
    const uint32_t requests = static_cast<uint32_t>(a.request_count);
    const uint32_t segment = item % p.segments, tile = item / p.segments / requests;
    const uint32_t req = item / p.segments - tile * requests, tg = tile * 64 * TT, tb = tg + wave * 16 * TT;
    if (tile >= p.tiles) return;
    const uint64_t start = a.request_slot_offsets[req], end = a.request_slot_offsets[req + 1];
    if (start > end || end > a.sequence_slot_count || tg >= end - start) return;
    uint32_t q0, q1;
    wgt_queries_of(a, req, &q0, &q1);
    // (A segment of the request's queries: its sums go to the workspace.)
    const uint32_t share = (q1 - q0 + p.segments - 1) / p.segments;
    q0 = q1 - q0 > segment * share ? q0 + segment * share : q1;
    q1 = q1 - q0 > share ? q0 + share : q1;
    // (A length that does not hold has been reported: its row weighs nothing.)
    const uint64_t most = end - start < p.max_length ? end - start : p.max_length;
    // The tokens that any of these queries attends, and the first that attends
    // this tile: every wave looks at its share of the lengths.
    uint32_t longest = 0, q_from = q1;
    for (uint32_t q = q0 + tid; q < q1; q += 256) {
        const uint64_t n64 = a.query_sequence_lengths[q];
        const uint32_t n = n64 <= most ? static_cast<uint32_t>(n64) : 0;
        longest = n > longest ? n : longest;
        if (n > tg && q < q_from) q_from = q;
    }
#pragma unroll
    for (uint32_t s = 1; s < 64; s <<= 1) {
        const uint32_t x = __shfl_xor(longest, s), y = __shfl_xor(q_from, s);
        longest = x > longest ? x : longest;
        q_from = y < q_from ? y : q_from;
    }
    if (lane == 0) {
        extents[0][wave] = longest;
        extents[1][wave] = q_from;
    }
    __syncthreads();
    for (uint32_t i = 0; i < 4; ++i) {
        longest = extents[0][i] > longest ? extents[0][i] : longest;
        q_from = extents[1][i] < q_from ? extents[1][i] : q_from;
    }
    longest = __builtin_amdgcn_readfirstlane(longest);
    q_from = __builtin_amdgcn_readfirstlane(q_from);
    float sum[TT][4] = {};
    if (tg < longest) {
        const uint64_t kbase = reinterpret_cast<uint64_t>(a.pool) + a.key_offset + kvh * a.key_head_stride;
        const uint64_t at = wgt_rows_at(a, kbase, start, tb, longest, false);
        sglkv_u16x8 kf[TT][DKC];
#pragma unroll
        for (uint32_t b = 0; b < TT; ++b) wgt_load_rows<DKC>(at, b, g, r, kf[b]);
        // Rows rho = (query - q_from) * group + head. A thread's pieces of a stage are
        // rows own + SIDE i; a row past the last is the first, weighed 0.
        const uint32_t count = (q1 - q_from) * a.group, dq = ROWS / a.group, dh = ROWS - dq * a.group;
        const uint32_t piece = 16 * (tid % PIECES), own = tid / PIECES;
        const uint64_t qbase = reinterpret_cast<uint64_t>(a.queries) + piece;
        const uint32_t head0 = kvh * a.group;
        uint32_t rq[LOADS + 1], rh[LOADS + 1];  // the last: row tid's, for its statistics
#pragma unroll
        for (uint32_t i = 0; i <= LOADS; ++i) {
            const uint32_t rho = i < LOADS ? own + SIDE * i : tid & (ROWS - 1);
            rq[i] = rho / a.group;
            rh[i] = rho - rq[i] * a.group;
        }
        sglkv_u16x8 ahead[LOADS];
        info next;
        auto load = [&] {
            const uint32_t last = q1 - q_from;
#pragma unroll
            for (uint32_t i = 0; i <= LOADS; ++i) {
                const bool in = rq[i] < last;
                const uint64_t q = q_from + (in ? rq[i] : 0), row = q * a.query_heads + head0 + (in ? rh[i] : 0);
                if (i < LOADS) {
                    ahead[i] = sel_load(qbase + row * (64 * DKC));
                } else if (tid < ROWS) {
                    const float2 x = reinterpret_cast<const float2 *>(p.joined)[row];
                    const uint64_t n = a.query_sequence_lengths[q];
                    next = info{x.x, x.y, in && n <= most ? n : 0};
                }
                rq[i] += dq;
                rh[i] += dh;
                if (rh[i] >= a.group) {
                    rh[i] -= a.group;
                    ++rq[i];
                }
            }
        };
        auto put = [&](uint32_t stage) {
#pragma unroll
            for (uint32_t i = 0; i < LOADS; ++i)
                *reinterpret_cast<sglkv_u16x8 *>(stages[stage] + (own + SIDE * i) * PITCH + piece) = ahead[i];
            if (tid < ROWS) infos[stage][tid] = next;
        };
        load();
        put(0);
        __syncthreads();
        uint32_t stage = 0;
        for (uint32_t done = 0; done < count; done += ROWS, stage ^= 1) {
            const bool more = done + ROWS < count;
            if (more) load();
#pragma unroll
            for (uint32_t n = 0; n < ROWS / 16; ++n) {
                const info x = infos[stage][16 * n + r];
                const uint64_t past = x.length > tb ? x.length - tb : 0;
                const uint32_t limit = past < 16 * TT ? static_cast<uint32_t>(past) : 16 * TT;
                if (!__ballot(limit > 0)) continue;
                const bool whole = !__ballot(limit < 16 * TT);
                const uint8_t *from = stages[stage] + (16 * n + r) * PITCH + 16 * g;
                sglkv_u16x8 qf[DKC];
#pragma unroll
                for (uint32_t c = 0; c < DKC; ++c) qf[c] = *reinterpret_cast<const sglkv_u16x8 *>(from + 64 * c);
                sglkv_f32x4 sc[TT];
#pragma unroll
                for (uint32_t b = 0; b < TT; ++b) sc[b] = sglkv_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (uint32_t c = 0; c < DKC; ++c)
#pragma unroll
                    for (uint32_t b = 0; b < TT; ++b)
                        sc[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(attn_as_bf16(kf[b][c]), attn_as_bf16(qf[c]), sc[b], 0,
                                                                        0, 0);
                if (whole) {
#pragma unroll
                    for (uint32_t b = 0; b < TT; ++b)
#pragma unroll
                        for (uint32_t e = 0; e < 4; ++e)
                            sum[b][e] =
                                fmaf(__builtin_amdgcn_exp2f(fmaf(sc[b][e], a.scale_log2, -x.m)), x.inv, sum[b][e]);
                } else {
#pragma unroll
                    for (uint32_t b = 0; b < TT; ++b)
#pragma unroll
                        for (uint32_t e = 0; e < 4; ++e) {
                            // (Factor and exponent both: 1 / l is NaN or infinite where the scores are.)
                            const bool in = 16 * b + 4 * g + e < limit;
                            const float y = in ? fmaf(sc[b][e], a.scale_log2, -x.m) : -INFINITY;
                            sum[b][e] = fmaf(__builtin_amdgcn_exp2f(y), in ? x.inv : 0.0f, sum[b][e]);
                        }
                }
            }
            if (more) {
                put(stage ^ 1);
                __syncthreads();
            }
        }
    } else if (p.segments == 1) {
        return;
    }
    // The 16 lanes of a token join; a segment writes all of its tokens.
#pragma unroll
    for (uint32_t b = 0; b < TT; ++b)
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) {
            float x = sum[b][e];
            x += __uint_as_float(sel_join<1>(__float_as_uint(x)));
            x += __uint_as_float(sel_join<2>(__float_as_uint(x)));
            x += __uint_as_float(sel_join<4>(__float_as_uint(x)));
            x += __uint_as_float(sel_join<8>(__float_as_uint(x)));
            const uint32_t t = tb + 16 * b + 4 * g + e;
            if (r != 0) continue;
            const uint64_t to = kvh * a.sequence_slot_count + start + t;
            if (p.segments > 1) {
                if (t < end - start) p.partial_sums[segment * a.kv_heads * a.sequence_slot_count + to] = x;
            } else if (t < longest) {
                p.weights[to] += x;
            }
        }
}

// The segments' sums, in order, added to the weights: a thread to a position of
// a request.
__device__ __forceinline__ void wgt_segments_body(const sglkv_weights_params &p) {
    const sglkv_attn_params &a = p.a;
    uint32_t bx = blockIdx.x;
    const uint32_t kvh = bx % a.kv_heads;
    bx /= a.kv_heads;
    const uint32_t blocks = (p.max_length + SGLKV_WEIGHTS_THREADS - 1) / SGLKV_WEIGHTS_THREADS;
    const uint32_t req = bx / blocks;
    const uint64_t t = static_cast<uint64_t>(bx - req * blocks) * SGLKV_WEIGHTS_THREADS + threadIdx.x;
    const uint64_t start = a.request_slot_offsets[req], end = a.request_slot_offsets[req + 1];
    if (start > end || end > a.sequence_slot_count || t >= end - start || t >= p.max_length) return;
    const uint64_t at = kvh * a.sequence_slot_count + start + t;
    float x = 0.0f;
    for (uint32_t s = 0; s < p.segments; ++s) x += p.partial_sums[s * a.kv_heads * a.sequence_slot_count + at];
    if (x != 0.0f) p.weights[at] += x;  // (NaN is added; nothing leaves a position as it is)
}

// Accumulation from kept scores: a workgroup has SGLKV_WEIGHTS_APPLY tokens of a
// (request, KV head), a thread every SGLKV_WEIGHTS_THREADS-th of them, its
// (query, head)s in turn.
__device__ __forceinline__ void wgt_apply_body(const sglkv_weights_params &p) {
    constexpr uint32_t THREADS = SGLKV_WEIGHTS_THREADS, EACH = SGLKV_WEIGHTS_APPLY / THREADS, ROWS = THREADS / 16;
    __shared__ float2 joined[ROWS];
    __shared__ uint32_t limits[ROWS];
    const sglkv_attn_params &a = p.a;
    const uint32_t tid = threadIdx.x;
    uint32_t bx = blockIdx.x;
    const uint32_t kvh = bx % a.kv_heads;
    bx /= a.kv_heads;
    const uint32_t tile = bx % p.tiles, req = bx / p.tiles, tb = tile * SGLKV_WEIGHTS_APPLY;
    const uint64_t start = a.request_slot_offsets[req], end = a.request_slot_offsets[req + 1];
    if (start > end || end > a.sequence_slot_count || tb >= end - start) return;
    uint32_t q0, q1;
    wgt_queries_of(a, req, &q0, &q1);
    const uint64_t most = end - start < p.max_length ? end - start : p.max_length;
    const uint32_t count = (q1 - q0) * a.group;
    float sum[EACH] = {};
    uint32_t longest = 0;
    for (uint32_t base = 0; base < count; base += ROWS) {
        const uint32_t here = count - base < ROWS ? count - base : ROWS;
        __syncthreads();
        // 16 lanes to a row: its splits' statistics joined.
        const uint32_t i = tid / 16, v = tid % 16;
        if (i < here) {
            const uint32_t q = q0 + (base + i) / a.group, h = (base + i) % a.group;
            const uint64_t row = static_cast<uint64_t>(q) * a.query_heads + kvh * a.group + h;
            const float2 x = a.splits == 1 ? reinterpret_cast<const float2 *>(a.partial)[row] : wgt_joined(a, row, v, 16);
            if (v == 0) {
                const uint64_t n = a.query_sequence_lengths[q];
                limits[i] = n <= most && a.query_request_indices[q] == req ? static_cast<uint32_t>(n) : 0;
                joined[i] = x;
            }
        }
        __syncthreads();
        uint32_t q = q0 + base / a.group, h = base % a.group;
#pragma unroll 4
        for (uint32_t j = 0; j < here; ++j) {
            const float *scores = p.scores + (static_cast<uint64_t>(q) * a.query_heads + kvh * a.group + h) * p.score_stride;
            if (++h == a.group) {
                h = 0;
                ++q;
            }
            const uint32_t limit = limits[j];
            const float2 stats = joined[j];
            longest = limit > longest ? limit : longest;
#pragma unroll
            for (uint32_t e = 0; e < EACH; ++e) {
                const uint32_t t = tb + THREADS * e + tid;
                if (t < limit) sum[e] = fmaf(__builtin_amdgcn_exp2f(scores[t] - stats.x), stats.y, sum[e]);
            }
        }
    }
#pragma unroll
    for (uint32_t e = 0; e < EACH; ++e) {
        const uint32_t t = tb + THREADS * e + tid;
        if (t < longest) p.weights[kvh * a.sequence_slot_count + start + t] += sum[e];
    }
}

// ---- The kept positions -----------------------------------------------------

// A request's slots and length; false (length 0) where its metadata does not
// hold, which sets the error word when `report`.
__device__ __forceinline__ uint64_t evt_request(const sglkv_evict_params &p, uint64_t req, bool report, uint64_t *start) {
    const uint64_t s = p.request_slot_offsets[req], e = p.request_slot_offsets[req + 1], n = p.request_lengths[req];
    *start = s;
    if (s <= e && e <= p.sequence_slot_count && n <= e - s && n <= p.max_length) return n;
    if (report) atomicOr(p.flag, SGLKV_FLAG_ATTN_SEQUENCE);
    return 0;
}

// Keys that order as the sums do: NaN above every number, and above it the
// positions that are always kept.
__device__ __forceinline__ uint32_t evt_key(float x) {
    if (x != x) return ~0u - 1;
    const uint32_t b = __float_as_uint(x + 0.0f);  // (-0 is 0)
    return b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | (1u << 31));
}

__device__ __forceinline__ void evt_select_body(const sglkv_evict_params &p) {
    __shared__ sel_pick_state state;
    const uint32_t head = blockIdx.x % p.heads;
    const uint64_t req = blockIdx.x / p.heads;
    uint64_t start;
    const uint64_t len = evt_request(p, req, head == 0 && threadIdx.x == 0, &start);
    const float *weights = p.weights + head * p.sequence_slot_count + start;
    sel_pick<uint32_t, SGLKV_EVICT_THREADS / 64, 16>(
        len, p.max_kept,
        [&](uint64_t i) { return i < p.first_tokens || i + p.last_tokens >= len ? ~0u : evt_key(weights[i]); },
        p.kept + (req * p.heads + head) * p.max_kept, state);
}

// ---- The copy ---------------------------------------------------------------
//
// A workgroup copies p.rows destination rows of a request for block_heads heads
// of one tensor (grid y: head blocks, z: tensors). It resolves each (row,
// head)'s kept position to the two addresses once, into LDS; then `lanes`
// threads move a head chunk, W bytes each, U chunks in flight. Bound by the bytes
// moved: 32 requests cut to 2,048 positions, 8 heads of 256 bytes, keys and values
// (537 MB read and written) take 110 us, 4.9 TB/s, the rate of a large plain copy.
// That wants 16 rows to a workgroup (32: 112 us, 64: 123) and loads and stores that
// pass the caches by (64 rows: 127 us with plain ones).
template <typename V>
__device__ __forceinline__ void evt_compact_body(const sglkv_evict_params &p) {
    typedef __attribute__((address_space(1))) const V src_t;
    typedef __attribute__((address_space(1))) V dst_t;
    __shared__ uint64_t from[SGLKV_COMPACT_CHUNKS], to[SGLKV_COMPACT_CHUNKS];
    constexpr uint32_t U = 8;
    const uint32_t tid = threadIdx.x, tensor = blockIdx.z;
    const uint32_t tile = blockIdx.x % p.row_tiles;
    const uint64_t req = blockIdx.x / p.row_tiles;
    const uint32_t h0 = blockIdx.y * p.block_heads, heads = p.heads - h0 < p.block_heads ? p.heads - h0 : p.block_heads;
    uint64_t start;
    const bool report = tile == 0 && h0 == 0 && tensor == 0 && tid == 0;
    if (report && req == 0 && p.scale_dst)
        for (uint32_t t = 0; t < p.tensors; ++t) p.scale_dst[t] = p.scale_src[t];
    const uint64_t len = evt_request(p, req, report, &start);
    const uint64_t d0 = p.to_offsets[req], d1 = p.to_offsets[req + 1];
    const bool ranged = d0 <= d1 && d1 <= p.to_slot_count;
    if (!ranged) {
        if (report) atomicOr(p.flag, SGLKV_FLAG_ATTN_SEQUENCE);
        return;
    }
    const uint64_t room = d1 - d0, r0 = static_cast<uint64_t>(tile) * p.rows;
    // Positions of the destination that no list reaches: their sums begin at 0.
    if (p.to_weights && tensor == 0)
        for (uint64_t row = p.max_kept + r0; row < room; row += static_cast<uint64_t>(p.row_tiles) * p.rows)
            for (uint32_t i = tid; i < p.rows * heads; i += SGLKV_COMPACT_THREADS) {
                const uint32_t h = i / p.rows, j = i - h * p.rows;
                if (row + j < room) p.to_weights[(h0 + h) * p.to_slot_count + d0 + row + j] = 0.0f;
            }
    const uint32_t rows = p.max_kept - r0 < p.rows ? static_cast<uint32_t>(p.max_kept - r0) : p.rows;
    // One head's rows side by side: the lists and sums are read in runs.
    for (uint32_t i = tid; i < rows * heads; i += SGLKV_COMPACT_THREADS) {
        const uint32_t h = i / rows, j = i - h * rows;
        const uint64_t row = r0 + j;
        const uint32_t *list = p.kept + (req * p.heads + h0 + h) * p.max_kept;
        const uint32_t kept = list[row];
        uint64_t src = SGLKV_INVALID_OFFSET, dst = SGLKV_INVALID_OFFSET;
        float weight = 0.0f;
        if (kept != SGLKV_SELECT_NONE) {
            if (kept >= len || row >= room) {
                atomicOr(p.flag, SGLKV_FLAG_ATTN_SEQUENCE);
            } else {
                const uint64_t s = p.sequence_slots[start + kept], d = p.to_slots[d0 + row];
                if (s >= p.src.slot_count || d >= p.dst.slot_count) {
                    atomicOr(p.flag, SGLKV_FLAG_ATTN_SLOT);
                } else {
                    const uint32_t sp = static_cast<uint32_t>(s) / p.src.page_size, dp = static_cast<uint32_t>(d) / p.dst.page_size;
                    src = p.src.plane[tensor] + sp * p.src.stride[tensor] +
                          (static_cast<uint32_t>(s) - sp * p.src.page_size) * p.src.pos_mult[tensor] +
                          (h0 + h) * p.src.head_stride[tensor];
                    dst = p.dst.plane[tensor] + dp * p.dst.stride[tensor] +
                          (static_cast<uint32_t>(d) - dp * p.dst.page_size) * p.dst.pos_mult[tensor] +
                          (h0 + h) * p.dst.head_stride[tensor];
                }
                if (p.to_weights && tensor == 0) weight = p.weights[(h0 + h) * p.sequence_slot_count + start + kept];
            }
        }
        from[j * heads + h] = src;
        to[j * heads + h] = dst;
        if (p.to_weights && tensor == 0 && row < room) p.to_weights[(h0 + h) * p.to_slot_count + d0 + row] = weight;
    }
    __syncthreads();
    const uint32_t lanes = p.lanes[tensor], vectors = p.vectors[tensor], side = SGLKV_COMPACT_THREADS / lanes;
    const uint32_t v0 = tid % lanes, chunks = rows * heads;
    for (uint32_t c0 = tid / lanes; c0 < chunks; c0 += side * U)
        for (uint32_t v = v0; v < vectors; v += lanes) {
            V x[U];
            uint64_t at[U];
#pragma unroll
            for (uint32_t u = 0; u < U; ++u) {
                const uint32_t c = c0 + side * u;
                const uint64_t s = c < chunks ? from[c] : SGLKV_INVALID_OFFSET;
                at[u] = c < chunks ? to[c] : SGLKV_INVALID_OFFSET;
                if (s != SGLKV_INVALID_OFFSET) x[u] = __builtin_nontemporal_load(reinterpret_cast<src_t *>(s + v * sizeof(V)));
            }
#pragma unroll
            for (uint32_t u = 0; u < U; ++u)
                if (at[u] != SGLKV_INVALID_OFFSET) __builtin_nontemporal_store(x[u], reinterpret_cast<dst_t *>(at[u] + v * sizeof(V)));
        }
}

}  // namespace

extern "C" __global__ __launch_bounds__(64) void sglkv_weight_stats_v16(sglkv_weights_params p) { wgt_stats_body<true>(p); }
extern "C" __global__ __launch_bounds__(64) __attribute__((amdgpu_waves_per_eu(2))) void
sglkv_weight_stats_v2(sglkv_weights_params p) {
    wgt_stats_body<false>(p);
}
extern "C" __global__ __launch_bounds__(64) void sglkv_accumulate_weights_v16(sglkv_weights_params p) {
    wgt_accumulate_body<true>(p);
}
extern "C" __global__ __launch_bounds__(64) __attribute__((amdgpu_waves_per_eu(2))) void
sglkv_accumulate_weights_v2(sglkv_weights_params p) {
    wgt_accumulate_body<false>(p);
}

extern "C" __global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(3))) void sglkv_weight_rows64(sglkv_weights_params p) {
    wgt_tile_stats_body<2, 4>(p);
}
extern "C" __global__ __launch_bounds__(64) __attribute__((amdgpu_waves_per_eu(2))) void sglkv_weight_few64(sglkv_weights_params p) {
    wgt_rows_body<2, 2>(p);
}
extern "C" __global__ __launch_bounds__(64) __attribute__((amdgpu_waves_per_eu(2))) void sglkv_weight_scores64(sglkv_weights_params p) {
    wgt_scores_body<64>(p);
}
extern "C" __global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(3))) void sglkv_accumulate_rows64(sglkv_weights_params p) {
    wgt_tile_accumulate_body<2, 4>(p);
}
extern "C" __global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(3))) void sglkv_weight_rows128(sglkv_weights_params p) {
    wgt_tile_stats_body<4, 4>(p);
}
extern "C" __global__ __launch_bounds__(64) __attribute__((amdgpu_waves_per_eu(2))) void sglkv_weight_few128(sglkv_weights_params p) {
    wgt_rows_body<4, 2>(p);
}
extern "C" __global__ __launch_bounds__(64) __attribute__((amdgpu_waves_per_eu(2))) void sglkv_weight_scores128(sglkv_weights_params p) {
    wgt_scores_body<128>(p);
}
extern "C" __global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(3))) void sglkv_accumulate_rows128(sglkv_weights_params p) {
    wgt_tile_accumulate_body<4, 4>(p);
}
extern "C" __global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) void sglkv_weight_rows256(sglkv_weights_params p) {
    wgt_tile_stats_body<8, 2>(p);
}
extern "C" __global__ __launch_bounds__(64) __attribute__((amdgpu_waves_per_eu(2))) void sglkv_weight_few256(sglkv_weights_params p) {
    wgt_rows_body<8, 1>(p);
}
extern "C" __global__ __launch_bounds__(64) __attribute__((amdgpu_waves_per_eu(2))) void sglkv_weight_scores256(sglkv_weights_params p) {
    wgt_scores_body<256>(p);
}
extern "C" __global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(3))) void sglkv_accumulate_rows256(sglkv_weights_params p) {
    wgt_tile_accumulate_body<8, 2>(p);
}
extern "C" __global__ __launch_bounds__(SGLKV_WEIGHTS_THREADS) void sglkv_add_segments(sglkv_weights_params p) {
    wgt_segments_body(p);
}
extern "C" __global__ __launch_bounds__(SGLKV_WEIGHTS_THREADS) void sglkv_join_statistics(sglkv_weights_params p) {
    wgt_join_body(p);
}
extern "C" __global__ __launch_bounds__(SGLKV_WEIGHTS_THREADS) void sglkv_apply_scores(sglkv_weights_params p) {
    wgt_apply_body(p);
}

extern "C" __global__ __launch_bounds__(SGLKV_EVICT_THREADS) void sglkv_select_tokens(sglkv_evict_params p) {
    evt_select_body(p);
}

extern "C" __global__ __launch_bounds__(SGLKV_COMPACT_THREADS) void sglkv_compact_tokens_v16(sglkv_evict_params p) {
    evt_compact_body<sglkv_v4u>(p);
}
extern "C" __global__ __launch_bounds__(SGLKV_COMPACT_THREADS) void sglkv_compact_tokens_v4(sglkv_evict_params p) {
    evt_compact_body<uint32_t>(p);
}
extern "C" __global__ __launch_bounds__(SGLKV_COMPACT_THREADS) void sglkv_compact_tokens_v2(sglkv_evict_params p) {
    evt_compact_body<uint16_t>(p);
}
extern "C" __global__ __launch_bounds__(SGLKV_COMPACT_THREADS) void sglkv_compact_tokens_v1(sglkv_evict_params p) {
    evt_compact_body<uint8_t>(p);
}
