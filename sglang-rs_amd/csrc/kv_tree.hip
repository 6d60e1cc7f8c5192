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

// Any head dims, page size and alignment (32 requests of 300 to 8,192 tokens whose
// rows the tiles could read: 2,254 us, in tiles 147): a wave to 16 query heads and
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

// ---- Tiles: head dims 64, 128 or 256 on 16-byte rows --------------------------
//
// A workgroup of four waves owns a tile: up to 32 RW (query, head) rows of one
// request and KV head. RW (times SHARE) waves make a token group, which computes
// 32 RW rows over blocks of B tokens; the 4 / (RW SHARE) groups of a workgroup take
// the blocks in turn and join their outputs through LDS at the end, so that small
// trees, which are bound by the rows' bytes, keep every wave busy.
//
// One pass: s = K q^T and o^T += V^T p^T on 32x32x16 products, whose layouts leave
// a row's scores in one lane pair, so that the running maximum and sum stay in
// registers; rows go straight to LDS a block ahead. The weights enter as hi + lo
// bf16 pairs, which costs half as many products again and 6 vector instructions a
// pair of weights. Measured with 32 query heads on 8 KV heads of 128 dims:
// - 32 requests of 300 to 8,192 tokens with up to 24 drafts: 147 us, 4.0 TB/s of
//   rows, bound by waits for them and by how evenly splits fall on workgroups;
// - 6 of 9,000 to 32,768 with up to 120: 377 to 401 us, 534 to 568 TFLOP/s not
//   counting the lo halves, bound by vector and matrix instructions, which follow
//   each other in a wave (the matrix pipes are busy 41 % of the time);
// - one of 2,048 with 16: 16.7 us, of which the merge's launch takes 4 and what a
//   workgroup does before its first block and behind its last 7.

template <uint32_t D, uint32_t RW>
struct tree_tl {
    typedef attn_tl<D> A;                                 // the swizzles of a row's pieces
    static constexpr uint32_t ROW = 2 * D;                // bytes of one token's head slice
    static constexpr uint32_t PIECES = D / 8;             // 16-byte pieces per row
    static constexpr uint32_t TPL = 1024 / ROW;           // tokens per load
    static constexpr uint32_t SHARE = D > 128 ? 2 : 1;    // waves that share 32 rows, each with D / SHARE outputs
    static constexpr uint32_t GW = RW * SHARE;            // waves of a token group
    static constexpr uint32_t TW = 4 / GW;                // token groups
    static constexpr uint32_t B = SGLKV_TREE_BLOCK(D, RW);
    static constexpr uint32_t N = B / GW;                 // tokens of a block that a wave loads
    static constexpr uint32_t LPW = N / TPL;              // its K loads (and V loads)
    static constexpr uint32_t V = B * ROW;                // V rows' offset in a stage
    static constexpr uint32_t STAGE = 2 * V;
    static constexpr uint32_t KC = D / 16;                // q.k steps
    static constexpr uint32_t NT = D / SHARE / 32;        // 32-dim output tiles of a wave
    static constexpr uint32_t TB = B / 32;                // 32-token score tiles
    static constexpr uint32_t AHEAD = 4;                  // products that the K reads run ahead
    static constexpr uint32_t OWN = 16 * NT / TW;         // outputs of a lane after the groups are joined
    static constexpr uint32_t RING = 2 * TW * STAGE;      // 256 bytes of raw slots for each wave and stage
    static constexpr uint32_t UNION = RING + 2048;        // which drafts the tile attends at all
    static constexpr uint32_t WORDS = UNION + 8 * (SGLKV_TREE_MAX_WORDS + 2);  // four words for each wave, and eight held
    static constexpr uint32_t TABLE = WORDS + 96;         // each wave's rows (tree_row)
    static constexpr uint32_t VBUF = D > 128 && TW == 1 ? 1 : 2;  // steps whose values there are registers for
    static_assert(TABLE + 4096 == SGLKV_TREE_LDS_BYTES(D, RW), "the host sizes the same LDS");
    static_assert(N <= 32 && LPW * TPL == N && TW * GW == 4 && OWN * TW == 16 * NT && OWN % 4 == 0, "whole loads and shares");
    static_assert(4 * 16 * NT * 256 <= RING, "the outputs are joined in the stages");
};

// One wave's slots of a block: the low words of tokens [0, N) and then the high
// ones (lane l: token l % N, word l / N % 2), without registers: into the ring,
// 256 bytes at `at`.
__device__ __forceinline__ void tree_load_slots(uint64_t address, uint32_t at) {
    uint32_t save;
    asm volatile(
        "s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %2, off\n\ts_mov_b32 m0, %0"
        : "=&s"(save)
        : "s"(at), "v"(address)
        : "memory");
}
// A wave's slots of the block from token `tb` on; `base`: the request's first slot
// and the lane's word of it.
template <uint32_t D, uint32_t RW>
__device__ __forceinline__ void tree_slots(uint64_t base, uint32_t last, uint32_t tb, uint32_t gw, uint32_t lane, uint32_t at) {
    typedef tree_tl<D, RW> T;
    const uint32_t tok = tb + T::N * gw + lane % T::N;
    tree_load_slots(base + 8ull * (tok < last ? tok : last), at);
}
template <uint32_t COUNT>
__device__ __forceinline__ void tree_wait() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(COUNT) : "memory");
}
template <uint32_t LPW>
__device__ __forceinline__ void tree_load_rows(const uint64_t *a, uint32_t at) {
    if constexpr (LPW == 8) {
        attn_tile_load4(a, at);
        attn_tile_load4(a + 4, at + 4096);
    } else if constexpr (LPW == 4) {
        attn_tile_load4(a, at);
    } else {
        static_assert(LPW == 2, "two, four or eight loads");
        attn_tile_load2(a, at);
    }
}

// The kernel's parameters, read again by whoever asks (as attn_tile_params).
__device__ __forceinline__ const sglkv_tree_params &tree_params() {
    typedef const __attribute__((address_space(4))) sglkv_tree_params kernarg;
    kernarg *k = (kernarg *)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(k));
    return *(const sglkv_tree_params *)k;
}

// Every line of them on its way into the scalar cache at once, where the first use
// of each would wait for memory by itself.
__device__ __forceinline__ void tree_touch() {
    uint32_t x[6];
    static_assert(sizeof(sglkv_tree_params) > 320 && sizeof(sglkv_tree_params) <= 384, "six lines of 64 bytes");
    asm volatile(
        "s_load_dword %0, %6, 0\n\ts_load_dword %1, %6, 64\n\ts_load_dword %2, %6, 128\n\ts_load_dword %3, %6, 192\n\t"
        "s_load_dword %4, %6, 256\n\ts_load_dword %5, %6, 320\n\ts_waitcnt lgkmcnt(0)"
        : "=&s"(x[0]), "=&s"(x[1]), "=&s"(x[2]), "=&s"(x[3]), "=&s"(x[4]), "=&s"(x[5])
        : "s"(__builtin_amdgcn_kernarg_segment_ptr()));
}

// What a pass over the tile's tokens needs: [t0, t1) of the request, all tokens
// below `common` attended by every row, those below `whole` by some row whole.
struct tree_pass {
    uint64_t start;
    uint32_t t0, t1, last;  // last: the request's last slot
    uint32_t common, whole;
};

// A row of the tile, kept in LDS: the loop has no registers for what it needs at
// its last blocks alone. Its mask's first two words, what it attends whole, how far
// it reaches (0: no row, or one that attends nothing), its query and that's number
// in the tile.
struct tree_row {
    uint64_t low, high;
    uint32_t context, reach, query, number;
};
static_assert(sizeof(tree_row) == 32, "32 rows a wave in a KiB");
__device__ __forceinline__ uint64_t tree_word(const tree_row &r, uint32_t i) {
    uint64_t w = i == 0 ? r.low : i == 1 ? r.high : 0;
    if (i >= 2) {
        const sglkv_tree_params &p = tree_params();
        if (i < p.mask_words) w = p.masks[static_cast<uint64_t>(r.query) * p.mask_words + i];
    }
    return w;
}
// The 64 bits of the row's mask from bit `at` on.
__device__ __forceinline__ uint64_t tree_bits(const tree_row &r, uint32_t at) {
    const uint32_t i = at >> 6, s = at & 63;
    const uint64_t a = tree_word(r, i);
    return s == 0 ? a : a >> s | tree_word(r, i + 1) << (64 - s);
}

template <uint32_t D, uint32_t RW>
struct tree_state {
    float m_run, l_part;               // row l % 32 (both half-waves hold the same m; l is this half's share)
    sglkv_f32x16 o[tree_tl<D, RW>::NT];  // o[n][i]: dim 32n + 8(i/4) + 4(l/32) + i%4 of the wave's dims of the row
};

// x of lane J of each PIECES lanes.
template <uint32_t PIECES, uint32_t J>
__device__ __forceinline__ uint64_t tree_of_lane(uint64_t x) {
    uint32_t half[2];
#pragma unroll
    for (uint32_t e = 0; e < 2; ++e) {
        const int v = static_cast<int>(x >> (32 * e));
        if constexpr (PIECES < 16) half[e] = __builtin_amdgcn_ds_swizzle(v, (J << 5) | (32 - PIECES));
        else half[e] = __builtin_amdgcn_update_dpp(v, v, 0x150 + J, 0xF, 0xF, false);  // (row_newbcast: within 16 lanes)
    }
    return static_cast<uint64_t>(half[1]) << 32 | half[0];
}
template <uint32_t N, typename F, uint32_t J = 0>
__device__ __forceinline__ void tree_each(F &f) {
    f(std::integral_constant<uint32_t, J>());
    if constexpr (J + 1 < N) tree_each<N, F, J + 1>(f);
}

// A wave's share of a block's rows into its group's stage, from the slots in its
// ring. A token that no row attends, or whose slot is outside the pool, reads the
// zero row.
template <uint32_t D, uint32_t RW>
__device__ __forceinline__ void tree_issue(const sglkv_attn_params &held, const tree_pass &pass, uint64_t kbase, uint64_t vbase,
                                           const uint32_t *ring, const uint64_t *seen, uint32_t tb, uint32_t gw, uint32_t lane,
                                           uint32_t stage_at) {
    typedef tree_tl<D, RW> T;
    const sglkv_attn_params &p = D > 64 ? tree_params().a : held;  // (no scalar registers left to hold them)
    if (D > 64) asm volatile("" : "+v"(lane));  // (what it computes from the lane is not held across the block)
    static_assert((T::LPW & (T::LPW - 1)) == 0 && T::LPW <= T::PIECES && T::LPW <= 16, "a lane for each load of a token's lanes");
    // Load j of a token's PIECES lanes reads the place that lane j of them has worked out.
    const uint32_t c = lane / T::PIECES, pos = lane % T::PIECES, own = T::TPL * (pos % T::LPW) + c;
    uint32_t low = ring[own];
    const uint32_t high = ring[T::N + own], tok = tb + T::N * gw + own;
    bool ok = true;
    if (!(tb + T::B <= pass.t1 && tb + T::B <= pass.whole)) {
        const uint32_t place = tok - pass.whole;
        ok = tok < pass.t1 && (tok < pass.whole || (place < 64 * SGLKV_TREE_MAX_WORDS && (seen[place >> 6] >> (place & 63)) & 1));
    }
    if (ok && (high != 0 || low >= static_cast<uint32_t>(p.slot_count))) {  // (host: below 2^32)
        atomicOr(tree_params().a.flag, SGLKV_FLAG_ATTN_SLOT);
        ok = false;
    }
    low = ok ? low : 0u;
    // K and V share the token's offset (the host's rule, as for paged attention's tiles).
    const uint64_t off = static_cast<uint64_t>(low >> p.page_shift) * p.page_stride32 +
                         __umul24(low & ((1u << p.page_shift) - 1), p.key_token_stride32);
    const uint64_t zero = reinterpret_cast<uint64_t>(p.zero_row);
    uint64_t kat, vat, ka[T::LPW], va[T::LPW];
    attn_sel64x2(ok, kbase + off, vbase + off, zero, kat, vat);
    auto each = [&](auto j) {
        const uint32_t t = T::N * gw + T::TPL * j() + c;
        ka[j()] = tree_of_lane<T::PIECES, j()>(kat) + 16 * (pos ^ T::A::kswz(t));
        va[j()] = tree_of_lane<T::PIECES, j()>(vat) + 16 * (pos ^ T::A::vswz(t));
    };
    tree_each<T::LPW>(each);
    const uint32_t at = stage_at + 1024 * T::LPW * gw;
    tree_load_rows<T::LPW>(ka, at);
    tree_load_rows<T::LPW>(va, at + T::V);
}

// One block from its stage: scores, softmax, o += p.v, as paged attention's tiles
// compute it (attn_tile_block). masked: `bits` says which of the block's tokens
// the lane's row attends.
template <uint32_t D, uint32_t RW>
__device__ __forceinline__ void tree_block(const sglkv_attn_params &p, const uint8_t *st_lds,
                                           const sglkv_u16x8 (&qf)[tree_tl<D, RW>::KC], uint64_t bits, bool masked, uint32_t lane,
                                           uint32_t part, tree_state<D, RW> &st) {
    typedef tree_tl<D, RW> T;
    const uint32_t t = lane & 31, h = lane >> 5;
    sglkv_f32x16 s[T::TB];
#pragma unroll
    for (uint32_t b = 0; b < T::TB; ++b) s[b] = sglkv_f32x16{};
    auto kread = [&](uint32_t i) {
        return *reinterpret_cast<const sglkv_u16x8 *>(st_lds + T::ROW * (32 * (i % T::TB) + t) +
                                                      16 * ((2 * (i / T::TB) + h) ^ T::A::kswz(t)));
    };
    __builtin_amdgcn_s_setprio(1);
    sglkv_u16x8 kf[T::AHEAD];
#pragma unroll
    for (uint32_t i = 0; i < T::AHEAD; ++i) kf[i] = kread(i);
#pragma unroll
    for (uint32_t i = 0; i < T::KC * T::TB; ++i) {
        __builtin_amdgcn_sched_barrier(0);
        const sglkv_u16x8 a = kf[i % T::AHEAD];
        s[i % T::TB] = attn_mfma32(a, qf[i / T::TB], s[i % T::TB]);
        if (i + T::AHEAD < T::KC * T::TB) kf[i % T::AHEAD] = kread(i + T::AHEAD);
    }
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(0);
    if (masked) {
        // Bitwise selects: a bit's sign extension keeps the score or makes it -inf.
        const uint64_t own = bits >> (4 * h);
#pragma unroll
        for (uint32_t b = 0; b < T::TB; ++b) {
            const uint32_t half = static_cast<uint32_t>(b ? own >> 32 : own);
#pragma unroll
            for (uint32_t i = 0; i < 16; ++i) {
                const uint32_t keep = static_cast<uint32_t>(__builtin_amdgcn_sbfe(static_cast<int32_t>(half), 8 * (i >> 2) + (i & 3), 1));
                s[b][i] = __uint_as_float((__float_as_uint(s[b][i]) & keep) | (0xFF800000u & ~keep));
            }
        }
    }
    float mx = s[0][0];
#pragma unroll
    for (uint32_t b = 0; b < T::TB; ++b)
#pragma unroll
        for (uint32_t i = 0; i < 16; i += 2) mx = attn_max3(mx, s[b][i], s[b][i + 1]);
    mx = fmaxf(mx, attn_xor32(mx)) * p.scale_log2;
    if (__builtin_amdgcn_readfirstlane(__ballot(mx > st.m_run + 8.0f) != 0 ? 1u : 0u)) {
        const float m_new = fmaxf(st.m_run, mx);
        const float alpha = exp2f(st.m_run - m_new);
        st.l_part *= alpha;
        st.m_run = m_new;
#pragma unroll
        for (uint32_t n = 0; n < T::NT; ++n)
#pragma unroll
            for (uint32_t i = 0; i < 16; ++i) st.o[n][i] *= alpha;
    }
    // V^T operand of 32-dim tile n, 16-token step `step`: tokens 16 step +
    // 4h + L/4 and + 8 (the same vswz), dims 32n + 16c + 4(L%4).
    const uint32_t L = lane & 15, c = (lane >> 4) & 1, t0 = 4 * h + (L >> 2);
    auto vread = [&](uint32_t n, uint32_t step) {
        const uint32_t pc = (4 * (T::NT * part + n) + 2 * c + ((L & 3) >> 1)) ^ T::A::vswz(t0);
        const uint8_t *at = st_lds + T::V + T::ROW * (16 * step + t0) + 16 * pc + 8 * (L & 1);
        const attn_i16x4 lo = attn_lat_vtr(at), hi = attn_lat_vtr(at + 8 * T::ROW);
        return sglkv_u16x8{(uint16_t)lo[0], (uint16_t)lo[1], (uint16_t)lo[2], (uint16_t)lo[3],
                           (uint16_t)hi[0], (uint16_t)hi[1], (uint16_t)hi[2], (uint16_t)hi[3]};
    };
    float psum = 0.0f;
    auto weights = [&](uint32_t step, sglkv_u16x8 &phi, sglkv_u16x8 &plo) {
        attn_u32x4 hi, lo;
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            const uint32_t e = 8 * (step & 1) + 2 * i;
            const float a = __builtin_amdgcn_exp2f(__builtin_fmaf(s[step >> 1][e], p.scale_log2, -st.m_run));
            const float b = __builtin_amdgcn_exp2f(__builtin_fmaf(s[step >> 1][e + 1], p.scale_log2, -st.m_run));
            psum += a;
            psum += b;
            hi[i] = attn_pack_bf16(a, b);
            lo[i] = attn_pack_bf16(a - __uint_as_float(hi[i] << 16), b - __uint_as_float(hi[i] & 0xFFFF0000u));
        }
        phi = __builtin_bit_cast(sglkv_u16x8, hi);
        plo = __builtin_bit_cast(sglkv_u16x8, lo);
    };
    sglkv_u16x8 phi[2], plo[2], v[T::VBUF][T::NT];
    if (T::VBUF == 2) {
#pragma unroll
        for (uint32_t n = 0; n < T::NT; ++n) v[0][n] = vread(n, 0);
    }
    weights(0, phi[0], plo[0]);
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (uint32_t step = 0; step < 2 * T::TB; ++step) {
        const uint32_t x = step & 1;
        __builtin_amdgcn_sched_barrier(0);
        if (T::VBUF == 1 || step + 1 < 2 * T::TB) {
#pragma unroll
            for (uint32_t n = 0; n < T::NT; ++n) v[(x + 1) % T::VBUF][n] = vread(n, T::VBUF == 2 ? step + 1 : step);
        }
#pragma unroll
        for (uint32_t n = 0; n < T::NT; ++n) st.o[n] = attn_mfma32(v[x % T::VBUF][n], phi[x], st.o[n]);
#pragma unroll
        for (uint32_t n = 0; n < T::NT; ++n) st.o[n] = attn_mfma32(v[x % T::VBUF][n], plo[x], st.o[n]);
        if (step + 1 < 2 * T::TB) {
            weights(step + 1, phi[x ^ 1], plo[x ^ 1]);
#pragma unroll
            for (uint32_t n = 0; n < 2 * T::NT; ++n) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);                      // a product
                __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);                      // an LDS read
                __builtin_amdgcn_sched_group_barrier(0x402, T::NT == 4 ? 6 : 16, 0);  // vector and exp instructions
            }
        }
    }
    __builtin_amdgcn_s_setprio(0);
    st.l_part += psum;
}

// Tokens [t0, t1) of the tile's request for the wave's 32 rows: `reach` bounds
// them, `least` is the fewest tokens that one of them attends whole.
template <uint32_t D, uint32_t RW>
__device__ __forceinline__ void tree_run(const sglkv_tree_params &p, const tree_pass &pass, uint64_t kbase, uint64_t vbase,
                                         uint32_t w, uint32_t lane, uint8_t *lds, uint32_t lds_at, uint32_t least,
                                         uint32_t reach,
                                         const sglkv_u16x8 (&qf)[tree_tl<D, RW>::KC], tree_state<D, RW> &st) {
    typedef tree_tl<D, RW> T;
    const sglkv_attn_params &a = p.a;
    const uint32_t tw = w / T::GW, gw = w % T::GW;
    const uint64_t *seen = reinterpret_cast<const uint64_t *>(lds + T::UNION);
    const uint64_t slot_base = reinterpret_cast<uint64_t>(a.sequence_slots + pass.start) + 4 * (lane / T::N % 2);
    const uint32_t stage_at = lds_at + 2 * T::STAGE * tw, ring_at = lds_at + T::RING + 512 * w;
    const uint8_t *stage = lds + 2 * T::STAGE * tw;
    const uint32_t *ring = reinterpret_cast<const uint32_t *>(lds + T::RING + 512 * w);
    const uint32_t all = (pass.t1 - pass.t0 + T::B - 1) / T::B;
    // Blocks of each group (a group short of one loads zeros), and those that this wave's rows attend.
    const uint32_t nb = (all + T::TW - 1) / T::TW;
    const uint32_t first = pass.t0 + tw * T::B;
    const uint32_t end = reach < pass.t1 ? reach : pass.t1;
    const uint32_t mine = end <= first ? 0 : (end - first + T::B * T::TW - 1) / (T::B * T::TW);
    auto block = [&](uint32_t k) { return first + k * T::B * T::TW; };
    auto slots = [&](uint32_t k) { tree_slots<D, RW>(slot_base, pass.last, block(k), gw, lane, ring_at + 256 * (k & 1)); };
    auto rows = [&](uint32_t k) {
        tree_issue<D, RW>(a, pass, kbase, vbase, ring + 64 * (k & 1), seen, block(k), gw, lane, stage_at + T::STAGE * (k & 1));
    };
    st.m_run = -3.402823466e+38f;
    st.l_part = 0.0f;
#pragma unroll
    for (uint32_t n = 0; n < T::NT; ++n) st.o[n] = sglkv_f32x16{};
    // The first two blocks' slots have arrived (the caller's tree_slots), and everything that the compiler loaded: it
    // puts no wait into the loop, where rows are in flight.
    __builtin_amdgcn_s_waitcnt(0x0F70);
    rows(0);
    slots(2);
    rows(1);
    tree_wait<2 * T::LPW + 1>();  // block 0's rows have landed; block 1's are on their way
    if constexpr (T::GW > 1) asm volatile("s_barrier" ::: "memory");
    for (uint32_t k = 0;;) {
        if (k < mine) {
            const uint32_t tb = block(k);
            const bool masked = tb + T::B > least;
            uint64_t bits = 0;
            if (masked) {
                const tree_row &row = reinterpret_cast<const tree_row *>(lds + T::TABLE)[32 * w + (lane & 31)];
                if (tb >= row.context) {
                    bits = tree_bits(row, tb - row.context);
                } else {
                    const uint32_t left = row.context - tb;
                    bits = left >= 64 ? ~0ull : ((1ull << left) - 1) | row.low << left;
                }
            }
            tree_block<D, RW>(a, stage + T::STAGE * (k & 1), qf, bits, masked, lane, gw % T::SHARE, st);
        }
        if (++k >= nb) break;
        if constexpr (T::GW == 1) {
            // The wave's own stages: the slots of k + 1 are older than the rows of k.
            tree_wait<2 * T::LPW>();
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // block k - 1's stage is read
            slots(k + 2);
            rows(k + 1);
            tree_wait<2 * T::LPW + 1>();
        } else {
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
            slots(k + 2);
            rows(k + 1);
        }
    }
    tree_wait<0>();  // (rows behind the last block, too)
}

// The first query of the launch whose request index is at least x[0], and x[1]:
// each step, the wave's lanes look at 64 places of what is left.
__device__ __forceinline__ void tree_find(const sglkv_attn_params &a, uint32_t lane, uint32_t request, uint32_t *first, uint32_t *end) {
    const uint32_t count = static_cast<uint32_t>(a.query_count);  // (host: below 2^31)
    uint32_t lo[2] = {0, 0}, hi[2] = {count, count};
    while (lo[0] < hi[0] || lo[1] < hi[1]) {
#pragma unroll
        for (uint32_t x = 0; x < 2; ++x) {
            const uint32_t step = (hi[x] - lo[x] + 63) / 64, at = lo[x] + lane * step;
            const bool in = step && at < hi[x];
            const uint32_t v = in ? a.query_request_indices[at] : 0xFFFFFFFFu;
            const uint32_t c = __popcll(__ballot(in && v < request + x));
            hi[x] = lo[x] + c * step < hi[x] ? lo[x] + c * step : hi[x];
            if (c) lo[x] += (c - 1) * step + 1;
        }
    }
    *first = lo[0];
    *end = lo[1] > lo[0] ? lo[1] : lo[0];
}

// x joined over 32 lanes whose halves of the wave are alike.
template <typename F>
__device__ __forceinline__ uint32_t tree_join(uint32_t x, F join) {
    x = join(x, sel_join<1>(x));
    x = join(x, sel_join<2>(x));
    x = join(x, sel_join<4>(x));
    x = join(x, sel_join<8>(x));
    return __builtin_amdgcn_readfirstlane(join(x, sel_join<16>(x)));
}
__device__ __forceinline__ uint32_t tree_most(uint32_t x) {
    return tree_join(x, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
}

__device__ __forceinline__ uint32_t tree_any(uint32_t x) {
    return tree_join(x, [](uint32_t a, uint32_t b) { return a | b; });
}

// The sum of x over the lanes up to this one.
__device__ __forceinline__ uint32_t tree_upto(uint32_t x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, false);  // (row_shr: within 16 lanes)
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);  // (the last lane of 16 to the next 16)
    return x + __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);  // (lane 31 to the upper half)
}

// ---- A launch's tiles ----
//
// Request r has T_r tiles of its queries and n_r tokens, cut into ceil(n_r / c) even
// splits, with the smallest c (whole units: a block for each token group) that leaves
// at most as many (request, split, tile)s as w times the workgroups resident at once.
// w is the least that holds the tiles, or one more where there are tiles for half the
// workgroups and the longer way takes less, at 10 blocks for what a workgroup does
// before its first and the mean share and half a split in place of a split where they
// follow each other (64 requests of 300 to 4,096 tokens with up to 12 drafts: 161 us
// with w = 1, 148 with 2; 30 of 300 to 2,000 with up to 120: 124 and 147). The host
// does not know the lengths. They are numbered without a gap, since a workgroup that
// finds nothing to do holds its place until the ones before it on its CU are done:
// 32 requests of 300 to 8,192 tokens took 265 us with every other workgroup empty,
// 163 us without; with half as many pairs 209, with twice 167.
// A request of one split has its outputs from there; the others' are merged.
// Each workgroup finds c and its own place, a lane to a request. Past
// SGLKV_TREE_BALANCED requests or SGLKV_TREE_LISTED queries c is the host's, and
// tiles beyond the average request's are taken by the same workgroups.

// The tokens of a request with slots [s, e) that the launch can reach (at most max_length).
__device__ __forceinline__ uint32_t tree_tokens(const sglkv_tree_params &p, uint64_t s, uint64_t e) {
    const uint64_t n = s <= e && e <= p.a.sequence_slot_count ? e - s : 0;
    return static_cast<uint32_t>(n < p.max_length ? n : p.max_length);
}
__device__ __forceinline__ uint32_t tree_splits(uint32_t n, uint32_t c) { return n > c ? (n + c - 1) / c : 1; }
// Tokens of a split of a request of n tokens.
__device__ __forceinline__ uint32_t tree_chunk(const sglkv_tree_params &p, uint32_t n, uint32_t c) {
    const uint32_t k = tree_splits(n, c);
    return ((n + k - 1) / k + p.unit - 1) / p.unit * p.unit;
}

// A workgroup's place: its request's queries [first, end) from tile `tile` on, every
// tile_step-th, and the split (alone: there is one, whose outputs need no merge).
// Queries [loose, loose_end) belong to no request.
struct tree_place {
    uint32_t request, split, chunk, first, end, tile, tile_step, loose, loose_end, alone;
};

// Where each request's queries begin and end, in LDS (the last entry: those of no
// request), and whether the indices ever fall.
__device__ __forceinline__ void tree_list(const sglkv_attn_params &a, uint32_t tid, uint32_t *begins, uint32_t *ends) {
    const uint32_t count = static_cast<uint32_t>(a.query_count), requests = static_cast<uint32_t>(a.request_count);
    constexpr uint32_t U = 4;
    uint32_t x[U], y[U];
    auto load = [&](uint32_t i0) {
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) {
            const uint32_t at = i0 + 256 * u + tid, i = at < count ? at : count - 1;
            x[u] = a.query_request_indices[i];
            y[u] = a.query_request_indices[i ? i - 1 : 0];
        }
    };
    load(0);  // (on their way over the barrier)
    if (tid <= requests) begins[tid] = ends[tid] = 0;
    __syncthreads();
    for (uint32_t i0 = 0; i0 < count;) {
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) {
            const uint32_t i = i0 + 256 * u + tid, own = x[u] < requests ? x[u] : requests, before = y[u] < requests ? y[u] : requests;
            if (i >= count) continue;
            if (i == 0 || own != before) {
                begins[own] = i;
                if (i) ends[before] = i;
            }
            if (i + 1 == count) ends[own] = count;
            if (y[u] > x[u] && blockIdx.x == 0) atomicOr(a.flag, SGLKV_FLAG_ATTN_REQUEST);
        }
        i0 += 256 * U;
        if (i0 < count) load(i0);
    }
    __syncthreads();
}

// False: no (request, split, tile) has this number. (Loose queries are there all the same.)
__device__ __forceinline__ bool tree_balance(const sglkv_tree_params &p, uint32_t number, uint32_t tid, uint32_t lane,
                                             uint32_t *begins, tree_place *at) {
    const sglkv_attn_params &a = p.a;
    uint32_t *const ends = begins + SGLKV_TREE_BALANCED + 1;
    const uint32_t requests = static_cast<uint32_t>(a.request_count), unit = p.unit;
    const uint64_t *const range = a.request_slot_offsets + (lane < requests ? lane : requests - 1);
    const uint64_t from = range[0], to = range[1];
    tree_list(a, tid, begins, ends);
    const uint32_t n = lane < requests ? tree_tokens(p, from, to) : 0;
    auto sum = [](uint32_t x) {
        x += sel_join<1>(x);
        x += sel_join<2>(x);
        x += sel_join<4>(x);
        x += sel_join<8>(x);
        x += sel_join<16>(x);
        return static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(x + sel_join<32>(x)));
    };
    const uint32_t first = lane < requests ? begins[lane] : 0, end = lane < requests ? ends[lane] : 0;
    const uint32_t tiles = end > first ? (end - first + p.tile_queries - 1) / p.tile_queries : 0;
    at->loose = __builtin_amdgcn_readfirstlane(begins[requests]);
    at->loose_end = __builtin_amdgcn_readfirstlane(ends[requests]);
    const uint32_t all_tiles = sum(tiles), fills = all_tiles > p.pairs ? (all_tiles + p.pairs - 1) / p.pairs : 1;
    float work = static_cast<float>(tiles) * static_cast<float>(n);
    work += __uint_as_float(sel_join<1>(__float_as_uint(work)));
    work += __uint_as_float(sel_join<2>(__float_as_uint(work)));
    work += __uint_as_float(sel_join<4>(__float_as_uint(work)));
    work += __uint_as_float(sel_join<8>(__float_as_uint(work)));
    work += __uint_as_float(sel_join<16>(__float_as_uint(work)));
    work += __uint_as_float(sel_join<32>(__float_as_uint(work)));
    uint32_t most = n;
    most = most > sel_join<32>(most) ? most : sel_join<32>(most);
    most = tree_most(most);
    const uint32_t by_records = ((most + a.splits - 1) / a.splits) / unit + 1;
    const uint32_t share = static_cast<uint32_t>(work / static_cast<float>(p.pairs)) / unit;
    uint32_t c = 0, own = 0;
    for (uint32_t w = fills, best = 0xFFFFFFFFu; w <= (2 * all_tiles > p.pairs ? fills + 1 : fills); ++w) {
        // From what an even share would be, in steps of a sixteenth.
        uint32_t d = share / w + 1, count;
        d = d > by_records ? d : by_records;
        d = d > p.least ? d : p.least;
        for (;; d += d / 16 + 1) {
            count = tiles * tree_splits(n, d * unit);
            if (sum(count) <= p.pairs * w) break;  // (at d past the longest request: the tiles alone)
        }
        const uint32_t cost = (w == 1 ? d : share + d / 2) + 10 * w;
        if (cost < best) {
            best = cost;
            c = d;
            own = count;
        }
    }
    c *= unit;
    const uint32_t upto = tree_upto(own);
    const uint64_t here = __ballot(number < upto);
    if (!here) return false;
    const uint32_t l = __builtin_ctzll(here), within = number - __builtin_amdgcn_readlane(upto - own, l);
    const uint32_t of = __builtin_amdgcn_readlane(tiles, l);
    at->request = l;
    at->split = within / of;
    at->tile = within - at->split * of;
    at->tile_step = 1u << 30;  // (one tile each)
    at->first = __builtin_amdgcn_readlane(first, l);
    at->end = __builtin_amdgcn_readlane(end, l);
    at->chunk = tree_chunk(p, __builtin_amdgcn_readlane(n, l), c);
    at->alone = __builtin_amdgcn_readlane(n, l) <= c;
    return true;
}

// The same where there are too many for that.
__device__ __forceinline__ bool tree_number(const sglkv_tree_params &p, uint32_t number, uint32_t tid, uint32_t lane, tree_place *at) {
    const sglkv_attn_params &a = p.a;
    const uint32_t requests = static_cast<uint32_t>(a.request_count), of_slot = requests * a.splits, count = static_cast<uint32_t>(a.query_count);
    const uint32_t slot = number / of_slot, u = number - slot * of_slot, every = gridDim.x / a.kv_heads;
    // The workgroup's share of the check that the indices never fall.
    if (blockIdx.x % a.kv_heads == 0)
        for (uint64_t q = static_cast<uint64_t>(number) * 256 + tid; q < count; q += static_cast<uint64_t>(every) * 256)
            if (q && a.query_request_indices[q - 1] > a.query_request_indices[q]) atomicOr(a.flag, SGLKV_FLAG_ATTN_REQUEST);
    tree_find(a, lane, requests, &at->loose, &at->loose_end);
    at->loose_end = count;
    if (slot >= p.tile_slots) return false;
    at->split = u / requests;
    at->request = u - at->split * requests;
    at->tile = slot;
    at->tile_step = p.tile_slots;
    const uint64_t *const range = a.request_slot_offsets + at->request;
    const uint32_t n = tree_tokens(p, range[0], range[1]), c = static_cast<uint32_t>(a.chunk_tokens);
    at->chunk = tree_chunk(p, n, c);
    at->alone = n <= c;
    tree_find(a, lane, at->request, &at->first, &at->end);
    return true;
}

// The lane's row number among the tile's and its head: worked out anew (the lane
// passes through an empty asm) rather than held across the loop.
template <uint32_t D, uint32_t RW>
__device__ __forceinline__ uint32_t tree_row_of(const sglkv_attn_params &a, uint32_t w, uint32_t lane, uint32_t *head) {
    typedef tree_tl<D, RW> T;
    asm volatile("" : "+v"(lane));
    const uint32_t r = 32 * (w % T::GW / T::SHARE) + (lane & 31), number = r / a.group;
    *head = r - number * a.group;
    return number;
}

// The rows' outputs (one split) or records, the token groups joined; rows that do
// not reach past t0, or whose query is not number `only` (if any), write nothing.
template <uint32_t D, uint32_t RW>
__device__ __forceinline__ void tree_write(uint32_t w, uint32_t lane, uint8_t *lds, uint32_t kvh, uint32_t split, uint32_t t0,
                                           uint32_t only, const tree_state<D, RW> &st) {
    typedef tree_tl<D, RW> T;
    const sglkv_attn_params &a = tree_params().a;
    const uint32_t tw = w / T::GW, gw = w % T::GW, part = gw % T::SHARE;
    float l = st.l_part + __shfl_xor(st.l_part, 32), m = st.m_run;
    float v[T::OWN];
    if constexpr (T::TW > 1) {
        // The groups' statistics, then their outputs, at one maximum.
        float2 *ml = reinterpret_cast<float2 *>(lds + T::RING);
        float *outs = reinterpret_cast<float *>(lds);
        __syncthreads();  // (the stages and rings are no longer read)
        if (lane < 32) ml[32 * w + lane] = make_float2(m, l);
        __syncthreads();
        float top = m, sum = 0.0f;
        float2 group[T::TW];
#pragma unroll
        for (uint32_t g = 0; g < T::TW; ++g) {
            group[g] = ml[32 * (T::GW * g + gw) + (lane & 31)];
            top = fmaxf(top, group[g].x);
        }
#pragma unroll
        for (uint32_t g = 0; g < T::TW; ++g) sum += group[g].y * exp2f(group[g].x - top);
        const float scale = exp2f(m - top);
#pragma unroll
        for (uint32_t n = 0; n < T::NT; ++n)
#pragma unroll
            for (uint32_t i = 0; i < 16; ++i) outs[64 * (16 * (T::NT * w + n) + i) + lane] = st.o[n][i] * scale;
        __syncthreads();
#pragma unroll
        for (uint32_t i = 0; i < T::OWN; ++i) {
            v[i] = 0.0f;
#pragma unroll
            for (uint32_t g = 0; g < T::TW; ++g) v[i] += outs[64 * (16 * T::NT * (T::GW * g + gw) + T::OWN * tw + i) + lane];
        }
        m = top;
        l = sum;
    } else {
#pragma unroll
        for (uint32_t i = 0; i < T::OWN; ++i) v[i] = st.o[i / 16][i % 16];
    }
    uint32_t rh;
    const uint32_t number = tree_row_of<D, RW>(a, w, lane, &rh);
    const tree_row &row = reinterpret_cast<const tree_row *>(lds + T::TABLE)[32 * w + (lane & 31)];
    if (row.reach <= t0 || (only != 0xFFFFFFFFu && number != only)) return;
    const uint64_t qrow = static_cast<uint64_t>(row.query) * a.query_heads + kvh * a.group + rh;
    // Value 4 i + e of the lane: dim 8 (i + OWN tw / 4) + 4 (lane / 32) + e of the wave's dims.
    const uint32_t dim = D / T::SHARE * part + 2 * T::OWN * tw + 4 * (lane >> 5);
    if (__builtin_amdgcn_readfirstlane(reinterpret_cast<const uint32_t *>(lds + T::WORDS)[23])) {  // (its request is not split)
        const float linv = 1.0f / l;
        uint16_t *out = a.output + qrow * D + dim;
#pragma unroll
        for (uint32_t i = 0; i < T::OWN / 4; ++i) {
            sglkv_u16x4 x;
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) x[e] = attn_to_bf16(v[4 * i + e] * linv);
            *reinterpret_cast<sglkv_u16x4 *>(out + 8 * i) = x;  // (host: 8-byte aligned output)
        }
        return;
    }
    const uint64_t rec = qrow * a.splits + split;
    uint32_t wave = w;
    asm volatile("" : "+v"(lane), "+s"(wave));  // (no comparison of them held across the loops)
    if (lane < 32 && wave < T::GW && wave % T::SHARE == 0) {
        float *ml = attn_rec_ml(a, rec);
        ml[0] = m;
        ml[1] = l;
    }
    float *out = attn_rec_o(a, rec) + dim;
#pragma unroll
    for (uint32_t i = 0; i < T::OWN / 4; ++i)
        *reinterpret_cast<sglkv_f32x4 *>(out + 8 * i) = sglkv_f32x4{v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]};
}

// The first two blocks' slots of a wave, into its ring.
template <uint32_t D, uint32_t RW>
__device__ __forceinline__ void tree_first_slots(const sglkv_attn_params &a, uint64_t from, uint64_t to, uint32_t t0, uint32_t w,
                                                 uint32_t lane, uint32_t lds_at) {
    typedef tree_tl<D, RW> T;
    const uint64_t base = reinterpret_cast<uint64_t>(a.sequence_slots + from) + 4 * (lane / T::N % 2);
    const uint32_t last = static_cast<uint32_t>(to - from < 1ull << 31 ? to - from : 1ull << 31) - 1;
    const uint32_t tb = t0 + w / T::GW * T::B, at = lds_at + T::RING + 512 * w;
    tree_slots<D, RW>(base, last, tb, w % T::GW, lane, at);
    tree_slots<D, RW>(base, last, tb + T::B * T::TW, w % T::GW, lane, at + 256);
}

// The queries of no request: those that attend something are reported, and all give
// zeros (with several splits the merge writes them). Every workgroup takes a share.
__device__ __forceinline__ void tree_loose(uint32_t number, uint32_t kvh, uint32_t tid, uint32_t first, uint32_t end) {
    const sglkv_tree_params &p = tree_params();
    const sglkv_attn_params &a = p.a;
    for (uint32_t q = first + number; q < end; q += gridDim.x / a.kv_heads) {
        if (kvh == 0 && tid == 0) {
            uint64_t any = a.query_sequence_lengths[q];
            for (uint32_t i = 0; i < p.mask_words; ++i) any |= p.masks[static_cast<uint64_t>(q) * p.mask_words + i];
            if (any) atomicOr(a.flag, SGLKV_FLAG_ATTN_REQUEST);
        }
        if (kvh == 0 && tid == 0) p.used[q] = 0;
        if (a.splits > 1) continue;
        uint16_t *out = a.output + (static_cast<uint64_t>(q) * a.query_heads + kvh * a.group) * a.dv;
        for (uint32_t i = 4 * tid; i < a.group * a.dv; i += 1024) *reinterpret_cast<sglkv_u16x4 *>(out + i) = sglkv_u16x4{0, 0, 0, 0};
    }
}

template <uint32_t D, uint32_t RW>
__device__ __forceinline__ void tree_tile_body() {
    typedef tree_tl<D, RW> T;
    extern __shared__ __attribute__((aligned(16))) uint8_t tree_tile_lds[];
    tree_touch();
    const sglkv_tree_params &p = tree_params();
    const sglkv_attn_params &a = p.a;
    uint8_t *lds = tree_tile_lds;
    uint32_t *words = reinterpret_cast<uint32_t *>(lds + T::WORDS);
    uint64_t *seen = reinterpret_cast<uint64_t *>(lds + T::UNION);
    const uint32_t lds_at = attn_lat_lds_at(lds);
    const uint32_t tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    // The KV heads of a tile side by side, one to an XCD where there are eight.
    const uint32_t number = blockIdx.x / a.kv_heads, kvh = blockIdx.x - number * a.kv_heads;
    tree_place at = {};
    const bool any = __builtin_amdgcn_readfirstlane(p.balanced ? tree_balance(p, number, tid, lane, reinterpret_cast<uint32_t *>(lds), &at)
                                                               : tree_number(p, number, tid, lane, &at));
    __syncthreads();  // (the list is read: rows go there)
    if (at.loose < at.loose_end) tree_loose(number, kvh, tid, at.loose, at.loose_end);
    if (!any) return;
    auto uniform = [](uint32_t x) { return static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(x)); };
    const uint32_t req = uniform(at.request), split = uniform(at.split), chunk = uniform(at.chunk);
    const uint32_t t0 = split * chunk;
    words[19] = chunk;
    words[23] = uniform(at.alone);
    // Held in LDS, not in registers that the loops need; every wave writes them and reads its own.
    words[16] = uniform(at.end);
    words[17] = uniform(at.tile_step);
    for (uint32_t q0 = uniform(at.first + at.tile * p.tile_queries); q0 < uniform(words[16]);) {
        sglkv_u16x8 qf[T::KC];
        {
            // The lane's row: its query, head, mask and reach.
            const sglkv_tree_params &p = tree_params();
            const sglkv_attn_params &a = p.a;
            const uint32_t left = uniform(words[16]) - q0;
            const uint32_t nq = left < p.tile_queries ? left : p.tile_queries;
            words[18] = nq;
            const uint64_t *const range = a.request_slot_offsets + req;
            const uint64_t from = range[0], to = range[1];
            // The first two blocks' slots, on their way with what says which of them count.
            if (from < to && to <= a.sequence_slot_count) tree_first_slots<D, RW>(a, from, to, t0, w, lane, lds_at);
            // For the passes, which look at them where a row reaches into the range, so that it is one. (No slot behind
            // 2^31 is reached.)
            words[20] = static_cast<uint32_t>(from);
            words[21] = static_cast<uint32_t>(from >> 32);
            words[22] = static_cast<uint32_t>(to - from < 1ull << 31 ? to - from : 1ull << 31) - 1;
            if (tid < SGLKV_TREE_MAX_WORDS) seen[tid] = 0;
            uint32_t rh;
            tree_row row;
            row.number = tree_row_of<D, RW>(a, w, lane, &rh);
            const bool has = row.number < nq;
            row.query = q0 + (has ? row.number : 0);
            const uint64_t qrow = static_cast<uint64_t>(row.query) * a.query_heads + kvh * a.group + rh;
            const uint64_t *mask = p.masks + static_cast<uint64_t>(row.query) * p.mask_words;
            row.low = mask[0];
            row.high = p.mask_words > 1 ? mask[1] : 0;
            const uint64_t length = a.query_sequence_lengths[row.query];
            const uint32_t index = a.query_request_indices[row.query];
#pragma unroll
            for (uint32_t c = 0; c < T::KC; ++c)
                qf[c] = *reinterpret_cast<const sglkv_u16x8 *>(a.queries + qrow * D + 16 * c + 8 * (lane >> 5));
            uint32_t wave = w, own = split;
            asm volatile("" : "+s"(wave), "+s"(own));  // (no comparison of them held across the loops)
            uint32_t drafts = row.high ? 128 - __builtin_clzll(row.high) : row.low ? 64 - __builtin_clzll(row.low) : 0;
            for (uint32_t i = 2; i < p.mask_words; ++i) {
                const uint64_t m = mask[i];
                if (m) drafts = 64 * i + 64 - __builtin_clzll(m);
            }
            const bool any = has && (length != 0 || drafts != 0);
            uint32_t bad = 0;
            if (any) {
                if (index != req)
                    bad = SGLKV_FLAG_ATTN_REQUEST;
                else if (from > to || to > a.sequence_slot_count || length > to - from || length + drafts > to - from ||
                         length + drafts > p.max_length)
                    bad = SGLKV_FLAG_ATTN_SEQUENCE;
                if (bad && (own | kvh) == 0) atomicOr(a.flag, bad);
            }
            const bool live = any && !bad;
            // What the merge needs to know of each query: its records, or that its outputs are there.
            if (has && rh == 0 && (own | kvh) == 0 && wave < T::GW)
                tree_params().used[row.query] = uniform(words[23]) ? SGLKV_SELECT_NONE
                                    : live             ? (static_cast<uint32_t>(length) + drafts + uniform(words[19]) - 1) / uniform(words[19])
                                                       : 0u;
            row.context = live ? static_cast<uint32_t>(length) : 0;
            row.reach = live ? row.context + drafts : 0;
            reinterpret_cast<tree_row *>(lds + T::TABLE)[32 * w + (lane & 31)] = row;  // (the wave's own: no barrier)
            if (has && !live && uniform(words[23]) && wave < T::GW) {
                // Nothing attended: zeros (those of requests that are split are the merge's).
                uint16_t *out = a.output + qrow * D + D / T::SHARE * (w % T::SHARE) + 4 * (lane >> 5);
#pragma unroll
                for (uint32_t i = 0; i < 4 * T::NT; ++i) *reinterpret_cast<sglkv_u16x4 *>(out + 8 * i) = sglkv_u16x4{0, 0, 0, 0};
            }
        }
        // One pass with every row; the tile is done unless its values are not finite. A token that one row attends
        // and another does not has weight 0 in the other's product, and 0 times an infinite or NaN value is NaN. So
        // when a wave whose rows attend different tokens holds an output that is not finite, the queries are done
        // again one by one: no row then meets a token that it does not attend.
        for (uint32_t only = 0xFFFFFFFFu;;) {
            const sglkv_tree_params &p = tree_params();
            const sglkv_attn_params &a = p.a;
            tree_pass pass;
            uint32_t wave_reach, wave_least;
            {
                const tree_row &row = reinterpret_cast<const tree_row *>(lds + T::TABLE)[32 * w + (lane & 31)];
                const bool on = row.reach != 0 && (only == 0xFFFFFFFFu || row.number == only);
                const uint32_t context = row.context;
                // The waves' extremes, exchanged.
                wave_reach = tree_most(on ? row.reach : 0);
                const uint32_t most = tree_most(on ? context : 0), least = tree_most(on ? ~context : 0);
                wave_least = ~least;
                if (lane == 0) *reinterpret_cast<sglkv_v4u *>(words + 4 * w) = sglkv_v4u{wave_reach, most, least, 0};
                __syncthreads();
                sglkv_v4u x = *reinterpret_cast<const sglkv_v4u *>(words);
#pragma unroll
                for (uint32_t i = 1; i < 4; ++i) {
                    const sglkv_v4u y = *reinterpret_cast<const sglkv_v4u *>(words + 4 * i);
#pragma unroll
                    for (uint32_t e = 0; e < 3; ++e) x[e] = y[e] > x[e] ? y[e] : x[e];
                }
                const uint32_t farthest = __builtin_amdgcn_readfirstlane(x[0]);
                pass.whole = __builtin_amdgcn_readfirstlane(x[1]);
                pass.common = ~__builtin_amdgcn_readfirstlane(x[2]);
                pass.t0 = t0;
                pass.t1 = farthest <= t0 ? t0 : farthest - t0 < uniform(words[19]) ? farthest : t0 + uniform(words[19]);
                if (pass.t1 > t0) {
                    pass.start = static_cast<uint64_t>(uniform(words[21])) << 32 | uniform(words[20]);
                    pass.last = uniform(words[22]);
                    // The drafts behind `whole` that some row attends.
                    for (uint32_t i = 0; i < p.mask_words; ++i) {
                        uint64_t m = 0;
                        if (on && pass.whole - context < 64 * p.mask_words) m = tree_bits(row, pass.whole - context + 64 * i);
                        // (joined over the wave first: the compiler's own way, lane by lane, took 1.5 us)
                        const uint64_t any = static_cast<uint64_t>(tree_any(static_cast<uint32_t>(m >> 32))) << 32 |
                                             tree_any(static_cast<uint32_t>(m));
                        uint32_t l = lane;
                        asm volatile("" : "+v"(l));
                        if (any && l == 0)
                            atomicOr(reinterpret_cast<unsigned long long *>(seen + i), static_cast<unsigned long long>(any));
                    }
                    if (only != 0xFFFFFFFFu) tree_first_slots<D, RW>(a, pass.start, pass.start + pass.last + 1, t0, w, lane, lds_at);
                    __syncthreads();
                }
            }
            bool redo = false;
            if (pass.t1 > t0) {
                tree_state<D, RW> st;
                const uint64_t pool = reinterpret_cast<uint64_t>(a.pool);
                tree_run<D, RW>(tree_params(), pass, pool + a.key_offset + kvh * a.key_head_stride,
                                pool + a.value_offset + kvh * a.value_head_stride, w, lane, lds, lds_at, wave_least, wave_reach, qf,
                                st);
                if (only == 0xFFFFFFFFu && pass.t1 > pass.common) {
                    float odd = 0.0f;
#pragma unroll
                    for (uint32_t n = 0; n < T::NT; ++n)
#pragma unroll
                        for (uint32_t i = 0; i < 16; ++i) odd = __builtin_fmaf(st.o[n][i], 0.0f, odd);
                    const tree_row &row = reinterpret_cast<const tree_row *>(lds + T::TABLE)[32 * w + (lane & 31)];
                    redo = __syncthreads_or(odd != 0.0f && row.reach > t0) != 0;  // (NaN != 0)
                }
                if (!redo) tree_write<D, RW>(w, lane, lds, kvh, split, t0, only, st);
            }
            if (only == 0xFFFFFFFFu && !redo) break;
            if (++only == uniform(words[18])) break;  // (from the whole tile to query 0)
            __syncthreads();
            if (tid < SGLKV_TREE_MAX_WORDS) seen[tid] = 0;
        }
        tree_wait<0>();  // (slots that nothing was read for)
        __syncthreads();  // (the next tile's loads go where this one's outputs were joined)
        const uint32_t left = uniform(words[16]) - q0, step = uniform(words[17]);
        if (step >= left) break;  // (a tile has a query or more)
        q0 += step * tree_params().tile_queries;
    }
}

}  // namespace

extern "C" __global__ __launch_bounds__(64) void sglkv_tree_attention_v16(sglkv_tree_params p) { tree_body<true>(p); }
extern "C" __global__ __launch_bounds__(64) __attribute__((amdgpu_waves_per_eu(2))) void sglkv_tree_attention_v2(
    sglkv_tree_params p) {
    tree_body<false>(p);
}

#define SGLKV_TREE_TILE(D, RW, WAVES)                                                                              \
    extern "C" __global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(WAVES))) void                 \
    sglkv_tree_tile##D##_##RW(sglkv_tree_params) {                                                                 \
        tree_tile_body<D, RW>();                                                                                   \
    }
SGLKV_TREE_TILE(64, 1, 2)
SGLKV_TREE_TILE(64, 2, 2)
SGLKV_TREE_TILE(64, 4, 2)
SGLKV_TREE_TILE(128, 1, 1)
SGLKV_TREE_TILE(128, 2, 2)
SGLKV_TREE_TILE(128, 4, 2)
SGLKV_TREE_TILE(256, 1, 1)
SGLKV_TREE_TILE(256, 2, 2)

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
    uint32_t used = 0;
    bool whole = false;  // one split, which has written the output
    if (p.unit) {
        // (The tiles have left it: going over the query's metadata again took as long as the merge.)
        if (inside) used = p.used[item / a.query_heads];
        whole = used == SGLKV_SELECT_NONE;
        if (whole) used = 0;
        if (used > a.splits) used = a.splits;  // (indices that fall, which are reported: never past the records)
    } else {
        tree_query t;
        if (inside && tree_metadata(p, item / a.query_heads, false, &t)) used = static_cast<uint32_t>((t.reach + a.chunk_tokens - 1) / a.chunk_tokens);
    }
    const bool any = used != 0;
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
        if (!inside || whole || !place.merges) continue;
        const float linv = any ? 1.0f / l : 0.0f;
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e)
            if (d + e < a.dv) a.output[item * a.dv + d + e] = attn_to_bf16(acc[e] * linv);
    }
}
