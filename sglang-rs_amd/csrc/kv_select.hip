// kv_select.hip -- attention over the pages of a long context that matter,
// for gfx950: each page's key bounds, the choice of pages for each (query, KV
// head), and softmax attention over the chosen pages alone. It reads the pools,
// slot lists and query metadata that kv_attention.hip reads.
//
// For a page with keys k_t, low_d = min_t k_td and high_d = max_t k_td, any
// query q has
//     q . k_t <= sum_d max(q_d, 0) high_d + min(q_d, 0) low_d
// for every token t of the page: the page's score, which takes 2 dk values
// instead of page_size * dk to compute.

namespace {

typedef __attribute__((address_space(1))) const sglkv_u16x8 sel_vec_t;

__device__ __forceinline__ sglkv_u16x8 sel_load(uint64_t at) { return *reinterpret_cast<sel_vec_t *>(at); }

__device__ __forceinline__ float sel_f32(uint16_t bits) { return __uint_as_float(static_cast<uint32_t>(bits) << 16); }

// A value from lane `lane ^ MASK`, MASK a power of two: within a row of 16
// lanes (permutes and mirrors of the vector unit; mirrors reverse 8 or 16
// lanes, which serves sums and extremes whose lower bits are already joined),
// then across rows.
template <uint32_t MASK>
__device__ __forceinline__ uint32_t sel_join(uint32_t x) {
    if constexpr (MASK == 1) return __builtin_amdgcn_update_dpp(x, x, 0xB1, 0xF, 0xF, true);   // quad 1 0 3 2
    if constexpr (MASK == 2) return __builtin_amdgcn_update_dpp(x, x, 0x4E, 0xF, 0xF, true);   // quad 2 3 0 1
    if constexpr (MASK == 4) return __builtin_amdgcn_update_dpp(x, x, 0x141, 0xF, 0xF, true);  // mirror of 8
    if constexpr (MASK == 8) return __builtin_amdgcn_update_dpp(x, x, 0x140, 0xF, 0xF, true);  // mirror of 16
    if constexpr (MASK == 16) return __float_as_uint(attn_xor16(__uint_as_float(x)));
    return __float_as_uint(attn_xor32(__uint_as_float(x)));
}

template <uint32_t MASK>
__device__ __forceinline__ double sel_join(double x) {
    const uint64_t b = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = sel_join<MASK>(static_cast<uint32_t>(b)), hi = sel_join<MASK>(static_cast<uint32_t>(b >> 32));
    return __builtin_bit_cast(double, (static_cast<uint64_t>(hi) << 32) | lo);
}

// The sum over each group of LANES (a power of two) adjacent lanes, in all of
// them, by the same tree for every group.
template <uint32_t LANES>
__device__ __forceinline__ double sel_sum(double x) {
    if constexpr (LANES > 1) x += sel_join<1>(x);
    if constexpr (LANES > 2) x += sel_join<2>(x);
    if constexpr (LANES > 4) x += sel_join<4>(x);
    if constexpr (LANES > 8) x += sel_join<8>(x);
    if constexpr (LANES > 16) x += sel_join<16>(x);
    if constexpr (LANES > 32) x += sel_join<32>(x);
    return x;
}

// This workgroup's place among items * inner_count of them. XCDs take workgroups in
// turn: eight items go side by side, each with all its inner_count parts on one
// XCD, whose L2 then shares what the parts read in common. Which of the eight
// goes to which XCD turns from eight to eight, so that work that grows with the
// item within a power of two of them does not pile up on one.
__device__ __forceinline__ void sel_place(uint32_t inner_count, uint32_t *item, uint32_t *inner) {
    const uint32_t b = blockIdx.x, k = b / 8, eight = k / inner_count;
    *inner = k - eight * inner_count;
    *item = 8 * eight + ((b + blockIdx.y + 5 * eight + eight / 8) & 7);
}

// ---- Page key bounds ------------------------------------------------------
//
// One wave per (page, KV head). NaN carries into both bounds (minimum and
// maximum of IEEE 754-2019), so that a page with one is not passed over.

__device__ __forceinline__ bool bounds_item(const sglkv_bounds_params &p, uint64_t *page, uint32_t *head,
                                            uint32_t *tokens) {
    const uint64_t item = static_cast<uint64_t>(blockIdx.x) * (blockDim.x / 64) +
                          __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    if (item >= p.count * p.heads) return false;
    const uint64_t i = item / p.heads;
    *head = static_cast<uint32_t>(item - i * p.heads);
    *page = p.pages[i];
    *tokens = p.counts[i];
    const bool ok = *page < p.page_count && *tokens <= p.page_size;
    if (!ok && *head == 0 && (threadIdx.x & 63) == 0)
        atomicOr(p.flag, *page < p.page_count ? SGLKV_FLAG_SPAN : SGLKV_FLAG_PAGE);
    return ok && *tokens > 0;
}

// LANES lanes to a token's row, 8 dims each; 64 / LANES tokens side by side. Bound by
// the keys' bytes: 6,250 pages of 16 tokens, 8 heads of 128 dims (205 MB read, 26
// written) take 43 us, 5.4 TB/s. Loads that would only repeat the last token are
// left out (47 us with them), and all pass the caches by (50 us without).
template <uint32_t LANES>
__device__ __forceinline__ void bounds_body(const sglkv_bounds_params &p) {
    uint64_t page;
    uint32_t head, tokens;
    if (!bounds_item(p, &page, &head, &tokens)) return;
    constexpr uint32_t GROUPS = 64 / LANES, U = 8;
    const uint32_t lane = threadIdx.x & 63, v = lane % LANES, group = lane / LANES;
    const uint64_t rows = reinterpret_cast<uint64_t>(p.pool) + page * p.page_stride + p.key_offset +
                          head * p.key_head_stride;
    uint16_t *const out = p.bounds + (page * p.heads + head) * 2 * p.dk;
    for (uint32_t d = 8 * v; d < p.dk; d += 8 * LANES) {  // (the lanes of one row alike, up to the row's end)
        float low[8], high[8];
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) {
            low[e] = INFINITY;
            high[e] = -INFINITY;
        }
        // U loads of GROUPS tokens in flight; past the last token of one, the last again.
        for (uint32_t t0 = 0; t0 < tokens; t0 += GROUPS * U) {
            sglkv_u16x8 r[U];
#pragma unroll
            for (uint32_t u = 0; u < U; ++u) {
                if (t0 + GROUPS * u >= tokens) break;
                const uint32_t t = t0 + GROUPS * u + group < tokens ? t0 + GROUPS * u + group : tokens - 1;
                r[u] = __builtin_nontemporal_load(reinterpret_cast<sel_vec_t *>(rows + static_cast<uint64_t>(t) * p.key_token_stride + 2 * d));
            }
#pragma unroll
            for (uint32_t u = 0; u < U; ++u) {
                if (t0 + GROUPS * u >= tokens) break;
#pragma unroll
                for (uint32_t e = 0; e < 8; ++e) {
                    low[e] = __builtin_elementwise_minimum(low[e], sel_f32(r[u][e]));
                    high[e] = __builtin_elementwise_maximum(high[e], sel_f32(r[u][e]));
                }
            }
        }
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) {
#pragma unroll
            for (uint32_t m = LANES; m < 64; m <<= 1) {
                low[e] = __builtin_elementwise_minimum(low[e], __shfl_xor(low[e], m));
                high[e] = __builtin_elementwise_maximum(high[e], __shfl_xor(high[e], m));
            }
        }
        if (group == 0) {
            sglkv_u16x8 lo, hi;
#pragma unroll
            for (uint32_t e = 0; e < 8; ++e) {
                lo[e] = static_cast<uint16_t>(__float_as_uint(low[e]) >> 16);  // (a bf16 value: exact)
                hi[e] = static_cast<uint16_t>(__float_as_uint(high[e]) >> 16);
            }
            *reinterpret_cast<sglkv_u16x8 *>(out + d) = lo;
            *reinterpret_cast<sglkv_u16x8 *>(out + p.dk + d) = hi;
        }
    }
}

// Rows of any width and alignment: a lane takes a dim of every token.
__device__ __forceinline__ void bounds_body_element(const sglkv_bounds_params &p) {
    uint64_t page;
    uint32_t head, tokens;
    if (!bounds_item(p, &page, &head, &tokens)) return;
    const uint64_t rows = reinterpret_cast<uint64_t>(p.pool) + page * p.page_stride + p.key_offset +
                          head * p.key_head_stride;
    uint16_t *const out = p.bounds + (page * p.heads + head) * 2 * p.dk;
    for (uint32_t d = threadIdx.x & 63; d < p.dk; d += 64) {
        float low = INFINITY, high = -INFINITY;
        for (uint32_t t = 0; t < tokens; ++t) {
            const float x = sel_f32(*reinterpret_cast<__attribute__((address_space(1))) const uint16_t *>(
                rows + static_cast<uint64_t>(t) * p.key_token_stride + 2 * d));
            low = __builtin_elementwise_minimum(low, x);
            high = __builtin_elementwise_maximum(high, x);
        }
        out[d] = static_cast<uint16_t>(__float_as_uint(low) >> 16);
        out[p.dk + d] = static_cast<uint16_t>(__float_as_uint(high) >> 16);
    }
}

// ---- The pages of a (query, KV head) ---------------------------------------
//
// Scores are summed in 64 bits: a product of two bf16 values has 16 bits, so
// the sums of up to 1,024 of them are exact unless they span over 2^27 in
// magnitude, and the choice does not depend on the order of summation. They are
// kept as keys that order like them: unsigned, NaN above every number, and
// pages that are always in above that.

constexpr uint64_t kSelForced = ~0ull, kSelNaN = ~0ull - 1;

__device__ __forceinline__ uint64_t sel_key(double score) {
    if (score != score) return kSelNaN;
    const uint64_t b = __builtin_bit_cast(uint64_t, score + 0.0);  // (-0 is 0)
    return b ^ (static_cast<uint64_t>(static_cast<int64_t>(b) >> 63) | (1ull << 63));
}

// A query's sequence: where its slots start and its length (0: none, or its
// metadata does not hold, which sets the error word when `report`).
__device__ __forceinline__ void sel_sequence(const sglkv_attn_params &p, uint64_t max_length, uint64_t q, bool report,
                                             uint64_t *start, uint64_t *len) {
    *start = *len = 0;
    const uint64_t n = p.query_sequence_lengths[q];
    if (n == 0) return;
    const uint32_t r = p.query_request_indices[q];
    if (r >= p.request_count) {
        if (report) atomicOr(p.flag, SGLKV_FLAG_ATTN_REQUEST);
        return;
    }
    const uint64_t s = p.request_slot_offsets[r], e = p.request_slot_offsets[r + 1];
    if (s > e || e > p.sequence_slot_count || n > e - s || n > max_length) {
        if (report) atomicOr(p.flag, SGLKV_FLAG_ATTN_SEQUENCE);
        return;
    }
    *start = s;
    *len = n;
}

// Pool page of logical page j (whose slots start at sequence_slots[start]),
// of which `tokens` are read; false (and the error word) where the slot is no
// page's first or the tokens pass the pool's slots.
__device__ __forceinline__ bool sel_page(const sglkv_attn_params &p, uint64_t start, uint64_t j, uint64_t tokens,
                                         uint64_t *page) {
    const uint64_t slot = p.sequence_slots[start + j * p.page_size];
    uint64_t in_page;
    attn_split_slot(p, slot, page, &in_page);
    if (slot < p.slot_count && tokens <= p.slot_count - slot && in_page == 0) return true;
    atomicOr(p.flag, SGLKV_FLAG_ATTN_SLOT);
    return false;
}

// The q.k bound of `pages` logical pages from `first` for one (query, KV
// head), as keys handed to store(i, key). A page takes LANES lanes, 8 dims
// each (NV times, past 8 LANES dims); a workgroup of SGLKV_SELECT_THREADS
// threads; the query heads' vectors lie in LDS (qs, 64 bits each).
template <uint32_t LANES, uint32_t NV, bool VEC, class Store>
__device__ __forceinline__ void sel_scores(const sglkv_select_params &p, uint32_t head, uint64_t start, uint64_t len,
                                           uint64_t first, uint64_t last, const uint16_t *qs, Store store) {
    constexpr uint32_t SIDE = SGLKV_SELECT_THREADS / LANES;  // pages side by side
    const uint32_t v = threadIdx.x % LANES, mine = threadIdx.x / LANES, dk = p.a.dk, qstride = SGLKV_SELECT_QSTRIDE(dk);
    const uint64_t count = (len + p.a.page_size - 1) / p.a.page_size;
    for (uint64_t j0 = first; j0 < last; j0 += SIDE) {
        const uint64_t j = j0 + mine;
        const bool live = j < last;
        const uint64_t left = len - j * p.a.page_size;
        uint64_t page = 0;
        bool ok = false;
        if (live) ok = sel_page(p.a, start, j, left < p.a.page_size ? left : p.a.page_size, &page);
        const uint64_t row = reinterpret_cast<uint64_t>(p.bounds) + (page * p.a.kv_heads + head) * 4 * dk;
        sglkv_u16x8 low[NV], high[NV];
#pragma unroll
        for (uint32_t n = 0; n < NV; ++n) {
            const uint32_t d = 8 * (v + LANES * n);
            low[n] = attn_load8<VEC>(row, d, dk, ok);
            high[n] = attn_load8<VEC>(row + 2 * dk, d, dk, ok);
        }
        double best = -INFINITY;
        for (uint32_t g = 0; g < p.a.group; ++g) {
            double sum = 0.0;
#pragma unroll
            for (uint32_t n = 0; n < NV; ++n) {
                const uint32_t d = 8 * (v + LANES * n);
                if (d < dk)
#pragma unroll
                    for (uint32_t e = 0; e < 8; ++e) {
                        const float q = sel_f32(qs[g * qstride + d + e]);  // (a NaN stays in the second product)
                        sum += static_cast<double>(q > 0.0f ? q : 0.0f) * static_cast<double>(sel_f32(high[n][e]));
                        sum += static_cast<double>(q > 0.0f ? 0.0f : q) * static_cast<double>(sel_f32(low[n][e]));
                    }
            }
            sum = sel_sum<LANES>(sum);
            best = !(sum <= best) && best == best ? sum : best;  // (NaN stays)
        }
        if (live && v == 0)
            store(j, j < p.first_pages || j + p.last_pages >= count ? kSelForced : ok ? sel_key(best) : 0);
    }
}

// The query heads of KV head `head` into LDS, zeros behind their dims.
__device__ __forceinline__ void sel_stage_queries(const sglkv_attn_params &p, uint64_t q, uint32_t head, uint16_t *qs) {
    const uint16_t *from = p.queries + (q * p.query_heads + static_cast<uint64_t>(head) * p.group) * p.dk;
    const uint32_t stride = SGLKV_SELECT_QSTRIDE(p.dk);
    for (uint32_t i = threadIdx.x; i < p.group * stride; i += SGLKV_SELECT_THREADS) {
        const uint32_t g = i / stride, d = i - g * stride;
        qs[i] = d < p.dk ? from[g * p.dk + d] : 0;
    }
}

constexpr uint32_t kSelBuckets = 1024;

struct sel_pick_state {
    uint32_t histogram[kSelBuckets];
    uint64_t low[16], high[16], lo, hi;
    uint32_t special[16], above[16], equal[16];
    uint32_t need, done;
};

// Writes the indices of the `keep` largest of keys load(0..n), ties to the
// lowest index, ascending, to out[0..keep), SGLKV_SELECT_NONE behind them.
// A workgroup of WAVES waves, each with a run of indices, whose keys stay in
// registers where a thread has EACH or fewer: one round trip to memory, where five
// passes over the keys each waited for their own (32 requests of up to 10,000 floats
// on 8 heads: 22 us of 32). Each round counts the keys of [lo, hi] in 1,024 equal steps and
// goes on in the step where the count from above reaches `keep`, until a step is
// taken whole or holds one key alone (lo == hi, of which the lowest indices are
// taken): two rounds on most scores. Forced entries and NaN, the two
// largest keys, are counted apart: they would stretch the steps over the whole
// type. Counting uses LDS atomics, whose order does not show.
template <typename Key, uint32_t WAVES, uint32_t EACH, class Load>
__device__ __forceinline__ void sel_pick(uint64_t n, uint64_t keep, Load load, uint32_t *out, sel_pick_state &s) {
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid / 64);
    constexpr uint32_t THREADS = 64 * WAVES, U = EACH < 8 ? EACH : 8;
    constexpr Key kSpecial = static_cast<Key>(~static_cast<Key>(0)) - 1;
    if (n <= keep) {
        for (uint64_t i = tid; i < keep; i += THREADS) out[i] = i < n ? static_cast<uint32_t>(i) : SGLKV_SELECT_NONE;
        return;
    }
    const uint64_t run = (n + THREADS - 1) / THREADS * 64, i0 = wave * run, i1 = i0 + run < n ? i0 + run : n;
    const bool fits = n <= static_cast<uint64_t>(THREADS) * EACH;
    Key held[EACH];
    if (fits)
#pragma unroll
        for (uint32_t j = 0; j < EACH; ++j) {
            const uint64_t i = i0 + 64 * j + lane;
            held[j] = i < i1 ? load(i) : 0;
        }
    // f(index, key) for the wave's run, 64 at a time (the last ones may pass i1).
    auto each = [&](auto f) {
        if (fits) {
#pragma unroll
            for (uint32_t j = 0; j < EACH; ++j)
                if (i0 + 64 * j < i1) f(i0 + 64 * j + lane, held[j]);
        } else {
            for (uint64_t base = i0; base < i1; base += 64 * U) {
                Key x[U];
#pragma unroll
                for (uint32_t u = 0; u < U; ++u) {
                    const uint64_t i = base + 64 * u + lane;
                    x[u] = load(i < i1 ? i : i1 - 1);
                }
#pragma unroll
                for (uint32_t u = 0; u < U; ++u)
                    if (base + 64 * u < i1) f(base + 64 * u + lane, x[u]);
            }
        }
    };
    Key low = static_cast<Key>(~static_cast<Key>(0)), high = 0;
    uint32_t special = 0;
    each([&](uint64_t i, Key k) {
        const bool in = i < i1, ordinary = in && k < kSpecial;
        special += __popcll(__ballot(in && !ordinary));
        low = ordinary && k < low ? k : low;
        high = ordinary && k > high ? k : high;
    });
#pragma unroll
    for (uint32_t m = 1; m < 64; m <<= 1) {
        const Key l = __shfl_xor(low, m), h = __shfl_xor(high, m);
        low = l < low ? l : low;
        high = h > high ? h : high;
    }
    if (lane == 0) {
        s.low[wave] = low;
        s.high[wave] = high;
        s.special[wave] = special;
    }
    __syncthreads();
    if (tid == 0) {
        uint64_t lo = s.low[0], hi = s.high[0];
        uint32_t count = s.special[0];
        for (uint32_t w = 1; w < WAVES; ++w) {
            lo = s.low[w] < lo ? s.low[w] : lo;
            hi = s.high[w] > hi ? s.high[w] : hi;
            count += s.special[w];
        }
        const bool enough = count >= keep;
        s.lo = enough ? static_cast<uint64_t>(kSpecial) : lo;
        s.hi = enough ? static_cast<uint64_t>(kSpecial) + 1 : hi;
        s.need = static_cast<uint32_t>(enough ? keep : keep - count);
        s.done = s.lo == s.hi;
    }
    __syncthreads();
    // `need` of the keys in [lo, hi] are taken, and all above.
    while (!s.done) {
        const uint64_t lo = s.lo, hi = s.hi;
        const uint32_t bits = 64 - __builtin_clzll(hi - lo), shift = bits > 10 ? bits - 10 : 0;
        for (uint32_t b = tid; b < kSelBuckets; b += THREADS) s.histogram[b] = 0;
        __syncthreads();
        each([&](uint64_t i, Key k) {
            if (i < i1 && k >= lo && k <= hi) atomicAdd(&s.histogram[(k - lo) >> shift], 1u);
        });
        __syncthreads();
        if (wave == 0) {
            // Lane l holds buckets B (63 - l) .. + B - 1: sums from the top down.
            constexpr uint32_t B = kSelBuckets / 64;
            const uint32_t b0 = B * (63 - lane);
            uint32_t c[B], sum = 0;
#pragma unroll
            for (uint32_t b = 0; b < B; ++b) c[b] = s.histogram[b0 + B - 1 - b];
#pragma unroll
            for (uint32_t b = 0; b < B; ++b) sum += c[b];
            uint32_t upto = sum;
#pragma unroll
            for (uint32_t m = 1; m < 64; m <<= 1) {
                const uint32_t x = __shfl_up(upto, m);
                if (lane >= m) upto += x;
            }
            const uint32_t need = s.need;
            uint32_t before = upto - sum;
            if (before < need && upto >= need) {  // (one lane: the counts reach `need`)
                uint32_t down = 0, here = c[0];
#pragma unroll
                for (uint32_t b = 1; b < B; ++b)
                    if (down + 1 == b && before + here < need) {
                        before += here;
                        here = c[b];
                        down = b;
                    }
                const uint64_t from = lo + (static_cast<uint64_t>(b0 + B - 1 - down) << shift), width = (1ull << shift) - 1;
                s.need = need - before;
                s.lo = from;
                s.hi = hi - from < width ? hi : from + width;
                s.done = here == need - before || shift == 0 || s.lo == s.hi;
            }
        }
        __syncthreads();
    }
    const uint64_t lo = s.lo, hi = s.hi;
    const uint32_t need = s.need;
    // Count, then write in order.
    uint32_t above = 0, equal = 0;
    each([&](uint64_t i, Key k) {
        above += __popcll(__ballot(i < i1 && k > hi));
        equal += __popcll(__ballot(i < i1 && k >= lo && k <= hi));
    });
    if (lane == 0) {
        s.above[wave] = above;
        s.equal[wave] = equal;
    }
    __syncthreads();
    uint32_t at = 0, ties = 0;
    for (uint32_t w = 0; w < wave; ++w) {
        at += s.above[w];
        ties += s.equal[w];
    }
    at += ties < need ? ties : need;
    each([&](uint64_t i, Key k) {
        const bool in = i < i1, tie = in && k >= lo && k <= hi;
        const uint64_t eq = __ballot(tie);
        const uint32_t rank = ties + __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(eq >> 32),
                                                               __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(eq), 0));
        const bool take = in && (k > hi || (tie && rank < need));
        const uint64_t taken = __ballot(take);
        if (take)
            out[at + __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(taken >> 32),
                                               __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(taken), 0))] =
                static_cast<uint32_t>(i);
        at += __popcll(taken);
        ties += __popcll(eq);
    });
}

// Scores of a chunk of a (query, KV head)'s pages into the workspace.
template <uint32_t LANES, uint32_t NV, bool VEC>
__device__ __forceinline__ void sel_scores_body(const sglkv_select_params &p) {
    extern __shared__ __attribute__((aligned(16))) uint8_t sel_lds[];
    uint16_t *qs = reinterpret_cast<uint16_t *>(sel_lds);
    const uint32_t chunks = p.heads / p.a.kv_heads;
    const uint32_t chunk = blockIdx.x % chunks, item = blockIdx.x / chunks;
    const uint32_t head = item % p.a.kv_heads;
    const uint64_t q = item / p.a.kv_heads;
    uint64_t start, len;
    sel_sequence(p.a, p.max_length, q, false, &start, &len);
    const uint64_t count = (len + p.a.page_size - 1) / p.a.page_size;
    const uint64_t first = static_cast<uint64_t>(chunk) * p.chunk_pages;
    if (first >= count || count <= p.max_pages) return;  // (nothing to choose from)
    sel_stage_queries(p.a, q, head, qs);
    __syncthreads();
    uint64_t *keys = p.keys + (q * p.a.kv_heads + head) * p.sequence_pages;
    sel_scores<LANES, NV, VEC>(p, head, start, len, first, first + p.chunk_pages < count ? first + p.chunk_pages : count, qs,
                          [&](uint64_t j, uint64_t key) { keys[j] = key; });
}

// The same for keys of 64, 128 or 256 dims on 16-byte rows, as a matrix product in
// 64 bits. A page's row is its 2 D bounds, low then high; a query head's, min(q, 0)
// then max(q, 0). v_mfma_f64_4x4x4 multiplies four 4 x 4 blocks: lane l holds, of
// page l % 4 and of query head l % 4, element l / 4 of 16, and gets block (l / 4)
// % 4's share of page l / 16's product with head l % 4. So a lane's 16 bytes of a
// row, for 16 lanes to a row, are eight steps, no lane holds more of a query than
// its 16th, and only four shares are left to add across lanes. (With a row's dims
// spread over lanes and 64-bit vector multiply-adds the query took 128 registers,
// one or two waves fitted a SIMD, and the sums across 16 lanes took as long as the
// products: 64 ragged sequences of up to 2,048 pages, 8 KV heads of 4 query heads,
// dims 128, 136 us.) 4 NG query heads a turn; more take several turns over the
// chunk, whose maxima wait in LDS. Those sequences take 77 to 81 us for 293 MB, 3.7
// TB/s, where a plain streaming read of them takes 45 (loads that keep the rows in the
// caches, 83; slots found row by row, 113): bound by issue before bytes. Waves wait
// for their turn to issue in 0.42 of their cycles and for anything else in 0.36: each
// element is converted to 64 bits, and the products are small. Sixteen pages
// a wave's step at 64 and 128 dims, 8 at 256 for the registers; 8 at 128 took 97 us.
__device__ __forceinline__ double sel_ror(double x, bool by8) {
    const uint64_t b = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = static_cast<uint32_t>(b), hi = static_cast<uint32_t>(b >> 32);
    const uint32_t rl = by8 ? __builtin_amdgcn_update_dpp(lo, lo, 0x128, 0xF, 0xF, true)
                            : __builtin_amdgcn_update_dpp(lo, lo, 0x124, 0xF, 0xF, true);
    const uint32_t rh = by8 ? __builtin_amdgcn_update_dpp(hi, hi, 0x128, 0xF, 0xF, true)
                            : __builtin_amdgcn_update_dpp(hi, hi, 0x124, 0xF, 0xF, true);
    return __builtin_bit_cast(double, (static_cast<uint64_t>(rh) << 32) | rl);
}

// The larger of two scores, NaN above every number.
__device__ __forceinline__ double sel_larger(double a, double b) { return a != a || b <= a ? a : b; }

template <uint32_t D, uint32_t NG>
__device__ __forceinline__ void sel_scores_fast_body(const sglkv_select_params &p) {
    constexpr uint32_t NV = D / 64, U = D == 256 ? 2 : 4;  // vectors of a lane; steps of four pages that a wave takes at once
    extern __shared__ __attribute__((aligned(16))) double sel_best[];  // the chunk's maxima, if there are several turns
    const uint32_t chunks = p.heads / p.a.kv_heads;
    // A workgroup's waves take block_heads KV heads (1, 2 or 4) of the same pages, whose
    // bounds lie side by side, and the workgroups of the other heads run on the same
    // XCD: a page's slot, a line of its own in a long slot list, is then fetched once.
    // So do those of near_queries queries in a row, as many as a request has on
    // average: drafted tokens read the same bounds (24.7 us for five queries each of
    // 24 sequences of up to 1,250 pages on 2 heads of 64 dims; 26.2 without).
    uint32_t item, inner;
    sel_place(p.a.kv_heads / p.block_heads * p.near_queries, &item, &inner);
    const uint32_t chunk = item % chunks, block = inner / p.near_queries;
    const uint64_t q = static_cast<uint64_t>(item / chunks) * p.near_queries + inner % p.near_queries;
    if (q >= p.a.query_count) return;
    const uint32_t lane = threadIdx.x & 63, slot4 = lane >> 2, in4 = lane & 3;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const uint32_t head = block * p.block_heads + wave % p.block_heads;
    const uint32_t part = wave / p.block_heads, parts = 4 / p.block_heads;  // of the pages
    uint64_t start, len;
    sel_sequence(p.a, p.max_length, q, false, &start, &len);
    const uint32_t page_size = static_cast<uint32_t>(p.a.page_size);
    const uint32_t count = static_cast<uint32_t>((len + page_size - 1) / page_size);
    const uint32_t first = chunk * p.chunk_pages;
    if (first >= count || count <= p.max_pages) return;  // (nothing to choose from)
    const uint32_t last = first + p.chunk_pages < count ? first + p.chunk_pages : count;
    double *best_of = sel_best + (wave % p.block_heads) * p.chunk_pages;
    const uint64_t bounds = reinterpret_cast<uint64_t>(p.bounds) + head * (4ull * D);
    const uint64_t page_bytes = p.a.kv_heads * (4ull * D);
    uint64_t *keys = p.keys + (q * p.a.kv_heads + head) * p.sequence_pages;
    // The wave's pages, in turns of 4 U: number w is page first + 4 U part + w / (4 U) *
    // 4 U parts + w % (4 U). Lane l finds the bounds row of number base + l: 64 pages'
    // slots are one load. A slot that is no page's first is reported; its row is page
    // 0's and its key 0.
    constexpr uint32_t STEP = 4 * U;
    const uint32_t TURN = STEP * parts, begin = first + STEP * part;
    auto page_of = [&](uint32_t w) { return begin + w / STEP * TURN + w % STEP; };
    auto slot_of = [&](uint32_t base) {
        const uint32_t j = page_of(base + lane);
        return p.a.sequence_slots[start + static_cast<uint64_t>(j < last ? j : last - 1) * page_size];
    };
    auto row_of = [&](uint32_t base, uint64_t slot, uint64_t *bad) {
        const uint32_t j = page_of(base + lane) < last ? page_of(base + lane) : last - 1;
        const uint64_t left = len - static_cast<uint64_t>(j) * page_size, tokens = left < page_size ? left : page_size;
        uint64_t page, in_page;
        attn_split_slot(p.a, slot, &page, &in_page);
        const bool ok = slot < p.a.slot_count && tokens <= p.a.slot_count - slot && in_page == 0;
        *bad = __ballot(!ok);
        if (!ok) atomicOr(p.a.flag, SGLKV_FLAG_ATTN_SLOT);
        return bounds + (ok ? page : 0) * page_bytes;
    };
    auto load = [&](uint64_t rows, uint32_t w, sglkv_u16x8 (&row)[U][NV]) {
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) {
            const uint64_t at = __shfl(rows, w + 4 * u + in4) + 16 * slot4;
#pragma unroll
            for (uint32_t n = 0; n < NV; ++n) row[u][n] = __builtin_nontemporal_load(reinterpret_cast<sel_vec_t *>(at + 256 * n));
        }
    };
    const uint32_t turns = (p.a.group + 4 * NG - 1) / (4 * NG);
    for (uint32_t turn = 0; turn < turns; ++turn) {
        if (begin >= last) break;
        uint64_t bad, bad_next = 0;
        uint64_t rows = row_of(0, slot_of(0), &bad), rows_next = 0;
        uint64_t slot = slot_of(64);
        sglkv_u16x8 row[U][NV];
        load(rows, 0, row);
        // Element 8 (slot4 + 16 n) + e of query head g0 + 4 m + l % 4's row of parts.
        double qv[NG][NV][8];
#pragma unroll
        for (uint32_t m = 0; m < NG; ++m) {
            const uint32_t g = turn * 4 * NG + 4 * m + in4;
            const uint64_t from = reinterpret_cast<uint64_t>(p.a.queries) +
                                  2 * (q * p.a.query_heads + head * p.a.group + (g < p.a.group ? g : 0)) * D;
#pragma unroll
            for (uint32_t n = 0; n < NV; ++n) {
                const uint32_t at = 8 * (slot4 + 16 * n);
                const sglkv_u16x8 x = sel_load(from + 2 * (at & (D - 1)));
#pragma unroll
                for (uint32_t e = 0; e < 8; ++e) {
                    const float f = sel_f32(x[e]);  // (a NaN stays with the low bounds)
                    qv[m][n][e] = at < D ? (f > 0.0f ? 0.0f : f) : (f > 0.0f ? f : 0.0f);
                }
            }
        }
        uint32_t w = 0;  // of the 64
        for (uint32_t base = 0, j0 = begin; j0 < last; j0 += TURN) {
            // The next turn's rows load while this one's are multiplied.
            sglkv_u16x8 next[U][NV];
            if (w + STEP < 64) {
                load(rows, w + STEP, next);
            } else {
                rows_next = row_of(base + 64, slot, &bad_next);
                slot = slot_of(base + 128);
                load(rows_next, 0, next);
            }
            __builtin_amdgcn_sched_barrier(0);
            double sum[U][NG] = {};
#pragma unroll
            for (uint32_t n = 0; n < NV; ++n)
#pragma unroll
                for (uint32_t e = 0; e < 8; ++e)
#pragma unroll
                    for (uint32_t u = 0; u < U; ++u) {
                        const double x = sel_f32(row[u][n][e]);
#pragma unroll
                        for (uint32_t m = 0; m < NG; ++m)
                            sum[u][m] = __builtin_amdgcn_mfma_f64_4x4x4f64(x, qv[m][n][e], sum[u][m], 0, 0, 0);
                    }
            // Page l / 16 of step u; lane 16 i + u of them writes page j0 + 4 u + i.
            double mine = 0.0;
            uint32_t mine_bad = 0;
#pragma unroll
            for (uint32_t u = 0; u < U; ++u) {
                double best = -INFINITY;
#pragma unroll
                for (uint32_t m = 0; m < NG; ++m) {
                    double x = sum[u][m];
                    x += sel_ror(x, true);
                    x += sel_ror(x, false);
                    if (turn * 4 * NG + 4 * m + in4 < p.a.group) best = sel_larger(best, x);
                }
                best = sel_larger(best, sel_join<1>(best));
                best = sel_larger(best, sel_join<2>(best));
                if ((lane & 15) == u) {
                    mine = best;
                    mine_bad = bad >> (w + 4 * u + (lane >> 4)) & 1;
                }
            }
            const uint32_t j = j0 + 4 * (lane & 15) + (lane >> 4);
            if ((lane & 15) < U && j < last) {
                if (turn > 0) mine = sel_larger(best_of[j - first], mine);
                if (turn + 1 < turns)
                    best_of[j - first] = mine;
                else
                    keys[j] = j < p.first_pages || j + p.last_pages >= count ? kSelForced : mine_bad ? 0 : sel_key(mine);
            }
            w += STEP;
            if (w == 64) {
                w = 0;
                base += 64;
                rows = rows_next;
                bad = bad_next;
            }
#pragma unroll
            for (uint32_t u = 0; u < U; ++u)
#pragma unroll
                for (uint32_t n = 0; n < NV; ++n) row[u][n] = next[u][n];
        }
    }
}

// The pages of a (query, KV head) from the workspace's keys.
__device__ __forceinline__ void sel_pick_body(const sglkv_select_params &p) {
    __shared__ sel_pick_state state;
    const uint32_t head = blockIdx.x % p.a.kv_heads;
    const uint64_t q = blockIdx.x / p.a.kv_heads;
    uint64_t start, len;
    sel_sequence(p.a, p.max_length, q, head == 0 && threadIdx.x == 0, &start, &len);
    const uint64_t count = (len + p.a.page_size - 1) / p.a.page_size;
    const uint64_t *keys = p.keys + (q * p.a.kv_heads + head) * p.sequence_pages;
    sel_pick<uint64_t, SGLKV_SELECT_THREADS / 64, 8>(count, p.max_pages, [&](uint64_t i) { return keys[i]; },
                                                     p.selected + (q * p.a.kv_heads + head) * p.max_pages, state);
}

// ---- Attention over the selected pages --------------------------------------

// The work of this workgroup: `pages` entries of its list from entry e0, in
// the order of the list, `tokens` tokens in all.
struct sel_work {
    attn_work w;
    uint64_t start, len;
    uint32_t e0, pages, tokens;
};

// Lane l's entry e0 + l of the list as its pool page, for this split of the
// list; the lists ascend, so only the sequence's last page, the last entry,
// holds fewer than page_size tokens. An entry that is no page of the sequence
// or does not ascend sets the error word, and the split counts as empty.
__device__ __forceinline__ uint64_t sel_decode(const sglkv_select_params &p, uint32_t lane, sel_work *s) {
    // (The head groups and value blocks of a (query, KV head) side by side: they read the same rows.)
    uint32_t bx = blockIdx.x;
    const uint32_t dblk = bx % p.a.dv_blocks;
    bx /= p.a.dv_blocks;
    const uint32_t hg = bx % p.a.head_groups;
    bx /= p.a.head_groups;
    const uint32_t kvh = bx % p.a.kv_heads;
    const uint64_t q = bx / p.a.kv_heads;
    const uint32_t split = blockIdx.y;
    s->w.q = q;
    s->w.kvh = kvh;
    s->w.h0 = kvh * p.a.group + hg * SGLKV_ATTN_HEADS;
    const uint32_t heads = p.a.group - hg * SGLKV_ATTN_HEADS;
    s->w.nh = heads < SGLKV_ATTN_HEADS ? heads : SGLKV_ATTN_HEADS;
    s->w.d0 = dblk * SGLKV_ATTN_DV;
    s->w.dblk = dblk;
    s->w.split = split;
    sel_sequence(p.a, p.max_length, q, lane == 0 && split == 0 && hg == 0 && dblk == 0 && kvh == 0, &s->start, &s->len);
    s->e0 = split * p.chunk_pages;
    s->pages = s->tokens = 0;
    const uint32_t e = s->e0 + lane;
    const uint32_t *list = p.selected + (q * p.a.kv_heads + kvh) * p.max_pages;
    const bool inside = s->len > 0 && lane < p.chunk_pages && e < p.max_pages;
    const uint32_t j = inside ? list[e] : SGLKV_SELECT_NONE;
    const uint32_t before = inside && e > 0 ? list[e - 1] : 0;
    const uint64_t listed = __ballot(j != SGLKV_SELECT_NONE);
    const uint64_t count = (s->len + p.a.page_size - 1) / p.a.page_size;
    uint64_t page = 0;
    bool bad = false;
    if (j != SGLKV_SELECT_NONE) {
        bad = j >= count || (e > 0 && before >= j);
        if (bad) {
            atomicOr(p.a.flag, SGLKV_FLAG_ATTN_SEQUENCE);
        } else {
            const uint64_t left = s->len - static_cast<uint64_t>(j) * p.a.page_size;
            bad = !sel_page(p.a, s->start, j, left < p.a.page_size ? left : p.a.page_size, &page);
        }
    }
    if (__ballot(bad) != 0 || listed == 0) return page;
    // (The listed ones are the first: NONE before a page does not ascend.)
    s->pages = __popcll(listed);
    const uint32_t last = __shfl(j, s->pages - 1);
    const uint64_t left = s->len - static_cast<uint64_t>(last) * p.a.page_size;
    s->tokens = static_cast<uint32_t>((s->pages - 1) * p.a.page_size + (left < p.a.page_size ? left : p.a.page_size));
    return page;
}

// A split without tokens: zeros where it is the only one, else a record that
// the merge leaves out (a maximum of -inf, which no split with tokens has).
__device__ __forceinline__ void sel_empty(const sglkv_select_params &p, const sel_work &s, uint32_t lane, uint32_t dims) {
    const sglkv_attn_params &a = p.a;
    if (a.splits == 1) {
        for (uint32_t i = lane; i < s.w.nh * dims; i += 64) {
            const uint32_t h = i / dims, d = s.w.d0 + i % dims;
            if (d < a.dv) a.output[(s.w.q * a.query_heads + s.w.h0 + h) * a.dv + d] = 0;
        }
    } else if (s.w.dblk == 0 && lane < s.w.nh) {
        float *ml = attn_rec_ml(a, (s.w.q * a.query_heads + s.w.h0 + lane) * a.splits + s.w.split);
        ml[0] = -INFINITY;
        ml[1] = 0.0f;
    }
}

// Any head dims, page size and alignment: a wave to 16 query heads and
// SGLKV_ATTN_DV value dims, 32 tokens a step, as the generic body of paged
// attention (attn_body), whose layouts of the matrix products it shares.
template <bool VEC>
__device__ __forceinline__ void sel_attend_body(const sglkv_select_params &p) {
    extern __shared__ __attribute__((aligned(16))) uint16_t sel_attend_lds[];
    __shared__ uint64_t pages[SGLKV_SELECT_CHUNK_PAGES];
    const sglkv_attn_params &a = p.a;
    const uint32_t lane = threadIdx.x, g = lane >> 4, r = lane & 15;
    sel_work s;
    pages[lane] = sel_decode(p, lane, &s);
    if (s.tokens == 0) {
        sel_empty(p, s, lane, SGLKV_ATTN_DV);
        return;
    }
    const attn_work &w = s.w;
    const uint32_t qstride = a.dk_pad + 8;
    uint16_t *qs = sel_attend_lds, *vt = sel_attend_lds + SGLKV_ATTN_HEADS * qstride;
    attn_stage_queries(a, w, lane, qs, qstride);  // (and a barrier: pages[] too)
    const uint64_t pool = reinterpret_cast<uint64_t>(a.pool);
    const uint64_t kbase = pool + a.key_offset + w.kvh * a.key_head_stride;
    const uint64_t vbase = pool + a.value_offset + w.kvh * a.value_head_stride;
    attn_state st;
    attn_state_init(st);
    for (uint32_t tb = 0; tb < s.tokens; tb += SGLKV_ATTN_TOKENS) {
        uint64_t krow[2], vrow[2];
        bool valid[2];
#pragma unroll
        for (uint32_t b = 0; b < 2; ++b) {
            const uint32_t tok = tb + 8 * (r >> 2) + 4 * b + (r & 3);
            valid[b] = tok < s.tokens;
            uint64_t e, pos;
            attn_split_slot(a, valid[b] ? tok : 0, &e, &pos);
            const uint64_t page = pages[e] * a.page_stride;
            krow[b] = kbase + page + pos * a.key_token_stride;
            vrow[b] = vbase + page + pos * a.value_token_stride;
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

// Head dims 64, 128 or 256 of keys and values alike, 16-byte rows, pages of 8
// tokens or more (a power of two), at most 16 query heads a KV head: the staged
// layout of paged attention (attn_stg: rows straight from the pool into LDS, two
// stages of 32 tokens, one wave a workgroup), which its loads' addresses are
// cheaper for. Lane l keeps the pool page of entry l, so a load's page and first
// token are one scalar base, and what a lane adds to it (its token of the load and
// its swizzled piece) is the same for every block: kept at dims 64 and 128, and
// at dims 256, whose accumulators leave no registers for it, made again from the
// lane's part and the load's, which do not share bits (attn_stg's swizzles are
// exclusive ors). LDS holds the two stages and nothing else, which leaves room
// for five workgroups a CU at dims 128. Bound by the rows' bytes: 64 queries' lists of
// 32 pages of 64 tokens, 8 KV heads, dims 128 (521 MB) take 88 us, 5.9 TB/s (the
// generic body: 227); 120 drafted queries' 45 pages of 16 tokens, 2 heads of 256 dims
// (144 MB), 35 us, 4.1 TB/s, with fewer waves than fill the card (generic: 127).
// Four loads: lane l's 16 bytes from base[i] + off[i] to LDS at at + 1024 i +
// 16 l (non-temporal). (The leading s_nop covers the vector write of a base just
// before.)
__device__ __forceinline__ void sel_load4(const uint64_t (&base)[4], const uint32_t *off, uint32_t at) {
    uint32_t save;
    asm volatile(
        "s_nop 4\n\ts_mov_b32 %0, m0\n\t"
        "s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %6 nt\n\t"
        "s_add_u32 m0, %1, 1024\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %3, %7 nt\n\t"
        "s_add_u32 m0, %1, 2048\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %4, %8 nt\n\t"
        "s_add_u32 m0, %1, 0xc00\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %5, %9 nt\n\t"
        "s_mov_b32 m0, %0"
        : "=&s"(save)
        : "s"(at), "v"(off[0]), "v"(off[1]), "v"(off[2]), "v"(off[3]), "s"(base[0]), "s"(base[1]), "s"(base[2]),
          "s"(base[3])
        : "scc");
}

template <uint32_t D>
__device__ __forceinline__ void sel_staged_body(const sglkv_select_params &p) {
    typedef attn_stg<D> S;
    extern __shared__ __attribute__((aligned(16))) uint8_t sel_stg_lds[];
    const sglkv_attn_params &a = p.a;
    const uint32_t lane = threadIdx.x, g = lane >> 4, r = lane & 15;
    sel_work s;
    const uint64_t mine = sel_decode(p, lane, &s);
    if (s.tokens == 0) {
        sel_empty(p, s, lane, D);
        return;
    }
    const attn_work &w = s.w;
    const uint32_t page_lo = static_cast<uint32_t>(mine);  // (the host keeps pages below 2^32)
    sglkv_u16x8 qf[S::KC];
#pragma unroll
    for (uint32_t c = 0; c < S::KC; ++c) {
        qf[c] = sglkv_u16x8{0, 0, 0, 0, 0, 0, 0, 0};
        if (r < w.nh)
            qf[c] = *reinterpret_cast<const sglkv_u16x8 *>(a.queries + (w.q * a.query_heads + w.h0 + r) * D + 32 * c + 8 * g);
    }
    const uint64_t pool = reinterpret_cast<uint64_t>(a.pool);
    const uint64_t kbase = pool + a.key_offset + w.kvh * a.key_head_stride;
    const uint64_t vbase = pool + a.value_offset + w.kvh * a.value_head_stride;
    const uint32_t mask = (1u << a.page_shift) - 1, stride = a.key_token_stride32;
    const uint32_t c = lane / S::PIECES, pc = lane % S::PIECES;
    // Load j takes tokens TPL j + c of a block: its base is the page of token TPL j
    // and that token's place in it, the lane's part token c and piece pc.
    const uint32_t lane_row = __umul24(c, stride), lane_k = S::kpos(c, pc), lane_v = S::vpos(c, pc);
    auto koff_of = [&](uint32_t j) { return lane_row + 16 * (lane_k ^ S::kpos(S::TPL * j, 0)); };
    auto voff_of = [&](uint32_t j) { return lane_row + 16 * (lane_v ^ S::vpos(S::TPL * j, 0)); };
    constexpr uint32_t KEPT = D == 256 ? 1 : S::LOADS;
    uint32_t koff[KEPT], voff[KEPT];
    if constexpr (D != 256)
#pragma unroll
        for (uint32_t j = 0; j < S::LOADS; ++j) {
            koff[j] = koff_of(j);
            voff[j] = voff_of(j);
        }
    const uint32_t nb = (s.tokens + kLatB - 1) / kLatB, full = s.tokens / kLatB;
    auto stage_at = [&](uint32_t b) { return attn_lat_lds_at(sel_stg_lds) + (b & 1) * S::STAGE; };
    auto token_base = [&](uint32_t token) {
        const uint32_t page = __builtin_amdgcn_readlane(page_lo, token >> a.page_shift);
        return static_cast<uint64_t>(page) * a.page_stride32 + static_cast<uint64_t>(token & mask) * stride;
    };
    auto issue = [&](uint32_t b) {
        const uint32_t t0 = kLatB * b, at = stage_at(b);
        const uint64_t zero = reinterpret_cast<uint64_t>(a.zero_row) + 16 * pc;
#pragma unroll
        for (uint32_t h = 0; h < S::LOADS / 4; ++h) {
            uint32_t ko[4], vo[4];
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                ko[i] = D == 256 ? koff_of(4 * h + i) : koff[D == 256 ? 0 : 4 * h + i];
                vo[i] = D == 256 ? voff_of(4 * h + i) : voff[D == 256 ? 0 : 4 * h + i];
            }
            if (b < full) {
                uint64_t kb[4], vb[4];
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    const uint64_t off = token_base(t0 + S::TPL * (4 * h + i));
                    kb[i] = kbase + off;
                    vb[i] = vbase + off;
                }
                sel_load4(kb, ko, at + 4096 * h);
                sel_load4(vb, vo, at + S::V + 4096 * h);
            } else {  // the last block: tokens past the end read the zero row
                uint64_t x[8];
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    const uint32_t t = t0 + S::TPL * (4 * h + i);
                    const uint64_t off = token_base(t < s.tokens ? t : t0);
                    attn_sel64x2(t + c < s.tokens, kbase + off + ko[i], vbase + off + vo[i], zero, x[i], x[4 + i]);
                }
                attn_lat_load4v<1024>(x, at + 4096 * h);
                attn_lat_load4v<1024>(x + 4, at + S::V + 4096 * h);
            }
        }
    };
    // The queries (which the compiler counts) are there before the loop, whose
    // waits count the rows alone.
    __builtin_amdgcn_s_waitcnt(0x0F70);
    issue(0);
    attn_state_n<S::NJ> st;
    attn_state_init(st);
    for (uint32_t k = 0; k < nb; ++k) {
        // Block k-1's reads are done before block k+1's rows take its stage; then
        // block k's rows, older than block k+1's, have landed.
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (k + 1 < nb) {
            issue(k + 1);
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * S::LOADS) : "memory");
        } else {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
        const uint8_t *kst = sel_stg_lds + (k & 1) * S::STAGE;
        const uint32_t left = s.tokens - kLatB * k;
        attn_stg_block<D>(a, g, r, qf, kst, left < kLatB ? left : kLatB, st);
    }
    attn_finish(a, w, g, r, st);
}

}  // namespace

extern "C" __global__ __launch_bounds__(256) void sglkv_page_bounds_8(sglkv_bounds_params p) { bounds_body<8>(p); }
extern "C" __global__ __launch_bounds__(256) void sglkv_page_bounds_16(sglkv_bounds_params p) { bounds_body<16>(p); }
extern "C" __global__ __launch_bounds__(256) void sglkv_page_bounds_32(sglkv_bounds_params p) { bounds_body<32>(p); }
extern "C" __global__ __launch_bounds__(256) void sglkv_page_bounds_64(sglkv_bounds_params p) { bounds_body<64>(p); }
extern "C" __global__ __launch_bounds__(256) void sglkv_page_bounds_element(sglkv_bounds_params p) {
    bounds_body_element(p);
}

extern "C" __global__ __launch_bounds__(SGLKV_SELECT_THREADS) void sglkv_page_scores_8(sglkv_select_params p) {
    sel_scores_body<8, 1, true>(p);
}
extern "C" __global__ __launch_bounds__(SGLKV_SELECT_THREADS) void sglkv_page_scores_16(sglkv_select_params p) {
    sel_scores_body<16, 1, true>(p);
}
extern "C" __global__ __launch_bounds__(SGLKV_SELECT_THREADS) void sglkv_page_scores_32(sglkv_select_params p) {
    sel_scores_body<32, 1, true>(p);
}
extern "C" __global__ __launch_bounds__(SGLKV_SELECT_THREADS) void sglkv_page_scores_64(sglkv_select_params p) {
    sel_scores_body<64, 2, true>(p);
}
extern "C" __global__ __launch_bounds__(SGLKV_SELECT_THREADS) void sglkv_page_scores_element(sglkv_select_params p) {
    sel_scores_body<64, 2, false>(p);
}
// Keys of 64, 128 or 256 dims; 4, 8 or 16 query heads a turn.
extern "C" __global__ __launch_bounds__(SGLKV_SELECT_THREADS) void sglkv_page_scores64_4(sglkv_select_params p) {
    sel_scores_fast_body<64, 1>(p);
}
extern "C" __global__ __launch_bounds__(SGLKV_SELECT_THREADS) void sglkv_page_scores64_8(sglkv_select_params p) {
    sel_scores_fast_body<64, 2>(p);
}
extern "C" __global__ __launch_bounds__(SGLKV_SELECT_THREADS) void sglkv_page_scores64_16(sglkv_select_params p) {
    sel_scores_fast_body<64, 4>(p);
}
extern "C" __global__ __launch_bounds__(SGLKV_SELECT_THREADS) void sglkv_page_scores128_4(sglkv_select_params p) {
    sel_scores_fast_body<128, 1>(p);
}
extern "C" __global__ __launch_bounds__(SGLKV_SELECT_THREADS) void sglkv_page_scores128_8(sglkv_select_params p) {
    sel_scores_fast_body<128, 2>(p);
}
extern "C" __global__ __launch_bounds__(SGLKV_SELECT_THREADS) void sglkv_page_scores128_16(sglkv_select_params p) {
    sel_scores_fast_body<128, 4>(p);
}
extern "C" __global__ __launch_bounds__(SGLKV_SELECT_THREADS) void sglkv_page_scores256_4(sglkv_select_params p) {
    sel_scores_fast_body<256, 1>(p);
}
extern "C" __global__ __launch_bounds__(SGLKV_SELECT_THREADS) void sglkv_page_scores256_8(sglkv_select_params p) {
    sel_scores_fast_body<256, 2>(p);
}
extern "C" __global__ __launch_bounds__(SGLKV_SELECT_THREADS) void sglkv_pick_pages(sglkv_select_params p) {
    sel_pick_body(p);
}

extern "C" __global__ __launch_bounds__(64) void sglkv_selected_attention_v16(sglkv_select_params p) {
    sel_attend_body<true>(p);
}
extern "C" __global__ __launch_bounds__(64) __attribute__((amdgpu_waves_per_eu(2))) void
sglkv_selected_attention_v2(sglkv_select_params p) {
    sel_attend_body<false>(p);
}

// (Two waves a SIMD: the accumulators stay in vector registers.)
extern "C" __global__ __launch_bounds__(64) __attribute__((amdgpu_waves_per_eu(2))) void
sglkv_selected_attention_staged64(sglkv_select_params p) {
    sel_staged_body<64>(p);
}
extern "C" __global__ __launch_bounds__(64) __attribute__((amdgpu_waves_per_eu(2))) void
sglkv_selected_attention_staged128(sglkv_select_params p) {
    sel_staged_body<128>(p);
}
extern "C" __global__ __launch_bounds__(64) __attribute__((amdgpu_waves_per_eu(2))) void
sglkv_selected_attention_staged256(sglkv_select_params p) {
    sel_staged_body<256>(p);
}

// Merges the split records of a (query, head), one wave each. Lane s weighs split
// s once (64 at a time); then sets of ceil(dv / 4) lanes, 4 dims a lane, add every
// so many splits' rows, eight in flight, and join. An empty split weighs nothing
// (its row holds anything); a (query, head) of nothing else is zeros.
extern "C" __global__ __launch_bounds__(64) void sglkv_selected_attention_combine(sglkv_select_params p) {
    const sglkv_attn_params &a = p.a;
    const uint64_t item = blockIdx.x;
    const uint32_t lane = threadIdx.x, opad = SGLKV_ATTN_OPAD(a.dv);
    const float2 *ml = reinterpret_cast<const float2 *>(attn_rec_ml(a, item * a.splits));
    const float *rows = attn_rec_o(a, item * a.splits);
    const uint32_t wide = (a.dv + 3) / 4, lanes = wide <= 16 ? 16 : wide <= 32 ? 32 : 64, sets = 64 / lanes;
    const uint32_t set = lane / lanes, v = lane % lanes;
    for (uint32_t d0 = 0; d0 < a.dv; d0 += 4 * lanes) {
        const uint32_t d = d0 + 4 * v < opad ? d0 + 4 * v : 0;
        float m = -INFINITY, l = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (uint32_t s0 = 0; s0 < a.splits; s0 += 64) {
            const uint32_t here = a.splits - s0 < 64 ? a.splits - s0 : 64;
            const float2 mine = lane < here ? ml[s0 + lane] : make_float2(-INFINITY, 0.0f);
            float top = fmaxf(m, mine.x);
#pragma unroll
            for (uint32_t x = 1; x < 64; x <<= 1) top = fmaxf(top, __shfl_xor(top, x));
            if (top == -INFINITY) continue;
            const float w = __builtin_amdgcn_exp2f(mine.x - top), back = __builtin_amdgcn_exp2f(m - top);
            float sum = mine.x == -INFINITY ? 0.0f : w * mine.y;
#pragma unroll
            for (uint32_t x = 1; x < 64; x <<= 1) sum += __shfl_xor(sum, x);
            l = l * back + sum;
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) o[e] *= back;
            m = top;
            // (All lanes make every round: a weight's lane may belong to a set whose own splits
            // are done. 8 sets divides 64, so `at` is a lane, and those past `here` hold 0.)
            for (uint32_t base = 0; base < here; base += 8 * sets) {
                float4 x[8];
#pragma unroll
                for (uint32_t i = 0; i < 8; ++i) {
                    const uint32_t at = base + set + i * sets;
                    x[i] = *reinterpret_cast<const float4 *>(rows + static_cast<uint64_t>(s0 + (at < here ? at : here - 1)) * opad + d);
                }
#pragma unroll
                for (uint32_t i = 0; i < 8; ++i) {
                    const float ws = __shfl(w, base + set + i * sets);
                    if (ws != 0.0f) {
                        o[0] = fmaf(ws, x[i].x, o[0]);
                        o[1] = fmaf(ws, x[i].y, o[1]);
                        o[2] = fmaf(ws, x[i].z, o[2]);
                        o[3] = fmaf(ws, x[i].w, o[3]);
                    }
                }
            }
        }
        for (uint32_t x = lanes; x < 64; x <<= 1)
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) o[e] += __shfl_xor(o[e], x);
        const float linv = m == -INFINITY ? 0.0f : 1.0f / l;
        if (set == 0)
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e)
                if (d0 + 4 * v + e < a.dv) a.output[item * a.dv + d0 + 4 * v + e] = attn_to_bf16(o[e] * linv);
    }
}
