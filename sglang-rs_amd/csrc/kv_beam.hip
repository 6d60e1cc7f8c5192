// kv_beam.hip -- beam search's choice: of each request's beams b and tokens v, the
// K with the largest scores[b] + x_bv - log sum_u exp(x_bu).
//
// Within a beam the order is that of its logits, so a row needs its K largest
// logits, their maximum m and l = sum exp(x - m): one pass over the data. A
// workgroup reads a split of a row into registers; the splits' results, K of them
// each, are joined by one workgroup a request in 64 bits.

namespace {

// A logit and its token as one key: larger logits first, then lower tokens; 0 for
// one that takes no part (-inf, NaN). -0 is 0.
__device__ __forceinline__ uint64_t beam_key(float x, uint32_t token) {
    if (!(x > -INFINITY)) return 0;
    const uint32_t b = __float_as_uint(x + 0.0f);
    return static_cast<uint64_t>(b & 0x80000000u ? ~b : b | 0x80000000u) << 32 | ~token;
}
__device__ __forceinline__ float beam_logit(uint64_t key) {
    const uint32_t o = static_cast<uint32_t>(key >> 32);
    return __uint_as_float(o & 0x80000000u ? o & 0x7FFFFFFFu : ~o);
}
__device__ __forceinline__ uint32_t beam_token(uint64_t key) { return ~static_cast<uint32_t>(key); }

__device__ __forceinline__ float beam_value(float x) { return x; }
__device__ __forceinline__ float beam_value(uint16_t x) { return __uint_as_float(static_cast<uint32_t>(x) << 16); }

__device__ __forceinline__ uint64_t beam_larger(uint64_t a, uint64_t b) { return a > b ? a : b; }

// Keys that order as the logits, in 32 bits (the upper half of beam_key's).
__device__ __forceinline__ uint32_t beam_order32(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return x > -INFINITY ? (b & 0x80000000u ? ~b : b | 0x80000000u) : 0u;
}

// The `kept` first of n keys in LDS, in order: a key's place is the number of
// larger ones (keys differ; 0 is none). n is at most a few for each thread.
template <uint32_t THREADS>
__device__ __forceinline__ void beam_rank(const uint64_t *keys, uint32_t n, uint32_t kept, uint64_t *out) {
    for (uint32_t i = threadIdx.x % THREADS; i < n; i += THREADS) {
        const uint64_t own = keys[i];
        uint32_t place = 0;
        for (uint32_t j = 0; j < n; ++j) place += keys[j] > own ? 1u : 0u;
        if (own != 0 && place < kept) out[place] = own;
    }
}

// 16 bytes of a row as floats.
__device__ __forceinline__ void beam_unpack(sglkv_v4u v, float (&x)[8]) {
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
        x[2 * i] = __uint_as_float(v[i] << 16);
        x[2 * i + 1] = __uint_as_float(v[i] & 0xFFFF0000u);
    }
}
__device__ __forceinline__ void beam_unpack(sglkv_v4u v, float (&x)[4]) {
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) x[i] = __uint_as_float(v[i]);
}

// A split of a row: its 16-byte vectors in registers, and a row's few elements
// before the first and behind the last multiple of 16 bytes with its first split.
template <typename E>
__device__ __forceinline__ void beam_rows_body(const sglkv_beam_params &p) {
    constexpr uint32_t W = SGLKV_BEAM_THREADS / 64, PER = 16 / sizeof(E), VECTORS = SGLKV_BEAM_OWN / PER, N = SGLKV_BEAM_OWN + 1;
    __shared__ float2 part[W];
    __shared__ uint32_t edge[W], count;
    __shared__ uint64_t best[2][W], list[SGLKV_BEAM_LIST];
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const uint32_t split = blockIdx.x % p.splits;
    const uint64_t row = blockIdx.x / p.splits;
    const uint64_t at = reinterpret_cast<uint64_t>(p.logits) + row * p.row_stride * sizeof(E);
    const uint32_t before = static_cast<uint32_t>((16 - at % 16) % 16 / sizeof(E)), lead = before < p.vocab ? before : p.vocab;
    const uint32_t vectors = (p.vocab - lead) / PER, tail = p.vocab - lead - PER * vectors;
    const uint32_t first = split * (SGLKV_BEAM_CHUNK / PER) + tid;
    typedef __attribute__((address_space(1))) const sglkv_v4u vec_t;
    typedef __attribute__((address_space(1))) const E elt_t;
    sglkv_v4u raw[VECTORS];
#pragma unroll
    for (uint32_t i = 0; i < VECTORS; ++i) {
        const uint32_t v = first + i * SGLKV_BEAM_THREADS;
        // (A vector past the row's is read at its start, or where the row has none not at all.)
        raw[i] = sglkv_v4u{0, 0, 0, 0};
        if (vectors) raw[i] = __builtin_nontemporal_load(reinterpret_cast<vec_t *>(at + lead * sizeof(E)) + (v < vectors ? v : 0));
    }
    float x[N];
    // Element i of the thread: its token.
    auto token = [&](uint32_t i) {
        if (i == N - 1) return tid < lead ? tid : PER * vectors + tid;
        return lead + PER * (first + i / PER * SGLKV_BEAM_THREADS) + i % PER;
    };
    x[N - 1] = -INFINITY;
    if (split == 0 && tid < lead + tail) x[N - 1] = beam_value(reinterpret_cast<elt_t *>(at)[token(N - 1)]);
#pragma unroll
    for (uint32_t i = 0; i < VECTORS; ++i) {
        float v[PER];
        beam_unpack(raw[i], v);
        const bool in = first + i * SGLKV_BEAM_THREADS < vectors;
#pragma unroll
        for (uint32_t e = 0; e < PER; ++e) x[PER * i + e] = in ? v[e] : -INFINITY;
    }
    // The thread's maximum and sum; a NaN stays in the sum (fmaxf drops it from the maximum).
    float own = x[N - 1];
#pragma unroll
    for (uint32_t i = 0; i + 1 < N; i += 2) own = attn_max3(own, x[i], x[i + 1]);
    float m = own;
#pragma unroll
    for (uint32_t d = 1; d < 64; d <<= 1) m = fmaxf(m, __shfl_xor(m, d));
    // At one maximum for the wave (0 where it has none: its terms are 0, or NaN if it is +inf).
    const float log2e = 1.4426950408889634f, top = m > -INFINITY ? m : 0.0f;
    float l = 0.0f;
#pragma unroll
    for (uint32_t i = 0; i < N; ++i) l += __builtin_amdgcn_exp2f((x[i] - top) * log2e);
#pragma unroll
    for (uint32_t d = 1; d < 64; d <<= 1) l += __shfl_xor(l, d);
    // A bound that at least `kept` of the wave's tokens reach: the kept-th largest of its threads' maxima, to 16 bits.
    // The largest of the waves' bounds is one for the workgroup.
    const uint32_t mine = beam_order32(own);
    uint32_t bound = 0;
    if (p.kept <= 64) {
#pragma unroll
        for (uint32_t bit = 31; bit >= 16; --bit) {
            const uint32_t more = bound | 1u << bit;
            if (__popcll(__ballot(mine >= more)) >= p.kept) bound = more;
        }
    }
    if (lane == 0) {
        part[wave] = make_float2(m, l);
        edge[wave] = bound;
    }
    if (tid == 0) count = 0;
    __syncthreads();
    const uint64_t out = row * p.splits + split;
    if (tid == 0) {
        m = part[0].x;
#pragma unroll
        for (uint32_t w = 1; w < W; ++w) m = fmaxf(m, part[w].x);
        l = 0.0f;
#pragma unroll
        for (uint32_t w = 0; w < W; ++w)
            l += part[w].x > -INFINITY || part[w].y != part[w].y ? part[w].y * __builtin_amdgcn_exp2f((part[w].x - m) * log2e) : 0.0f;
        reinterpret_cast<float2 *>(p.partial)[out] = make_float2(m, l);
    }
#pragma unroll
    for (uint32_t w = 0; w < W; ++w) bound = edge[w] > bound ? edge[w] : bound;
    // What reaches the bound, ranked among itself: `kept` tokens and a few more, unless many are equal.
    if (mine >= bound && mine != 0) {
#pragma unroll
        for (uint32_t i = 0; i < N; ++i)
            if (beam_order32(x[i]) >= bound && x[i] > -INFINITY) {
                const uint32_t place = atomicAdd(&count, 1u);
                if (place < SGLKV_BEAM_LIST) list[place] = beam_key(x[i], token(i));
            }
    }
    __syncthreads();
    const uint32_t n = count;
    uint64_t *const to = p.candidates + out * p.kept;
    if (n <= SGLKV_BEAM_LIST) {
        beam_rank<SGLKV_BEAM_THREADS>(list, n, p.kept, to);
        for (uint32_t k = n + tid; k < p.kept; k += SGLKV_BEAM_THREADS) to[k] = 0;
        return;
    }
    // The largest keys, one after another.
    uint64_t next = 0;
#pragma unroll
    for (uint32_t i = 0; i < N; ++i) next = beam_larger(next, beam_key(x[i], token(i)));
    for (uint32_t k = 0; k < p.kept; ++k) {
        uint64_t largest = next;
#pragma unroll
        for (uint32_t d = 1; d < 64; d <<= 1) largest = beam_larger(largest, __shfl_xor(largest, d));
        if (lane == 0) best[k & 1][wave] = largest;
        __syncthreads();
        largest = best[k & 1][0];
#pragma unroll
        for (uint32_t w = 1; w < W; ++w) largest = beam_larger(largest, best[k & 1][w]);
        if (tid == 0) to[k] = largest;
        if (largest != 0 && largest == next) {
            next = 0;
#pragma unroll
            for (uint32_t i = 0; i < N; ++i) {
                const uint64_t key = beam_key(x[i], token(i));
                next = key < largest ? beam_larger(next, key) : next;
            }
        }
    }
}

// A double as a key of the same order (no NaN).
__device__ __forceinline__ uint64_t beam_order(double x) {
    const uint64_t b = __builtin_bit_cast(uint64_t, x + 0.0);
    return b >> 63 ? ~b : b | 1ull << 63;
}

// A beam's joined statistics: a token's score is offset + (logit - top). An offset
// of NaN: the beam takes no part (a logit of NaN or +inf, none above -inf, or a
// score that is not finite).
struct beam_base {
    double offset;
    float top;
};
__device__ __forceinline__ double beam_score(const beam_base &b, uint64_t key) {
    return b.offset + (static_cast<double>(beam_logit(key)) - b.top);
}
// Its ordered key, 0 if it is not finite (whose difference from itself is NaN).
__device__ __forceinline__ uint64_t beam_score_key(const beam_base &b, uint64_t key) {
    const double total = beam_score(b, key);
    return key != 0 && total - total == 0.0 ? beam_order(total) : 0;
}

// A wave joins the splits of a row, lane l split l (the host has at most 64): its
// statistics, and its `kept` largest keys at out[0..kept), where there are as many.
__device__ __forceinline__ beam_base beam_join_row(const sglkv_beam_params &p, uint64_t row, uint32_t lane, uint64_t *list,
                                                   uint64_t *out) {
    const uint32_t kept = p.kept, all = p.splits * kept;
    const uint64_t first = row * p.splits, at = first + (lane < p.splits ? lane : 0);
    const uint64_t *keys = p.candidates + first * kept, *mine = p.candidates + at * kept;
    const float2 own = reinterpret_cast<const float2 *>(p.partial)[at];
    const float score = p.scores[row];
    // Every split's last key is reached by `kept` of the row's.
    uint64_t bound = mine[kept - 1];
    float m = own.x;
    const bool odd = __ballot(own.y != own.y || own.x == INFINITY) != 0;
#pragma unroll
    for (uint32_t d = 1; d < 64; d <<= 1) {
        m = fmaxf(m, __shfl_xor(m, d));
        bound = beam_larger(bound, __shfl_xor(bound, d));
    }
    double sum = lane < p.splits && own.y > 0.0f ? static_cast<double>(own.y) * exp(static_cast<double>(own.x) - m) : 0.0;
#pragma unroll
    for (uint32_t d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d);
    beam_base base;
    base.top = m;
    base.offset = odd || m == -INFINITY ? NAN : static_cast<double>(score) - log(sum);
    uint32_t n = 0;
    for (uint32_t i = lane; i < ((all + 63) & ~63u); i += 64) {
        const uint64_t key = i < all ? keys[i] : 0;
        const bool in = key != 0 && key >= bound;
        const uint64_t who = __ballot(in);
        const uint32_t place = n + __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(who >> 32),
                                                             __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(who), 0));
        if (in && place < SGLKV_BEAM_LIST) list[place] = key;
        n += __popcll(who);
    }
    __builtin_amdgcn_wave_barrier();
    if (n <= SGLKV_BEAM_LIST) {
        beam_rank<64>(list, n, kept, out);
    } else {
        // The splits' lists descend: their heads are compared, and the largest is taken.
        uint32_t next = 0;
        uint64_t head = lane < p.splits ? mine[0] : 0;
        for (uint32_t k = 0; k < kept; ++k) {
            uint64_t top = head;
#pragma unroll
            for (uint32_t d = 1; d < 64; d <<= 1) top = beam_larger(top, __shfl_xor(top, d));
            if (lane == 0) out[k] = top;
            if (top != 0 && head == top) head = ++next < kept ? mine[next] : 0;
        }
    }
    __builtin_amdgcn_wave_barrier();
    return base;
}

// A workgroup a request: its waves join the beams' splits, then the beams are
// joined: up to SGLKV_BEAM_FINALS continuations by their rank among each other,
// more by the first wave, which takes the best of the lists' heads, lane l those of
// beams l, l + 64, ....
__device__ __forceinline__ void beam_join_body(const sglkv_beam_params &p) {
    constexpr uint32_t W = SGLKV_BEAM_JOIN_THREADS / 64;
    __shared__ beam_base bases[SGLKV_BEAM_MAX_BEAMS];
    __shared__ uint32_t place[SGLKV_BEAM_MAX_BEAMS];
    __shared__ uint64_t lists[W][SGLKV_BEAM_LIST], finals[SGLKV_BEAM_FINALS], orders[SGLKV_BEAM_FINALS];
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t request = blockIdx.x, kept = p.kept, all = p.beams * kept;
    const uint64_t rows = static_cast<uint64_t>(request) * p.beams, out = static_cast<uint64_t>(request) * kept;
    const bool few = all <= SGLKV_BEAM_FINALS;
    for (uint32_t b = wave; b < p.beams; b += W) {
        uint64_t *list = few ? finals + b * kept : p.lists + (rows + b) * kept;
        for (uint32_t k = lane; k < kept; k += 64) list[k] = 0;
        __builtin_amdgcn_wave_barrier();
        const beam_base base = beam_join_row(p, rows + b, lane, lists[wave], list);
        if (lane == 0) {
            bases[b] = base;
            place[b] = 0;
        }
    }
    __syncthreads();
    if (few) {
        const uint32_t b = tid / kept;
        const uint64_t key = tid < all ? finals[tid] : 0, own = tid < all ? beam_score_key(bases[b], key) : 0;
        if (tid < all) orders[tid] = own;
        const uint32_t count = __syncthreads_count(own != 0);
        uint32_t rank = 0;
        for (uint32_t j = 0; j < all; ++j) rank += orders[j] > own || (orders[j] == own && j < tid) ? 1u : 0u;
        if (own != 0 && rank < kept) {
            p.best_scores[out + rank] = static_cast<float>(beam_score(bases[b], key));
            p.best_parents[out + rank] = static_cast<uint32_t>(rows) + b;
            p.best_tokens[out + rank] = beam_token(key);
        }
        for (uint32_t k = count + tid; k < kept; k += SGLKV_BEAM_JOIN_THREADS) {
            p.best_scores[out + k] = -INFINITY;
            p.best_parents[out + k] = p.best_tokens[out + k] = 0xFFFFFFFFu;
        }
        return;
    }
    if (wave != 0) return;
    // The lane's best beam: its score's key (0: none) and its list's head.
    uint64_t best, head;
    uint32_t beam;
    auto look = [&]() {
        best = 0;
        for (uint32_t b = lane; b < p.beams; b += 64) {
            const uint64_t key = place[b] < kept ? p.lists[(rows + b) * kept + place[b]] : 0, o = beam_score_key(bases[b], key);
            if (o > best) {
                best = o;
                beam = b;
                head = key;
            }
        }
    };
    look();
    for (uint32_t k = 0; k < kept; ++k) {
        uint64_t top = best;
#pragma unroll
        for (uint32_t d = 1; d < 64; d <<= 1) top = beam_larger(top, __shfl_xor(top, d));
        uint32_t lowest = top != 0 && best == top ? beam : 0xFFFFFFFFu;
#pragma unroll
        for (uint32_t d = 1; d < 64; d <<= 1) {
            const uint32_t x = __shfl_xor(lowest, d);
            lowest = x < lowest ? x : lowest;
        }
        if (lowest == 0xFFFFFFFFu) {
            if (lane == 0) {
                p.best_scores[out + k] = -INFINITY;
                p.best_parents[out + k] = p.best_tokens[out + k] = 0xFFFFFFFFu;
            }
        } else if (best == top && beam == lowest) {
            p.best_scores[out + k] = static_cast<float>(beam_score(bases[beam], head));
            p.best_parents[out + k] = static_cast<uint32_t>(rows) + beam;
            p.best_tokens[out + k] = beam_token(head);
            ++place[beam];
            look();
        }
    }
}

}  // namespace

extern "C" __global__ __launch_bounds__(SGLKV_BEAM_THREADS) void sglkv_beam_rows_bf16(sglkv_beam_params p) {
    beam_rows_body<uint16_t>(p);
}
extern "C" __global__ __launch_bounds__(SGLKV_BEAM_THREADS) void sglkv_beam_rows_f32(sglkv_beam_params p) {
    beam_rows_body<float>(p);
}
extern "C" __global__ __launch_bounds__(SGLKV_BEAM_JOIN_THREADS) void sglkv_beam_join(sglkv_beam_params p) { beam_join_body(p); }
