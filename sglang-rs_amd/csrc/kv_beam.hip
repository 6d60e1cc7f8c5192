// kv_beam.hip -- beam search's choice: of each request's beams b and tokens v, the
// K with the largest scores[b] + x_bv - log sum_u exp(x_bu).
//
// Within a beam the order is that of its logits, so a row needs its K largest
// logits, their maximum m and l = sum exp(x - m): one pass over the data. A
// workgroup reads a split of a row into registers; the splits' results, K of them
// each, are joined by one workgroup a request in 64 bits. What can be among the K is
// found by a bound (the K-th largest of the threads' maxima) and ranked, where K
// rounds of maxima took 99 us for 64 requests of 4 beams, 128,256 tokens and K = 8:
// now 16.8 (66 MB, 3.9 TB/s; loads and what is counted of each logit share the time)
// and 5.7 for the join; 1 request of 4 beams of 32,000: 5.7 and 5.2, each a chain of
// joins over lanes, LDS and barriers. Many kept have no such bound: with K = 64 the
// first batch takes 1,150 us, with 128 2,150.

namespace {

template <int M>
struct beam_mask {
    static constexpr int value = M;
};

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

// x joined over the wave's lanes, in every lane: each step takes what lane l ^ 1,
// 2, 4, ... has, without a round trip through LDS.
template <typename T, typename F>
__device__ __forceinline__ T beam_all(T x, F join) {
    auto other = [](auto mask, T v) {
        constexpr int MASK = decltype(mask)::value;
        if constexpr (sizeof(T) == 4) {
            return __builtin_bit_cast(T, sel_join<MASK>(__builtin_bit_cast(uint32_t, v)));
        } else {
            const uint64_t b = __builtin_bit_cast(uint64_t, v);
            return __builtin_bit_cast(T, static_cast<uint64_t>(sel_join<MASK>(static_cast<uint32_t>(b >> 32))) << 32 |
                                             sel_join<MASK>(static_cast<uint32_t>(b)));
        }
    };
    x = join(x, other(beam_mask<1>(), x));
    x = join(x, other(beam_mask<2>(), x));
    x = join(x, other(beam_mask<4>(), x));
    x = join(x, other(beam_mask<8>(), x));
    x = join(x, other(beam_mask<16>(), x));
    return join(x, other(beam_mask<32>(), x));
}
template <typename T>
__device__ __forceinline__ T beam_sum(T x) {
    return beam_all(x, [](T a, T b) { return a + b; });
}
__device__ __forceinline__ float beam_max(float x) {
    return beam_all(x, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ uint64_t beam_max(uint64_t x) { return beam_all(x, beam_larger); }

// Keys that order as the logits, in 32 bits (the upper half of beam_key's).
__device__ __forceinline__ uint32_t beam_order32(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return x > -INFINITY ? (b & 0x80000000u ? ~b : b | 0x80000000u) : 0u;
}

// The `kept` first of n keys in LDS, in order: a key's place is the number of
// larger ones (keys differ). n is at most a few for each thread; the list has room
// for whole fours, which are read together.
template <uint32_t THREADS>
__device__ __forceinline__ void beam_rank(const uint64_t *keys, uint32_t n, uint32_t kept, uint64_t *out) {
    for (uint32_t i = threadIdx.x % THREADS; i < n; i += THREADS) {
        const uint64_t own = keys[i];
        uint32_t place = 0;
        for (uint32_t j = 0; j < n; j += 4) {
            uint64_t other[4];
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) other[e] = keys[j + e];
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) place += j + e < n && other[e] > own ? 1u : 0u;
        }
        if (place < kept) out[place] = own;
    }
}

// Element e of 16 bytes of a row.
__device__ __forceinline__ float beam_element(uint16_t, sglkv_v4u v, uint32_t e) {
    return __uint_as_float(e & 1 ? v[e / 2] & 0xFFFF0000u : v[e / 2] << 16);
}
__device__ __forceinline__ float beam_element(float, sglkv_v4u v, uint32_t e) { return __uint_as_float(v[e]); }

// A split of a row, SGLKV_BEAM_CHUNK tokens a round, and with the row's first split
// its few elements before the first and behind the last multiple of 16 bytes.
//  - A round takes each lane's maximum and its sum at that maximum, nothing else.
//  - Then a bound that `kept` tokens reach: a wave's kept-th largest of its lanes'
//    maxima, to 16 bits; the largest of the waves'. Lanes that reach it are few, and
//    their tokens are read again, by all threads: some `kept` reach it, which are
//    ranked among themselves.
template <typename E>
__device__ __forceinline__ void beam_rows_body(const sglkv_beam_params &p) {
    constexpr uint32_t W = SGLKV_BEAM_THREADS / 64, PER = 16 / sizeof(E), VECTORS = SGLKV_BEAM_OWN / PER;
    constexpr uint32_t ROUND = SGLKV_BEAM_CHUNK / PER;  // vectors of a round
    __shared__ float2 part[W];
    __shared__ uint32_t edge[W], lanes, count, who[SGLKV_BEAM_THREADS];
    __shared__ uint64_t best[2][W], list[SGLKV_BEAM_LIST + 4];
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, kept = p.kept;
    const uint32_t split = blockIdx.x % p.splits;
    const uint64_t row = blockIdx.x / p.splits;
    const uint64_t at = reinterpret_cast<uint64_t>(p.logits) + row * p.row_stride * sizeof(E);
    const uint32_t before = static_cast<uint32_t>((16 - at % 16) % 16 / sizeof(E)), lead = before < p.vocab ? before : p.vocab;
    const uint32_t vectors = (p.vocab - lead) / PER, tail = p.vocab - lead - PER * vectors;
    const uint32_t begin = split * p.rounds * ROUND;
    const uint32_t left = begin < vectors ? (vectors - begin + ROUND - 1) / ROUND : 0, rounds = left < p.rounds ? left : p.rounds;
    typedef __attribute__((address_space(1))) const sglkv_v4u vec_t;
    typedef __attribute__((address_space(1))) const E elt_t;
    vec_t *const row_vectors = reinterpret_cast<vec_t *>(at + lead * sizeof(E));
    // (Every load is made, so that the compiler counts those in flight: behind the row, the last vector's again.)
    auto load = [&](uint32_t round, sglkv_v4u (&raw)[VECTORS]) {
#pragma unroll
        for (uint32_t i = 0; i < VECTORS; ++i) {
            const uint32_t v = begin + round * ROUND + tid + i * SGLKV_BEAM_THREADS;
            raw[i] = __builtin_nontemporal_load(row_vectors + (v < vectors ? v : vectors - 1));
        }
    };
    auto odd_token = [&](uint32_t thread) { return thread < lead ? thread : PER * vectors + thread; };
    const bool has_odd = split == 0 && tid < lead + tail;
    float odd = -INFINITY;
    if (has_odd) odd = beam_value(reinterpret_cast<elt_t *>(at)[odd_token(tid)]);
    if (tid == 0) lanes = count = 0;
    const float log2e = 1.4426950408889634f;
    // (At 0 where there is no maximum yet: its terms are 0, or NaN if it is +inf. A NaN stays in the sum.)
    float m = odd;
    // (Of the rounds' sums: up to 64 of 32 logits, whose running sum in 32 bits would be off by a rounding for each logit.)
    double total = __builtin_amdgcn_exp2f((odd - (odd > -INFINITY ? odd : 0.0f)) * log2e);
    auto work = [&](uint32_t round, sglkv_v4u (&raw)[VECTORS]) {
        if (begin + (round + 1) * ROUND > vectors) {
            const uint32_t none = sizeof(E) == 2 ? 0xFF80FF80u : 0xFF800000u;  // -inf
#pragma unroll
            for (uint32_t i = 0; i < VECTORS; ++i)
                if (begin + round * ROUND + tid + i * SGLKV_BEAM_THREADS >= vectors) raw[i] = sglkv_v4u{none, none, none, none};
        }
        float higher = m;
#pragma unroll
        for (uint32_t v = 0; v < VECTORS; ++v) {
#pragma unroll
            for (uint32_t e = 0; e < PER; e += 2)
                higher = attn_max3(higher, beam_element(E(), raw[v], e), beam_element(E(), raw[v], e + 1));
        }
        const float top = higher > -INFINITY ? higher : 0.0f;
        const float scale = __builtin_amdgcn_exp2f((m > -INFINITY ? m - top : 0.0f) * log2e);
        m = higher;
        float sum = 0.0f;
        // (The floats are made anew from the 16 bytes: kept, they would take as many registers again.)
#pragma unroll
        for (uint32_t v = 0; v < VECTORS; ++v) {
            asm volatile("" : "+v"(raw[v]));
#pragma unroll
            for (uint32_t e = 0; e < PER; ++e) sum += __builtin_amdgcn_exp2f((beam_element(E(), raw[v], e) - top) * log2e);
        }
        total = __builtin_fma(total, static_cast<double>(scale), static_cast<double>(sum));
    };
    if (rounds) {
        // The next round's loads are in flight while one is worked on.
        sglkv_v4u raw[VECTORS], next[VECTORS];
        load(0, raw);
        uint32_t round = 0;
        for (; round + 1 < rounds; ++round) {
            load(round + 1, next);
            work(round, raw);
#pragma unroll
            for (uint32_t v = 0; v < VECTORS; ++v) raw[v] = next[v];
        }
        work(round, raw);
    }
    float l = static_cast<float>(total);
    const uint32_t mine = beam_order32(m);
    uint32_t bound = 0;
    if (kept <= 64) {
#pragma unroll
        for (uint32_t bit = 31; bit >= 16; --bit) {
            const uint32_t more = bound | 1u << bit;
            if (__popcll(__ballot(mine >= more)) >= kept) bound = more;
        }
    }
    // The lanes' sums at the wave's maximum, the waves' at the workgroup's.
    auto at_maximum = [&](float own_m, float own_l, float top) {
        return own_m > -INFINITY ? own_l * __builtin_amdgcn_exp2f((own_m - top) * log2e) : own_l;
    };
    const float wave_m = beam_max(m);
    const float wave_l = beam_sum(at_maximum(m, l, wave_m));
    if (lane == 0) {
        part[wave] = make_float2(wave_m, wave_l);
        edge[wave] = bound;
    }
    __syncthreads();
#pragma unroll
    for (uint32_t w = 0; w < W; ++w) bound = edge[w] > bound ? edge[w] : bound;
    if (mine != 0 && mine >= bound) who[atomicAdd(&lanes, 1u)] = tid;
    const uint64_t out = row * p.splits + split;
    if (tid == 0) {
        m = part[0].x;
#pragma unroll
        for (uint32_t w = 1; w < W; ++w) m = fmaxf(m, part[w].x);
        l = 0.0f;
#pragma unroll
        for (uint32_t w = 0; w < W; ++w) l += at_maximum(part[w].x, part[w].y, m);
        reinterpret_cast<float2 *>(p.partial)[out] = make_float2(m, l);
    }
    __syncthreads();
    // Compared as floats, of which none below the lowest finite one takes part.
    const float reach = bound == 0 ? -3.402823466e+38f : __uint_as_float(bound & 0x80000000u ? bound & 0x7FFFFFFFu : ~bound);
    auto take = [&](float x, uint32_t t) {
        if (!(x >= reach)) return;
        const uint32_t place = atomicAdd(&count, 1u);
        if (place < SGLKV_BEAM_LIST) list[place] = beam_key(x, t);
    };
    const uint32_t each = rounds * VECTORS + 1;  // a lane's vectors, and its odd element
    for (uint32_t i = tid; i < lanes * each; i += SGLKV_BEAM_THREADS) {
        const uint32_t of = i / each, j = i - of * each, thread = who[of], v = begin + thread + j * SGLKV_BEAM_THREADS;
        if (j + 1 == each) {
            if (split == 0 && thread < lead + tail) take(beam_value(reinterpret_cast<elt_t *>(at)[odd_token(thread)]), odd_token(thread));
        } else if (v < vectors) {
            const sglkv_v4u x = row_vectors[v];
            float most = beam_element(E(), x, 0);
#pragma unroll
            for (uint32_t e = 1; e < PER; ++e) most = fmaxf(most, beam_element(E(), x, e));
            if (most >= reach) {
#pragma unroll
                for (uint32_t e = 0; e < PER; ++e) take(beam_element(E(), x, e), lead + PER * v + e);
            }
        }
    }
    __syncthreads();
    const uint32_t n = count;
    uint64_t *const to = p.candidates + out * kept;
    if (n <= SGLKV_BEAM_LIST) {
        beam_rank<SGLKV_BEAM_THREADS>(list, n, kept, to);
        for (uint32_t k = n + tid; k < kept; k += SGLKV_BEAM_THREADS) to[k] = 0;
        return;
    }
    // Many equal ones, or more kept than a wave has lanes: the largest keys, one after another; each thread's next one
    // from its tokens in memory.
    auto scan = [&](uint64_t below) {
        uint64_t most = 0;
        auto look = [&](uint32_t t) {
            const uint64_t key = beam_key(beam_value(reinterpret_cast<elt_t *>(at)[t]), t);
            most = key < below ? beam_larger(most, key) : most;
        };
        if (has_odd) look(odd_token(tid));
#pragma unroll 1
        for (uint32_t i = 0; i < rounds * VECTORS; ++i) {
            const uint32_t v = begin + tid + i * SGLKV_BEAM_THREADS;
            if (v >= vectors) break;
#pragma unroll 1
            for (uint32_t e = 0; e < PER; ++e) look(lead + PER * v + e);
        }
        return most;
    };
    uint64_t following = scan(~0ull);
    for (uint32_t k = 0; k < kept; ++k) {
        uint64_t largest = beam_max(following);
        if (lane == 0) best[k & 1][wave] = largest;
        __syncthreads();
        largest = best[k & 1][0];
#pragma unroll
        for (uint32_t w = 1; w < W; ++w) largest = beam_larger(largest, best[k & 1][w]);
        if (tid == 0) to[k] = largest;
        if (largest != 0 && largest == following) following = scan(largest);
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
    uint64_t key[4];
    auto load = [&](uint32_t i0) {
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) key[e] = i0 + 64 * e + lane < all ? keys[i0 + 64 * e + lane] : 0;
    };
    load(0);
    // Every split's last key is reached by `kept` of the row's.
    const uint64_t bound = beam_max(mine[kept - 1]);
    const bool odd = __ballot(own.y != own.y || own.x == INFINITY) != 0;
    const float m = beam_max(own.x);
    const double sum =
        beam_sum(lane < p.splits && own.y > 0.0f ? static_cast<double>(own.y) * exp(static_cast<double>(own.x) - m) : 0.0);
    beam_base base;
    base.top = m;
    base.offset = odd || m == -INFINITY ? NAN : static_cast<double>(score) - log(sum);
    uint32_t n = 0;
    for (uint32_t i0 = 0;;) {
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) {
            const bool in = key[e] != 0 && key[e] >= bound;
            const uint64_t who = __ballot(in);
            const uint32_t place = n + __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(who >> 32),
                                                                 __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(who), 0));
            if (in && place < SGLKV_BEAM_LIST) list[place] = key[e];
            n += __popcll(who);
        }
        if ((i0 += 256) >= all) break;
        load(i0);
    }
    __builtin_amdgcn_wave_barrier();
    if (n <= SGLKV_BEAM_LIST) {
        beam_rank<64>(list, n, kept, out);
    } else {
        // The splits' lists descend: their heads are compared, and the largest is taken.
        uint32_t next = 0;
        uint64_t head = lane < p.splits ? mine[0] : 0;
        for (uint32_t k = 0; k < kept; ++k) {
            const uint64_t top = beam_max(head);
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
    __shared__ uint64_t lists[W][SGLKV_BEAM_LIST + 4], finals[SGLKV_BEAM_FINALS], orders[SGLKV_BEAM_FINALS];
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
        for (uint32_t j = 0; j < all; j += 4) {
            uint64_t other[4];
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) other[e] = orders[j + e];
            // (Equal ones before the lane's own are larger than it, by 1.)
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) rank += j + e < all && other[e] + (j + e < tid ? 1 : 0) > own ? 1u : 0u;
        }
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
        const uint64_t top = beam_max(best);
        const uint32_t lowest = beam_all(top != 0 && best == top ? beam : 0xFFFFFFFFu, [](uint32_t a, uint32_t b) { return a < b ? a : b; });
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
