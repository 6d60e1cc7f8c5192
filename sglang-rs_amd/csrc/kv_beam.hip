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

template <typename E>
__device__ __forceinline__ void beam_rows_body(const sglkv_beam_params &p) {
    constexpr uint32_t W = SGLKV_BEAM_THREADS / 64, N = SGLKV_BEAM_OWN;
    __shared__ float part[W];
    __shared__ uint64_t best[2][W];
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const uint32_t split = blockIdx.x % p.splits;
    const uint64_t row = blockIdx.x / p.splits;
    const E *at = static_cast<const E *>(p.logits) + row * p.row_stride;
    const uint32_t first = split * SGLKV_BEAM_CHUNK + tid;
    float x[N];
#pragma unroll
    for (uint32_t i = 0; i < N; ++i) {
        const uint32_t v = first + i * SGLKV_BEAM_THREADS;
        x[i] = v < p.vocab ? beam_value(at[v]) : -INFINITY;
    }
    // The maximum; a NaN stays (fmaxf would drop it).
    float m = -INFINITY, odd = 0.0f;
#pragma unroll
    for (uint32_t i = 0; i < N; ++i) {
        m = fmaxf(m, x[i]);
        odd = x[i] != x[i] ? x[i] : odd;
    }
#pragma unroll
    for (uint32_t d = 1; d < 64; d <<= 1) {
        m = fmaxf(m, __shfl_xor(m, d));
        odd += __shfl_xor(odd, d);
    }
    if (lane == 0) part[wave] = odd != odd ? odd : m;
    __syncthreads();
    m = part[0];
#pragma unroll
    for (uint32_t w = 1; w < W; ++w) m = m != m || part[w] != part[w] ? NAN : fmaxf(m, part[w]);
    float l = 0.0f;
    const bool finite = m > -INFINITY && m < INFINITY;
    if (finite) {
#pragma unroll
        for (uint32_t i = 0; i < N; ++i) l += __expf(x[i] - m);
    }
#pragma unroll
    for (uint32_t d = 1; d < 64; d <<= 1) l += __shfl_xor(l, d);
    __syncthreads();
    if (lane == 0) part[wave] = l;
    __syncthreads();
    const uint64_t out = row * p.splits + split;
    if (tid == 0) {
        l = part[0];
        for (uint32_t w = 1; w < W; ++w) l += part[w];
        p.partial[2 * out] = m;
        p.partial[2 * out + 1] = l;
    }
    // The largest keys, one after another.
    uint64_t mine = 0;
#pragma unroll
    for (uint32_t i = 0; i < N; ++i) mine = beam_larger(mine, beam_key(x[i], first + i * SGLKV_BEAM_THREADS));
    for (uint32_t k = 0; k < p.kept; ++k) {
        uint64_t top = mine;
#pragma unroll
        for (uint32_t d = 1; d < 64; d <<= 1) top = beam_larger(top, __shfl_xor(top, d));
        if (lane == 0) best[k & 1][wave] = top;
        __syncthreads();
        top = best[k & 1][0];
#pragma unroll
        for (uint32_t w = 1; w < W; ++w) top = beam_larger(top, best[k & 1][w]);
        if (tid == 0) p.candidates[out * p.kept + k] = top;
        if (top != 0 && top == mine) {
            mine = 0;
#pragma unroll
            for (uint32_t i = 0; i < N; ++i) {
                const uint64_t key = beam_key(x[i], first + i * SGLKV_BEAM_THREADS);
                mine = key < top ? beam_larger(mine, key) : mine;
            }
        }
    }
}

// A double as a key of the same order (no NaN).
__device__ __forceinline__ uint64_t beam_order(double x) {
    const uint64_t b = __builtin_bit_cast(uint64_t, x + 0.0);
    return b >> 63 ? ~b : b | 1ull << 63;
}

// A workgroup a request: a wave joins a beam's splits, lane l split l (the host
// has at most 64); then the first wave joins the beams, lane l beams l, l + 64, ....
// Both join lists that descend: their heads are compared, the largest is taken.
__device__ __forceinline__ void beam_join_body(const sglkv_beam_params &p) {
    // A token's score is offset + (logit - top); an offset of NaN: the beam takes no part.
    __shared__ double offset[SGLKV_BEAM_MAX_BEAMS];
    __shared__ float tops[SGLKV_BEAM_MAX_BEAMS];
    __shared__ uint32_t place[SGLKV_BEAM_MAX_BEAMS];
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t request = blockIdx.x, kept = p.kept;
    const uint64_t rows = static_cast<uint64_t>(request) * p.beams;
    for (uint32_t b = wave; b < p.beams; b += SGLKV_BEAM_JOIN_THREADS / 64) {
        const uint64_t row = rows + b, at = row * p.splits + (lane < p.splits ? lane : 0);
        const float2 own = reinterpret_cast<const float2 *>(p.partial)[at];
        float m = own.x;
        const bool odd = __ballot(m != m || m == INFINITY) != 0;
#pragma unroll
        for (uint32_t d = 1; d < 64; d <<= 1) m = fmaxf(m, __shfl_xor(m, d));
        double sum = lane < p.splits && own.y > 0.0f ? static_cast<double>(own.y) * exp(static_cast<double>(own.x) - m) : 0.0;
#pragma unroll
        for (uint32_t d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d);
        if (lane == 0) {
            offset[b] = odd || m == -INFINITY ? NAN : static_cast<double>(p.scores[row]) - log(sum);
            tops[b] = m;
            place[b] = 0;
        }
        uint64_t *list = p.lists + row * kept;
        const uint64_t *mine = p.candidates + at * kept;
        uint32_t next = 0;
        uint64_t head = lane < p.splits ? mine[0] : 0;
        for (uint32_t k = 0; k < kept; ++k) {
            uint64_t top = head;
#pragma unroll
            for (uint32_t d = 1; d < 64; d <<= 1) top = beam_larger(top, __shfl_xor(top, d));
            if (lane == 0) list[k] = top;
            if (top != 0 && head == top) head = ++next < kept ? mine[next] : 0;
        }
    }
    __syncthreads();
    if (wave != 0) return;
    // The lane's best beam: its score as an ordered key (0: none) and its list's head.
    uint64_t best, head;
    uint32_t beam;
    auto score = [&](uint32_t b, uint64_t key) { return offset[b] + (static_cast<double>(beam_logit(key)) - tops[b]); };
    auto look = [&]() {
        best = 0;
        for (uint32_t b = lane; b < p.beams; b += 64) {
            const uint64_t key = place[b] < kept ? p.lists[(rows + b) * kept + place[b]] : 0;
            const double total = score(b, key);
            const uint64_t o = key != 0 && total - total == 0.0 ? beam_order(total) : 0;  // (infinite or NaN: no difference of 0)
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
        const uint64_t out = static_cast<uint64_t>(request) * kept + k;
        if (lowest == 0xFFFFFFFFu) {
            if (lane == 0) {
                p.best_scores[out] = -INFINITY;
                p.best_parents[out] = p.best_tokens[out] = 0xFFFFFFFFu;
            }
        } else if (best == top && beam == lowest) {
            p.best_scores[out] = static_cast<float>(score(beam, head));
            p.best_parents[out] = static_cast<uint32_t>(rows) + beam;
            p.best_tokens[out] = beam_token(head);
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
