// kv_branch.hip -- the cache's part of decoding along several continuations:
// accepted drafts' rows moved together (keep_drafts), and page tables of beams
// that go on from others (fork_sequences).

namespace {

typedef __attribute__((address_space(1))) const sglkv_v4u brn_src16;
typedef __attribute__((address_space(1))) sglkv_v4u brn_dst16;

// Offset of position `slot` in tensor t of the layer, heads aside; the slot is
// inside the pool.
__device__ __forceinline__ uint64_t brn_row(const sglkv_side &s, uint32_t tensor, uint32_t slot) {
    const uint32_t page = slot / s.page_size;
    return page * s.stride[tensor] + (slot - page * s.page_size) * s.pos_mult[tensor];
}

// ---- keep_drafts ------------------------------------------------------------
//
// Row i <- row kept[i] >= i, in place: destinations trail the sources. A thread
// owns the same piece of every row and takes the rows in the list's order, a few
// at a time (all read before any is written), so nothing is written before it is
// read and no thread waits for another.

template <typename V>
__device__ __forceinline__ void brn_keep_body(const sglkv_keep_params &p) {
    typedef __attribute__((address_space(1))) const V src_t;
    typedef __attribute__((address_space(1))) V dst_t;
    constexpr uint32_t U = 8;
    __shared__ uint64_t from[2][SGLKV_KEEP_ROWS], to[2][SGLKV_KEEP_ROWS];
    const uint32_t tid = threadIdx.x, layer = blockIdx.y;
    const uint64_t req = blockIdx.x / p.groups;
    const uint32_t group = blockIdx.x % p.groups;
    const bool report = layer == 0 && group == 0;
    const uint32_t *list = p.kept + req * p.max_kept;
    const uint64_t s = p.request_slot_offsets[req], e = p.request_slot_offsets[req + 1], context = p.request_lengths[req];
    // The whole list first: a request moves all of its rows or none.
    uint32_t bad = s > e || e > p.sequence_slot_count || context > e - s ? SGLKV_FLAG_ATTN_SEQUENCE : 0u;
    const uint64_t room = bad ? 0 : e - s - context;
    uint32_t count = 0;
    if (!bad)
        for (uint32_t i = tid; i < p.max_kept; i += SGLKV_KEEP_THREADS) {
            const uint32_t k = list[i], before = i ? list[i - 1] : 0;
            if (k == SGLKV_SELECT_NONE) continue;
            count = i + 1;
            if (k >= room || (i && before >= k)) {
                bad |= SGLKV_FLAG_ATTN_SEQUENCE;
            } else if (k != i) {
                if (p.sequence_slots[s + context + k] >= p.pool.slot_count ||
                    p.sequence_slots[s + context + i] >= p.pool.slot_count)
                    bad |= SGLKV_FLAG_ATTN_SLOT;
            }
        }
    if (bad && report) atomicOr(p.flag, bad);
    // (Entries behind NONE do not ascend: the last entry's place is the count.)
    uint32_t *const most = reinterpret_cast<uint32_t *>(from);
    if (tid == 0) *most = 0;
    if (__syncthreads_or(bad)) return;
    atomicMax(most, count);
    __syncthreads();
    count = *most;
    const uint64_t base = layer * p.pool.layer_stride;
    for (uint32_t r0 = 0; r0 < count; r0 += SGLKV_KEEP_ROWS) {
        const uint32_t rows = count - r0 < SGLKV_KEEP_ROWS ? count - r0 : SGLKV_KEEP_ROWS;
        __syncthreads();
        if (tid < rows) {
            const uint32_t i = r0 + tid, k = list[i];
#pragma unroll
            for (uint32_t t = 0; t < 2; ++t) {
                const bool moves = t < p.tensors && k != i;
                from[t][tid] = moves ? brn_row(p.pool, t, static_cast<uint32_t>(p.sequence_slots[s + context + k])) : SGLKV_INVALID_OFFSET;
                to[t][tid] = moves ? brn_row(p.pool, t, static_cast<uint32_t>(p.sequence_slots[s + context + i])) : 0;
            }
        }
        __syncthreads();
        const uint32_t first = p.heads * p.chunk_pieces[0];
        for (uint32_t piece = group * SGLKV_KEEP_THREADS + tid; piece < p.pieces; piece += p.groups * SGLKV_KEEP_THREADS) {
            const uint32_t t = piece >= first, x = t ? piece - first : piece, h = x / p.chunk_pieces[t];
            const uint64_t at = p.pool.plane[t] + base + h * p.pool.head_stride[t] + (x - h * p.chunk_pieces[t]) * sizeof(V);
            for (uint32_t r = 0; r < rows; r += U) {
                V v[U];
#pragma unroll
                for (uint32_t u = 0; u < U; ++u) {
                    const uint64_t o = r + u < rows ? from[t][r + u] : SGLKV_INVALID_OFFSET;
                    if (o != SGLKV_INVALID_OFFSET) v[u] = *reinterpret_cast<src_t *>(at + o);
                }
#pragma unroll
                for (uint32_t u = 0; u < U; ++u)
                    if (r + u < rows && from[t][r + u] != SGLKV_INVALID_OFFSET) *reinterpret_cast<dst_t *>(at + to[t][r + u]) = v[u];
            }
        }
    }
}

// ---- fork_sequences ---------------------------------------------------------

// What sequence s needs: its parent's tokens, pages of these, new pages.
struct brn_need {
    uint32_t parent;
    uint64_t length, full, pages, need;
    uint32_t fresh;  // new pages, a copied last page first among them
    bool copies;
};
__device__ __forceinline__ brn_need brn_sequence(const sglkv_fork_params &p, uint32_t s, const uint32_t *first) {
    brn_need n;
    n.parent = p.parents[s];
    const bool live = n.parent != SGLKV_FORK_NONE;
    n.length = live ? p.lengths[n.parent] : 0;
    n.full = n.length / p.pool.page_size;
    n.pages = n.full + (n.length % p.pool.page_size != 0);
    const uint64_t end = n.length + p.append;
    n.need = live ? end / p.pool.page_size + (end % p.pool.page_size != 0) : 0;
    n.copies = live && n.pages > n.full && __hip_atomic_load(first + n.parent, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) != s;
    n.fresh = static_cast<uint32_t>(n.need - n.pages) + (n.copies ? 1u : 0u);
    return n;
}

// One workgroup: who is whose first child, how many new pages come before each
// sequence's, and whether all of that holds.
__device__ __forceinline__ void brn_plan_body(const sglkv_fork_params &p) {
    constexpr uint32_t T = SGLKV_FORK_PLAN_THREADS;
    __shared__ uint64_t sums[T / 64];
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const uint64_t room = p.table_pages * p.pool.page_size;  // (host: no overflow)
    for (uint32_t i = tid; i < p.old_sequences; i += T) {
        __hip_atomic_store(p.first + i, SGLKV_FORK_NONE, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __hip_atomic_store(p.children + i, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    for (uint32_t i = tid; i < (p.page_count + 31) / 32; i += T) p.freed[i] = 0;
    uint32_t bad = 0;
    const uint64_t free_count = *p.free_count;
    if (free_count > p.page_count) bad |= SGLKV_FLAG_ATTN_SEQUENCE;
    for (uint32_t i = tid; i < p.old_sequences; i += T)
        if (p.lengths[i] > room) bad |= SGLKV_FLAG_ATTN_SEQUENCE;
    __threadfence();
    __syncthreads();
    for (uint32_t s = tid; s < p.sequences; s += T) {
        const uint32_t parent = p.parents[s];
        if (parent == SGLKV_FORK_NONE) continue;
        if (parent >= p.old_sequences) {
            bad |= SGLKV_FLAG_ATTN_REQUEST;
            continue;
        }
        atomicMin(p.first + parent, s);
        atomicAdd(p.children + parent, 1u);
        const uint64_t length = p.lengths[parent];
        if (length > room || p.append > room - length) bad |= SGLKV_FLAG_ATTN_SEQUENCE;
    }
    __threadfence();
    if (__syncthreads_or(bad)) {
        if (bad) atomicOr(p.flag, bad);
        if (tid == 0) p.head[0] = 0;
        return;
    }
    // New pages before each sequence's: sums over the waves, round by round.
    uint64_t taken = 0;
    for (uint32_t s0 = 0; s0 < p.sequences; s0 += T) {
        const uint32_t s = s0 + tid, own = s < p.sequences ? brn_sequence(p, s, p.first).fresh : 0;
        uint64_t sum = own;
#pragma unroll
        for (uint32_t d = 1; d < 64; d <<= 1) {
            const uint64_t x = __shfl_up(sum, d);
            sum += lane >= d ? x : 0;
        }
        if (lane == 63) sums[wave] = sum;
        __syncthreads();
        uint64_t before = taken, all = 0;
        for (uint32_t w = 0; w < T / 64; ++w) {
            if (w < wave) before += sums[w];
            all += sums[w];
        }
        // (Numbers past the free ones are not used: the call is refused.)
        if (s < p.sequences) p.before[s] = static_cast<uint32_t>(before + sum - own);
        taken += all;
        __syncthreads();
    }
    if (taken > free_count) bad |= SGLKV_FLAG_OUT_OF_PAGES;
    else
        for (uint64_t i = free_count - taken + tid; i < free_count; i += T)
            if (static_cast<uint32_t>(p.free_pages[i]) >= p.page_count) bad |= SGLKV_FLAG_PAGE;
    const bool refused = __syncthreads_or(bad) != 0;
    if (bad) atomicOr(p.flag, bad);
    if (tid == 0) {
        p.head[0] = refused ? 0 : 1;
        p.head[1] = static_cast<uint32_t>(taken);
    }
}

// New page number k of the call.
__device__ __forceinline__ uint32_t brn_fresh(const sglkv_fork_params &p, uint64_t free_count, uint32_t k) {
    return static_cast<uint32_t>(p.free_pages[free_count - 1 - k]);
}

// The new tables, the references, the pages that are freed: a workgroup to each
// new sequence, then to each old one.
__device__ __forceinline__ void brn_tables_body(const sglkv_fork_params &p) {
    if (p.head[0] == 0) return;
    const uint32_t tid = threadIdx.x;
    if (blockIdx.x < p.sequences) {
        const uint32_t s = blockIdx.x;
        const brn_need n = brn_sequence(p, s, p.first);
        const uint64_t free_count = *p.free_count;
        const uint64_t begin = n.copies ? n.full : n.pages;  // new pages from here on
        if (tid == 0) p.forked_lengths[s] = n.length;
        for (uint64_t j = tid; j < p.table_pages; j += SGLKV_FORK_THREADS) {
            int32_t page = -1;
            if (j >= begin && j < n.need) {
                page = static_cast<int32_t>(brn_fresh(p, free_count, p.before[s] + static_cast<uint32_t>(j - begin)));
                p.references[page] = 1;
            } else if (j < n.pages) {
                page = p.tables[n.parent * p.table_pages + j];
                if (static_cast<uint32_t>(page) >= p.page_count) {
                    atomicOr(p.flag, SGLKV_FLAG_PAGE);
                    page = -1;
                }
            }
            p.forked_tables[s * p.table_pages + j] = page;
        }
        return;
    }
    const uint32_t old = blockIdx.x - p.sequences, children = p.children[old];
    const uint64_t length = p.lengths[old], full = length / p.pool.page_size, pages = full + (length % p.pool.page_size != 0);
    for (uint64_t j = tid; j < pages; j += SGLKV_FORK_THREADS) {
        const uint32_t page = static_cast<uint32_t>(p.tables[old * p.table_pages + j]);
        // A row of its own less; one more for each child that shares the page.
        const int32_t change = static_cast<int32_t>(j < full ? children : children ? 1 : 0) - 1;
        if (change == 0) continue;
        if (page >= p.page_count) {
            atomicOr(p.flag, SGLKV_FLAG_PAGE);
            continue;
        }
        const uint32_t was = atomicAdd(p.references + page, static_cast<uint32_t>(change));
        // (No other row's change can follow the one that reaches 0: a row that goes on adds before
        // or after, and its own reference keeps the count above 0 until it is subtracted.)
        if (was + static_cast<uint32_t>(change) == 0) atomicOr(p.freed + page / 32, 1u << (page % 32));
    }
}

// The last pages' rows: a workgroup to each (sequence, layer, tensor), which
// copies the chunks of the heads (head-major pages) or all rows at once.
__device__ __forceinline__ void brn_copy_body(const sglkv_fork_params &p) {
    if (p.head[0] == 0) return;
    const uint32_t s = blockIdx.x, layer = blockIdx.y, t = blockIdx.z, tid = threadIdx.x;
    const brn_need n = brn_sequence(p, s, p.first);
    if (!n.copies) return;
    const uint32_t source = static_cast<uint32_t>(p.tables[n.parent * p.table_pages + n.full]);
    if (source >= p.page_count) return;  // (reported with the tables)
    const uint32_t to = brn_fresh(p, *p.free_count, p.before[s]);
    const uint64_t base = p.pool.plane[t] + layer * p.pool.layer_stride;
    const uint64_t rows = n.length - n.full * p.pool.page_size;
    // A head's rows lie together, and so do a token-major page's whole rows.
    const uint64_t bytes = rows * p.chunk[t];
    for (uint32_t h = 0; h < p.heads; ++h) {
        const uint64_t from_at = base + source * p.pool.stride[t] + h * p.pool.head_stride[t];
        const uint64_t to_at = base + to * p.pool.stride[t] + h * p.pool.head_stride[t];
        uint64_t done = 0;
        if (p.wide) {
            // Both are misaligned alike: 16 bytes at a time from the first multiple of 16.
            const uint64_t lead = (16 - from_at % 16) % 16, head = lead < bytes ? lead : bytes;
            const uint64_t vectors = (bytes - head) / 16;
            for (uint64_t i = tid; i < head; i += SGLKV_FORK_THREADS)
                reinterpret_cast<sglkv_gdst *>(to_at)[i] = reinterpret_cast<sglkv_gsrc *>(from_at)[i];
            for (uint64_t i = tid; i < vectors; i += SGLKV_FORK_THREADS)
                reinterpret_cast<brn_dst16 *>(to_at + head)[i] = reinterpret_cast<brn_src16 *>(from_at + head)[i];
            done = head + 16 * vectors;
        }
        for (uint64_t i = done + tid; i < bytes; i += SGLKV_FORK_THREADS)
            reinterpret_cast<sglkv_gdst *>(to_at)[i] = reinterpret_cast<sglkv_gsrc *>(from_at)[i];
    }
}

// One workgroup: the freed pages behind what is left of the free ones, ascending.
__device__ __forceinline__ void brn_free_body(const sglkv_fork_params &p) {
    constexpr uint32_t T = SGLKV_FORK_PLAN_THREADS;
    __shared__ uint32_t sums[T / 64];
    if (p.head[0] == 0) return;
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, words = (p.page_count + 31) / 32;
    uint64_t end = *p.free_count - p.head[1];
    for (uint32_t w0 = 0; w0 < words; w0 += T) {
        uint32_t bits = w0 + tid < words ? p.freed[w0 + tid] : 0;
        const uint32_t own = __popc(bits);
        uint32_t sum = own;
#pragma unroll
        for (uint32_t d = 1; d < 64; d <<= 1) {
            const uint32_t x = __shfl_up(sum, d);
            sum += lane >= d ? x : 0;
        }
        if (lane == 63) sums[wave] = sum;
        __syncthreads();
        uint64_t at = end + sum - own;
        uint32_t all = 0;
        for (uint32_t w = 0; w < T / 64; ++w) {
            if (w < wave) at += sums[w];
            all += sums[w];
        }
        for (; bits; bits &= bits - 1, ++at)
            if (at < p.page_count) p.free_pages[at] = static_cast<int32_t>(32 * (w0 + tid) + __builtin_ctz(bits));
        end += all;
        __syncthreads();
    }
    // (More than the pool has: the caller's counts and its free pages contradict each other.)
    if (tid == 0) {
        if (end > p.page_count) atomicOr(p.flag, SGLKV_FLAG_PAGE);
        *p.free_count = end < p.page_count ? end : p.page_count;
    }
}

}  // namespace

extern "C" __global__ __launch_bounds__(SGLKV_KEEP_THREADS) void sglkv_keep_drafts_v16(sglkv_keep_params p) {
    brn_keep_body<sglkv_v4u>(p);
}
extern "C" __global__ __launch_bounds__(SGLKV_KEEP_THREADS) void sglkv_keep_drafts_v4(sglkv_keep_params p) {
    brn_keep_body<uint32_t>(p);
}
extern "C" __global__ __launch_bounds__(SGLKV_KEEP_THREADS) void sglkv_keep_drafts_v1(sglkv_keep_params p) {
    brn_keep_body<uint8_t>(p);
}

extern "C" __global__ __launch_bounds__(SGLKV_FORK_PLAN_THREADS) void sglkv_fork_plan(sglkv_fork_params p) { brn_plan_body(p); }
extern "C" __global__ __launch_bounds__(SGLKV_FORK_THREADS) void sglkv_fork_tables(sglkv_fork_params p) { brn_tables_body(p); }
extern "C" __global__ __launch_bounds__(SGLKV_FORK_THREADS) void sglkv_fork_copy(sglkv_fork_params p) { brn_copy_body(p); }
extern "C" __global__ __launch_bounds__(SGLKV_FORK_PLAN_THREADS) void sglkv_fork_free(sglkv_fork_params p) { brn_free_body(p); }
