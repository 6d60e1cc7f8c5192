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
// read and no thread waits for another. Bytes bound it where there are many (64
// requests of 8 rows, 32 layers, 57 MB in and out: 15.7 us, 3.7 TB/s, three quarters
// of the waves' time waiting for rows of 2 KiB; packed rows of 649 bytes, which go
// byte by byte: 28.9 for 21 MB), else three loads one after another: list, slots,
// rows (3 requests, 24 layers: 4.9 us, 7.1 with its launch).

template <typename V>
__device__ __forceinline__ void brn_keep_body(const sglkv_keep_params &p) {
    typedef __attribute__((address_space(1))) const V src_t;
    typedef __attribute__((address_space(1))) V dst_t;
    constexpr uint32_t U = 8;
    __shared__ uint64_t from[2][SGLKV_KEEP_ROWS], to[2][SGLKV_KEEP_ROWS];  // (an entry that stays: from[0] says so)
    __shared__ uint32_t most;
    const uint32_t tid = threadIdx.x, layer = blockIdx.y;
    const uint64_t req = blockIdx.x / p.groups;
    const uint32_t group = blockIdx.x % p.groups;
    const bool report = layer == 0 && group == 0;
    const uint32_t *list = p.kept + req * p.max_kept;
    // (The list does not wait for the request's range, so that the slots are a second step and the rows a third.)
    uint32_t k = tid < p.max_kept ? list[tid] : SGLKV_SELECT_NONE, before = tid && tid < p.max_kept ? list[tid - 1] : 0;
    const uint64_t s = p.request_slot_offsets[req], e = p.request_slot_offsets[req + 1], context = p.request_lengths[req];
    if (tid == 0) most = 0;
    uint32_t bad = s > e || e > p.sequence_slot_count || context > e - s ? SGLKV_FLAG_ATTN_SEQUENCE : 0u;
    const uint64_t room = bad ? 0 : e - s - context;
    // Where entry i's row goes from and to, if it moves; what is wrong with it.
    auto place = [&](uint32_t i, uint32_t k, uint32_t before) {
        const uint32_t at = i % SGLKV_KEEP_ROWS;
        from[0][at] = SGLKV_INVALID_OFFSET;
        if (k == SGLKV_SELECT_NONE) return 0u;
        if (k >= room || (i && before >= k)) return SGLKV_FLAG_ATTN_SEQUENCE;
        if (k == i) return 0u;
        const uint64_t source = p.sequence_slots[s + context + k], dest = p.sequence_slots[s + context + i];
        if (source >= p.pool.slot_count || dest >= p.pool.slot_count) return SGLKV_FLAG_ATTN_SLOT;
#pragma unroll
        for (uint32_t t = 0; t < 2; ++t)
            if (t < p.tensors) {
                from[t][at] = brn_row(p.pool, t, static_cast<uint32_t>(source));
                to[t][at] = brn_row(p.pool, t, static_cast<uint32_t>(dest));
            }
        return 0u;
    };
    // The whole list first, from its end: a request moves all of its rows or none, and the first entries' places stay.
    // (Entries behind NONE do not ascend: the last entry's place is the count.)
    uint32_t count = 0;
    for (uint32_t i0 = p.max_kept > SGLKV_KEEP_ROWS ? (p.max_kept - 1) / SGLKV_KEEP_ROWS * SGLKV_KEEP_ROWS : 0; i0; i0 -= SGLKV_KEEP_ROWS) {
        const uint32_t i = i0 + tid;
        if (i >= p.max_kept) continue;
        const uint32_t own = list[i];
        bad |= place(i, own, list[i - 1]);
        if (own != SGLKV_SELECT_NONE && i >= count) count = i + 1;
    }
    bad |= place(tid, k, before);
    if (k != SGLKV_SELECT_NONE && tid >= count) count = tid + 1;
    if (bad && report) atomicOr(p.flag, bad);
    if (__syncthreads_or(bad)) return;
    if (count) atomicMax(&most, count);
    __syncthreads();
    count = most;
    const uint64_t base = layer * p.pool.layer_stride;
    for (uint32_t r0 = 0; r0 < count; r0 += SGLKV_KEEP_ROWS) {
        const uint32_t rows = count - r0 < SGLKV_KEEP_ROWS ? count - r0 : SGLKV_KEEP_ROWS;
        if (r0) {
            __syncthreads();
            if (tid < rows) (void)place(r0 + tid, list[r0 + tid], 0);
            __syncthreads();
        }
        const uint32_t first = p.heads * p.chunk_pieces[0];
        for (uint32_t piece = group * SGLKV_KEEP_THREADS + tid; piece < p.pieces; piece += p.groups * SGLKV_KEEP_THREADS) {
            const uint32_t t = piece >= first, x = t ? piece - first : piece, h = x / p.chunk_pieces[t];
            const uint64_t at = p.pool.plane[t] + base + h * p.pool.head_stride[t] + (x - h * p.chunk_pieces[t]) * sizeof(V);
            for (uint32_t r = 0; r < rows; r += U) {
                V v[U];
#pragma unroll
                for (uint32_t u = 0; u < U; ++u) {
                    if (r + u < rows && from[0][r + u] != SGLKV_INVALID_OFFSET)
                        v[u] = __builtin_nontemporal_load(reinterpret_cast<src_t *>(at + from[t][r + u]));
                }
#pragma unroll
                for (uint32_t u = 0; u < U; ++u)
                    if (r + u < rows && from[0][r + u] != SGLKV_INVALID_OFFSET)
                        __builtin_nontemporal_store(v[u], reinterpret_cast<dst_t *>(at + to[t][r + u]));
            }
        }
    }
}

// ---- fork_sequences ---------------------------------------------------------
//
// The book-keeping is a chain of short steps: who has which children, how many new
// pages come before each sequence's (a sum), the tables, the references, the freed
// pages in order. Few sequences take one workgroup, which has all of it in LDS;
// many take three launches. The copies are a launch of their own: bytes. Measured:
// 1 request of 4 beams 9.2 us and 3.1 for the copies, 64 of 4 11.8 and 34.4 (166 MB
// in and out, 4.8 TB/s, 0.82 of this library's stream copy: waves wait to issue for
// 0.71 of their time, each vector with a 64-bit address of its own).

// What a sequence needs: its parent's tokens, pages of these, entries that it has
// from its parent (`held`: these pages and, for the lowest child, reserved ones
// behind them), new pages.
struct brn_need {
    uint64_t length, full, pages, held, need;
    uint32_t parent, fresh;  // fresh: new pages, a copied last page first among them
    bool copies;
};
// `takes`: the sequence takes over its parent's last page, as the lowest child of a
// parent that holds it alone. `reserved`: where its parent's reserved pages end, if it
// has them (0: it has none).
__device__ __forceinline__ brn_need brn_sequence(const sglkv_fork_params &p, uint32_t parent, uint64_t length, bool takes,
                                                 uint32_t reserved) {
    brn_need n;
    const bool live = parent != SGLKV_FORK_NONE;
    n.parent = parent;
    n.length = live ? length : 0;
    const uint64_t end = n.length + p.append;
    if (end >> 32 == 0) {  // (a 64-bit division takes a hundred instructions)
        const uint32_t size = p.pool.page_size, l = static_cast<uint32_t>(n.length), e = static_cast<uint32_t>(end);
        n.full = l / size;
        n.pages = n.full + (l % size != 0);
        n.need = live ? e / size + (e % size != 0) : 0;
    } else {
        n.full = n.length / p.pool.page_size;
        n.pages = n.full + (n.length % p.pool.page_size != 0);
        n.need = live ? end / p.pool.page_size + (end % p.pool.page_size != 0) : 0;
    }
    n.copies = n.pages > n.full && !takes;
    n.held = n.pages > reserved ? n.pages : reserved;
    n.fresh = (n.need > n.held ? static_cast<uint32_t>(n.need - n.held) : 0u) + (n.copies ? 1u : 0u);
    return n;
}

// Whether more than old row r holds entry `full` of it, a page that is not full:
// other rows or the caller, by the references of before the call. No child may
// write to it then.
__device__ __forceinline__ bool brn_shared(const sglkv_fork_params &p, uint64_t r, uint64_t full) {
    const uint32_t page = static_cast<uint32_t>(p.tables[r * p.table_pages + full]);
    return page < p.page_count && p.references[page] > 1;
}

// Entries of old row r that are pages: its own `pages` and, with keep_reserved, those
// behind them. What ends these is -1, or reported. (A step for each reserved page:
// few. The host bounds the row.)
__device__ __forceinline__ uint32_t brn_held(const sglkv_fork_params &p, uint64_t r, uint64_t pages) {
    const int32_t *row = p.tables + r * p.table_pages;
    for (uint64_t j = pages; j < p.table_pages; ++j)
        if (static_cast<uint32_t>(row[j]) >= p.page_count) {
            if (row[j] != -1) atomicOr(p.flag, SGLKV_FLAG_PAGE);
            return static_cast<uint32_t>(j);
        }
    return static_cast<uint32_t>(p.table_pages);
}

// Exclusive sums over a workgroup of 1,024 threads in their order, and the total.
// `sums`: a word for each wave; a barrier before and behind.
__device__ __forceinline__ uint64_t brn_sum(uint64_t own, uint64_t *sums, uint64_t *all) {
    constexpr uint32_t W = SGLKV_FORK_PLAN_THREADS / 64;
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    uint64_t sum = own;
#pragma unroll
    for (uint32_t d = 1; d < 64; d <<= 1) {
        const uint64_t x = __shfl_up(sum, d);
        sum += lane >= d ? x : 0;
    }
    if (lane == 63) sums[wave] = sum;
    __syncthreads();
    uint64_t before = 0, total = 0;
#pragma unroll
    for (uint32_t w = 0; w < W; ++w) {
        before += w < wave ? sums[w] : 0;
        total += sums[w];
    }
    *all = total;
    __syncthreads();
    return before + sum - own;
}

// New page number k of the call.
__device__ __forceinline__ uint32_t brn_fresh(const sglkv_fork_params &p, uint64_t free_count, uint32_t k) {
    return static_cast<uint32_t>(p.free_pages[free_count - 1 - k]);
}

// Entry j of sequence s's new row. `old`: its parent's entry j; fresh(k): new page
// number k of the call.
template <typename F>
__device__ __forceinline__ int32_t brn_entry(const sglkv_fork_params &p, const brn_need &n, uint64_t j, int32_t old, F fresh,
                                             uint32_t before) {
    const bool behind = j >= n.held;
    if (behind ? j < n.need : n.copies && j == n.full) {
        const uint32_t page = fresh(before + (behind ? (n.copies ? 1u : 0u) + static_cast<uint32_t>(j - n.held) : 0u));
        p.references[page] = 1;
        return static_cast<int32_t>(page);
    }
    if (behind) return -1;
    if (static_cast<uint32_t>(old) < p.page_count) return old;
    atomicOr(p.flag, SGLKV_FLAG_PAGE);
    return -1;
}

// Entry j of an old row of `length` tokens that `children` go on from: a row of its
// own less, and one more for each child that shares the page (its last one, if it
// is not full: for the child that takes it over; a reserved one: for the lowest).
// True: the page is held by nothing any more. (No other row's change can follow the
// one that reaches 0: a row that goes on holds its own reference until then.)
__device__ __forceinline__ bool brn_release(const sglkv_fork_params &p, uint64_t length, uint64_t j, uint32_t children, int32_t entry) {
    const uint64_t next = (j + 1) * p.pool.page_size;
    const uint32_t count = children & ~SGLKV_FORK_SHARED;
    const bool goes_on = count && (count == children || j * p.pool.page_size >= length);
    const int32_t change = static_cast<int32_t>(next <= length ? count : goes_on ? 1 : 0) - 1;
    if (change == 0) return false;
    const uint32_t page = static_cast<uint32_t>(entry);
    if (page >= p.page_count) {
        atomicOr(p.flag, SGLKV_FLAG_PAGE);
        return false;
    }
    return atomicAdd(p.references + page, static_cast<uint32_t>(change)) + static_cast<uint32_t>(change) == 0;
}

// The copy of a last page to page `to`, if its source is one.
__device__ __forceinline__ sglkv_page_copy brn_copy_of(const sglkv_fork_params &p, const brn_need &n, uint32_t to) {
    sglkv_page_copy c;
    c.source = static_cast<uint32_t>(p.tables[n.parent * p.table_pages + n.full]);
    c.to = to;
    c.rows = c.source < p.page_count ? static_cast<uint32_t>(n.length - n.full * p.pool.page_size) : 0;
    return c;
}

// The freed pages of 32 for each thread behind the `end` free ones, ascending.
__device__ __forceinline__ void brn_append(const sglkv_fork_params &p, uint32_t word, uint32_t bits, uint64_t at) {
    for (; bits; bits &= bits - 1, ++at)
        if (at < p.page_count) p.free_pages[at] = static_cast<int32_t>(32 * word + __builtin_ctz(bits));
}
__device__ __forceinline__ void brn_free_count(const sglkv_fork_params &p, uint64_t end) {
    // (More than the pool has: the caller's counts and its free pages contradict each other.)
    if (end > p.page_count) atomicOr(p.flag, SGLKV_FLAG_PAGE);
    *p.free_count = end < p.page_count ? end : p.page_count;
}

// Everything but the copies of few sequences, in one workgroup.
__device__ __forceinline__ void brn_small_body(const sglkv_fork_params &p) {
    constexpr uint32_t T = SGLKV_FORK_PLAN_THREADS, N = SGLKV_FORK_SMALL_SEQUENCES, U = 4;
    extern __shared__ uint32_t brn_bits[];  // a bit for each page that is freed
    __shared__ uint64_t sums[T / 64];
    __shared__ uint32_t parents[N], lengths[N], first[N], children[N], held[N], before[N], place[N], top[T];  // top: the first new pages
    const uint32_t tid = threadIdx.x, words = (p.page_count + 31) / 32;
    const uint32_t width = static_cast<uint32_t>(p.table_pages), room = width * p.pool.page_size;  // (host: below 2^31)
    const uint32_t old_entries = p.old_sequences * width, new_entries = p.sequences * width;
    // The first entries of the old tables, ahead of what says which of them count.
    int32_t early[U];
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) early[u] = p.tables[tid + T * u < old_entries ? tid + T * u : 0];
    const uint64_t free_count = *p.free_count;
    uint32_t bad = free_count > p.page_count ? SGLKV_FLAG_ATTN_SEQUENCE : 0u;
    for (uint32_t i = tid; i < p.old_sequences; i += T) {
        const uint64_t length = p.lengths[i];
        if (length > room) bad |= SGLKV_FLAG_ATTN_SEQUENCE;
        lengths[i] = static_cast<uint32_t>(length);
        first[i] = SGLKV_FORK_NONE;
        children[i] = 0;
    }
    for (uint32_t s = tid; s < p.sequences; s += T) parents[s] = p.parents[s];
    for (uint32_t i = tid; i < words; i += T) brn_bits[i] = 0;
    if (free_count <= p.page_count && tid < free_count) top[tid] = static_cast<uint32_t>(p.free_pages[free_count - 1 - tid]);
    __syncthreads();
    // (The new tables' first entries, too.)
    int32_t old[U];
    auto parent_entry = [&](uint32_t i) {
        const uint32_t s = i < new_entries ? i / width : 0, parent = parents[s];
        return i < new_entries && parent < p.old_sequences ? p.tables[parent * width + (i - s * width)] : -1;
    };
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) old[u] = parent_entry(T * u + tid);
    auto fresh = [&](uint32_t k) { return k < T ? top[k] : brn_fresh(p, free_count, k); };
    for (uint32_t i = tid; i < p.old_sequences; i += T) {
        const uint32_t length = lengths[i], full = length / p.pool.page_size, pages = full + (full * p.pool.page_size != length);
        held[i] = pages;
        if (length > room) continue;
        if (pages != full && brn_shared(p, i, full)) atomicOr(children + i, SGLKV_FORK_SHARED);
        if (p.keep_reserved) held[i] = brn_held(p, i, pages);
    }
    for (uint32_t s = tid; s < p.sequences; s += T) {
        const uint32_t parent = parents[s];
        if (parent == SGLKV_FORK_NONE) continue;
        if (parent >= p.old_sequences) {
            bad |= SGLKV_FLAG_ATTN_REQUEST;
            continue;
        }
        atomicMin(first + parent, s);
        atomicAdd(children + parent, 1u);
        if (lengths[parent] > room || p.append > room - lengths[parent]) bad |= SGLKV_FLAG_ATTN_SEQUENCE;
    }
    if (__syncthreads_or(bad)) {
        if (bad) atomicOr(p.flag, bad);
        if (tid == 0) p.head[0] = p.head[2] = 0;
        return;
    }
    auto need = [&](uint32_t s) {
        const uint32_t parent = parents[s];
        const bool live = parent != SGLKV_FORK_NONE;
        const bool lowest = live && first[parent] == s;
        return brn_sequence(p, parent, live ? lengths[parent] : 0, !live || (lowest && !(children[parent] & SGLKV_FORK_SHARED)),
                            lowest ? held[parent] : 0);
    };
    // New pages, and copies, before each sequence's.
    uint64_t done = 0;
    for (uint32_t s0 = 0; s0 < p.sequences; s0 += T) {
        const uint32_t s = s0 + tid;
        uint64_t own = 0, all;
        if (s < p.sequences) {
            const brn_need n = need(s);
            own = n.fresh | static_cast<uint64_t>(n.copies) << 32;
        }
        const uint64_t at = done + brn_sum(own, sums, &all);
        if (s < p.sequences) {
            before[s] = static_cast<uint32_t>(at);
            place[s] = static_cast<uint32_t>(at >> 32);
        }
        done += all;
    }
    const uint32_t taken = static_cast<uint32_t>(done), copies = static_cast<uint32_t>(done >> 32);
    if (taken > free_count) {
        bad = SGLKV_FLAG_OUT_OF_PAGES;
    } else {
        for (uint32_t i = tid; i < taken; i += T)
            if (fresh(i) >= p.page_count) bad |= SGLKV_FLAG_PAGE;
    }
    const bool refused = __syncthreads_or(bad) != 0;
    if (tid == 0) {
        p.head[0] = refused ? 0 : 1;
        p.head[2] = refused ? 0 : copies;
    }
    if (refused) {
        if (bad) atomicOr(p.flag, bad);
        return;
    }
    for (uint32_t s = tid; s < p.sequences; s += T) {
        const brn_need n = need(s);
        p.forked_lengths[s] = n.length;
        if (n.copies) p.copies[place[s]] = brn_copy_of(p, n, fresh(before[s]));
    }
    for (uint32_t i0 = 0; i0 < new_entries; i0 += U * T) {
        if (i0)
#pragma unroll
            for (uint32_t u = 0; u < U; ++u) old[u] = parent_entry(i0 + T * u + tid);
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) {
            const uint32_t i = i0 + T * u + tid, s = i / width;
            if (i < new_entries) p.forked_tables[i] = brn_entry(p, need(s), i - s * width, old[u], fresh, before[s]);
        }
    }
    for (uint32_t i0 = 0; i0 < old_entries; i0 += U * T)
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) {
            const uint32_t i = i0 + T * u + tid, r = i / width, j = i - r * width;
            if (i >= old_entries || j >= held[r]) continue;
            const int32_t entry = i0 == 0 ? early[u] : p.tables[i];
            if (brn_release(p, lengths[r], j, children[r], entry)) atomicOr(brn_bits + entry / 32, 1u << (entry % 32));
        }
    __syncthreads();
    uint64_t end = free_count - taken;
    for (uint32_t w0 = 0; w0 < words; w0 += T) {
        const uint32_t bits = w0 + tid < words ? brn_bits[w0 + tid] : 0;
        uint64_t all;
        const uint64_t at = end + brn_sum(__popc(bits), sums, &all);
        brn_append(p, w0 + tid, bits, at);
        end += all;
    }
    if (tid == 0) brn_free_count(p, end);
}

// The same in three launches. One workgroup: who is whose first child, how many new
// pages come before each sequence's, and whether all of that holds.
__device__ __forceinline__ uint32_t brn_load(const uint32_t *at) {
    return __hip_atomic_load(at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ brn_need brn_sequence(const sglkv_fork_params &p, uint32_t s) {
    const uint32_t parent = p.parents[s];
    if (parent == SGLKV_FORK_NONE) return brn_sequence(p, parent, 0, true, 0);
    const bool lowest = brn_load(p.first + parent) == s;
    const bool takes = lowest && !(brn_load(p.children + parent) & SGLKV_FORK_SHARED);
    return brn_sequence(p, parent, p.lengths[parent], takes, p.keep_reserved && lowest ? brn_load(p.held + parent) : 0);
}
__device__ __forceinline__ void brn_plan_body(const sglkv_fork_params &p) {
    constexpr uint32_t T = SGLKV_FORK_PLAN_THREADS;
    __shared__ uint64_t sums[T / 64];
    const uint32_t tid = threadIdx.x;
    const uint64_t room = p.table_pages * p.pool.page_size;  // (host: no overflow)
    uint32_t bad = 0;
    const uint64_t free_count = *p.free_count;
    if (free_count > p.page_count) bad |= SGLKV_FLAG_ATTN_SEQUENCE;
    for (uint32_t i = tid; i < p.old_sequences; i += T) {
        __hip_atomic_store(p.first + i, SGLKV_FORK_NONE, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        const uint64_t length = p.lengths[i], full = length / p.pool.page_size;
        if (length > room) bad |= SGLKV_FLAG_ATTN_SEQUENCE;
        const bool shared = length <= room && full * p.pool.page_size != length && brn_shared(p, i, full);
        __hip_atomic_store(p.children + i, shared ? SGLKV_FORK_SHARED : 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (p.keep_reserved && length <= room)
            __hip_atomic_store(p.held + i, brn_held(p, i, full + (full * p.pool.page_size != length)), __ATOMIC_RELAXED,
                               __HIP_MEMORY_SCOPE_AGENT);
    }
    for (uint32_t i = tid; i < (p.page_count + 31) / 32; i += T) p.freed[i] = 0;
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
        if (tid == 0) p.head[0] = p.head[2] = 0;
        return;
    }
    // (Numbers past the free pages' are not used: the call is refused.)
    uint64_t taken = 0;
    for (uint32_t s0 = 0; s0 < p.sequences; s0 += T) {
        const uint32_t s = s0 + tid;
        uint64_t all;
        const uint64_t at = taken + brn_sum(s < p.sequences ? brn_sequence(p, s).fresh : 0, sums, &all);
        if (s < p.sequences) p.before[s] = static_cast<uint32_t>(at);
        taken += all;
    }
    if (taken > free_count) {
        bad |= SGLKV_FLAG_OUT_OF_PAGES;
    } else {
        for (uint64_t i = free_count - taken + tid; i < free_count; i += T)
            if (static_cast<uint32_t>(p.free_pages[i]) >= p.page_count) bad |= SGLKV_FLAG_PAGE;
    }
    const bool refused = __syncthreads_or(bad) != 0;
    if (bad) atomicOr(p.flag, bad);
    uint64_t copies = 0;
    if (!refused)
        for (uint32_t s0 = 0; s0 < p.sequences; s0 += T) {
            const uint32_t s = s0 + tid;
            const brn_need n = brn_sequence(p, s < p.sequences ? s : 0);
            const bool own = s < p.sequences && n.copies;
            uint64_t all;
            const uint64_t at = copies + brn_sum(own, sums, &all);
            if (own) p.copies[at] = brn_copy_of(p, n, brn_fresh(p, free_count, p.before[s]));
            copies += all;
        }
    if (tid == 0) {
        p.head[0] = refused ? 0 : 1;
        p.head[1] = static_cast<uint32_t>(taken);
        p.head[2] = static_cast<uint32_t>(copies);
    }
}

// The new tables, the references, the pages that are freed: a workgroup to each
// new sequence, then to each old one.
__device__ __forceinline__ void brn_tables_body(const sglkv_fork_params &p) {
    if (p.head[0] == 0) return;
    const uint32_t tid = threadIdx.x;
    if (blockIdx.x < p.sequences) {
        const uint32_t s = blockIdx.x;
        const brn_need n = brn_sequence(p, s);
        const uint64_t free_count = *p.free_count;
        if (tid == 0) p.forked_lengths[s] = n.length;
        for (uint64_t j = tid; j < p.table_pages; j += SGLKV_FORK_THREADS) {
            const int32_t old = j < n.held ? p.tables[n.parent * p.table_pages + j] : -1;
            p.forked_tables[s * p.table_pages + j] =
                brn_entry(p, n, j, old, [&](uint32_t k) { return brn_fresh(p, free_count, k); }, p.before[s]);
        }
        return;
    }
    const uint32_t r = blockIdx.x - p.sequences, children = p.children[r];
    const uint64_t length = p.lengths[r], reserved = p.keep_reserved ? p.held[r] : 0;
    for (uint64_t j = tid; j * p.pool.page_size < length || j < reserved; j += SGLKV_FORK_THREADS) {
        const int32_t entry = p.tables[r * p.table_pages + j];
        if (brn_release(p, length, j, children, entry)) atomicOr(p.freed + entry / 32, 1u << (entry % 32));
    }
}

// One workgroup: the freed pages behind what is left of the free ones, ascending.
__device__ __forceinline__ void brn_free_body(const sglkv_fork_params &p) {
    constexpr uint32_t T = SGLKV_FORK_PLAN_THREADS;
    __shared__ uint64_t sums[T / 64];
    if (p.head[0] == 0) return;
    const uint32_t tid = threadIdx.x, words = (p.page_count + 31) / 32;
    uint64_t end = *p.free_count - p.head[1];
    for (uint32_t w0 = 0; w0 < words; w0 += T) {
        const uint32_t bits = w0 + tid < words ? p.freed[w0 + tid] : 0;
        uint64_t all;
        const uint64_t at = end + brn_sum(__popc(bits), sums, &all);
        brn_append(p, w0 + tid, bits, at);
        end += all;
    }
    if (tid == 0) brn_free_count(p, end);
}

// The last pages' rows: a workgroup to each (copy, layer, tensor). A head's rows lie
// together on head-major pages, all heads' on token-major ones: `heads` stretches.
__device__ __forceinline__ void brn_copy_body(const sglkv_fork_params &p) {
    constexpr uint32_t T = SGLKV_FORK_THREADS, U = 8;
    // (A page's layers and tensors one after another; the workgroups without a copy come last.)
    const uint32_t parts = p.layers * p.tensors, number = blockIdx.x / parts, part = blockIdx.x - number * parts;
    const uint32_t layer = part / p.tensors, t = part - layer * p.tensors, tid = threadIdx.x;
    const sglkv_page_copy c = p.copies[number];
    if (number >= p.head[2]) return;
    const uint64_t base = p.pool.plane[t] + layer * p.pool.layer_stride, bytes = static_cast<uint64_t>(c.rows) * p.chunk[t];
    const uint64_t source = base + c.source * p.pool.stride[t], to = base + c.to * p.pool.stride[t];
    if (p.wide == 2) {
        // (Host: a page's part of a tensor is below 2^32 bytes.)
        const uint32_t vectors = static_cast<uint32_t>(bytes / 16), all = vectors * p.heads;
        for (uint32_t i0 = tid; i0 < all; i0 += U * T) {
            sglkv_v4u x[U];
            uint64_t at[U];
#pragma unroll
            for (uint32_t u = 0; u < U; ++u) {
                const uint32_t i = i0 + T * u < all ? i0 + T * u : i0, h = p.heads > 1 ? i / vectors : 0;
                at[u] = h * p.pool.head_stride[t] + 16ull * (i - h * vectors);
                x[u] = __builtin_nontemporal_load(reinterpret_cast<brn_src16 *>(source + at[u]));
            }
#pragma unroll
            for (uint32_t u = 0; u < U; ++u)
                if (i0 + T * u < all) __builtin_nontemporal_store(x[u], reinterpret_cast<brn_dst16 *>(to + at[u]));
        }
        return;
    }
    for (uint32_t h = 0; h < p.heads; ++h) {
        const uint64_t from_at = source + h * p.pool.head_stride[t], to_at = to + h * p.pool.head_stride[t];
        uint64_t done = 0;
        if (p.wide) {
            // Both are misaligned alike: 16 bytes at a time from the first multiple of 16.
            const uint64_t lead = (16 - from_at % 16) % 16, head = lead < bytes ? lead : bytes;
            const uint64_t vectors = (bytes - head) / 16;
            for (uint64_t i = tid; i < head; i += T)
                reinterpret_cast<sglkv_gdst *>(to_at)[i] = reinterpret_cast<sglkv_gsrc *>(from_at)[i];
            for (uint64_t i = tid; i < vectors; i += T)
                reinterpret_cast<brn_dst16 *>(to_at + head)[i] = reinterpret_cast<brn_src16 *>(from_at + head)[i];
            done = head + 16 * vectors;
        }
        for (uint64_t i = done + tid; i < bytes; i += T)
            reinterpret_cast<sglkv_gdst *>(to_at)[i] = reinterpret_cast<sglkv_gsrc *>(from_at)[i];
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

extern "C" __global__ __launch_bounds__(SGLKV_FORK_PLAN_THREADS) void sglkv_fork_small(sglkv_fork_params p) { brn_small_body(p); }
extern "C" __global__ __launch_bounds__(SGLKV_FORK_PLAN_THREADS) void sglkv_fork_plan(sglkv_fork_params p) { brn_plan_body(p); }
extern "C" __global__ __launch_bounds__(SGLKV_FORK_THREADS) void sglkv_fork_tables(sglkv_fork_params p) { brn_tables_body(p); }
extern "C" __global__ __launch_bounds__(SGLKV_FORK_THREADS) void sglkv_fork_copy(sglkv_fork_params p) { brn_copy_body(p); }
extern "C" __global__ __launch_bounds__(SGLKV_FORK_PLAN_THREADS) void sglkv_fork_free(sglkv_fork_params p) { brn_free_body(p); }
