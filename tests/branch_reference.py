"""Plain 64-bit restatements of decoding along several continuations for the
tests: attention by masks, accepted rows moved together, the best continuations
and forks of page tables, on numpy arrays."""
import numpy as np

from selection_reference import bf16, f64
from sgl_rocm_kv import hip
import sgl_rocm_kv as kv

NONE = 0xFFFFFFFF


class Trees:
    """Requests of contexts[r] tokens and drafts[r] drafted ones behind them in
    scattered pages, a query to each draft, with masks (bool [query][64 words])
    of random ancestors; `spare` slots that are never to be read lie behind each
    request's, `padding` queries that attend nothing behind the last."""

    def __init__(self, rng, pool, qheads, contexts, drafts, *, words=None, spare=0, padding=0):
        self.pool, self.qheads, self.contexts, self.drafts = pool, qheads, list(contexts), list(drafts)
        self.words = words or max(1, -(-max(drafts) // 64))
        page = pool.page
        lengths = [c + n for c, n in zip(contexts, drafts)]
        need = [-(-n // page) for n in lengths]
        assert sum(need) <= pool.pages
        pages, at, slots, offsets = rng.permutation(pool.pages), 0, [], [0]
        for n, c in zip(lengths, need):
            own = (pages[at:at + c, None] * page + np.arange(page)).reshape(-1)[:n]
            slots += [own, np.full(spare, (1 << 40) + 7)]
            offsets.append(offsets[-1] + n + spare)
            at += c
        self.slots = np.concatenate(slots).astype(np.uint64)
        self.offsets = np.asarray(offsets, np.uint64)
        self.requests = np.concatenate([np.repeat(np.arange(len(drafts)), drafts), np.full(padding, NONE)]).astype(np.uint32)
        self.lengths = np.concatenate([np.repeat(contexts, drafts), np.zeros(padding)]).astype(np.uint64)
        self.masks = np.zeros((len(self.requests), 64 * self.words), bool)
        q = 0
        for n in drafts:
            for i in range(n):
                if i:
                    self.masks[q + i] = self.masks[q + rng.integers(max(0, i - 5), i)]
                self.masks[q + i, i] = True
            q += n
        self.queries = bf16(rng.standard_normal((len(self.requests), qheads, pool.dk)))

    def upload(self):
        bits = np.packbits(self.masks, axis=1, bitorder="little").view(np.uint64)
        self.device = {n: hip.DeviceBuffer.from_array(np.ascontiguousarray(a)) for n, a in dict(
            queries=self.queries, query_request_indices=self.requests, query_sequence_lengths=self.lengths,
            request_slot_offsets=self.offsets, sequence_slots=self.slots, masks=bits).items()}
        return self.device

    def plan(self, longest=0):
        p = self.pool
        attention = kv.PagedAttentionPlan.for_layer(p.layout, p.layer, len(self.requests), len(self.contexts), len(self.slots),
                                                    self.qheads, p.dk ** -0.5, p.head_layout)
        return kv.TreeAttentionPlan.new(attention, mask_words=self.words, max_sequence_length=longest)

    def attended(self, q):
        """Slots that query q attends."""
        n = int(self.lengths[q])
        if n == 0 and not self.masks[q].any():
            return np.zeros(0, np.int64)
        start = int(self.offsets[self.requests[q]])
        places = np.concatenate([np.arange(n), n + np.flatnonzero(self.masks[q])])
        return self.slots[start + places].astype(np.int64)

    def attend(self):
        """(output, sum of w |v|) in float64."""
        pool, group = self.pool, self.qheads // self.pool.heads
        out = np.zeros((len(self.requests), self.qheads, pool.dv))
        absolute = np.zeros_like(out)
        keys, values = pool.rows(0), pool.rows(1)
        for q in range(len(self.requests)):
            slots = self.attended(q)
            if not len(slots):
                continue
            for h in range(pool.heads):
                k, v = f64(keys.get(slots, h)), f64(values.get(slots, h))
                s = f64(self.queries[q, h * group:(h + 1) * group]) @ k.T * pool.dk ** -0.5
                w = np.exp(s - s.max(axis=1, keepdims=True))
                w /= w.sum(axis=1, keepdims=True)
                out[q, h * group:(h + 1) * group] = w @ v
                absolute[q, h * group:(h + 1) * group] = w @ np.abs(v)
        return out, absolute


def best_beams(logits, scores, keep):
    """(scores, parents, tokens) of float64 logits [request][beam][token]: by the
    logits within a beam, by the score between beams, equal ones by (beam, token)."""
    requests, beams, vocab = logits.shape
    out = (np.full((requests, keep), -np.inf), np.full((requests, keep), NONE, np.uint32),
           np.full((requests, keep), NONE, np.uint32))
    for r in range(requests):
        entries = []
        for b in range(beams):
            x = logits[r, b]
            if np.isnan(x).any() or np.isposinf(x).any() or not np.isfinite(x).any() or not np.isfinite(scores[r, b]):
                continue
            top = x.max()
            log_sum = np.log(np.exp(x - top).sum())
            order = np.lexsort((np.arange(vocab), -x))[:keep]
            entries += [(scores[r, b] - log_sum + (x[v] - top), b, i, v) for i, v in enumerate(order) if np.isfinite(x[v])]
        entries.sort(key=lambda e: (-e[0], e[1], e[2]))
        for k, (total, b, _, v) in enumerate(entries[:keep]):
            out[0][r, k], out[1][r, k], out[2][r, k] = total, r * beams + b, v
    return out


class OutOfPages(Exception):
    pass


def fork(parents, lengths, tables, references, free, free_count, page, append, copy):
    """The state after fork_sequences, one sequence after another; copy(source,
    destination, rows) copies the first rows of a page. The arrays are not changed."""
    references, free, end = references.copy(), free.copy(), int(free_count)
    held = references > 0
    new_lengths = np.zeros(len(parents), np.uint64)
    new_tables = np.full((len(parents), tables.shape[1]), -1, np.int32)
    seen = set()
    for s, p in enumerate(parents):
        if p == NONE:
            continue
        n = int(lengths[p])
        new_lengths[s] = n
        for j in range(-(-(n + append) // page)):
            last = j == n // page and n % page > 0
            if j * page >= n or (last and p in seen):
                end -= 1
                if end < 0:
                    raise OutOfPages
                new_tables[s, j] = free[end]
                if last:
                    copy(tables[p, j], free[end], n % page)
            else:
                new_tables[s, j] = tables[p, j]
            references[new_tables[s, j]] += 1
        seen.add(p)
    for n, table in zip(lengths, tables):
        for j in range(-(-int(n) // page)):
            references[table[j]] -= 1
    for number in np.flatnonzero(held & (references == 0)):
        free[end] = number
        end += 1
    return new_lengths, new_tables, references, free, end
