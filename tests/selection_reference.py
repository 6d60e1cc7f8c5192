"""Plain 64-bit restatements of page selection for the tests: page key bounds,
the lists, and attention over listed pages, on numpy arrays."""
import numpy as np

import oracle
import sgl_rocm_kv as kv
from sgl_rocm_kv import hip

NONE = 0xFFFFFFFF


def bf16(values):
    """bf16 bits of float32 values."""
    a = np.asarray(values, np.float32)
    return oracle.f32_to_bf16(a.reshape(-1)).reshape(a.shape)


def f64(bits):
    return (bits.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


class Pool:
    """A bf16 pool of `pages` pages, its seeded contents on the host and the
    device, and the rows of one layer by slot."""

    def __init__(self, rng, *, page, heads, dk, dv=None, pages, layers=2, layer=1, hnd=False, shift=0, spread=1.0):
        dv = dk if dv is None else dv
        kb, vb = heads * dk * 2, heads * dv * 2
        runtime = kv.KvCacheRuntimeLayout("bf16", page, layers, heads, dk, 2, layers * (kb + vb), layers * (kb + vb) * page)
        self.layout = (kv.PagedKvCacheLayout.new(runtime, pages) if dk == dv
                       else kv.PagedKvCacheLayout.new_with_tensor_pair(runtime, pages, kb, vb))
        self.page, self.heads, self.dk, self.dv, self.pages, self.layer, self.hnd = page, heads, dk, dv, pages, layer, hnd
        n = self.layout.total_byte_len // 2
        self.bits = bf16(spread * rng.standard_normal(n))
        self.shift = shift  # bytes between the allocation and the pool
        self.upload()

    def upload(self):
        raw = np.concatenate([np.zeros(self.shift, np.uint8), self.bits.view(np.uint8)])
        self.buffer = hip.DeviceBuffer.from_array(raw)

    @property
    def head_layout(self):
        return kv.HND if self.hnd else kv.NHD

    def view(self):
        return self.layout.pool_view(self.buffer.ptr + self.shift, self.buffer.nbytes - self.shift, self.layer,
                                     self.head_layout, heads=self.heads)

    def rows(self, tensor):
        """[slot][head][dim] bits of the layer's keys (0) or values (1); a view that writes through."""
        start = self.layout.tensor_token_byte_range(0, self.layer, tensor, 0)[0] // 2
        stride = self.layout.runtime.page_size_bytes // 2
        d = (self.dk, self.dv)[tensor]
        region = self.bits.reshape(self.pages, stride)[:, start:start + self.page * self.heads * d]
        return _Rows(region, self, d)


class _Rows:
    def __init__(self, region, pool, d):
        shape = (pool.pages, pool.heads, pool.page, d) if pool.hnd else (pool.pages, pool.page, pool.heads, d)
        self.at = region.reshape(shape) if region.flags.c_contiguous else np.lib.stride_tricks.as_strided(
            region, shape, (region.strides[0],) + tuple(2 * int(np.prod(shape[i + 1:])) for i in (1, 2, 3)))
        self.pool = pool

    def get(self, slots, head):
        p, t = np.divmod(np.asarray(slots, np.int64), self.pool.page)
        return self.at[p, head, t] if self.pool.hnd else self.at[p, t, head]

    def put(self, slot, head, bits):
        p, t = divmod(int(slot), self.pool.page)
        self.at[(p, head, t) if self.pool.hnd else (p, t, head)] = bits


class Batch:
    """Requests of `lengths` tokens in scattered pages, `per` queries each (the
    last ones), with metadata on the host and the device."""

    def __init__(self, rng, pool, lengths, qheads, per=1, spare=0):
        self.pool, self.lengths, self.qheads = pool, [int(n) for n in lengths], qheads
        page = pool.page
        need = [-(-n // page) for n in self.lengths]
        assert sum(need) <= pool.pages
        pages, at = rng.permutation(pool.pages), 0
        slots, offsets = [], [0]
        for n, c in zip(self.lengths, need):
            own = (pages[at:at + c, None] * page + np.arange(page)).reshape(-1)[:n]
            slots += [own, np.full(spare, (1 << 40) + 7)]  # room behind a sequence, never to be read
            offsets.append(offsets[-1] + n + spare)
            at += c
        self.slots = np.concatenate(slots).astype(np.uint64) if sum(map(len, slots)) else np.zeros(1, np.uint64)
        self.offsets = np.asarray(offsets, np.uint64)
        counts = [min(per, n) if n else 1 for n in self.lengths]
        self.requests = np.repeat(np.arange(len(counts)), counts).astype(np.uint32)
        self.ends = np.concatenate([n - c + 1 + np.arange(c) if n else [0] for n, c in zip(self.lengths, counts)])
        self.ends = self.ends.astype(np.uint64)
        self.queries = bf16(rng.standard_normal((len(self.ends), qheads, pool.dk)))
        self.upload()

    def upload(self):
        self.device = dict(queries=hip.DeviceBuffer.from_array(self.queries),
                           query_request_indices=hip.DeviceBuffer.from_array(self.requests),
                           query_sequence_lengths=hip.DeviceBuffer.from_array(self.ends),
                           request_slot_offsets=hip.DeviceBuffer.from_array(self.offsets),
                           sequence_slots=hip.DeviceBuffer.from_array(self.slots))

    def plan(self, scale=None):
        p = self.pool
        return kv.PagedAttentionPlan.for_layer(p.layout, p.layer, len(self.ends), len(self.lengths), len(self.slots),
                                               self.qheads, p.dk ** -0.5 if scale is None else scale, p.head_layout)

    def own_slots(self, q):
        r = int(self.requests[q])
        return self.slots[int(self.offsets[r]):int(self.offsets[r]) + int(self.ends[q])].astype(np.int64)


def page_bounds(pool, page, count):
    """[head][low, high][dim] of a pool page's first `count` keys, as float64."""
    keys = np.stack([f64(pool.rows(0).get(page * pool.page + np.arange(count), h)) for h in range(pool.heads)])
    return np.stack([keys.min(axis=1), keys.max(axis=1)], axis=1)


def select(batch, bounds, keep, first=0, last=0):
    """[query][head][keep] lists from bounds [page][head][2][dim] (bits)."""
    pool, group = batch.pool, batch.qheads // batch.pool.heads
    out = np.full((len(batch.ends), pool.heads, keep), NONE, np.uint32)
    b = f64(bounds)
    with np.errstate(invalid="ignore"):
        for q, end in enumerate(batch.ends.astype(int)):
            if end == 0:
                continue
            pages = batch.own_slots(q)[::pool.page] // pool.page
            count = len(pages)
            j = np.arange(count)
            forced = (j < first) | (j + last >= count)
            for h in range(pool.heads):
                vectors = f64(batch.queries[q, h * group:(h + 1) * group])
                scores = (np.where(vectors > 0, vectors, 0.0)[:, None] * b[pages, h, 1] +
                          np.where(vectors > 0, 0.0, vectors)[:, None] * b[pages, h, 0]).sum(axis=2)
                score = np.where(np.isnan(scores).any(axis=0), np.nan, scores.max(axis=0))
                # Forced ones, then NaN, then by score; the lower page first among equals.
                order = np.lexsort((j, -np.where(np.isnan(score), 0.0, score), ~np.isnan(score), ~forced))
                best = np.sort(order[:keep])
                out[q, h, :len(best)] = best
    return out


def attend(batch, lists, scale=None):
    """(output, sum of w |v|) in float64 over listed pages [query][head][max]."""
    pool, group = batch.pool, batch.qheads // batch.pool.heads
    scale = pool.dk ** -0.5 if scale is None else scale
    out = np.zeros((len(batch.ends), batch.qheads, pool.dv))
    absolute = np.zeros_like(out)
    keys, values = pool.rows(0), pool.rows(1)
    for q, end in enumerate(batch.ends.astype(int)):
        for h in range(pool.heads):
            pages = lists[q, h][lists[q, h] != NONE].astype(np.int64)
            tokens = (pages[:, None] * pool.page + np.arange(pool.page)).reshape(-1)
            tokens = tokens[tokens < end]
            if not len(tokens):
                continue
            slots = batch.own_slots(q)[tokens]
            k, v = f64(keys.get(slots, h)), f64(values.get(slots, h))
            s = f64(batch.queries[q, h * group:(h + 1) * group]) @ k.T * scale
            w = np.exp(s - s.max(axis=1, keepdims=True))
            w /= w.sum(axis=1, keepdims=True)
            out[q, h * group:(h + 1) * group] = w @ v
            absolute[q, h * group:(h + 1) * group] = w @ np.abs(v)
    return out, absolute


def random_lists(rng, batch, keep):
    """Random pages of each (query, head), the newest always among them."""
    out = np.full((len(batch.ends), batch.pool.heads, keep), NONE, np.uint32)
    for q, end in enumerate(batch.ends.astype(int)):
        count = -(-end // batch.pool.page)
        for h in range(batch.pool.heads):
            n = min(keep, count)
            if n:
                best = np.sort(np.append(rng.choice(count - 1, n - 1, replace=False), count - 1))
                out[q, h, :n] = best
    return out
