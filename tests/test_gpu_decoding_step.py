"""GPU tests of decoding along several continuations as a loop uses it, enqueued in
a row on one stream without a wait: the best beams, their forks, the forks' slots
and attention over them; attention of drafted trees, the accepted drafts moved
together and attention over what stays. Then two chains at once, two contexts,
captured and replayed chains, and a pool whose offsets pass 32 bits.

Lists, tables and rows are compared exactly; scores and attention outputs have the
bounds of test_gpu_beams.py and test_gpu_tree.py."""
import ctypes

import numpy as np
import pytest

import branch_reference as ref
import sgl_rocm_kv as kv
from branch_reference import NONE, Trees
from selection_reference import Pool, bf16, f64
from sgl_rocm_kv import hip
from test_gpu_selection import _check, _filled, _say

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def k():
    if hip.device_count() == 0:
        pytest.fail("no GPU visible: the gpu tests need an MI355X")
    ctx = kv.RocmKvPairCopyKernels(0)
    yield ctx
    ctx.close()


def _all_layers(layout, base, nbytes, head_layout, heads):
    """A view of the first layer, and what leads to the others."""
    starts = [layout.tensor_token_byte_range(0, layer, 0, 0)[0] for layer in range(2)]
    return (layout.pool_view(base, nbytes, 0, head_layout, heads=heads),
            dict(layer_count=layout.runtime.num_layers, layer_stride_bytes=starts[1] - starts[0]))


def _attend(pool, queries, slots):
    """([head][dim], its sum of magnitudes) of one query over the rows at `slots`."""
    heads = len(queries) // pool.heads
    out, absolute = np.zeros((len(queries), pool.dv)), np.zeros((len(queries), pool.dv))
    for h in range(pool.heads):
        own = slice(h * heads, (h + 1) * heads)
        s = f64(queries[own]) @ f64(pool.rows(0).get(slots, h)).T * pool.dk ** -0.5
        w = np.exp(s - s.max(axis=1, keepdims=True))
        w /= w.sum(axis=1, keepdims=True)
        v = f64(pool.rows(1).get(slots, h))
        out[own], absolute[own] = w @ v, w @ np.abs(v)
    return out, absolute


class Step:
    """What the chains have in common: buffers by name, as they start and as they are."""

    def hold(self, **arrays):
        for name, a in arrays.items():
            self.start[name] = np.ascontiguousarray(a)
            self.held[name] = hip.DeviceBuffer.from_array(self.start[name])

    def reset(self):
        for name, a in self.start.items():
            self.held[name].upload(a)
        hip.synchronize()

    def got(self, name):
        a = self.start[name]
        return self.held[name].download().view(a.dtype).reshape(a.shape)

    def results(self):
        return [self.got(name) for name in self.written]


class Beams(Step):
    """A step of beam search: `beams` sequences of each request share all pages but the last."""

    written = ("best_scores", "best_parents", "best_tokens", "forked_lengths", "forked_tables", "page_references", "free_pages",
               "free_count", "slots", "output", "pool")

    def __init__(self, seed, *, page=16, heads=2, qheads=8, dk=128, hnd=False, lengths=(100, 33, 64), beams=4, vocab=3000,
                 free=40):
        rng = np.random.default_rng(seed)
        self.start, self.held = {}, {}
        self.beams, self.lengths, self.page = beams, lengths, page
        sequences = len(lengths) * beams
        full, tails = [n // page for n in lengths], [n % page > 0 for n in lengths]
        pages = sum(f + t * beams for f, t in zip(full, tails)) + free
        self.pool = pool = Pool(rng, page=page, heads=heads, dk=dk, pages=pages, hnd=hnd)
        self.table_pages = max(full) + 2
        order, at = rng.permutation(pages), 0
        tables, references = np.full((sequences, self.table_pages), -1, np.int32), np.zeros(pages, np.uint32)
        for r, n in enumerate(lengths):
            shared, at = order[at:at + full[r]], at + full[r]
            for b in range(beams):
                row = tables[r * beams + b]
                row[:full[r]] = shared
                if tails[r]:
                    row[full[r]], at = order[at], at + 1
                references[row[row >= 0]] += 1
        free_pages = np.full(pages, -1, np.int32)
        free_pages[:free] = order[at:]
        self.per = np.repeat(lengths, beams)  # a sequence's tokens, before and after
        spans = np.zeros(sequences, kv.SPAN_DTYPE)
        offsets = np.concatenate([[0], np.cumsum(self.per)]).astype(np.uint64)
        spans["row_start"], spans["token_count"] = offsets[:-1], self.per
        spans["page_table_start"] = np.arange(sequences) * self.table_pages
        self.logits = bf16(2.5 * rng.standard_normal((len(lengths), beams, vocab)))
        self.queries = bf16(rng.standard_normal((sequences, qheads, dk)))
        self.plan = kv.BeamPlan.new(request_count=len(lengths), beam_count=beams, vocab_size=vocab, max_kept=beams)
        self.forks = kv.ForkPlan.new(sequence_count=sequences, parent_count=sequences, table_pages=self.table_pages,
                                     page_size=page, page_count=pages, append_tokens=1)
        self.attention = kv.PagedAttentionPlan.for_layer(pool.layout, pool.layer, sequences, sequences, int(offsets[-1]), qheads,
                                                         dk ** -0.5, pool.head_layout)
        kept = (len(lengths), beams)
        self.hold(logits=self.logits, scores=(-20 * rng.random(kept)).astype(np.float32), best_scores=np.zeros(kept, np.float32),
                  best_parents=np.zeros(kept, np.uint32), best_tokens=np.zeros(kept, np.uint32),
                  beam_workspace=np.full(self.plan.workspace_required_bytes, 0xFF, np.uint8),
                  lengths=self.per.astype(np.uint64), page_tables=tables, forked_lengths=np.zeros(sequences, np.uint64),
                  forked_tables=np.zeros_like(tables), page_references=references, free_pages=free_pages,
                  free_count=np.asarray([free], np.uint64),
                  fork_workspace=np.full(self.forks.workspace_required_bytes, 0xFF, np.uint8), spans=spans,
                  slots=np.zeros(int(offsets[-1]), np.uint64), queries=self.queries,
                  requests=np.arange(sequences, dtype=np.uint32), offsets=offsets,
                  output=np.zeros((sequences, qheads, dk), np.uint16), pool=pool.bits)
        self.view, self.layers = _all_layers(pool.layout, self.held["pool"].ptr, self.held["pool"].nbytes, pool.head_layout, heads)

    def enqueue(self, k, stream):
        h = self.held
        k.select_beams(self.plan, kv.BeamBuffers(
            logits=h["logits"], scores=h["scores"], best_scores=h["best_scores"], best_parents=h["best_parents"],
            best_tokens=h["best_tokens"], workspace=h["beam_workspace"]), stream=stream)
        k.fork_sequences(self.forks, kv.ForkBuffers(
            parents=h["best_parents"], workspace=h["fork_workspace"],
            **{n: h[n] for n in ("lengths", "page_tables", "forked_lengths", "forked_tables", "page_references", "free_pages",
                                 "free_count")}), self.view, stream=stream, **self.layers)
        table, spans, slots = (kv.device_buffer(h[n].ptr, h[n].nbytes) for n in ("forked_tables", "spans", "slots"))
        k.resolve_spans(self.page, self.pool.pages, spans, len(self.per), table, self.start["forked_tables"].size,
                        len(self.start["slots"]), slots, stream)
        k.paged_attention_async(self.attention, queries=h["queries"], query_request_indices=h["requests"],
                                query_sequence_lengths=h["lengths"], request_slot_offsets=h["offsets"], sequence_slots=h["slots"],
                                pool=h["pool"], output=h["output"], stream=stream)

    def check(self):
        pool, s = self.pool, self.start
        scores, parents, tokens = ref.best_beams(f64(self.logits), s["scores"].astype(np.float64), self.beams)
        assert np.array_equal(self.got("best_parents"), parents) and np.array_equal(self.got("best_tokens"), tokens)
        assert (np.abs(self.got("best_scores") - scores) <= 2.0 ** -17 + 2.0 ** -24 * np.abs(scores)).all()
        copies = []
        want = ref.fork(parents.reshape(-1), s["lengths"], s["page_tables"], s["page_references"], s["free_pages"],
                        s["free_count"][0], self.page, 1, lambda *c: copies.append(c))
        for name, a in zip(("forked_lengths", "forked_tables", "page_references", "free_pages"), want):
            assert np.array_equal(self.got(name), a), name
        assert int(self.got("free_count")[0]) == want[4]
        # What a beam attends is its parent's, of before the step.
        output = f64(self.got("output"))
        for i, p in enumerate(parents.reshape(-1)):
            n = int(self.per[i])
            before = s["page_tables"][p][np.arange(n) // self.page].astype(np.int64) * self.page + np.arange(n) % self.page
            _check(output[i:i + 1], *(x[None] for x in _attend(pool, self.queries[i], before)))
        before, after = pool.bits.copy(), self.got("pool").copy()
        pool.bits = after  # the copied rows of the attended layer; the other rows are what they were
        rows = [[pool.rows(t) for t in (0, 1)]]
        pool.bits = before
        rows.append([pool.rows(t) for t in (0, 1)])
        for source, to, count in copies:
            for t in (0, 1):
                for h in range(pool.heads):
                    a, b = (int(p) * self.page + np.arange(count) for p in (to, source))
                    assert np.array_equal(rows[0][t].get(a, h), rows[1][t].get(b, h))


class Drafts(Step):
    """A step of checking drafted trees: one path of each is accepted."""

    written = ("output", "pool", "after")

    def __init__(self, seed, *, page=16, heads=2, qheads=8, dk=128, hnd=False, contexts=(100, 5, 300), drafts=(12, 24, 7)):
        rng = np.random.default_rng(seed)
        self.start, self.held = {}, {}
        pages = sum(-(-(c + n) // page) for c, n in zip(contexts, drafts)) + 2
        self.pool = pool = Pool(rng, page=page, heads=heads, dk=dk, pages=pages, hnd=hnd)
        self.trees = trees = Trees(rng, pool, qheads, contexts, drafts)
        at = np.concatenate([[0], np.cumsum(drafts)])
        self.last = [int(a + rng.integers(n)) for a, n in zip(at, drafts)]
        kept = np.full((len(drafts), 16), NONE, np.uint32)
        for r, q in enumerate(self.last):
            path = np.flatnonzero(trees.masks[q])[-16:]
            kept[r, :len(path)] = path
            trees.masks[q] = False  # (at most 16 of the path)
            trees.masks[q, path] = True
        self.lengths = [c + int((own != NONE).sum()) for c, own in zip(contexts, kept)]
        self.plan = trees.plan(max(c + n for c, n in zip(contexts, drafts)))
        self.keep = kv.DraftPlan.new(request_count=len(drafts), sequence_slot_count=len(trees.slots), max_kept=16)
        self.attention = kv.PagedAttentionPlan.for_layer(pool.layout, pool.layer, len(drafts), len(drafts), len(trees.slots),
                                                         qheads, dk ** -0.5, pool.head_layout)
        self.hold(pool=pool.bits, kept=kept, contexts=np.asarray(contexts, np.uint64), lengths=np.asarray(self.lengths, np.uint64),
                  requests=np.arange(len(drafts), dtype=np.uint32), queries=trees.queries[self.last],
                  output=np.zeros(trees.queries.shape, np.uint16), after=np.zeros((len(drafts), qheads, dk), np.uint16),
                  workspace=np.full(max(64, self.plan.workspace_required_bytes), 0xFF, np.uint8))
        trees.upload()
        self.view, self.layers = _all_layers(pool.layout, self.held["pool"].ptr, self.held["pool"].nbytes, pool.head_layout, heads)

    def enqueue(self, k, stream):
        h, d = self.held, self.trees.device
        k.tree_attention(self.plan, kv.TreeAttentionBuffers(**d, pool=h["pool"], output=h["output"], workspace=h["workspace"]),
                         stream=stream)
        own = dict(request_slot_offsets=d["request_slot_offsets"], sequence_slots=d["sequence_slots"])
        k.keep_drafts(self.keep, kv.DraftBuffers(**own, request_lengths=h["contexts"], kept=h["kept"]), self.view, stream=stream,
                      **self.layers)
        k.paged_attention_async(self.attention, **own, queries=h["queries"], query_request_indices=h["requests"],
                                query_sequence_lengths=h["lengths"], pool=h["pool"], output=h["after"], stream=stream)

    def check(self):
        want, absolute = self.trees.attend()
        _check(f64(self.got("output")), want, absolute)
        # The last accepted draft attends the same tokens, now in a row.
        _check(f64(self.got("after")), want[self.last], absolute[self.last])
        trees, pool = self.trees, self.pool
        before, after = pool.bits.copy(), self.got("pool").copy()
        old = [pool.rows(t) for t in (0, 1)]
        pool.bits = after
        new = [pool.rows(t) for t in (0, 1)]
        pool.bits = before
        for r, own in enumerate(self.start["kept"]):
            at = int(trees.offsets[r]) + trees.contexts[r]
            for i, draft in enumerate(own[own != NONE]):
                for t in (0, 1):
                    for h in range(pool.heads):
                        assert np.array_equal(new[t].get(trees.slots[at + i], h), old[t].get(trees.slots[at + int(draft)], h))


def _same(a, b):
    return all(np.array_equal(x.view(np.uint8), y.view(np.uint8)) for x, y in zip(a, b))


CHAINS = [(Beams, dict()), (Beams, dict(page=64, heads=8, qheads=32, lengths=(700, 64, 1, 130), beams=8, vocab=40000)),
          (Beams, dict(dk=64, heads=2, qheads=14, hnd=True, lengths=(50,), beams=1)),
          (Beams, dict(page=7, dk=40, lengths=(20, 21, 22), beams=128, vocab=300, free=600)),
          (Drafts, dict()), (Drafts, dict(page=64, heads=8, qheads=32, contexts=(700, 64, 0, 130), drafts=(61, 1, 64, 20))),
          (Drafts, dict(dk=64, heads=2, qheads=14, hnd=True)), (Drafts, dict(page=7, dk=40, qheads=6)),
          (Drafts, dict(dk=256, contexts=(50, 60), drafts=(100, 3)))]


@pytest.mark.parametrize("of,case", CHAINS, ids=lambda x: x.__name__ if isinstance(x, type) else "-".join(map(str, x.items())))
def test_a_step_of_all_calls(k, of, case):
    _say(f"decoding step: {of.__name__} {case}")
    chain, stream = of(1, **case), hip.Stream()
    hip.synchronize()
    chain.enqueue(k, stream)
    stream.synchronize()
    k.check_errors()
    chain.check()
    stream.destroy()


def test_chains_at_once_on_streams(k):
    """Chains with buffers of their own do not see each other, and a repeated run gives the same bits."""
    chains = [Beams(2), Drafts(3), Beams(4, page=64, heads=4, qheads=16, lengths=(1000, 90), beams=8), Drafts(5, dk=64, hnd=True)]
    streams = [hip.Stream() for _ in chains]
    want = []
    for chain in chains:
        chain.enqueue(k, None)
        hip.synchronize()
        want.append(chain.results())
    for i in range(4):
        for chain in chains:
            chain.reset()
        _say(f"decoding step: streams, run {i}")
        for chain, stream in zip(chains, streams):
            chain.enqueue(k, stream)
        hip.synchronize()
        for chain, w in zip(chains, want):
            assert _same(chain.results(), w)
    k.check_errors()
    for stream in streams:
        stream.destroy()


@pytest.mark.parametrize("of", [Beams, Drafts])
def test_two_contexts_share_nothing(k, of):
    other, chain = kv.RocmKvPairCopyKernels(0), of(6)
    chain.enqueue(k, None)
    hip.synchronize()
    want = chain.results()
    chain.reset()
    chain.enqueue(other, None)
    hip.synchronize()
    assert _same(chain.results(), want)
    other.check_errors()
    k.check_errors()
    other.close()


@pytest.mark.parametrize("of,case", [CHAINS[1], CHAINS[3], CHAINS[5]], ids=["beams", "many_beams", "drafts"])
def test_captured_chain_replays(k, of, case):
    """The chain in a graph: every replay gives the eager run's bits, with the same chain run eagerly in between."""
    chain, stream = of(7, **case), hip.Stream()
    chain.enqueue(k, None)
    hip.synchronize()
    want = chain.results()
    h, vp = hip.lib(), ctypes.c_void_p
    h.hipStreamBeginCapture.argtypes = [vp, ctypes.c_int]
    h.hipStreamEndCapture.argtypes = [vp, ctypes.POINTER(vp)]
    h.hipGraphInstantiate.argtypes = [ctypes.POINTER(vp), vp, vp, vp, ctypes.c_size_t]
    h.hipGraphLaunch.argtypes = [vp, vp]
    h.hipGraphExecDestroy.argtypes = [vp]
    h.hipGraphDestroy.argtypes = [vp]
    graph, execution = vp(), vp()
    _say(f"decoding step: {of.__name__} under graph capture")
    hip.check(h.hipStreamBeginCapture(stream.handle, 0), "hipStreamBeginCapture")
    chain.enqueue(k, stream)
    hip.check(h.hipStreamEndCapture(stream.handle, ctypes.byref(graph)), "hipStreamEndCapture")
    hip.check(h.hipGraphInstantiate(ctypes.byref(execution), graph, None, None, 0), "hipGraphInstantiate")
    for i in range(4):
        chain.reset()
        hip.check(h.hipGraphLaunch(execution, stream.handle), "hipGraphLaunch")
        stream.synchronize()
        assert _same(chain.results(), want), f"replay {i}"
        chain.reset()
        chain.enqueue(k, None)  # eager work between the replays
        hip.synchronize()
        assert _same(chain.results(), want), f"eager {i}"
    k.check_errors()
    hip.check(h.hipGraphExecDestroy(execution), "hipGraphExecDestroy")
    hip.check(h.hipGraphDestroy(graph), "hipGraphDestroy")
    stream.destroy()


@pytest.mark.parametrize("hnd,dk", [(False, 128), (True, 64), (False, 256), (False, 40)])
def test_offsets_past_32_bits(k, hnd, dk):
    """A pool of more than 8 GiB whose used pages lie at both its ends and across every 4 GiB gives what a small pool
    with the same rows gives: attention, the rows moved together, and the copied pages."""
    rng = np.random.default_rng(8)
    page, heads, qheads, pages = 64, 8, 16, 24
    contexts, drafts = (500, 60, 260), (30, 5, 64)
    small = Pool(rng, page=page, heads=heads, dk=dk, pages=pages, layers=16, layer=13, hnd=hnd)
    stride = small.layout.total_byte_len // pages
    many = (9 << 30) // stride
    big = kv.PagedKvCacheLayout.new(small.layout.runtime, many)
    at = np.concatenate([np.arange(many - 8, many), *((g << 30) // stride + np.arange(-3, 3) for g in (4, 8)), np.arange(4)])
    _say(f"decoding step: {many} pages of {stride} bytes, dims {dk}")
    held = hip.DeviceBuffer(big.total_byte_len)
    raw = small.bits.view(np.uint8).reshape(pages, stride)
    for i, p in enumerate(at):
        held.upload(raw[i], int(p) * stride)
    trees = Trees(rng, small, qheads, contexts, drafts)
    trees.upload()
    kept = np.full((3, 4), NONE, np.uint32)
    kept[0, :3], kept[1, :2], kept[2, :4] = (3, 17, 29), (0, 4), (1, 40, 62, 63)
    # Two sequences of the first requests' pages, each taken twice: one more page with copied rows for each.
    own = [trees.slots[int(trees.offsets[r])::page][:-(-contexts[r] // page)].astype(np.int64) // page for r in (0, 1)]
    spare = np.setdiff1d(np.arange(pages), trees.slots.astype(np.int64) // page)[:2]

    def run(layout, pool, index):
        device = dict(trees.device, sequence_slots=hip.DeviceBuffer.from_array(
            (index[trees.slots.astype(np.int64) // page] * page + trees.slots.astype(np.int64) % page).astype(np.uint64)))
        attention = kv.PagedAttentionPlan.for_layer(layout, 13, len(trees.requests), 3, len(trees.slots), qheads, dk ** -0.5,
                                                    small.head_layout)
        plan = kv.TreeAttentionPlan.new(attention, mask_words=trees.words)
        output = _filled(attention.output_required_bytes)
        k.tree_attention(plan, kv.TreeAttentionBuffers(**device, pool=pool, output=output,
                                                       workspace=_filled(max(64, plan.workspace_required_bytes), 0xFF)))
        view, layers = _all_layers(layout, pool.ptr, pool.nbytes, small.head_layout, heads)
        drafts_plan = kv.DraftPlan.new(request_count=3, sequence_slot_count=len(trees.slots), max_kept=4)
        k.keep_drafts(drafts_plan, kv.DraftBuffers(
            request_lengths=hip.DeviceBuffer.from_array(np.asarray(contexts, np.uint64)), sequence_slots=device["sequence_slots"],
            request_slot_offsets=device["request_slot_offsets"], kept=hip.DeviceBuffer.from_array(kept)), view, **layers)
        count = layout.total_byte_len // stride
        tables, references, free = np.full((2, 9), -1, np.int32), np.zeros(count, np.uint32), np.full(count, -1, np.int32)
        for i, o in enumerate(own):
            tables[i, :len(o)] = index[o]
            references[index[o]] += 1
        free[:2] = index[spare]
        given = {n: hip.DeviceBuffer.from_array(a) for n, a in dict(
            parents=np.asarray([0, 0, 1, 1], np.uint32), lengths=np.asarray(contexts[:2], np.uint64), page_tables=tables,
            forked_lengths=np.zeros(4, np.uint64), forked_tables=np.zeros((4, 9), np.int32), page_references=references,
            free_pages=free, free_count=np.asarray([2], np.uint64)).items()}
        forks = kv.ForkPlan.new(sequence_count=4, parent_count=2, table_pages=9, page_size=page, page_count=count)
        k.fork_sequences(forks, kv.ForkBuffers(**given, workspace=_filled(forks.workspace_required_bytes, 0xFF)), view, **layers)
        hip.synchronize()
        k.check_errors()
        forked = given["forked_tables"].download().view(np.int32).reshape(4, 9)
        return output.download(), forked

    want, small_tables = run(small.layout, small.buffer, np.arange(pages))
    got, big_tables = run(big, held, at)
    assert np.array_equal(got, want)
    assert np.array_equal(big_tables, np.where(small_tables < 0, small_tables, at[small_tables]))
    assert set(small_tables[[1, 3], [len(o) - 1 for o in own]]) == set(spare)
    _check(f64(want.view(np.uint16).reshape(trees.queries.shape[0], qheads, dk)), *trees.attend())
    after = small.buffer.download().reshape(pages, stride)
    assert not np.array_equal(after, raw)
    for i, p in enumerate(at):
        assert np.array_equal(held.download(stride, int(p) * stride), after[i]), p
    held.free()
