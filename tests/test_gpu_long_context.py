"""GPU tests of page selection and eviction used together, as a decode loop uses
them: sums of attention weights, the positions kept, their copy into fresh pages,
those pages' bounds, each head's pages and attention over them, enqueued in a row
on one stream without a wait; in two chains at once; captured and replayed; and on
a pool whose offsets pass 32 bits.

Sums and attention outputs have the bounds of test_gpu_eviction.py and
test_gpu_selection.py, each step judged on the inputs that it got; lists, rows and
bounds are compared exactly."""
import ctypes

import numpy as np
import pytest

import selection_reference as ref
import sgl_rocm_kv as kv
from selection_reference import NONE, Batch, Pool, f64
from sgl_rocm_kv import hip
from test_gpu_eviction import _check_weights, _kept, _weights
from test_gpu_selection import _check, _filled, _say

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def k():
    if hip.device_count() == 0:
        pytest.fail("no GPU visible: the gpu tests need an MI355X")
    ctx = kv.RocmKvPairCopyKernels(0)
    yield ctx
    ctx.close()


class Chain:
    """The six calls over one batch, with every buffer of their own."""

    def __init__(self, seed, *, page=16, heads=2, qheads=8, dk=128, lengths=(600, 1, 260, 37), keep=128, listed=3, per=4,
                 hnd=False):
        rng = np.random.default_rng(seed)
        pages = sum(-(-n // page) for n in lengths) + 2
        self.keep, self.listed, self.lengths = keep, listed, lengths
        self.kept_lengths = [min(n, keep) for n in lengths]
        self.pool = Pool(rng, page=page, heads=heads, dk=dk, pages=pages, hnd=hnd)
        self.batch = Batch(rng, self.pool, lengths, qheads, per)
        self.short_pool = Pool(rng, page=page, heads=heads, dk=dk, hnd=hnd,
                               pages=sum(-(-n // page) for n in self.kept_lengths) + 3)
        self.short = Batch(rng, self.short_pool, self.kept_lengths, qheads)
        self.start = rng.random((heads, len(self.batch.slots))).astype(np.float32)
        self.sums = hip.DeviceBuffer.from_array(self.start)
        self.moved = _filled(4 * heads * len(self.short.slots))
        self.before = self.short_pool.bits.copy()
        self.bounds_start = np.full((self.short_pool.pages, heads, 2, dk), 0x1234, np.uint16)
        self.bounds = hip.DeviceBuffer.from_array(self.bounds_start)
        self.page_list = np.concatenate([self.short.own_slots(q)[::page] // page for q in range(len(lengths))])
        self.counts = np.concatenate([np.minimum(page, n - page * np.arange(-(-n // page))) for n in self.kept_lengths])
        self.page_buffers = [hip.DeviceBuffer.from_array(a.astype(np.uint32)) for a in (self.page_list, self.counts)]

        self.weight_plan = kv.WeightAccumulationPlan.new(self.batch.plan(), max_sequence_length=max(lengths))
        self.weight_buffers = kv.WeightAccumulationBuffers(
            **self.batch.device, pool=self.pool.buffer, weights=self.sums,
            workspace=_filled(self.weight_plan.workspace_required_bytes, 0xFF))
        self.eviction = kv.EvictionPlan.new(
            request_count=len(lengths), kv_head_count=heads, sequence_slot_count=len(self.batch.slots), max_kept=keep,
            destination_slot_count=len(self.short.slots), first_tokens=4, last_tokens=16)
        self.kept = _filled(self.eviction.kept_required_bytes)
        self.eviction_buffers = kv.EvictionBuffers(
            request_lengths=hip.DeviceBuffer.from_array(np.asarray(lengths, np.uint64)),
            request_slot_offsets=self.batch.device["request_slot_offsets"],
            sequence_slots=self.batch.device["sequence_slots"], weights=self.sums, kept=self.kept,
            destination_slot_offsets=self.short.device["request_slot_offsets"],
            destination_slots=self.short.device["sequence_slots"], destination_weights=self.moved,
            workspace=_filled(self.eviction.workspace_required_bytes, 0xFF))
        self.selection = kv.PageSelectionPlan.new(self.short.plan(), max_pages=listed, first_pages=1, last_pages=1)
        self.selected = _filled(self.selection.selected_required_bytes)
        self.output = _filled(self.selection.attention.output_required_bytes)
        self.selection_buffers = kv.PageSelectionBuffers(
            **self.short.device, pool=self.short_pool.buffer, bounds=self.bounds, selected=self.selected, output=self.output,
            workspace=_filled(self.selection.workspace_required_bytes, 0xFF))

    def enqueue(self, k, stream):
        k.accumulate_weights(self.weight_plan, self.weight_buffers, stream=stream)
        k.select_tokens(self.eviction, self.eviction_buffers, stream=stream)
        k.compact_tokens(self.eviction, self.eviction_buffers, self.pool.view(), self.short_pool.view(), stream=stream)
        k.page_bounds(self.short_pool.view(), pages=self.page_buffers[0], counts=self.page_buffers[1],
                      page_count=len(self.page_list), bounds=self.bounds, stream=stream)
        k.select_pages(self.selection, self.selection_buffers, stream=stream)
        k.selected_attention(self.selection, self.selection_buffers, stream=stream)

    def reset(self):
        """Everything that a run writes, as it was before the first."""
        self.sums.upload(self.start)
        self.bounds.upload(self.bounds_start)
        self.short_pool.buffer.upload(self.before)
        for held in (self.kept, self.moved, self.selected, self.output):
            held.fill(0xA5)
        hip.synchronize()

    def results(self):
        return [held.download().copy() for held in (self.sums, self.kept, self.moved, self.short_pool.buffer, self.bounds,
                                                    self.selected, self.output)]

    def check(self):
        heads, pool, short = self.pool.heads, self.pool, self.short
        sums, kept, moved, rows, bounds, selected, output = self.results()
        sums = sums.view(np.float32).reshape(self.start.shape)
        _check_weights(sums, _weights(self.batch, self.start))
        kept = kept.view(np.uint32).reshape(len(self.lengths), heads, self.keep)
        assert np.array_equal(kept, _kept(sums, self.lengths, self.batch.offsets, self.keep, 4, 16))
        # The copy, from what was there before it.
        self.short_pool.bits = self.before.copy()
        want_moved = np.zeros((heads, len(short.slots)), np.float32)
        for r, n in enumerate(self.lengths):
            own, to = int(self.batch.offsets[r]), int(short.offsets[r])
            for h in range(heads):
                for i, t in enumerate(kept[r, h][kept[r, h] != NONE]):
                    for tensor in (0, 1):
                        self.short_pool.rows(tensor).put(short.slots[to + i], h,
                                                         pool.rows(tensor).get(self.batch.slots[own + t], h))
                    want_moved[h, to + i] = sums[h, own + t]
        assert np.array_equal(rows.view(np.uint16), self.short_pool.bits)
        assert np.array_equal(moved.view(np.float32).reshape(want_moved.shape), want_moved)
        bounds = bounds.view(np.uint16).reshape(self.bounds_start.shape)
        want = f64(self.bounds_start)
        for p, c in zip(self.page_list, self.counts):
            want[p] = ref.page_bounds(self.short_pool, p, c)
        assert np.array_equal(f64(bounds), want)
        selected = selected.view(np.uint32).reshape(len(self.lengths), heads, self.listed)
        assert np.array_equal(selected, ref.select(short, bounds, self.listed, 1, 1))
        _check(f64(output.view(np.uint16).reshape(len(self.lengths), short.qheads, pool.dv)), *ref.attend(short, selected))


def _same(a, b):
    return all(np.array_equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("case", [
    dict(), dict(page=64, heads=8, qheads=32, lengths=(2000, 300, 64), keep=512, listed=5, per=1),
    dict(heads=2, qheads=14, dk=64, lengths=(900, 30, 129), keep=200, per=5, hnd=True),
    dict(page=48, heads=1, qheads=3, dk=40, lengths=(300, 7), keep=100, listed=2),
    dict(page=16, heads=2, qheads=4, dk=256, lengths=(150, 90), keep=64, per=1000)])
def test_a_step_of_all_calls(k, case):
    _say(f"long context: {case}")
    chain, stream = Chain(1, **case), hip.Stream()
    hip.synchronize()
    chain.enqueue(k, stream)
    stream.synchronize()
    k.check_errors()
    chain.check()
    stream.destroy()


def test_two_chains_at_once_on_two_streams(k):
    """Chains with buffers of their own do not see each other, and a repeated run gives the same bits."""
    chains = [Chain(2), Chain(3, page=64, heads=4, qheads=16, lengths=(3000, 100, 700), keep=256, listed=4, per=1)]
    streams = [hip.Stream(), hip.Stream()]
    want = []
    for chain in chains:
        chain.enqueue(k, None)
        hip.synchronize()
        want.append(chain.results())
    for i in range(4):
        for chain in chains:
            chain.reset()
        _say(f"long context: two streams, run {i}")
        for chain, stream in zip(chains, streams):
            chain.enqueue(k, stream)
        hip.synchronize()
        assert all(_same(chain.results(), w) for chain, w in zip(chains, want))
    k.check_errors()
    for stream in streams:
        stream.destroy()


def test_two_contexts_share_nothing(k):
    other = kv.RocmKvPairCopyKernels(0)
    chain = Chain(4)
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


def test_captured_chain_replays(k):
    """The chain in a graph: every replay gives the eager run's bits, with the same chain run
    eagerly in between, from inputs that the graph's buffers get before it."""
    chain, stream = Chain(5, page=64, heads=4, qheads=16, lengths=(1500, 100, 1, 700), keep=256, listed=4, per=2), hip.Stream()
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
    _say("long context: the chain under graph capture")
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


@pytest.mark.parametrize("hnd,dk,per", [(False, 128, 1), (True, 64, 3), (False, 128, 10 ** 6), (False, 40, 1)])
def test_offsets_past_32_bits(k, hnd, dk, per):
    """A pool of more than 8 GiB whose used pages lie at both its ends and across every 4 GiB
    gives what a small pool with the same rows gives."""
    rng = np.random.default_rng(6)
    page, heads, qheads, lengths = 64, 8, 16, (700, 130, 400)
    small = Pool(rng, page=page, heads=heads, dk=dk, pages=24, layers=16, layer=13, hnd=hnd)
    stride = small.layout.total_byte_len // 24
    pages = (9 << 30) // stride
    runtime = small.layout.runtime
    big = kv.PagedKvCacheLayout.new(runtime, pages)
    # Where the small pool's pages lie: the last ones, the ones round 4 and 8 GiB, the first.
    at = np.concatenate([np.arange(pages - 8, pages), *((g << 30) // stride + np.arange(-3, 3) for g in (4, 8)), np.arange(4)])
    _say(f"long context: {pages} pages of {stride} bytes, dims {dk}")
    held = hip.DeviceBuffer(big.total_byte_len)
    raw = small.bits.view(np.uint8).reshape(24, stride)
    for i, p in enumerate(at):
        held.upload(raw[i], int(p) * stride)
    batch = Batch(rng, small, lengths, qheads, per)
    start = rng.random((heads, len(batch.slots))).astype(np.float32)
    moved_slots = (at[batch.slots.astype(np.int64) // page] * page + batch.slots.astype(np.int64) % page).astype(np.uint64)
    small_view, big_view = small.view(), big.pool_view(held.ptr, held.nbytes, 13, small.head_layout, heads=heads)
    own = batch.own_slots
    listed = np.concatenate([np.unique(own(q) // page) for q in np.flatnonzero(np.append(batch.requests[1:] != batch.requests[:-1], True))])

    def run(view, layout, slots, pool, index):
        device = dict(batch.device, sequence_slots=hip.DeviceBuffer.from_array(slots))
        plan = kv.PagedAttentionPlan.for_layer(layout, 13, len(batch.ends), len(lengths), len(slots), qheads, dk ** -0.5,
                                               small.head_layout)
        weight_plan = kv.WeightAccumulationPlan.new(plan)
        sums = hip.DeviceBuffer.from_array(start)
        k.accumulate_weights(weight_plan, kv.WeightAccumulationBuffers(
            **device, pool=pool, weights=sums, workspace=_filled(weight_plan.workspace_required_bytes, 0xFF)))
        bounds = _filled(layout.total_byte_len // stride * heads * 4 * dk)
        entries = index[listed].astype(np.uint32)
        k.page_bounds(view, pages=hip.DeviceBuffer.from_array(entries), page_count=len(entries), bounds=bounds,
                      counts=hip.DeviceBuffer.from_array(np.full(len(entries), page, np.uint32)))
        hip.synchronize()
        selection = kv.PageSelectionPlan.new(plan, max_pages=4)
        selected, output = _filled(selection.selected_required_bytes), _filled(selection.attention.output_required_bytes)
        buffers = kv.PageSelectionBuffers(**device, pool=pool, bounds=bounds, selected=selected, output=output,
                                          workspace=_filled(selection.workspace_required_bytes, 0xFF))
        k.select_pages(selection, buffers)
        k.selected_attention(selection, buffers)
        hip.synchronize()
        k.check_errors()
        return [x.download() for x in (sums, selected, output)]

    want = run(small_view, small.layout, batch.slots, small.buffer, np.arange(24))
    got = run(big_view, big, moved_slots, held, at)
    assert _same(got, want)
    _check_weights(got[0].view(np.float32).reshape(start.shape), _weights(batch, start))
    # The copy: rows of the big pool into the small one's pages and back into the big one's.
    keep = 40
    plan = kv.EvictionPlan.new(request_count=3, kv_head_count=heads, sequence_slot_count=len(batch.slots), max_kept=keep,
                               destination_slot_count=3 * keep)
    lists = _kept(start, lengths, batch.offsets, keep, 0, 4)
    names = dict(request_lengths=np.asarray(lengths, np.uint64), request_slot_offsets=batch.offsets, kept=lists,
                 destination_slot_offsets=keep * np.arange(4, dtype=np.uint64))
    spare = np.setdiff1d(np.arange(24 * page), batch.slots.astype(np.int64))[:3 * keep]
    given = {n: hip.DeviceBuffer.from_array(v) for n, v in names.items()}
    for slots, to, source, destination in (
            (moved_slots, spare, big_view, small_view),
            (moved_slots, at[spare // page] * page + spare % page, big_view, big_view)):
        k.compact_tokens(plan, kv.EvictionBuffers(
            **given, sequence_slots=hip.DeviceBuffer.from_array(slots),
            destination_slots=hip.DeviceBuffer.from_array(to.astype(np.uint64))), source, destination)
        hip.synchronize()
    k.check_errors()
    for r in range(3):
        for h in range(heads):
            for i, t in enumerate(lists[r, h][lists[r, h] != NONE]):
                for tensor in (0, 1):
                    small.rows(tensor).put(spare[keep * r + i], h,
                                           small.rows(tensor).get(batch.slots[int(batch.offsets[r]) + t], h))
    assert np.array_equal(small.buffer.download().view(np.uint16), small.bits)
    after = small.bits.view(np.uint8).reshape(24, stride)
    for i, p in enumerate(at):
        assert np.array_equal(held.download(stride, int(p) * stride), after[i]), p
    held.free()
