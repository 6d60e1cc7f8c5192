"""GPU tests of eviction by accumulated attention weight (accumulate_weights,
select_tokens, compact_tokens) against 64-bit restatements.

Weights. A position's sum adds softmax weights w = 2^(x - m) / l, x = q.k scale
log2(e), in fp32. With u = 2^-24 (half a step), S = max |q| |k| scale log2(e)
over a row and N products a dot product (dk <= 1,024), the matrix product's sum
is off by at most N u S; x - m is one fused operation, another u (S + |m|) <= 2 u
S; exp2 (1 ulp) and its argument's error e turn into a factor 1 + 0.7 e + 2 u; l,
a sum of at most 2^17 such terms in runs of at most 2^11 (a lane's), gets at most
(2^11 + 10) u on top of them and 1/l and the last product 2 u more; and a position's
sum of M weights, all of one sign, M u. Random signs make the real errors the
square root of these; here S < 64, N = 128, so that 0.7 (N + 2) u S alone would
allow 5,900 u = 3.5e-4. The bound asked is 2e-5 of the position's sum, a
seventeenth of it, and 1e-9 for positions that get nothing.

Lists are whole numbers and rows are copied: both are compared exactly."""
import numpy as np
import pytest

import selection_reference as ref
import sgl_rocm_kv as kv
from selection_reference import NONE, Batch, Pool, bf16, f64
from sgl_rocm_kv import hip
from test_gpu_selection import _filled, _say

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def k():
    if hip.device_count() == 0:
        pytest.fail("no GPU visible: the gpu tests need an MI355X")
    ctx = kv.RocmKvPairCopyKernels(0)
    yield ctx
    ctx.close()


# ---- accumulation ---------------------------------------------------------------------------

def _weights(batch, start, scale=None):
    """The sums in float64 after one call on `start` [head][slot]."""
    pool, group = batch.pool, batch.qheads // batch.pool.heads
    scale = pool.dk ** -0.5 if scale is None else scale
    out = start.astype(np.float64)
    keys = pool.rows(0)
    for q, end in enumerate(batch.ends.astype(int)):
        if end == 0:
            continue
        slots = batch.own_slots(q)
        first = int(batch.offsets[batch.requests[q]])
        for h in range(pool.heads):
            s = f64(batch.queries[q, h * group:(h + 1) * group]) @ f64(keys.get(slots, h)).T * scale
            w = np.exp(s - s.max(axis=1, keepdims=True))
            out[h, first:first + end] += (w / w.sum(axis=1, keepdims=True)).sum(axis=0)
    return out


def _run_weights(k, batch, start, scale=None, longest=0, calls=1, stream=None):
    plan = kv.WeightAccumulationPlan.new(batch.plan(scale), max_sequence_length=longest)
    assert plan.weights_required_bytes == start.nbytes
    held = hip.DeviceBuffer.from_array(start)
    buffers = kv.WeightAccumulationBuffers(**batch.device, pool=batch.pool.buffer, pool_offset=batch.pool.shift, weights=held,
                                           workspace=_filled(plan.workspace_required_bytes, 0xFF))
    for _ in range(calls):
        k.accumulate_weights(plan, buffers, stream=stream)
    hip.synchronize()
    return held.download().view(np.float32).reshape(start.shape)


def _check_weights(got, want, label=""):
    ratio = np.abs(got - want) / (2e-5 * np.abs(want) + 1e-9)
    _say(f"weights {label}: largest error {np.abs(got - want).max():.3g}, {ratio.max():.3f} of the bound")
    assert ratio.max() <= 1.0


@pytest.mark.parametrize("page,heads,qheads,dk,dv,hnd,shift,lengths,per", [
    (64, 8, 32, 128, 128, False, 0, (3000,), 1),
    (64, 8, 32, 128, 128, True, 0, (1500, 64, 65, 1, 0), 1),
    (16, 2, 14, 64, 64, True, 0, (900, 17, 300), 5),
    (16, 2, 8, 256, 256, True, 0, (700, 31), 5),
    (1, 2, 4, 64, 64, False, 0, (300, 1, 2), 1),
    (48, 3, 9, 128, 128, False, 0, (600, 50), 2),
    (16, 1, 40, 64, 64, False, 0, (400,), 1),
    (64, 1, 128, 576, 512, False, 0, (500, 130), 1),
    (16, 2, 4, 20, 24, False, 0, (200,), 1),
    (16, 2, 4, 97, 113, True, 0, (200, 40), 3),
    (16, 2, 8, 128, 128, False, 2, (300,), 1),
    (16, 4, 16, 128, 128, False, 0, (200, 61, 1, 130), 10 ** 6),  # whole prompts
    (16, 2, 14, 64, 64, True, 0, (257, 100), 10 ** 6),
    (16, 1, 8, 256, 256, False, 0, (120, 33), 10 ** 6),
    (16, 2, 2, 128, 128, False, 0, (600, 40), 17),
    (16, 1, 33, 64, 64, False, 0, (300,), 40),                     # 33 query heads: three groups of 16
    (64, 8, 64, 128, 128, False, 0, tuple(range(100, 2100, 100)), 1),
    (16, 2, 4, 128, 128, False, 0, (3, 100, 0, 1, 64, 65, 2, 90), 20),   # tiles of queries of several requests
    (16, 2, 14, 64, 64, False, 0, (3, 100, 0, 1, 64, 65, 2, 90, 30), 11),
    (8, 1, 130, 64, 64, False, 0, (200, 31), 3),                         # a query's heads pass a tile
    (8, 1, 70, 256, 256, True, 0, (200, 31), 2),
    (16, 1, 1, 128, 128, False, 0, (5000,), 1),
    (16, 1, 2, 256, 256, False, 0, (700, 300), 300),
    (4, 8, 8, 64, 64, True, 0, (10, 20, 30, 4000), 2),
])
def test_weights(k, page, heads, qheads, dk, dv, hnd, shift, lengths, per):
    rng = np.random.default_rng(page + dk)
    pool = Pool(rng, page=page, heads=heads, dk=dk, dv=dv, pages=sum(-(-n // page) for n in lengths) + 2, hnd=hnd,
                shift=shift)
    batch = Batch(rng, pool, lengths, qheads, per, spare=3)
    start = rng.random((heads, len(batch.slots))).astype(np.float32)
    _say(f"weights page={page} heads={heads}x{qheads} dk={dk} hnd={hnd} lengths={lengths[:5]} per={per}")
    got = _run_weights(k, batch, start, longest=max(lengths))
    k.check_errors()
    want = _weights(batch, start)
    _check_weights(got, want)
    assert (got[want == start] == start[want == start]).all()  # untouched positions


@pytest.mark.parametrize("dk", [64, 128, 256])
def test_weights_of_a_long_slot_list(k, dk):
    """A plan for 4.4 million positions, whose scores are not kept: the few rows' way."""
    rng = np.random.default_rng(dk)
    pool = Pool(rng, page=16, heads=1, dk=dk, pages=60)
    batch = Batch(rng, pool, (500, 60, 300), 20, 1, spare=1_500_000)
    assert 4 * 60 * len(batch.slots) > 256 << 20
    start = rng.random((1, len(batch.slots))).astype(np.float32)
    _say(f"weights of a long slot list, dims {dk}")
    got = _run_weights(k, batch, start)
    k.check_errors()
    want = _weights(batch, start)
    _check_weights(got, want)
    assert (got[want == start] == start[want == start]).all()


@pytest.mark.parametrize("dk,qheads,per", [(128, 8, 1), (128, 8, 40), (64, 40, 2), (40, 6, 2)])
def test_weights_of_a_padded_batch(k, dk, qheads, per):
    """Queries of length 0 between the requests' and behind them (index UINT32_MAX) add nothing."""
    rng = np.random.default_rng(dk + per)
    pool = Pool(rng, page=16, heads=2, dk=dk, pages=80)
    batch = Batch(rng, pool, (500, 60, 0, 300), qheads, per)
    start = rng.random((2, len(batch.slots))).astype(np.float32)
    want = _weights(batch, start)
    batch.requests = np.concatenate([batch.requests, np.full(9, NONE, np.uint32)])
    batch.ends = np.concatenate([batch.ends, np.zeros(9, np.uint64)])
    padding = np.full((9, *batch.queries.shape[1:]), 0x7FC0, np.uint16)  # NaN
    batch.queries = np.concatenate([batch.queries, padding])
    batch.upload()
    _say(f"weights of a padded batch, dims {dk}")
    got = _run_weights(k, batch, start)
    k.check_errors()
    _check_weights(got, want)


def test_weights_refusals(k):
    rng = np.random.default_rng(12)
    pool = Pool(rng, page=8, heads=2, dk=64, pages=4)
    batch = Batch(rng, pool, (20,), 4)
    plan = kv.WeightAccumulationPlan.new(batch.plan())
    sums, workspace = _filled(plan.weights_required_bytes), _filled(plan.workspace_required_bytes)
    sound = dict(batch.device, pool=pool.buffer, weights=sums, workspace=workspace)

    def refused(variant, name, **more):
        with pytest.raises(kv.KvError) as e:
            k.accumulate_weights(plan, kv.WeightAccumulationBuffers(**{**sound, **more}))
        assert (e.value.variant, e.value.name) == (variant, name)

    host = np.zeros(1 << 16, np.uint8)
    for name in sound:
        refused("DeviceMismatch", name, **{name: kv.device_buffer(host.ctypes.data, host.nbytes)})
        refused("AllocationOutOfBounds", name, **{name + "_offset": 1 << 20})
    for name in ("queries", "query_request_indices", "query_sequence_lengths", "request_slot_offsets", "sequence_slots",
                 "weights", "workspace"):
        big = _filled(1 << 16)
        refused("InvalidArgument", "alignment", **{name: big, name + "_offset": 1})
    assert (sums.download() == 0xA5).all()
    k.check_errors()


def test_weights_of_one_call_add_up_and_repeat(k):
    """Two calls add twice; the same call gives the same bits; a row's weights sum to 1."""
    rng = np.random.default_rng(2)
    for d, per in ((128, 1), (64, 60), (256, 3)):
        pool = Pool(rng, page=16, heads=2, dk=d, pages=200)
        batch = Batch(rng, pool, (1500, 700, 64), 8, per)
        zero = np.zeros((2, len(batch.slots)), np.float32)
        once = _run_weights(k, batch, zero)
        assert np.array_equal(once, _run_weights(k, batch, zero))
        _check_weights(_run_weights(k, batch, zero, calls=3), 3 * once.astype(np.float64))
        assert abs(once.sum(dtype=np.float64) - 8 * len(batch.ends)) < 2e-5 * 8 * len(batch.ends)
    k.check_errors()


def test_weights_large_scores(k):
    """Scores of hundreds: the maximum is taken out before the exponential. A row's weights are then
    a few ones; scores S = 400 log2(e) allow 0.7 * 130 * 2^-24 * 577 = 3.2e-3 (see above): asked 3.2e-3."""
    rng = np.random.default_rng(3)
    pool = Pool(rng, page=16, heads=2, dk=128, pages=80)
    batch = Batch(rng, pool, (1000,), 8, 4)
    zero = np.zeros((2, len(batch.slots)), np.float32)
    got, want = _run_weights(k, batch, zero, scale=3.0), _weights(batch, zero, scale=3.0)
    assert np.isfinite(got).all() and (np.abs(got - want) <= 3.2e-3 * np.abs(want) + 1e-9).all()
    k.check_errors()


def test_weights_do_not_read_what_no_query_attends(k):
    """NaN keys behind the longest query of a request, and padding queries between others."""
    rng = np.random.default_rng(4)
    for d, per in ((128, 1), (64, 40)):
        pool = Pool(rng, page=16, heads=2, dk=d, pages=60)
        batch = Batch(rng, pool, (500, 300), 8, per)
        batch.ends[batch.requests == 0] -= 7
        batch.ends[0] = 0
        batch.upload()
        start = np.ones((2, len(batch.slots)), np.float32)
        want = _weights(batch, start)
        rows = pool.rows(0)
        for t in range(493, 500):
            for h in (0, 1):
                rows.put(batch.slots[t], h, 0x7FC0)
        pool.upload()
        got = _run_weights(k, batch, start)
        if per == 1:  # its only query is padding: request 0 gets nothing
            assert (got[:, :500] == 1).all()
        _check_weights(got, want, f"dims {d}")
        assert (got[:, 493:500] == 1).all()
    k.check_errors()


def test_weights_nan_keys_reach_only_their_request(k):
    rng = np.random.default_rng(5)
    pool = Pool(rng, page=16, heads=2, dk=128, pages=60)
    batch = Batch(rng, pool, (500, 300), 8)
    pool.rows(0).put(batch.slots[77], 1, 0x7FC0)
    pool.upload()
    zero = np.zeros((2, len(batch.slots)), np.float32)
    got, want = _run_weights(k, batch, zero), _weights(batch, zero)
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.isnan(got[1, :500]).all()
    fine = ~np.isnan(want)
    _check_weights(got[fine], want[fine])
    k.check_errors()


@pytest.mark.parametrize("kind", ["query", "key", "infinity"])
@pytest.mark.parametrize("dk,heads,qheads,per", [
    (64, 2, 8, 40), (128, 2, 8, 40), (256, 2, 8, 40),     # many rows, a request's queries in one part
    (64, 2, 8, 200), (128, 2, 8, 200), (256, 2, 8, 200),  # in several
    (64, 2, 8, 5), (128, 2, 8, 2), (40, 2, 6, 30)])       # few rows; kept scores; any dims
def test_weights_nan_ends_where_its_queries_end(k, kind, dk, heads, qheads, per):
    """A NaN query, a NaN key and a query whose scores are all -inf make NaN of what their queries attend, and of
    nothing behind it: neither what longer queries attend further on nor what none does."""
    rng = np.random.default_rng(dk + per)
    pool = Pool(rng, page=16, heads=heads, dk=dk, pages=60)
    batch = Batch(rng, pool, (500, 300), qheads, per, spare=70)
    batch.ends[batch.requests == 0] -= 39  # (from 461 down: inside a wave's tokens)
    odd = int(np.flatnonzero(batch.requests == 0)[len(np.flatnonzero(batch.requests == 0)) // 2])
    if kind == "query":
        batch.queries[odd, 1, 3] = 0x7FC0
    elif kind == "key":
        pool.rows(0).put(batch.slots[int(batch.ends[odd]) - 1], 0, np.full(dk, 0x7FC0))
    else:  # a positive key everywhere, times -inf
        for slot in batch.slots[:500]:
            pool.rows(0).put(slot, 0, np.where(np.arange(dk) == 3, 0x3F80, pool.rows(0).get([slot], 0)[0]))
        batch.queries[odd, 1, 3] = 0xFF80
    batch.upload()
    pool.upload()
    start = rng.random((heads, len(batch.slots))).astype(np.float32)
    _say(f"weights with a {kind} of NaN, dims {dk}, {per} queries a request")
    with np.errstate(invalid="ignore"):
        want = _weights(batch, start)
    got = _run_weights(k, batch, start, longest=500)
    k.check_errors()
    assert np.isnan(want[0, int(batch.ends[odd]) - 1]) and not np.isnan(want[0, 461:]).any()
    assert np.array_equal(np.isnan(got), np.isnan(want))
    fine = ~np.isnan(want)
    _check_weights(got[fine], want[fine], f"{kind}, dims {dk}")
    same = want == start
    assert same[:, 461:500].all() and (got[same] == start[same]).all()


def test_weights_report_bad_metadata(k):
    rng = np.random.default_rng(6)
    pool = Pool(rng, page=16, heads=2, dk=64, pages=60, layers=1, layer=0)

    def case(change, per=1, longest=400):
        batch = Batch(rng, pool, (400, 300), 4, per)
        start = np.zeros((2, len(batch.slots)), np.float32)
        sound = _weights(batch, start)
        change(batch)
        batch.upload()
        got = _run_weights(k, batch, start, longest=longest)
        with pytest.raises(kv.KvError) as e:
            k.check_errors()
        assert e.value.variant == "DeviceMetadataInvalid"
        return got, sound, e.value.fields[0]

    def last(b): b.requests[-1] = 2
    def length(b): b.ends[0] = 401
    def slot(b): b.slots[32] = 60 * 16
    def falls(b): b.requests[:] = b.requests[::-1].copy()
    got, sound, flags = case(last)
    assert flags == 1 and (got[:, 400:] == 0).all()
    _check_weights(got[:, :400], sound[:, :400])
    for change, longest in ((length, 400), (lambda b: None, 399)):
        got, sound, flags = case(change, longest=longest)
        assert flags == 2 and (got[:, :400] == 0).all()
        _check_weights(got[:, 400:], sound[:, 400:])
    assert case(slot)[2] == 4
    assert case(falls, per=2)[2] & 1
    k.check_errors()


# ---- kept positions -------------------------------------------------------------------------

def _kept(weights, lengths, offsets, keep, first, last):
    """[request][head][keep] lists from weights [head][slot]."""
    out = np.full((len(lengths), len(weights), keep), NONE, np.uint32)
    for r, n in enumerate(lengths):
        j = np.arange(n)
        forced = (j < first) | (j + last >= n)
        for h in range(len(weights)):
            w = weights[h, int(offsets[r]):int(offsets[r]) + n].astype(np.float64)
            order = np.lexsort((j, -np.where(np.isnan(w), 0.0, w), ~np.isnan(w), ~forced))
            best = np.sort(order[:keep])
            out[r, h, :len(best)] = best
    return out


def _buffers(plan, lengths, offsets, weights, kept=None, **more):
    kept = _filled(plan.kept_required_bytes) if kept is None else kept
    return kv.EvictionBuffers(request_lengths=hip.DeviceBuffer.from_array(np.asarray(lengths, np.uint64)),
                              request_slot_offsets=hip.DeviceBuffer.from_array(np.asarray(offsets, np.uint64)),
                              weights=hip.DeviceBuffer.from_array(weights), kept=kept,
                              workspace=_filled(plan.workspace_required_bytes, 0xFF), **more), kept


def _run_kept(k, weights, lengths, offsets, keep, first=0, last=0, longest=0):
    plan = kv.EvictionPlan.new(request_count=len(lengths), kv_head_count=len(weights),
                               sequence_slot_count=weights.shape[1], max_kept=keep, first_tokens=first, last_tokens=last,
                               max_sequence_length=longest)
    buffers, kept = _buffers(plan, lengths, offsets, weights)
    k.select_tokens(plan, buffers)
    hip.synchronize()
    return kept.download().view(np.uint32).reshape(len(lengths), len(weights), keep)


def _offsets(lengths, spare=0):
    return np.concatenate([[0], np.cumsum([n + spare for n in lengths])]).astype(np.uint64)


@pytest.mark.parametrize("lengths,heads,keep,first,last", [
    ((5000,), 8, 1000, 4, 16), ((100, 0, 1, 33, 2000), 2, 32, 1, 2), ((70000, 3000), 1, 2048, 0, 0),
    ((1025, 1024, 1023), 3, 1024, 4, 4), ((300,), 4, 1, 0, 0), ((300,), 4, 7, 3, 4), ((2, 3), 1, 100, 50, 50),
    ((200001,), 1, 199999, 0, 0), (tuple(range(60, 90)), 5, 64, 0, 8)])
def test_kept(k, lengths, heads, keep, first, last):
    rng = np.random.default_rng(keep)
    offsets = _offsets(lengths, 3)
    weights = np.exp(3 * rng.standard_normal((heads, int(offsets[-1])))).astype(np.float32)
    _say(f"kept lengths={lengths[:5]} heads={heads} keep={keep}")
    got = _run_kept(k, weights, lengths, offsets, keep, first, last, max(lengths))
    k.check_errors()
    assert np.array_equal(got, _kept(weights, lengths, offsets, keep, first, last))


def test_kept_ties_signs_nan_and_infinities(k):
    rng = np.random.default_rng(7)
    lengths = (900, 64, 1300)
    offsets = _offsets(lengths)
    n = int(offsets[-1])
    few = rng.choice(np.array([0.5, 1.0, 1.0000001, 0.0, -0.0, -1.0, 3e-45, -3e-45], np.float32), (4, n))
    odd = few.copy()
    odd[rng.random(few.shape) < 0.02] = np.nan
    odd[rng.random(few.shape) < 0.02] = np.inf
    odd[rng.random(few.shape) < 0.02] = -np.inf
    odd.view(np.uint32)[0, 5] = 0xFFFFFFFF  # NaN of either sign and any payload
    for weights in (few, odd, np.zeros_like(few), np.full_like(few, np.nan)):
        for keep in (1, 40, 600):
            got = _run_kept(k, weights, lengths, offsets, keep, 0, min(keep, 2))
            assert np.array_equal(got, _kept(weights, lengths, offsets, keep, 0, min(keep, 2)))
    k.check_errors()


@pytest.mark.parametrize("values", [(0, 1), (0, 1, 2, 3), (0, 4), (1, 3), (-4, 0), (-2, -1, 2, 8), (np.inf, 0)])
def test_kept_ties_of_round_values(k, values):
    """Sums a power of two apart, whose largest alone are more than the list takes: a counting step that holds
    just the largest key. The longest request has more positions than a workgroup keeps in registers."""
    rng = np.random.default_rng(9)
    lengths = (40000, 900, 3000)
    offsets = _offsets(lengths)
    weights = rng.choice(np.asarray(values, np.float32), (2, int(offsets[-1])))
    _say(f"kept among sums of {values}")
    for keep in (1, 40, 200):
        got = _run_kept(k, weights, lengths, offsets, keep)
        assert np.array_equal(got, _kept(weights, lengths, offsets, keep, 0, 0))
    k.check_errors()


def test_kept_and_compact_do_not_look_at_the_reserved_workspace(k):
    """Neither a missing one nor one that is no device memory changes a result."""
    rng = np.random.default_rng(10)
    lengths, offsets = (300, 20), _offsets((300, 20))
    weights = rng.random((2, 320)).astype(np.float32)
    plan = kv.EvictionPlan.new(request_count=2, kv_head_count=2, sequence_slot_count=320, max_kept=30,
                               destination_slot_count=50)
    raw, held, view, at = _side(rng, page=16, heads=2, chunk=64, pages=20)
    want = _kept(weights, lengths, offsets, 30, 0, 0)
    host = np.zeros(64, np.uint8)
    for more in ({}, dict(workspace=kv.device_buffer(host.ctypes.data, 64), workspace_offset=1 << 40)):
        to_raw, to_held, to_view, to_at = _side(rng, page=16, heads=2, chunk=64, pages=4)
        given = dict(request_lengths=np.asarray(lengths, np.uint64), request_slot_offsets=offsets, weights=weights,
                     sequence_slots=np.arange(320, dtype=np.uint64), destination_slots=np.arange(50, dtype=np.uint64),
                     destination_slot_offsets=np.array([0, 30, 50], np.uint64))
        given = {n: hip.DeviceBuffer.from_array(a) for n, a in given.items()}
        kept, moved = _filled(plan.kept_required_bytes), _filled(plan.destination_weights_required_bytes)
        buffers = kv.EvictionBuffers(**given, kept=kept, destination_weights=moved, **more)
        k.select_tokens(plan, buffers)
        k.compact_tokens(plan, buffers, view, to_view)
        hip.synchronize()
        k.check_errors()
        assert np.array_equal(kept.download().view(np.uint32).reshape(want.shape), want)
        for h in (0, 1):
            for i, t in enumerate(want[0, h]):
                assert np.array_equal(to_held.download()[to_at(1, i, h)], raw[at(1, t, h)])


def test_kept_reports_bad_requests(k):
    rng = np.random.default_rng(8)
    lengths = (100, 50, 70)
    offsets = _offsets(lengths)
    weights = rng.random((2, 220)).astype(np.float32)
    want = _kept(weights, lengths, offsets, 9, 0, 1)
    for change, longest in (((101, 50, 70), 0), ((100, 50, 70), 99), ((2 ** 63, 50, 70), 0)):
        got = _run_kept(k, weights, change, offsets, 9, 0, 1, longest)
        with pytest.raises(kv.KvError) as e:
            k.check_errors()
        assert e.value.variant == "DeviceMetadataInvalid" and e.value.fields[0] == 2
        assert (got[0] == NONE).all() and np.array_equal(got[1:], want[1:])
    for bad in ([0, 100, 150, 221], [0, 2 ** 63, 150, 220]):
        _run_kept(k, weights, lengths, np.asarray(bad, np.uint64), 9, 0, 1)
        with pytest.raises(kv.KvError) as e:
            k.check_errors()
        assert e.value.fields[0] == 2


# ---- the copy -------------------------------------------------------------------------------

def _side(rng, *, page, heads, chunk, pages, tensors=2, hnd=False, shift=0, value_chunk=None):
    """A pool of one layer in bytes with room around its regions, its view, and (tensor, slot, head) -> bytes."""
    widths = [heads * chunk, heads * (value_chunk or chunk)][:tensors]
    offset = [32]
    offset.append(offset[0] + page * widths[0] + 16)
    stride = offset[tensors - 1] + page * widths[tensors - 1] + 16
    raw = rng.integers(0, 256, shift + stride * pages, dtype=np.uint8)
    held = hip.DeviceBuffer.from_array(raw)
    view = kv.pool_view(held.ptr + shift, held.nbytes - shift, page_size=page, page_stride_bytes=stride, page_count=pages,
                        tensor_offset=tuple(offset[:tensors]), row_bytes=widths[0], tensor_count=tensors, heads=heads,
                        head_layout=kv.HND if hnd else kv.NHD,
                        **({"value_row_bytes": widths[1]} if tensors == 2 and value_chunk else {}))

    def at(t, slot, h):
        c = widths[t] // heads
        p, i = divmod(int(slot), page)
        inside = (h * page + i) * c if hnd else i * widths[t] + h * c
        start = shift + p * stride + offset[t] + inside
        return slice(start, start + c)
    return raw, held, view, at


@pytest.mark.parametrize("heads,chunk,value_chunk,tensors,src,dst", [
    (8, 256, None, 2, dict(page=64, hnd=False), dict(page=64, hnd=False)),
    (2, 128, None, 2, dict(page=16, hnd=True), dict(page=16, hnd=True)),
    (4, 512, None, 2, dict(page=1, hnd=False), dict(page=16, hnd=True)),
    (20, 64, None, 2, dict(page=16, hnd=True), dict(page=48, hnd=False)),   # more heads than a workgroup takes
    (1, 1152, 1024, 2, dict(page=64), dict(page=16)),                       # an MLA pair
    (1, 649, None, 1, dict(page=64), dict(page=64)),                        # packed rows
    (3, 40, 24, 2, dict(page=7, hnd=True), dict(page=5)),
    (2, 34, None, 2, dict(page=8), dict(page=8, shift=2)),
    (2, 6, None, 2, dict(page=8, shift=1), dict(page=8)),
    (1, 16, None, 1, dict(page=8), dict(page=4)),
    (1, 8192, None, 2, dict(page=4), dict(page=4)),
])
def test_compact(k, heads, chunk, value_chunk, tensors, src, dst):
    rng = np.random.default_rng(chunk)
    lengths, keep = (300, 40, 0, 1, 200), 70
    offsets = _offsets(lengths, 2)
    n = int(offsets[-1])
    shape = dict(heads=heads, chunk=chunk, value_chunk=value_chunk, tensors=tensors)
    raw, _held, view, at = _side(rng, pages=-(-n // src["page"]) + 2, **shape, **src)
    slots = rng.permutation((-(-n // src["page"]) + 2) * src["page"])[:n].astype(np.uint64)
    # Destinations: room for what is kept, more, and (a request of one token) none to spare.
    room = [70, 55, 3, 1, 70]
    to_offsets = _offsets(room)
    m = int(to_offsets[-1])
    to_raw, to_held, to_view, to_at = _side(rng, pages=-(-m // dst["page"]) + 1, **shape, **dst)
    to_slots = rng.permutation((-(-m // dst["page"]) + 1) * dst["page"])[:m].astype(np.uint64)
    weights = rng.random((heads, n)).astype(np.float32)
    plan = kv.EvictionPlan.new(request_count=5, kv_head_count=heads, sequence_slot_count=n, destination_slot_count=m,
                               max_kept=keep, last_tokens=3)
    lists = _kept(weights, lengths, offsets, keep, 0, 3)
    to_weights = _filled(4 * heads * m)
    buffers, _ = _buffers(plan, lengths, offsets, weights, hip.DeviceBuffer.from_array(lists),
                          sequence_slots=hip.DeviceBuffer.from_array(slots),
                          destination_slot_offsets=hip.DeviceBuffer.from_array(to_offsets),
                          destination_slots=hip.DeviceBuffer.from_array(to_slots), destination_weights=to_weights)
    _say(f"compact heads={heads} chunk={chunk} src={src} dst={dst}")
    k.compact_tokens(plan, buffers, view, to_view)
    hip.synchronize()
    k.check_errors()
    want, want_weights = to_raw.copy(), np.zeros((heads, m), np.float32)
    for r in range(5):
        for h in range(heads):
            for i, t in enumerate(lists[r, h][lists[r, h] != NONE]):
                s, d = slots[int(offsets[r]) + t], to_slots[int(to_offsets[r]) + i]
                for tensor in range(tensors):
                    want[to_at(tensor, d, h)] = raw[at(tensor, s, h)]
                want_weights[h, int(to_offsets[r]) + i] = weights[h, int(offsets[r]) + t]
    assert np.array_equal(to_held.download(), want)
    assert np.array_equal(to_weights.download().view(np.float32).reshape(heads, m), want_weights)


def _small_compact(k, change=lambda v: None, weights=True):
    """Two requests of 20 and 12 tokens, 5 kept each, one pool, destinations behind the sources."""
    rng = np.random.default_rng(9)
    v = dict(lengths=np.array([20, 12], np.uint64), offsets=np.array([0, 20, 32], np.uint64),
             slots=rng.permutation(32).astype(np.uint64), to_offsets=np.array([0, 5, 10], np.uint64),
             to_slots=(32 + rng.permutation(16)[:10]).astype(np.uint64),
             kept=np.stack([np.sort(rng.choice(12, 5, replace=False)) for _ in range(4)]).reshape(2, 2, 5).astype(np.uint32))
    sums = rng.random((2, 32)).astype(np.float32)
    raw, held, view, at = _side(rng, page=16, heads=2, chunk=64, pages=3)
    want = raw.copy()
    for r in range(2):
        for h in range(2):
            for i, t in enumerate(v["kept"][r, h]):
                for tensor in (0, 1):
                    want[at(tensor, v["to_slots"][5 * r + i], h)] = raw[at(tensor, v["slots"][20 * r + t], h)]
    change(v)
    plan = kv.EvictionPlan.new(request_count=2, kv_head_count=2, sequence_slot_count=32, destination_slot_count=10,
                               max_kept=5)
    names = dict(request_lengths="lengths", request_slot_offsets="offsets", sequence_slots="slots", kept="kept",
                 destination_slot_offsets="to_offsets", destination_slots="to_slots")
    given = {n: hip.DeviceBuffer.from_array(v[x]) for n, x in names.items()}
    if weights:
        given.update(weights=hip.DeviceBuffer.from_array(sums), destination_weights=_filled(80))
    k.compact_tokens(plan, kv.EvictionBuffers(**given), view, view)
    hip.synchronize()
    return held.download(), want, raw, at, v


def test_compact_within_one_pool_and_without_weights(k):
    for weights in (True, False):
        got, want, *_ = _small_compact(k, weights=weights)
        k.check_errors()
        assert np.array_equal(got, want)


def test_compact_reports_bad_entries_and_copies_the_rest(k):
    def past(v): v["kept"][0, 0, 4] = 20
    def slot(v): v["slots"][int(v["kept"][0, 0, 4])] = 48
    def to_slot(v): v["to_slots"][4] = 1 << 33
    def length(v): v["lengths"][0] = 21
    def room(v): v["to_offsets"][:] = (0, 4, 9)
    def ranges(v): v["to_offsets"][:] = (0, 11, 10)
    for change, flag in ((past, 2), (slot, 4), (to_slot, 4), (length, 2), (ranges, 2)):
        got, want, raw, at, v = _small_compact(k, change)
        with pytest.raises(kv.KvError) as e:
            k.check_errors()
        assert e.value.variant == "DeviceMetadataInvalid" and e.value.fields[0] == flag, change.__name__
        if change is not ranges:  # request 1 is whole
            for h in (0, 1):
                for d in v["to_slots"][5:]:
                    assert np.array_equal(got[at(0, d, h)], want[at(0, d, h)]) and np.array_equal(got[at(1, d, h)], want[at(1, d, h)])
    got, *_ = _small_compact(k, room)
    with pytest.raises(kv.KvError) as e:
        k.check_errors()
    assert e.value.fields[0] == 2


def test_compact_copies_scales(k):
    rng = np.random.default_rng(10)
    raw, held, view, at = _side(rng, page=8, heads=1, chunk=64, pages=2)
    to_raw, to_held, to_view, to_at = _side(rng, page=8, heads=1, chunk=64, pages=2)
    import ctypes
    scales = [hip.DeviceBuffer.from_array(np.array(x, np.float32)) for x in ((0.5, 0.25), (1.0, 1.0))]
    for v, s in ((view, scales[0]), (to_view, scales[1])):
        v.scale = ctypes.cast(s.ptr, type(v.scale)) if not isinstance(v.scale, (int, type(None))) else s.ptr
    one = np.zeros(1, np.uint64)
    plan = kv.EvictionPlan.new(request_count=1, kv_head_count=1, sequence_slot_count=1, destination_slot_count=1, max_kept=1)
    given = dict(request_lengths=one + 1, request_slot_offsets=np.array([0, 1], np.uint64), sequence_slots=one + 9,
                 kept=np.zeros(1, np.uint32), destination_slot_offsets=np.array([0, 1], np.uint64), destination_slots=one + 3)
    buffers = kv.EvictionBuffers(**{n: hip.DeviceBuffer.from_array(a) for n, a in given.items()})
    k.compact_tokens(plan, buffers, view, to_view)
    k.check_errors()
    assert (scales[1].download().view(np.float32) == (0.5, 0.25)).all()
    assert np.array_equal(to_held.download()[to_at(0, 3, 0)], raw[at(0, 9, 0)])


def test_compact_refusals(k):
    rng = np.random.default_rng(11)
    raw, held, view, at = _side(rng, page=8, heads=2, chunk=64, pages=2)
    plan = kv.EvictionPlan.new(request_count=1, kv_head_count=2, sequence_slot_count=4, destination_slot_count=4, max_kept=4)
    slots = hip.DeviceBuffer.from_array(np.arange(4, dtype=np.uint64))
    given = dict(request_lengths=np.full(1, 4, np.uint64), request_slot_offsets=np.array([0, 4], np.uint64),
                 kept=np.zeros((1, 2, 4), np.uint32), destination_slot_offsets=np.array([0, 4], np.uint64))
    given = {n: hip.DeviceBuffer.from_array(a) for n, a in given.items()}

    def refused(variant, name, source=view, destination=view, **more):
        with pytest.raises(kv.KvError) as e:
            k.compact_tokens(plan, kv.EvictionBuffers(**{**given, "sequence_slots": slots, **more}), source, destination)
        assert (e.value.variant, e.value.name) == (variant, name)

    other = hip.DeviceBuffer.from_array(np.arange(4, dtype=np.uint64) + 8)
    refused("InvalidArgument", "in place", destination_slots=slots)
    refused("DeviceMismatch", "destination_slots")
    refused("AllocationOutOfBounds", "destination_slots", destination_slots=other, destination_slots_offset=8)
    refused("InvalidArgument", "alignment", destination_slots=kv.device_buffer(other.ptr + 1, 1 << 20))
    refused("DeviceMismatch", "destination_weights", destination_slots=other, weights=other)
    for change in (dict(heads=4, chunk=32), dict(heads=2, chunk=32), dict(heads=2, chunk=64, tensors=1),
                   dict(heads=2, chunk=64, value_chunk=32)):
        _, kept_alive, wrong, _ = _side(rng, page=8, pages=2, **change)
        refused("InvalidArgument", "views", destination=wrong, destination_slots=other)
    refused("InvalidArgument", "in place", destination_slots=other, weights=other, destination_weights=other)
    host = np.zeros(64, np.uint8)
    refused("DeviceMismatch", "kept", destination_slots=other, kept=kv.device_buffer(host.ctypes.data, 64))
