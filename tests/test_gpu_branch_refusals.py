"""GPU tests of calls that the operators for several continuations refuse because one write would meet another or a
read: nothing is launched, and what was there stays."""
import numpy as np
import pytest

import sgl_rocm_kv as kv
from sgl_rocm_kv import hip
from test_gpu_beams import _random
from test_gpu_branches import POOLS, Bytes, Drafts, _forks, _same
from test_gpu_selection import _filled
from test_gpu_tree import _make

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def k():
    if hip.device_count() == 0:
        pytest.fail("no GPU visible: the gpu tests need an MI355X")
    ctx = kv.RocmKvPairCopyKernels(0)
    yield ctx
    ctx.close()


def _refused(variant, name, call):
    with pytest.raises(kv.KvError) as e:
        call()
    assert (e.value.variant, e.value.name) == (variant, name)


# Of POOLS[0], page 16, rows of 2,048 bytes: a region of 32,768 bytes, K and V side by side.
@pytest.mark.parametrize("layers,stride", [(2, 0), (3, 1), (2, 16 * 2048 - 16), (2, 16 * 2048), (3, 16 * 2048 + 4096)])
def test_layers_that_overlap(k, layers, stride):
    """A row would be moved twice, or a layer's K while another's V is."""
    rng = np.random.default_rng(71)
    pool = Bytes(rng, pages=12, **POOLS[0])
    case = Drafts(rng, pool, (5, 9), (12, 17), [(1, 4), (2,)], 2)
    case.run(k)
    after = pool.device.download()
    plan = kv.DraftPlan.new(request_count=2, sequence_slot_count=len(case.slots), max_kept=2)
    _refused("InvalidArgument", "layer_stride",
             lambda: k.keep_drafts(plan, kv.DraftBuffers(**case.given), pool.view(), layer_count=layers, layer_stride_bytes=stride))
    hip.synchronize()
    assert np.array_equal(pool.device.download(), after)
    forks = _forks(31, POOLS[0], [40, 40], [0, 0], [1, 1])
    plan, buffers = forks.plan_and_buffers()
    _refused("InvalidArgument", "layer_stride",
             lambda: k.fork_sequences(plan, buffers, forks.pool.view(), layer_count=layers, layer_stride_bytes=stride))
    hip.synchronize()
    _same(forks.state(), forks.untouched())
    k.check_errors()


def test_layers_that_do_not(k):
    """K of all layers, then V of all: the stride is one region. One layer has no stride."""
    rng = np.random.default_rng(72)
    page, row, layers, pages = 16, 64, 3, 8
    region = page * row
    raw = rng.integers(0, 256, pages * 2 * layers * region, dtype=np.uint8)
    held = hip.DeviceBuffer.from_array(raw)
    view = kv.pool_view(held.ptr, held.nbytes, page_size=page, page_stride_bytes=2 * layers * region, page_count=pages,
                        tensor_offset=(0, layers * region), row_bytes=row, tensor_count=2, heads=1, head_layout=kv.NHD)
    plan = kv.DraftPlan.new(request_count=1, sequence_slot_count=40, max_kept=2)
    slots = rng.permutation(pages * page)[:40].astype(np.uint64)
    given = dict(request_lengths=np.asarray([30], np.uint64), request_slot_offsets=np.asarray([0, 40], np.uint64),
                 sequence_slots=slots, kept=np.asarray([3, 9], np.uint32))
    buffers = kv.DraftBuffers(**{n: hip.DeviceBuffer.from_array(a) for n, a in given.items()})
    k.keep_drafts(plan, buffers, view, layer_count=layers, layer_stride_bytes=region)
    hip.synchronize()
    k.check_errors()
    want = raw.reshape(pages, 2 * layers, page, row).copy()
    for i, draft in enumerate((3, 9)):
        to, source = int(slots[30 + i]), int(slots[30 + draft])
        want[to // page, :, to % page] = raw.reshape(want.shape)[source // page, :, source % page]
    assert np.array_equal(held.download(), want.reshape(-1))
    k.keep_drafts(plan, buffers, view, layer_count=1, layer_stride_bytes=0)
    hip.synchronize()
    k.check_errors()


def test_forked_tables_in_the_pool(k):
    """Inside the pool's pages they are refused; behind the last, in the same allocation, they are not."""
    case = _forks(33, POOLS[1], [40, 40], [0, 0], [1, 1])
    plan, _ = case.plan_and_buffers()
    pool, used = case.pool, case.pool.device.nbytes
    arena = hip.DeviceBuffer(used + 4096)
    arena.upload(np.concatenate([pool.raw, np.full(4096, 0xA5, np.uint8)]))
    view = pool.view()
    view.base, view.byte_len = arena.ptr, arena.nbytes

    def call(**change):
        k.fork_sequences(plan, kv.ForkBuffers(**{**case.device, **change}), view, **pool.call())

    for name in ("forked_lengths", "forked_tables"):
        n = case.device[name].nbytes
        for at in (0, used // 2 // 16 * 16, used - 16):
            _refused("InvalidArgument", "in place", lambda: call(**{name: kv.device_buffer(arena.ptr + at, n)}))
    hip.synchronize()
    assert np.array_equal(arena.download()[:used], pool.raw)
    tables = kv.device_buffer(arena.ptr + used, case.device["forked_tables"].nbytes)
    call(forked_tables=tables)
    hip.synchronize()
    k.check_errors()
    want = case.want()
    got = arena.download()
    assert np.array_equal(got[:used], want[5])
    assert np.array_equal(got[used:used + tables.byte_len].view(np.int32).reshape(want[1].shape), want[1])


@pytest.mark.parametrize("beams,vocab", [(4, 9000), (1, 50), (20, 700)])  # (20 x 20 continuations: the merge by lists)
def test_scores_in_place(k, beams, vocab):
    """As many continuations as beams: the best scores may take the scores' places."""
    case = _random(73, 40, beams, vocab, beams, "bf16")
    want = [a.copy() for a in case.run(k)]
    scores = np.concatenate([case.scores.reshape(-1).view(np.uint8), np.full(64, 0xA5, np.uint8)])
    case.given["scores"] = case.given["best_scores"] = hip.DeviceBuffer.from_array(scores)
    got = case.run(k)
    k.check_errors()
    assert all(np.array_equal(a, b) for a, b in zip(got, want))


def test_outputs_over_inputs(k):
    case = _random(74, 3, 4, 600, 8, "f32")
    shared = hip.DeviceBuffer(1 << 20)

    def call(**change):
        k.select_beams(case.plan, kv.BeamBuffers(**{**case.given, **change}))

    for written in ("best_scores", "best_parents", "best_tokens", "workspace"):
        for other in case.given:
            if other.endswith("_offset") or other == written:
                continue
            nbytes = getattr(case.plan, other + "_required_bytes")
            _refused("InvalidArgument", "in place", lambda: call(**{
                other: shared, written: kv.device_buffer(shared.ptr + nbytes // 16 * 16 - (16 if nbytes % 16 == 0 else 0), 1 << 19)}))
    _refused("InvalidArgument", "in place", lambda: call(scores=shared, best_scores=shared))  # (8 kept of 4 beams)
    square = _random(75, 3, 4, 600, 4, "f32")
    _refused("InvalidArgument", "in place", lambda: k.select_beams(square.plan, kv.BeamBuffers(**{
        **square.given, "logits": shared, "scores": shared, "best_scores": shared})))
    call()
    hip.synchronize()
    k.check_errors()


@pytest.mark.parametrize("dk", [128, 40])
def test_attention_over_its_inputs(k, dk):
    _, trees = _make(9, dk=dk, contexts=(50, 900), drafts=(10, 7))
    plan = trees.plan()
    sizes = {n: getattr(plan.attention, n + "_required_bytes") for n in (
        "query_request_indices", "query_sequence_lengths", "request_slot_offsets", "sequence_slots", "pool", "output")}
    sizes.update(queries=plan.attention.query_required_bytes, masks=plan.masks_required_bytes,
                 workspace=plan.workspace_required_bytes)
    given = dict(**trees.upload(), pool=trees.pool.buffer, output=_filled(sizes["output"]), workspace=_filled(sizes["workspace"]))
    assert set(sizes) == set(given) and all(sizes.values())
    shared = hip.DeviceBuffer(max(sizes.values()) + (1 << 22))
    for written in ("output", "workspace"):
        for other in given:
            if other == written:
                continue
            at = (sizes[other] - 1) // 16 * 16
            _refused("InvalidArgument", "in place", lambda: k.tree_attention(plan, kv.TreeAttentionBuffers(**{
                **given, other: shared, written: kv.device_buffer(shared.ptr + at, 1 << 21)})))
    k.tree_attention(plan, kv.TreeAttentionBuffers(**given))
    hip.synchronize()
    k.check_errors()
