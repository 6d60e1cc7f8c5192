"""GPU tests of tree attention against the 64-bit restatement in
branch_reference.py. The bound is that of tests/test_gpu_selection.py: u |want|
for the output's rounding (u = 2^-8, half a step of bf16), 2^-12 sum_i w_i |v_i|
for the hi + lo weights (2^-16) and the fp32 sums, and 1e-6."""
import numpy as np
import pytest

import sgl_rocm_kv as kv
from branch_reference import NONE, Trees
from selection_reference import Pool, f64
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


def _run(k, trees, longest=0, stream=None, keep=None):
    plan = trees.plan(longest)
    output = _filled(plan.attention.output_required_bytes + 64)
    buffers = kv.TreeAttentionBuffers(**trees.upload(), pool=trees.pool.buffer, pool_offset=trees.pool.shift, output=output,
                                      workspace=_filled(plan.workspace_required_bytes + 64, 0xFF))
    k.tree_attention(plan, buffers, stream=stream)
    hip.synchronize()
    raw = output.download()
    n = plan.attention.output_required_bytes
    assert (raw[n:] == 0xA5).all()
    return f64(raw[:n].view(np.uint16).reshape(len(trees.requests), trees.qheads, trees.pool.dv))


def _make(seed, *, page=16, heads=2, qheads=8, dk=128, dv=None, hnd=False, shift=0, contexts=(100,), drafts=(8,), words=None,
          spare=0, padding=0, extra=2):
    rng = np.random.default_rng(seed)
    pages = sum(-(-(c + n) // page) for c, n in zip(contexts, drafts)) + extra
    pool = Pool(rng, page=page, heads=heads, dk=dk, dv=dv, pages=pages, hnd=hnd, shift=shift)
    return rng, Trees(rng, pool, qheads, contexts, drafts, words=words, spare=spare, padding=padding)


SHAPES = [
    dict(contexts=(0,), drafts=(1,)),                                    # one token that attends itself
    dict(contexts=(1,), drafts=(1,)),
    dict(page=64, heads=8, qheads=32, contexts=(2000, 1, 63, 64, 65), drafts=(16, 1, 64, 24, 2), spare=3),
    dict(page=64, heads=8, qheads=32, contexts=(700, 333), drafts=(61, 33), hnd=True, padding=5),
    dict(heads=2, qheads=14, dk=64, contexts=(900, 17, 300, 0), drafts=(61, 5, 64, 7), hnd=True, padding=3),
    dict(heads=2, qheads=8, dk=256, contexts=(500, 31, 64), drafts=(13, 5, 64), hnd=True),
    dict(heads=2, qheads=8, dk=256, page=64, contexts=(1500, 2), drafts=(30, 3)),
    dict(heads=8, qheads=32, dk=64, page=32, contexts=(1000, 999), drafts=(16, 15)),
    dict(heads=1, qheads=8, contexts=(40, 41, 42, 43), drafts=(120, 70, 128, 65), spare=1),   # two mask words
    dict(heads=2, qheads=2, contexts=(64, 96), drafts=(1000, 1024), words=16),                # the most mask words
    dict(heads=2, qheads=8, contexts=(50,), drafts=(20,), words=5),                           # words that hold no bit
    dict(heads=1, qheads=1, dk=64, contexts=(500, 20), drafts=(9, 40)),
    dict(heads=2, qheads=66, dk=128, contexts=(130, 20), drafts=(9, 40)),                     # 33 query heads a KV head
    dict(heads=1, qheads=130, dk=64, contexts=(130, 20), drafts=(3, 4)),                      # 130
    dict(page=48, heads=3, qheads=9, contexts=(1000, 50), drafts=(24, 31)),                   # pages that are no power of two
    dict(page=1, heads=2, qheads=4, dk=64, contexts=(300, 2), drafts=(12, 33)),
    dict(page=4, heads=2, qheads=4, contexts=(300, 5), drafts=(12, 33), hnd=True),
    dict(heads=1, qheads=128, dk=576, dv=512, page=64, contexts=(300, 130), drafts=(3, 6)),   # latent rows
    dict(heads=1, qheads=4, dk=20, dv=24, contexts=(200, 33), drafts=(7, 20)),                # rows that 16-byte accesses cannot read
    dict(heads=2, qheads=6, dk=97, contexts=(333, 1), drafts=(11, 3)),
    dict(heads=2, qheads=8, dk=128, shift=2, contexts=(300,), drafts=(16,)),                  # a pool that is not 16-byte aligned
    dict(heads=2, qheads=8, dk=40, hnd=True, contexts=(300, 100), drafts=(16, 2)),
    dict(heads=2, qheads=8, contexts=(400, 3) * 32, drafts=(7, 2) * 32, padding=3),           # as many requests as one wave has lanes
    dict(heads=2, qheads=8, contexts=(400, 3, 0, 17, 200) * 14, drafts=(7, 2, 1, 1, 61) * 14, padding=9),      # and more
    dict(heads=1, qheads=8, dk=64, contexts=(900,) + (1,) * 129, drafts=(120,) + (1,) * 129, hnd=True, spare=1),
    dict(heads=1, qheads=4, dk=256, contexts=(1,) * 99 + (700,), drafts=(1,) * 99 + (64,)),
    dict(heads=1, qheads=128, contexts=(300, 20), drafts=(9, 40)),                            # a query to a tile
    dict(heads=1, qheads=64, dk=256, contexts=(300, 20), drafts=(9, 40), hnd=True),
    dict(heads=600, qheads=600, dk=64, page=1, contexts=(70, 5), drafts=(9, 3)),              # more KV heads than workgroups at once
    dict(heads=8, qheads=32, page=64, contexts=(9000,), drafts=(3,), padding=2),              # one long request
    dict(heads=1, qheads=1, dk=64, contexts=(30, 0, 7, 64, 1), drafts=(1000, 1020, 800, 1024, 700), words=16, spare=1),  # long lists
]


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(f"{a}{b}" for a, b in s.items()).replace(" ", "")[:80])
@pytest.mark.parametrize("hint", [True, False])
def test_against_the_definition(k, shape, hint):
    """Random trees; the longest reach given or not."""
    _, trees = _make(1, **shape)
    _say(f"tree attention {shape} hint={hint}")
    longest = max(c + n for c, n in zip(trees.contexts, trees.drafts)) if hint else 0
    got = _run(k, trees, longest)
    k.check_errors()
    _check(got, *trees.attend(), "tree")


@pytest.mark.parametrize("dk,hnd", [(64, False), (128, True), (256, False), (40, False)])
def test_any_mask(k, dk, hnd):
    """Masks that are no trees: empty ones, full ones, single bits, the last bit alone, and queries of one request that
    attend different numbers of tokens whole, in no order."""
    rng, trees = _make(2, dk=dk, hnd=hnd, contexts=(0, 200, 90, 400), drafts=(64, 64, 100, 7), heads=2, qheads=6)
    n = len(trees.requests)
    trees.masks &= rng.random(trees.masks.shape) < 0.4
    for q in range(n):
        d = trees.drafts[trees.requests[q]]
        if q % 5 == 0:
            trees.masks[q] = False
        if q % 7 == 0:
            trees.masks[q, :d] = True
        if q % 11 == 0:
            trees.masks[q] = False
            trees.masks[q, d - 1] = True
    for q in np.flatnonzero(trees.requests == 3):  # any length; the mask counts from there
        room = 407 - int(rng.integers(0, 408))
        trees.lengths[q] = room
        trees.masks[q] = False
        trees.masks[q, :max(0, min(128, 407 - room))] = rng.random(max(0, min(128, 407 - room))) < 0.5
    _say(f"tree attention, any mask, dk={dk}")
    got = _run(k, trees)
    k.check_errors()
    want, absolute = trees.attend()
    empty = [q for q in range(n) if not len(trees.attended(q))]
    assert len(empty) > 3 and (got[empty] == 0).all()
    _check(got, want, absolute, "any mask")


@pytest.mark.parametrize("shape", [dict(dk=64), dict(dk=128), dict(dk=256, hnd=True), dict(dk=40), dict(dk=128, qheads=64)],
                         ids=str)
@pytest.mark.parametrize("value", [0x7FC0, 0x7F80, 0xFF80, 0xFF7F])
def test_what_is_not_attended_does_not_show(k, shape, value):
    """NaN, infinities and the lowest value in rows that a query does not attend, those that others do among them."""
    _, trees = _make(3, contexts=(70, 130), drafts=(30, 64), spare=2, **{**dict(heads=2, qheads=8), **shape})
    want, absolute = trees.attend()
    clean = _run(k, trees)
    k.check_errors()
    # Draft 4 of each request and everything behind the drafts in their pages: what does not attend draft 4 stays.
    pool = trees.pool
    used = np.zeros(pool.pages * pool.page, bool)
    hit = np.zeros(len(trees.requests), bool)
    for r in range(2):
        start, c, n = int(trees.offsets[r]), trees.contexts[r], trees.drafts[r]
        used[trees.slots[start:start + c + n].astype(np.int64)] = True
        slot = int(trees.slots[start + c + 4])
        hit |= (trees.requests == r) & trees.masks[:, 4]
        for h in range(pool.heads):
            pool.rows(0).put(slot, h, value)
            pool.rows(1).put(slot, h, value)
    for slot in np.flatnonzero(~used):
        for h in range(pool.heads):
            pool.rows(0).put(slot, h, value)
            pool.rows(1).put(slot, h, value)
    pool.upload()
    _say(f"tree attention with {value:#x} where it is not attended, {shape}")
    got = _run(k, trees)
    k.check_errors()
    assert 0 < hit.sum() < len(hit)
    _check(got[~hit], want[~hit], absolute[~hit], "unattended")
    if value == 0xFF7F:  # (a weight of 0 takes nothing from a finite value)
        assert np.array_equal(got[~hit], clean[~hit])
    if value == 0x7FC0:
        assert np.isnan(got[hit]).all()


def test_attended_infinities(k):
    """An infinite value that some drafts attend is theirs alone. Their outputs are infinite or NaN: a weight w enters the
    product as hi = bf16(w) and lo = bf16(w - hi), and hi x inf + lo x inf is inf where lo > 0, else NaN (0 x inf, inf - inf)."""
    _, trees = _make(4, contexts=(40,), drafts=(20,))
    pool = trees.pool
    slot = int(trees.slots[40 + 3])
    for h in range(pool.heads):
        bits = pool.rows(1).get(slot, h).copy()
        bits[5] = 0x7F80
        pool.rows(1).put(slot, h, bits)
    pool.upload()
    got = _run(k, trees)
    with np.errstate(invalid="ignore"):
        want, absolute = trees.attend()
    on = trees.masks[:, 3]
    assert (np.isposinf(got[on][:, :, 5]) | np.isnan(got[on][:, :, 5])).all() and np.isfinite(got[~on]).all() and np.isfinite(np.delete(got, 5, axis=2)).all()
    keep = np.delete(np.arange(pool.dv), 5)
    _check(got[:, :, keep], want[:, :, keep], absolute[:, :, keep])


@pytest.mark.parametrize("dk", [128, 40])
def test_bad_metadata(k, dk):
    """What does not hold is reported, and gives zeros; the others are not disturbed."""
    def fresh():
        return _make(5, dk=dk, contexts=(90, 33, 64), drafts=(9, 5, 12), spare=1)[1]

    def expect(trees, flags, bad, longest=0):
        want, absolute = fresh().attend()
        got = _run(k, trees, longest)
        with pytest.raises(kv.KvError) as e:
            k.check_errors()
        assert (e.value.variant, e.value.fields[0]) == ("DeviceMetadataInvalid", flags), e.value
        assert (got[bad] == 0).all()
        good = np.setdiff1d(np.arange(len(want)), bad)
        _check(got[good], want[good], absolute[good])
        k.check_errors()

    third = np.arange(14, 26)
    trees = fresh()
    trees.requests[third] = 3
    expect(trees, 1, third)
    trees = fresh()
    trees.lengths[10] = 2 ** 63
    expect(trees, 2, [10])
    trees = fresh()
    trees.masks[11, 63] = True  # behind the request's slots
    expect(trees, 2, [11])
    trees = fresh()
    trees.lengths[25] += 2  # its mask's last bit is one behind the request's slots
    expect(trees, 2, [25])
    trees = fresh()
    reach = [int(n) + np.flatnonzero(m)[-1] + 1 for n, m in zip(trees.lengths, trees.masks)]
    expect(trees, 2, [q for q, n in enumerate(reach) if n > 92], longest=92)
    trees = fresh()
    trees.offsets[3] = len(trees.slots) + 1
    expect(trees, 2, third)
    trees = fresh()
    trees.offsets[1], trees.offsets[2] = trees.offsets[2], trees.offsets[1]  # the second request's range is no range
    bad = np.arange(9, 14)
    trees.lengths[third] = 0
    trees.masks[third] = False
    got = _run(k, trees)
    with pytest.raises(kv.KvError):
        k.check_errors()
    assert (got[bad] == 0).all() and (got[third] == 0).all()


@pytest.mark.parametrize("dk", [128, 40])
def test_a_slot_outside_the_pool(k, dk):
    """Reported where it is attended, and what does not attend it is right; not looked at where nobody attends it."""
    _, trees = _make(6, dk=dk, contexts=(50,), drafts=(10,))
    trees.masks[:, 7] = False
    trees.masks[7, 6] = True
    trees.slots[57] = 2 ** 32 + 3
    got = _run(k, trees)
    k.check_errors()
    want, absolute = trees.attend()
    _check(got, want, absolute)
    bad = _make(6, dk=dk, contexts=(50,), drafts=(10,))[1]
    bad.masks[:, 7] = trees.masks[:, 7]
    bad.masks[:, 8] = False
    bad.masks[2:5, 8] = True
    bad.masks[7, 6] = True
    bad.slots[57] = bad.pool.pages * bad.pool.page
    slot = bad.slots[58]
    want, absolute = bad.attend()
    bad.slots[58] = 2 ** 63
    got = _run(k, bad)
    with pytest.raises(kv.KvError) as e:
        k.check_errors()
    assert e.value.fields[0] == 4
    rest = np.delete(np.arange(10), [2, 3, 4])
    _check(got[rest], want[rest], absolute[rest])
    bad.slots[58] = slot
    got = _run(k, bad)
    k.check_errors()
    _check(got, want, absolute)


def test_queries_out_of_order_are_reported(k):
    _, trees = _make(7, contexts=(50, 60), drafts=(10, 10))
    trees.requests[:] = trees.requests[::-1].copy()
    _run(k, trees)
    with pytest.raises(kv.KvError) as e:
        k.check_errors()
    assert e.value.fields[0] & 1


def test_a_chain_is_paged_attention(k):
    """Drafts that each attend all before them: the outputs of paged attention at their lengths, within both bounds."""
    _, trees = _make(8, heads=8, qheads=32, page=64, contexts=(300, 1000), drafts=(5, 5))
    trees.masks[:] = False
    for q in range(10):
        trees.masks[q, :q % 5 + 1] = True
    got = _run(k, trees)
    plan = trees.plan().attention
    output = _filled(plan.output_required_bytes)
    ends = np.repeat(trees.contexts, 5) + np.tile(np.arange(5), 2) + 1
    given = {n: b for n, b in trees.device.items() if n != "masks"}
    given["query_sequence_lengths"] = hip.DeviceBuffer.from_array(ends.astype(np.uint64))
    k.paged_attention_async(plan, **given, pool=trees.pool.buffer, output=output)
    hip.synchronize()
    k.check_errors()
    chain = f64(output.download().view(np.uint16).reshape(got.shape))
    want, absolute = trees.attend()
    _check(got, want, absolute)
    _check(chain, want, absolute)


def test_refusals(k):
    _, trees = _make(9, contexts=(50,), drafts=(10,))
    plan = trees.plan()
    output = _filled(plan.attention.output_required_bytes)
    given = dict(**trees.upload(), pool=trees.pool.buffer, output=output, workspace=_filled(plan.workspace_required_bytes + 16))

    def refused(variant, name, **change):
        with pytest.raises(kv.KvError) as e:
            k.tree_attention(plan, kv.TreeAttentionBuffers(**{**given, **change}))
        assert (e.value.variant, e.value.name) == (variant, name)

    for name in ("queries", "query_request_indices", "query_sequence_lengths", "request_slot_offsets", "sequence_slots", "pool",
                 "output", "masks"):
        short = kv.device_buffer(given[name].ptr, given[name].nbytes - given[name].nbytes // 8 - 1)
        refused("AllocationOutOfBounds", name, **{name: short})
        refused("DeviceMismatch", name, **{name: kv.device_buffer(1 << 20, 1 << 40)})
    refused("InvalidArgument", "alignment", masks=kv.device_buffer(given["masks"].ptr + 4, 1 << 20))
    with pytest.raises(TypeError):
        kv.TreeAttentionBuffers(mask=given["masks"])
    plan._c.config.mask_words = 17
    refused("DimensionTooLarge", "mask_words")
    plan._c.config.mask_words = 0
    refused("ZeroDimension", "mask_words")
