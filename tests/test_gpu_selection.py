"""GPU tests of page selection (page_bounds, select_pages, selected_attention)
against the 64-bit restatements in selection_reference.py.

Bounds are values of the keys and the lists are whole numbers: both are compared
exactly. (The scores are sums of at most 2 * 576 products of two bf16 values of
16 bits each; with operands between 2^-12 and 2^3 in magnitude, as nearly all
normal ones are, every partial sum is a multiple of 2^-38 and below 2^14: 52
bits, exact in any order. A smaller operand moves a sum by less than 2^-52 of
it, and no two pages' scores here are that near unless the pages are equal,
which the tests of ties make them.)

Attention: the bound of tests/test_gpu_attention.py, u |want| for the rounding of
the output (u = 2^-8, half a step of bf16), 2^-12 sum_i w_i |v_i| for the hi + lo
weights (2^-16) and the fp32 sums, and 1e-6."""
import numpy as np
import pytest

import selection_reference as ref
import sgl_rocm_kv as kv
from selection_reference import NONE, Batch, Pool, bf16, f64
from sgl_rocm_kv import hip

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def k():
    if hip.device_count() == 0:
        pytest.fail("no GPU visible: the gpu tests need an MI355X")
    ctx = kv.RocmKvPairCopyKernels(0)
    yield ctx
    ctx.close()


def _say(msg):
    print(f"[gpu] {msg}", flush=True)


def _filled(nbytes, value=0xA5):
    return hip.DeviceBuffer.from_array(np.full(max(1, nbytes), value, np.uint8))


def _workspace(plan):
    # Whatever a workspace holds must not show: all NaN.
    return _filled(plan.workspace_required_bytes + 64, 0xFF)


# ---- bounds ---------------------------------------------------------------------------------

def _run_bounds(k, pool, pages, counts, start=None):
    """The bounds buffer [page][head][2][dim] after the call."""
    shape = (pool.pages, pool.heads, 2, pool.dk)
    start = np.full(shape, 0x1234, np.uint16) if start is None else start
    out = hip.DeviceBuffer.from_array(start)
    k.page_bounds(pool.view(), pages=hip.DeviceBuffer.from_array(np.asarray(pages, np.uint32)),
                  counts=hip.DeviceBuffer.from_array(np.asarray(counts, np.uint32)), page_count=len(pages), bounds=out)
    return out, lambda: out.download().view(np.uint16).reshape(shape)


@pytest.mark.parametrize("page,heads,dk,dv,hnd,shift", [
    (64, 8, 128, 128, False, 0), (16, 8, 128, 128, True, 0), (16, 2, 64, 64, False, 0), (48, 3, 256, 256, True, 0),
    (1, 4, 64, 64, False, 0), (64, 1, 576, 512, False, 0), (7, 2, 40, 40, False, 0), (5, 3, 20, 20, True, 0),
    (16, 2, 64, 64, False, 2), (33, 1, 97, 33, False, 0), (4, 2, 8, 8, True, 0), (100, 1, 1024, 1024, False, 0)])
def test_bounds(k, page, heads, dk, dv, hnd, shift):
    rng = np.random.default_rng(page * dk)
    pool = Pool(rng, page=page, heads=heads, dk=dk, dv=dv, pages=23, hnd=hnd, shift=shift)
    pages = rng.permutation(23)[:17]
    counts = rng.integers(0, page + 1, 17)
    counts[:3] = (page, 1, 0)
    _say(f"bounds page={page} heads={heads} dk={dk} hnd={hnd} shift={shift}")
    _, get = _run_bounds(k, pool, pages, counts)
    k.check_errors()
    got = get()
    for p in range(23):
        at = np.flatnonzero(pages == p)
        if len(at) and counts[at[0]]:
            assert np.array_equal(f64(got[p]), ref.page_bounds(pool, p, counts[at[0]])), p
        else:
            assert (got[p] == 0x1234).all(), p


def test_bounds_of_infinities_and_nan(k):
    """Infinities are bounds like any; a NaN makes both of its channel's NaN, also
    behind and before numbers; keys past the count are not read."""
    pool = Pool(np.random.default_rng(3), page=16, heads=2, dk=64, pages=4)
    rows = pool.rows(0)
    rows.at[1, 3, 0, 5] = 0x7F80
    rows.at[1, 9, 1, 6] = 0xFF80
    rows.at[1, 0, 0, 7] = rows.at[1, 11, 0, 8] = rows.at[2, 15, 1, 9] = 0x7FC0
    rows.at[3, 12, 0, 3] = 0x7FC0  # past the count
    pool.upload()
    _, get = _run_bounds(k, pool, [1, 2, 3], [16, 16, 12])
    k.check_errors()
    got = f64(get())
    want = np.stack([ref.page_bounds(pool, p, c) for p, c in ((1, 16), (2, 16), (3, 12))])
    assert np.array_equal(got[1:], want, equal_nan=True)
    assert np.isnan(got[1, 0, :, 7]).all() and np.isnan(got[1, 0, :, 8]).all() and np.isnan(got[2, 1, :, 9]).all()
    assert got[1, 0, 1, 5] == np.inf and got[1, 1, 0, 6] == -np.inf and np.isfinite(got[3]).all()


def test_bounds_bad_entries_are_reported_and_skipped(k):
    pool = Pool(np.random.default_rng(4), page=8, heads=2, dk=64, pages=5)
    for pages, counts, variant in (([1, 5, 2], [8, 8, 3], "DevicePageIndexOutOfRange"),
                                   ([1, 0xFFFFFFFF, 2], [8, 8, 3], "DevicePageIndexOutOfRange"),
                                   ([1, 4, 2], [8, 9, 3], "DeviceSpanOutOfRange")):
        _, get = _run_bounds(k, pool, pages, counts)
        with pytest.raises(kv.KvError) as e:
            k.check_errors()
        assert e.value.variant == variant
        got = get()
        assert np.array_equal(f64(got[1]), ref.page_bounds(pool, 1, 8))
        assert np.array_equal(f64(got[2]), ref.page_bounds(pool, 2, 3))
        assert (got[[0, 3, 4]] == 0x1234).all()
    k.check_errors()


# ---- selection ------------------------------------------------------------------------------

def _bounds(rng, pool):
    a = rng.standard_normal((2, pool.pages, pool.heads, pool.dk))
    return bf16(np.stack([a.min(axis=0), a.max(axis=0)], axis=2))


def _run_select(k, batch, bounds, keep, first=0, last=0, longest=0, stream=None):
    plan = kv.PageSelectionPlan.new(batch.plan(), max_pages=keep, first_pages=first, last_pages=last,
                                    max_sequence_length=longest)
    shape = (len(batch.ends), batch.pool.heads, keep)
    assert plan.selected_required_bytes == 4 * int(np.prod(shape))
    out = _filled(plan.selected_required_bytes)
    held = hip.DeviceBuffer.from_array(bounds) if isinstance(bounds, np.ndarray) else bounds
    buffers = kv.PageSelectionBuffers(**batch.device, bounds=held, selected=out, workspace=_workspace(plan))
    k.select_pages(plan, buffers, stream=stream)
    hip.synchronize()
    return out.download().view(np.uint32).reshape(shape)


@pytest.mark.parametrize("page,heads,qheads,dk,dv,lengths,per,keep,first,last", [
    (64, 8, 32, 128, 128, (5000,), 1, 8, 1, 1),
    (16, 2, 14, 64, 64, (700, 1, 33, 2000), 5, 9, 1, 2),
    (16, 2, 14, 64, 64, (700,), 333, 9, 1, 2),              # a prompt's queries
    (16, 4, 8, 128, 128, (1700, 300), 150, 12, 0, 1),
    (16, 8, 8, 128, 128, (1600, 900), 1, 33, 0, 0),
    (16, 1, 16, 256, 256, (3000, 16, 17), 3, 12, 2, 1),
    (1, 2, 4, 64, 64, (300, 0, 2), 1, 20, 4, 16),
    (48, 1, 128, 576, 512, (4000, 100), 1, 30, 0, 1),
    (8, 3, 6, 20, 20, (500,), 2, 11, 0, 1),           # rows that 16-byte accesses cannot read
    (8, 1, 3, 97, 97, (900, 64), 1, 40, 0, 0),
    (4, 2, 10, 1024, 1024, (100,), 1, 6, 1, 0),
    (16, 4, 4, 8, 8, (4000,), 1, 100, 0, 0),
    (64, 2, 80, 64, 64, (6400,), 1, 1, 0, 0),         # 40 query heads a KV head, one page
    (16, 64, 256, 64, 64, (640, 200, 1000), 1, 5, 1, 1),
    (2, 1, 2, 64, 64, (1100,), 150, 64, 1, 1),        # a chunk of a prompt
])
def test_select(k, page, heads, qheads, dk, dv, lengths, per, keep, first, last):
    rng = np.random.default_rng(dk + keep)
    pool = Pool(rng, page=page, heads=heads, dk=dk, dv=dv, pages=sum(-(-n // page) for n in lengths) + 3, layers=1,
                layer=0)
    batch = Batch(rng, pool, lengths, qheads, per, spare=5)
    bounds = _bounds(rng, pool)
    _say(f"select page={page} heads={heads}x{qheads} dk={dk} lengths={lengths} per={per} keep={keep}")
    got = _run_select(k, batch, bounds, keep, first, last, longest=max(lengths))
    k.check_errors()
    assert np.array_equal(got, ref.select(batch, bounds, keep, first, last))


def test_select_more_pages_than_a_workgroup_keeps(k):
    """20,001 pages: the picking workgroup reads its keys from memory."""
    rng = np.random.default_rng(5)
    pool = Pool(rng, page=2, heads=1, dk=64, pages=30100, layers=1, layer=0)
    batch = Batch(rng, pool, (40001, 20000), 2)
    bounds = _bounds(rng, pool)
    for keep in (1, 700):
        assert np.array_equal(_run_select(k, batch, bounds, keep, 0, 1), ref.select(batch, bounds, keep, 0, 1))
    k.check_errors()


def test_select_ties_go_to_the_lower_page(k):
    """Pages with the same bounds, also all of them, and zeros of both signs."""
    rng = np.random.default_rng(6)
    pool = Pool(rng, page=16, heads=2, dk=64, pages=130, layers=1, layer=0)
    batch = Batch(rng, pool, (1600, 300), 8)
    bounds = _bounds(rng, pool)
    kinds = bounds[:3].copy()
    few = kinds[rng.integers(0, 3, pool.pages)]
    for b in (few, np.broadcast_to(bounds[:1], bounds.shape), np.where(rng.random(bounds.shape) < 0.5, 0, 0x8000)):
        b = np.ascontiguousarray(b.astype(np.uint16))
        for keep in (7, 60):
            assert np.array_equal(_run_select(k, batch, b, keep), ref.select(batch, b, keep))
    k.check_errors()


@pytest.mark.parametrize("values", [(0, 1), (0, 1, 2, 3), (0, 4), (1, 3), (-4, 0), (-2, -1, 2, 8)])
@pytest.mark.parametrize("dk,lengths", [(64, (3200, 500)), (40, (3200, 500)), (64, (40000, 3200))])
def test_select_ties_of_round_scores(k, values, dk, lengths):
    """Scores a power of two apart, whose largest alone are more than the list takes: a counting step that holds
    just the largest key. The last lengths have more pages than a workgroup keeps in registers."""
    rng = np.random.default_rng(dk)
    pool = Pool(rng, page=8, heads=2, dk=dk, pages=sum(-(-n // 8) for n in lengths) + 2, layers=1, layer=0)
    batch = Batch(rng, pool, lengths, 4)
    batch.queries[:] = 0
    batch.queries[:, :, 0] = 0x3F80  # 1.0: a page's score is its bound
    batch.upload()
    bounds = np.zeros((pool.pages, 2, 2, dk), np.uint16)
    bounds[:, :, :, 0] = bf16(rng.choice(np.asarray(values, np.float32), (pool.pages, 2, 1)))
    _say(f"select among scores of {values}, dims {dk}, {lengths} tokens")
    for keep in (1, 7, 50):
        assert np.array_equal(_run_select(k, batch, bounds, keep), ref.select(batch, bounds, keep))
    k.check_errors()


def test_select_infinities_and_nan(k):
    """An infinite or NaN bound makes its page's score infinite or NaN; NaN ranks above every number,
    also where only some query heads see it."""
    rng = np.random.default_rng(7)
    pool = Pool(rng, page=16, heads=2, dk=64, pages=101, layers=1, layer=0)
    batch = Batch(rng, pool, (1600,), 8)
    batch.queries[:, :, 3] = bf16(np.abs(f64(batch.queries[:, :, 3]).astype(np.float32)) + 0.5)
    batch.queries[0, 1, 9] = 0  # 0 times infinity
    batch.upload()
    bounds = _bounds(rng, pool)
    own = batch.own_slots(0)[::16] // 16
    bounds[own[70], 0, 1, 3] = 0x7F80
    bounds[own[11], 0, 0, 3] = bounds[own[50], 1, 1, 3] = 0xFF80
    bounds[own[33], 0, 1, 7] = 0x7FC0
    bounds[own[34], 1, 0, 8] = 0xFFC0
    bounds[own[80], 0, 1, 9] = 0x7F80
    for keep in (1, 2, 3, 10, 99):
        got = _run_select(k, batch, bounds, keep, 0, 0)
        assert np.array_equal(got, ref.select(batch, bounds, keep))
    batch.queries[0, 0, 0] = 0x7FC0  # every page of KV head 0 is NaN
    batch.upload()
    assert np.array_equal(_run_select(k, batch, bounds, 5), ref.select(batch, bounds, 5))
    k.check_errors()


def test_select_reports_bad_metadata_and_lists_nothing(k):
    rng = np.random.default_rng(8)
    pool = Pool(rng, page=16, heads=2, dk=64, pages=60, layers=1, layer=0)
    bounds = _bounds(rng, pool)

    def case(change, longest=400):
        batch = Batch(rng, pool, (400, 300), 4)
        sound = ref.select(batch, bounds, 5, 0, 1)
        change(batch)
        batch.upload()
        got = _run_select(k, batch, bounds, 5, 0, 1, longest)
        with pytest.raises(kv.KvError) as e:
            k.check_errors()
        assert e.value.variant == "DeviceMetadataInvalid"
        assert np.array_equal(got[1], sound[1])
        return got, e.value.fields[0]

    def request(b): b.requests[0] = 2
    def length(b): b.ends[0] = 401
    def offsets(b): b.offsets[0] = 1 << 60
    def slot(b): b.slots[32] = 60 * 16
    def inside(b): b.slots[32] += 1
    got, flags = case(request)
    assert flags == 1 and (got[0] == NONE).all()
    for change in (length, offsets):
        got, flags = case(change)
        assert flags == 2 and (got[0] == NONE).all()
    got, flags = case(lambda b: None, longest=399)
    assert flags == 2 and (got[0] == NONE).all()
    for change in (slot, inside):
        assert case(change)[1] == 4
    k.check_errors()


# ---- attention ------------------------------------------------------------------------------

def _run_attend(k, batch, lists, scale=None, longest=0, stream=None):
    plan = kv.PageSelectionPlan.new(batch.plan(scale), max_pages=lists.shape[2], max_sequence_length=longest)
    out = _filled(plan.attention.output_required_bytes)
    pool = batch.pool
    buffers = kv.PageSelectionBuffers(**batch.device, pool=pool.buffer, pool_offset=pool.shift, output=out,
                                      selected=hip.DeviceBuffer.from_array(lists), workspace=_workspace(plan))
    k.selected_attention(plan, buffers, stream=stream)
    hip.synchronize()
    return f64(out.download().view(np.uint16).reshape(len(batch.ends), batch.qheads, pool.dv))


def _check(got, want, absolute, label=""):
    bound = 2.0 ** -8 * np.abs(want) + 2.0 ** -12 * absolute + 1e-6
    worst = (np.abs(got - want) / bound).max()
    _say(f"attention {label}: largest error {np.abs(got - want).max():.3g}, {worst:.3f} of the bound")
    assert worst <= 1.0  # (a NaN fails too)


@pytest.mark.parametrize("page,heads,qheads,dk,dv,hnd,shift,lengths,per,keep", [
    (64, 8, 32, 128, 128, False, 0, (5000,), 1, 32),
    (64, 8, 32, 128, 128, True, 0, (3000, 64, 65, 1, 0), 1, 12),
    (16, 2, 14, 64, 64, True, 0, (900, 17, 300), 5, 45),
    (16, 2, 8, 256, 256, True, 0, (1500, 31, 600), 5, 60),
    (32, 4, 4, 64, 64, False, 0, (999, 32, 33), 1, 8),
    (128, 1, 16, 128, 128, False, 0, (10000, 127), 1, 70),  # more pages than a split has lanes
    (8, 2, 6, 128, 128, False, 0, (500, 7), 3, 30),
    (8, 2, 6, 256, 256, True, 0, (500, 9), 3, 30),
    (16, 2, 32, 256, 256, False, 0, (500, 9), 1, 7),
    (1, 2, 4, 64, 64, False, 0, (300, 1, 2), 1, 130),
    (4, 2, 4, 128, 128, True, 0, (300, 5), 2, 40),
    (48, 3, 9, 128, 128, False, 0, (1000, 50), 2, 9),       # pages that are no power of two
    (16, 1, 40, 64, 64, False, 0, (400,), 1, 10),           # more query heads than a wave takes
    (64, 1, 128, 576, 512, False, 0, (1000, 130), 1, 6),    # latent rows
    (16, 2, 4, 20, 24, False, 0, (200,), 1, 5),             # rows that 16-byte accesses cannot read
    (16, 2, 4, 97, 113, True, 0, (200, 40), 1, 9),
    (16, 2, 8, 128, 128, False, 2, (300,), 1, 9),
    (16, 2, 8, 64, 128, False, 0, (300,), 1, 9),
    (16, 2, 8, 128, 64, True, 0, (300,), 1, 9),
    (64, 8, 64, 128, 128, False, 0, tuple(range(100, 3100, 100)), 1, 16),
])
def test_attend(k, page, heads, qheads, dk, dv, hnd, shift, lengths, per, keep):
    rng = np.random.default_rng(page + dk + keep)
    pool = Pool(rng, page=page, heads=heads, dk=dk, dv=dv, pages=sum(-(-n // page) for n in lengths) + 2, hnd=hnd,
                shift=shift)
    batch = Batch(rng, pool, lengths, qheads, per, spare=3)
    lists = ref.random_lists(rng, batch, keep)
    _say(f"attend page={page} heads={heads}x{qheads} {dk}/{dv} hnd={hnd} lengths={lengths[:5]} per={per} keep={keep}")
    want, absolute = ref.attend(batch, lists)
    _check(_run_attend(k, batch, lists, longest=max(lengths)), want, absolute)
    k.check_errors()


@pytest.mark.parametrize("heads,qheads,dk,dv,pages", [
    *[(2, 8, 64, 64, n) for n in (17, 21, 34, 51, 63, 81, 98)],
    *[(2, 8, 128, 128, n) for n in (33, 47, 63, 97, 127, 131)],
    (2, 8, 40, 40, 29), (2, 8, 40, 40, 50),                 # the generic body, four sets of lanes in the merge
    (2, 8, 97, 97, 35), (2, 8, 97, 97, 63),                 # and two
    (1, 4, 64, 20, 17), (1, 4, 64, 24, 97), (2, 8, 256, 256, 35), (1, 16, 576, 512, 33)])
def test_attend_in_any_number_of_splits(k, heads, qheads, dk, dv, pages):
    """A page to a split and none of them empty: every split's record counts, whichever of the merge's rounds and
    sets of lanes it falls to; and lists of all pages give paged attention's output."""
    rng = np.random.default_rng(dk + pages)
    pool = Pool(rng, page=64, heads=heads, dk=dk, dv=dv, pages=pages + 1)
    batch = Batch(rng, pool, (64 * pages - 9,), qheads)
    lists = np.ascontiguousarray(np.broadcast_to(np.arange(pages, dtype=np.uint32), (1, heads, pages)))
    # Lists of every page need no scores: the workspace is the records, an output row in fp32 (its dims in 32s) and
    # two floats for each (query head, split).
    plan = kv.PageSelectionPlan.new(batch.plan(), max_pages=pages)
    assert plan.workspace_required_bytes == qheads * pages * 4 * (-(-dv // 32) * 32 + 2)
    _say(f"attend {dk}/{dv} in {pages} splits")
    want, absolute = ref.attend(batch, lists)
    got = _run_attend(k, batch, lists)
    _check(got, want, absolute, f"{dk}/{dv} in {pages} splits")
    out = _filled(qheads * dv * 2)
    k.paged_attention(batch.plan(), **batch.device, pool=pool.buffer, output=out)
    paged = f64(out.download().view(np.uint16).reshape(1, qheads, dv))
    # (Both within the bound of the 64-bit form: twice it.)
    _check(got, paged, 2 * absolute + 16 * np.abs(paged))
    k.check_errors()


def test_attend_lists_of_any_kind(k):
    """Lists from elsewhere: empty ones, one page, no newest page, short ones in long buffers."""
    rng = np.random.default_rng(11)
    for page, d, hnd in ((16, 128, False), (64, 64, True), (32, 256, False), (12, 128, False)):
        pool = Pool(rng, page=page, heads=4, dk=d, pages=120, hnd=hnd)
        batch = Batch(rng, pool, (page * 40 + 3, page * 7, page * 50), 8)
        lists = np.full((3, 4, 200), NONE, np.uint32)
        lists[0, 0, :2] = (3, 39)
        lists[0, 1, :1] = 40          # the page of 3 tokens alone
        lists[1, 2, :7] = np.arange(7)
        lists[2, 0, :50] = np.arange(50)
        lists[2, 3, :1] = 0
        want, absolute = ref.attend(batch, lists)
        got = _run_attend(k, batch, lists)
        k.check_errors()
        _check(got, want, absolute, f"page {page} dims {d}")
        assert (got[0, 4:] == 0).all() and (got[1, :4] == 0).all()
        empty = np.full((3, 4, 2), NONE, np.uint32)
        assert (_run_attend(k, batch, empty) == 0).all()


def test_attend_all_pages_is_paged_attention(k):
    """Both against the oracle bound; here against each other, so twice it."""
    rng = np.random.default_rng(12)
    pool = Pool(rng, page=16, heads=2, dk=128, pages=200)
    batch = Batch(rng, pool, (1000, 1, 500), 8)
    count = -(-1000 // 16)
    lists = np.full((3, 2, count), NONE, np.uint32)
    for q, end in enumerate(batch.ends.astype(int)):
        lists[q, :, :-(-end // 16)] = np.arange(-(-end // 16))
    out = _filled(3 * 8 * 128 * 2)
    k.paged_attention(batch.plan(), **batch.device, pool=pool.buffer, output=out)
    paged = f64(out.download().view(np.uint16).reshape(3, 8, 128))
    absolute = ref.attend(batch, lists)[1]
    _check(_run_attend(k, batch, lists), paged, 2 * absolute + 16 * np.abs(paged))


def test_attend_does_not_read_what_is_masked(k):
    """NaN in every key and value that no list reaches (pages not listed, and the rest of a last page)."""
    rng = np.random.default_rng(13)
    for page, d in ((64, 128), (16, 64), (16, 256), (24, 128)):
        pool = Pool(rng, page=page, heads=2, dk=d, pages=40)
        batch = Batch(rng, pool, (page * 20 + 5, 3), 8)
        lists = ref.random_lists(rng, batch, 6)
        want, absolute = ref.attend(batch, lists)
        read = np.zeros((pool.pages * page, 2), bool)
        for q, end in enumerate(batch.ends.astype(int)):
            for h in range(2):
                for j in lists[q, h][lists[q, h] != NONE]:
                    read[batch.own_slots(q)[j * page:min(end, (j + 1) * page)], h] = True
        for t in (0, 1):
            rows = pool.rows(t)
            for slot, h in zip(*np.nonzero(~read)):
                rows.put(slot, h, 0x7FC0)
        pool.upload()
        _check(_run_attend(k, batch, lists), want, absolute, f"page {page} dims {d}")
    k.check_errors()


def test_attend_nan_and_infinite_values_are_carried(k):
    rng = np.random.default_rng(14)
    pool = Pool(rng, page=16, heads=1, dk=128, pages=40)
    batch = Batch(rng, pool, (600,), 4)
    lists = ref.random_lists(rng, batch, 20)
    slots = batch.own_slots(0)
    pool.rows(1).put(slots[16 * int(lists[0, 0, 2]) + 1], 0, np.full(128, 0x7FC0))
    pool.upload()
    got = _run_attend(k, batch, lists)
    assert np.isnan(got).all()


def test_attend_reports_bad_lists_and_slots(k):
    rng = np.random.default_rng(15)
    for page, d in ((16, 128), (12, 64)):
        pool = Pool(rng, page=page, heads=2, dk=d, pages=100)

        def case(change):
            batch = Batch(rng, pool, (page * 30 + 1, page * 9), 4)
            lists = ref.random_lists(rng, batch, 6)
            change(batch, lists)
            batch.upload()
            got = _run_attend(k, batch, lists)
            with pytest.raises(kv.KvError) as e:
                k.check_errors()
            assert e.value.variant == "DeviceMetadataInvalid"
            return got, e.value.fields[0]

        def past(b, l): l[0, 0, 5] = 31
        def far(b, l): l[0, 1, 2] = 0xFFFFFFFE
        def twice(b, l): l[0, 0, 3] = l[0, 0, 2]
        def falling(b, l): l[0, 0, [2, 3]] = l[0, 0, [3, 2]]
        def gap(b, l): l[0, 0, 2] = NONE
        for change in (past, far, twice, falling, gap):
            assert case(change)[1] == 2, change.__name__
        def slot(b, l): b.slots[int(l[0, 0, 0]) * page] = pool.pages * page
        def inside(b, l): b.slots[int(l[0, 0, 0]) * page] += 1
        for change in (slot, inside):
            assert case(change)[1] == 4, change.__name__
        def request(b, l): b.requests[0] = 9
        assert case(request)[1] == 1
    k.check_errors()


def test_select_then_attend_matches_the_definition(k):
    """The three calls in a row on one stream, as a decode step makes them."""
    rng = np.random.default_rng(16)
    pool = Pool(rng, page=16, heads=4, dk=128, pages=400, hnd=True)
    batch = Batch(rng, pool, (3000, 10, 900), 16)
    bounds = np.zeros((pool.pages, 4, 2, 128), np.uint16)
    pages = np.concatenate([batch.own_slots(q)[::16] // 16 for q in range(3)])
    counts = np.concatenate([np.minimum(16, n - 16 * np.arange(-(-n // 16))) for n in (3000, 10, 900)])
    held, get = _run_bounds(k, pool, pages, counts, bounds)
    lists = _run_select(k, batch, held, 20, 1, 2)
    want_bounds = get()
    assert np.array_equal(lists, ref.select(batch, want_bounds, 20, 1, 2))
    want, absolute = ref.attend(batch, lists)
    _check(_run_attend(k, batch, lists), want, absolute)
    k.check_errors()


def test_padded_batches_select_and_attend_nothing(k):
    """Queries of length 0 behind the batch, of any request index, get no pages and zeros."""
    rng = np.random.default_rng(17)
    pool = Pool(rng, page=16, heads=2, dk=64, pages=90)
    batch = Batch(rng, pool, (700, 90, 400), 8)
    bounds = _bounds(rng, pool)
    want = ref.select(batch, bounds, 6)
    want_output, absolute = ref.attend(batch, want)
    batch.requests = np.concatenate([batch.requests, np.array([0, 2, NONE, 7], np.uint32)])
    batch.ends = np.concatenate([batch.ends, np.zeros(4, np.uint64)])
    batch.queries = np.concatenate([batch.queries, np.full((4, 8, 64), 0x7FC0, np.uint16)])
    batch.upload()
    lists = _run_select(k, batch, bounds, 6)
    assert np.array_equal(lists[:3], want) and (lists[3:] == NONE).all()
    output = _run_attend(k, batch, lists)
    _check(output[:3], want_output, absolute)
    assert (output[3:] == 0).all()
    k.check_errors()


def test_refusals(k):
    rng = np.random.default_rng(18)
    pool = Pool(rng, page=8, heads=2, dk=64, pages=40)
    batch = Batch(rng, pool, (250,), 4)
    plan = kv.PageSelectionPlan.new(batch.plan(), max_pages=20)
    bounds = _filled(plan.bounds_required_bytes)
    selected, output = _filled(plan.selected_required_bytes), _filled(plan.attention.output_required_bytes)
    sound = dict(batch.device, pool=pool.buffer, bounds=bounds, selected=selected, output=output,
                 workspace=_workspace(plan))
    shared = ("queries", "query_request_indices", "query_sequence_lengths", "request_slot_offsets", "sequence_slots",
              "selected", "workspace")
    host = np.zeros(1 << 16, np.uint8)
    for call, own in ((k.select_pages, ("bounds",)), (k.selected_attention, ("pool", "output"))):
        def refused(variant, name, **more):
            with pytest.raises(kv.KvError) as e:
                call(plan, kv.PageSelectionBuffers(**{**sound, **more}))
            assert (e.value.variant, e.value.name) == (variant, name)
        for name in shared + own:
            refused("DeviceMismatch", name, **{name: kv.device_buffer(host.ctypes.data, host.nbytes)})
            refused("AllocationOutOfBounds", name, **{name + "_offset": 1 << 30})
            if name != "pool":
                big = _filled(1 << 18)
                with pytest.raises(kv.KvError) as e:
                    call(plan, kv.PageSelectionBuffers(**{**sound, name: big, name + "_offset": 1}))
                assert e.value.variant == "InvalidArgument"
    assert (selected.download() == 0xA5).all() and (output.download() == 0xA5).all()
    # page_bounds
    lists = dict(pages=_filled(64), counts=_filled(64), bounds=bounds)

    def refused_bounds(variant, name, **more):
        with pytest.raises(kv.KvError) as e:
            k.page_bounds(pool.view(), **{**lists, "page_count": 4, **more})
        assert (e.value.variant, e.value.name) == (variant, name)
    for name in lists:
        refused_bounds("DeviceMismatch", name, **{name: kv.device_buffer(host.ctypes.data, host.nbytes)})
    refused_bounds("AllocationOutOfBounds", "pages", page_count=17)
    refused_bounds("AllocationOutOfBounds", "bounds", bounds=_filled(64))
    k.page_bounds(pool.view(), **lists, page_count=0)
    assert (bounds.download() == 0xA5).all()
    k.check_errors()
